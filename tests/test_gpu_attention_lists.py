"""ATTENTION over lists that no other test has: row starts that fall, pages given back behind a window."""
import numpy as np
import pytest

from kv_helpers import BF16, F32, TYPE_NAMES, batch, to_type
from test_gpu_attention import check, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,length,hint", [(1, 900, 1), (5, 900, 5), (40, 300, 0), (200, 300, 0)])
def test_row_starts_that_fall(hl, dev, rows, length, hint):
    """Starts that go back to 0 for every other sequence, past the operands and below 0: all sequences are alike, so whichever
    one's results a row holds, they are the same; rows of no sequence stay."""
    import torch

    rng = np.random.default_rng(rows)
    cache, tables, gpu = setup(hl, dev, rng, np.array([length]), 2, 64, 16)
    seqs = 150
    many = np.repeat(tables, seqs, 0)
    starts = np.array([0, rows] * (seqs // 2) + [rows], dtype=np.int64)
    lens = np.full(seqs, length)
    q, qx = to_type(rng.standard_normal((rows + 2, 6, 64)), F32, dev)
    out, status = torch.full_like(q, 5.0), torch.zeros(1, dtype=torch.int32, device=dev)
    hl.attention(F32, gpu.cache, 0, gpu.batch(many, lens, starts, rows + 2, max_rows=hint), q, out, 6, status=status)
    check(F32, out.double().cpu().numpy(), cache, 0, tables, lens[:1], np.array([0, rows]), qx, 0, None)
    assert status.item() == 0
    starts[::2], starts[1::2] = -9, 1 << 30  # cut to all rows of the operands, the last two among them
    hl.attention(F32, gpu.cache, 0, gpu.batch(many, lens, starts, rows + 2, max_rows=hint), q, out, 6, status=status)
    check(F32, out.double().cpu().numpy(), cache, 0, tables, lens[:1], np.array([0, rows + 2]), qx, 0, None)


@pytest.mark.parametrize("t", [F32, BF16], ids=lambda t: TYPE_NAMES[t])
@pytest.mark.parametrize("dim,block,rows,window", [(64, 16, 1, 37), (64, 16, 1, 1), (128, 32, 5, 100), (256, 16, 4, 90), (128, 16, 60, 33), (64, 16, 150, 70),
                                                   (192, 64, 150, 200), (256, 16, 130, 16)])
def test_pages_behind_the_window(hl, dev, t, dim, block, rows, window):
    """The entries of pages that no row sees are -1 (a server gave them back): the same values and no status. One entry more, and
    the row that sees it is NaN and is reported."""
    import torch

    print("[case] attention window", TYPE_NAMES[t], dim, block, rows, window, flush=True)
    rng = np.random.default_rng(dim + rows + window)
    lens = np.array([rows + 700 + i for i in (0, 1, 5, 15, 16, 17, 31, 40)] + [rows + 5, rows])
    counts = np.full(len(lens), rows)
    cache, tables, gpu = setup(hl, dev, rng, lens, 2, dim, block)
    starts = batch(counts)
    q, qx = to_type(rng.standard_normal((len(lens) * rows, 4, dim)), t, dev)
    held = tables.copy()
    gone = np.maximum(lens - rows - window + 1, 0) // block  # whole pages before the first row's window
    for s, n in enumerate(gone):
        held[s, :n] = -1
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    for hint in (dict(), dict(max_rows=rows)):
        out = torch.full_like(q, 5.0)
        hl.attention(t, gpu.cache, 0, gpu.batch(held, lens, starts, **hint), q, out, 4, window=window, status=status)
        check(t, out.double().cpu().numpy(), cache, 0, tables, lens, starts, qx, window, None)
        assert status.item() == 0
    held[1, gone[1]] = -1  # a page that the second sequence's first row sees
    hl.attention(t, gpu.cache, 0, gpu.batch(held, lens, starts), q, out, 4, window=window, status=status)
    assert status.item() == hl.STATUS_BAD_INDEX
    nan = out.isnan().cpu().numpy().all((1, 2))
    assert nan[rows] and not nan[:rows].any() and not nan[2 * rows:].any()
