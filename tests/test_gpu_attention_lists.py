"""ATTENTION over lists that no other test has: row starts that fall."""
import numpy as np
import pytest

from kv_helpers import F32, to_type
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
