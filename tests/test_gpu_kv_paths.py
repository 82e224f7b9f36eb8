"""Forms of the cache's writes, reads and attention that depend on alignment, on rows a kv head and on the cache's size: each of
them against the definition, at the head_dims and types where it is a path of its own."""
import numpy as np
import pytest

from kv_helpers import BF16, F16, F32, TYPE_NAMES, Cache, batch, tables_for, to_type, write_ref
from test_gpu_attention import check, run, setup
from test_gpu_kv_cache import OnGpu, same_pool

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("t", [F32, F16, BF16], ids=lambda t: TYPE_NAMES[t])


@TYPES
@pytest.mark.parametrize("dim,kv,group,rows,window", [(192, 1, 6, 4, 0), (256, 2, 5, 4, 130), (256, 1, 17, 1, 0), (192, 1, 8, 4, 65), (256, 1, 5, 6, 0),
                                                      (128, 1, 8, 8, 0), (64, 2, 16, 3, 40), (96, 1, 33, 1, 0)])
def test_two_row_tiles(hl, dev, t, dim, kv, group, rows, window):
    """More rows a kv head than a tile of few rows has (16; 32 up to head_dim 128) and fewer than two of them, over few sequences: verify
    steps, whose second tile is partly empty; long enough to be joined, and in one piece."""
    print("[case] attention two tiles", TYPE_NAMES[t], dim, kv, group, rows, window, flush=True)
    rng = np.random.default_rng(dim + group + window)
    lens = np.array([rows, 70, 1333, 300, rows + 1])
    cache, tables, gpu = setup(hl, dev, rng, lens, kv, dim, 32)
    q = rng.standard_normal((rows * len(lens), kv * group, dim)) * 2
    run(hl, dev, gpu, cache, tables, lens, np.full(len(lens), rows), t, kv * group, q, window=window, max_rows=rows)
    run(hl, dev, gpu, cache, tables, lens, np.full(len(lens), rows), t, kv * group, q, window=window, max_rows=rows, max_kv=200)


@TYPES
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
def test_reads_past_the_caches(hl, dev, t, dim):
    """A table with room for more bytes than the L2 caches hold: the codes are read once, past them."""
    print("[case] attention large table", TYPE_NAMES[t], dim, flush=True)
    rng = np.random.default_rng(dim)
    lens = np.array([900, 33, 2100])
    cache, tables, gpu = setup(hl, dev, rng, lens, 2, dim, 16)
    room = np.full((3, (32 << 20) // (2 * 3 * 2 * dim) // 16 + 1), -1, dtype=np.int32)
    room[:, :tables.shape[1]] = tables
    q = rng.standard_normal((3, 8, dim))
    run(hl, dev, gpu, cache, room, lens, np.ones(3, int), t, 8, q, max_rows=1)


@TYPES
@pytest.mark.parametrize("dim,rows,length", [(64, 1, 700), (256, 4, 900), (128, 40, 60), (96, 200, 30), (128, 40, 3000), (192, 150, 1500)])
def test_unaligned_rows(hl, dev, t, dim, rows, length):
    """q at an odd offset in rows of an odd stride, out likewise: element by element; whole, split and joined. Rows of no sequence
    and elements between the rows stay."""
    import torch

    print("[case] attention unaligned", TYPE_NAMES[t], dim, rows, length, flush=True)
    rng = np.random.default_rng(dim + rows)
    kv, heads = 2, 6
    lens = np.array([rows + length, rows])
    cache, tables, gpu = setup(hl, dev, rng, lens, kv, dim, 16)
    starts = np.array([2, 2 + rows, 2 + 2 * rows], dtype=np.int32)
    n, wide = 2 * rows + 4, heads * dim + 9
    x = rng.standard_normal((n, wide))
    x[:2], x[2 + 2 * rows:] = np.nan, np.inf
    xd, xx = to_type(x, t, dev)
    out = torch.full((n, wide), 5.0, dtype=xd.dtype, device=dev)
    hl.attention(t, gpu.cache, 0, gpu.batch(tables, lens, starts, n), xd[:, 3:], out[:, 5:], heads, q_stride=wide, out_stride=wide)
    got = out.double().cpu().numpy()
    check(t, got[:, 5:5 + heads * dim].reshape(n, heads, dim).copy(), cache, 0, tables, lens, starts, xx[:, 3:3 + heads * dim].reshape(n, heads, dim), 0, None)
    assert np.all(got[:, :5] == 5.0) and np.all(got[:, 5 + heads * dim:] == 5.0)


@TYPES
@pytest.mark.parametrize("rows", [1, 90])
def test_q_and_out_in_one_row(hl, dev, t, rows):
    import torch

    rng = np.random.default_rng(rows)
    dim, kv, heads = 128, 2, 4
    lens = np.array([rows + 200, rows + 3])
    cache, tables, gpu = setup(hl, dev, rng, lens, kv, dim, 32)
    n, width = 2 * rows, heads * dim
    q, qx = to_type(rng.standard_normal((n, width)), t, dev)
    both = torch.full((n, 2 * width), 5.0, dtype=q.dtype, device=dev)
    both[:, width:] = q
    starts = batch([rows, rows])
    hl.attention(t, gpu.cache, 0, gpu.batch(tables, lens, starts), both[:, width:], both, heads, q_stride=2 * width, out_stride=2 * width)
    assert torch.equal(both[:, width:], q)
    check(t, both[:, :width].double().cpu().numpy().reshape(n, heads, dim), cache, 0, tables, lens, starts, qx.reshape(n, heads, dim), 0, None)


@TYPES
@pytest.mark.parametrize("dim,block", [(256, 32), (192, 64), (128, 64), (128, 128), (64, 128), (256, 128), (96, 128)])
def test_writes_of_unaligned_rows(hl, dev, t, dim, block):
    """Rows at an odd offset and stride into large pages: more elements than stay in registers between a page's maximum and its codes,
    which are read again; whole pages, parts of one, growth of the scale."""
    print("[case] kv_write unaligned", TYPE_NAMES[t], dim, block, flush=True)
    rng = np.random.default_rng(dim + block)
    heads, pages = 2, 16
    cache = Cache(pages, 1, heads, dim, block)
    cache.fill(rng)
    gpu = OnGpu(hl, dev, cache)
    lens = np.array([2 * block + 7, block - 1, 3 * block, 5])
    rows = lens.copy()
    room = np.array([3, 2, 4, 2]) * block
    tables = tables_for(rng, room, block, pages, 4, stray=99)
    stride = 2 * heads * dim + 3
    for loud in (1.0, 6.0, 0.3):
        starts = batch(rows) + 1
        n = int(starts[-1]) + 1
        x = rng.standard_normal((n, stride)) * loud
        x[0], x[-1] = np.nan, np.inf
        xd, xx = to_type(x, t, dev)
        k, v = xx[:, 1:1 + heads * dim].reshape(n, heads, dim), xx[:, 2 + heads * dim:2 + 2 * heads * dim].reshape(n, heads, dim)
        hl.kv_write(t, gpu.cache, 0, gpu.batch(tables, lens, starts, n), xd[:, 1:], xd[:, 2 + heads * dim:], k_stride=stride, v_stride=stride)
        write_ref(cache, 0, tables, lens, starts, k, v)
        same_pool(gpu, cache)
        rows = np.array([3, block // 2 + 1, 1, block])
        lens = np.minimum(lens + rows, room)
        rows = np.minimum(rows, lens)


@pytest.mark.parametrize("dim,block", [(64, 16), (192, 64)])
def test_read_into_one_row(hl, dev, dim, block):
    """k_out and v_out side by side, with a gap that stays."""
    import torch

    heads, rng = 3, np.random.default_rng(dim)
    cache = Cache(9, 1, heads, dim, block)
    cache.fill(rng)
    gpu = OnGpu(hl, dev, cache)
    lens = np.array([2 * block + 3, 5])
    tables = tables_for(rng, lens, block, 9, 3)
    width = heads * dim
    both = torch.full((int(lens.sum()), 2 * width + 5), 9.0, device=dev)
    hl.kv_read(gpu.cache, 0, gpu.batch(tables, lens, batch(lens)), both[:, 1:], both[:, width + 3:], k_stride=2 * width + 5, v_stride=2 * width + 5)
    got = both.cpu().numpy()
    want = [np.concatenate([cache.tokens(tables[s], n, 0)[j].transpose(1, 0, 2) for s, n in enumerate(lens)]).reshape(-1, width).astype(np.float32) for j in (0, 1)]
    assert np.array_equal(got[:, 1:1 + width], want[0]) and np.array_equal(got[:, width + 3:2 * width + 3], want[1])
    assert np.all(got[:, [0, width + 1, width + 2, 2 * width + 3, 2 * width + 4]] == 9.0)
