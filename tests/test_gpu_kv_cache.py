"""KV_WRITE into the 8-bit paged cache and kv_read on the GPU: codes and scales equal to the definition's."""
import numpy as np
import pytest

from kv_helpers import BF16, F16, F32, TYPE_NAMES, Cache, batch, tables_for, to_type, write_ref

pytestmark = pytest.mark.gpu


class OnGpu:
    """A numpy Cache's copy on the GPU, and batches over it."""

    def __init__(self, hl, dev, cache):
        import torch

        self.hl, self.dev, self.pool = hl, dev, torch.from_numpy(cache.bytes.copy()).to(dev)
        self.cache = hl.KvCache(self.pool, cache.n_pages, cache.layers, cache.heads, cache.dim, cache.block)

    def ints(self, x):
        import torch

        return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(self.dev)

    def batch(self, tables, lens, starts, n_rows=None, **kw):
        return self.hl.KvBatch(self.ints(tables), tables.shape[1], self.ints(lens), self.ints(starts), len(lens),
                               int(starts[-1]) if n_rows is None else n_rows, **kw)

    def bytes(self):
        return self.pool.cpu().numpy()


def same_pool(gpu, cache):
    """Equal bytes; the scales by value, since a NaN has many forms and zeros two, and with them the codes of a NaN block."""
    got = Cache(*cache.geometry)
    got.bytes[:] = gpu.bytes()
    a, b = got.scales, cache.scales
    assert np.array_equal(a, b, equal_nan=True), f"{np.argwhere(~((a == b) | (np.isnan(a) & np.isnan(b))))[:4]}"
    keep = ~np.isnan(b)
    assert np.array_equal(got.codes[keep], cache.codes[keep]), f"{np.argwhere((got.codes != cache.codes) & keep[..., None])[:4]}"
    end = got.scales_at()[1]
    assert np.array_equal(got.bytes[:, end:], cache.bytes[:, end:])


def write_both(hl, gpu, cache, t, layer, tables, lens, starts, k, v, dev, **kw):
    kd, kx = to_type(k, t, dev)
    vd, vx = to_type(v, t, dev)
    hl.kv_write(t, gpu.cache, layer, gpu.batch(tables, lens, starts, len(k), **kw), kd, vd)
    write_ref(cache, layer, tables, lens, starts, kx, vx)


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=lambda t: TYPE_NAMES[t])
@pytest.mark.parametrize("dim,block,heads", [(64, 16, 1), (96, 32, 3), (128, 64, 2), (192, 16, 5), (256, 128, 1), (256, 16, 4)])
def test_write(hl, dev, t, dim, block, heads):
    """Ragged batches onto pages that hold other bytes, three times in a row: prompts, then tokens that widen the scales or
    do not, from one token to more than a page, empty sequences among them."""
    print("[case] kv_write", TYPE_NAMES[t], dim, block, heads, flush=True)
    rng = np.random.default_rng(dim + block + heads + t)
    cache = Cache(24, 2, heads, dim, block)
    cache.fill(rng)
    lens = np.array([1, block, 2 * block + 5, 0, block - 1, 17], dtype=np.int64)
    tables = tables_for(rng, lens + 2 * block + 4, block, 24, 5)
    gpu = OnGpu(hl, dev, cache)
    rows = lens.copy()
    for loud in (1.0, 4.0, 0.2):
        starts = batch(rows)
        k, v = (rng.standard_normal((starts[-1], heads, dim)) * loud for _ in range(2))
        k[:, :, 3 % dim] *= 5
        write_both(hl, gpu, cache, t, 1, tables, lens, starts, k, v, dev)
        same_pool(gpu, cache)
        rows = np.array([1, 3, 1, 0, block + 2, 1])
        lens = lens + rows


def test_write_borders(hl, dev):
    """Values half way between two codes go to the even one, those a last bit away to the near one; in a scale that is
    a power of two, and in one whose multiples are not representable; growth that puts old codes on borders too."""
    import torch

    dim, block = 64, 16
    for top in (127.0, 127.0 * 2.0 ** -40, 254.0 / 3, 93.7):
        cache = Cache(3, 1, 1, dim, block)
        gpu = OnGpu(hl, dev, cache)
        s = np.float64(np.float32(top) / np.float32(127))
        i = np.arange(dim) - dim // 2
        x = np.zeros((2 * block, 1, dim))
        for r in range(2 * block):
            at = ((i + 2 * r % 90) + 0.5) * s
            x[r, 0] = np.clip(np.nextafter(np.float32(at), np.float32(np.inf) * (r % 3 - 1)) if r % 3 != 1 else np.float32(at), -top, top)
        x[:, 0, 0] = np.float32(top)
        tables, lens = np.array([[2, 0]], dtype=np.int32), np.array([2 * block])
        write_both(hl, gpu, cache, F32, 0, tables, lens, batch([2 * block]), x, -x, dev)
        same_pool(gpu, cache)
        # one more row at the place of the last, twice as loud: scale doubles, odd codes lie on borders
        more = np.zeros((1, 1, dim))
        more[0, 0, 5] = np.float32(2 * top)
        write_both(hl, gpu, cache, F32, 0, tables, lens, batch([1]), more, more, dev)
        same_pool(gpu, cache)
    assert torch.cuda.is_available()


def test_write_special_values(hl, dev):
    """Zeros, values below the smallest scale, subnormals, the largest finite ones; infinities and NaN mark their blocks
    and no other; a block restarts clean at its first token."""
    dim, block, heads = 64, 16, 2
    cache = Cache(8, 1, heads, dim, block)
    cache.fill(np.random.default_rng(3))
    gpu = OnGpu(hl, dev, cache)
    tables = np.array([[0, 1], [2, 3], [4, 5], [6, 7]], dtype=np.int32)
    lens = np.array([20, 20, 20, 20])
    k = np.zeros((80, heads, dim))
    v = np.ones((80, heads, dim))
    k[20:40] = 1e-30  # under the smallest scale
    k[40:60] = np.float32(3e38)
    k[60:80, 0, 0] = 1e-41
    v[3, 1, 7] = np.inf
    v[25, 0, 9] = np.nan
    v[59, 0, 1] = -np.inf
    write_both(hl, gpu, cache, F32, 0, tables, lens, batch([20] * 4), k, v, dev)
    same_pool(gpu, cache)
    assert np.isnan(cache.scales).sum() == 3
    # the NaN stays while its block grows, and goes where the block starts again
    lens = np.array([21, 17, 21, 1])
    write_both(hl, gpu, cache, F32, 0, tables, lens, batch([1] * 4), k[:4] + 1, v[5:9], dev)
    same_pool(gpu, cache)
    assert np.isnan(cache.scales).sum() == 3  # sequence 1 began its second page again: its NaN, at token 5, is in the first
    lens = np.array([22, 1, 22, 2])
    write_both(hl, gpu, cache, F32, 0, tables, lens, batch([1] * 4), k[:4] + 1, v[5:9], dev)
    same_pool(gpu, cache)
    assert np.isnan(cache.scales).sum() == 2 and np.isfinite(cache.scales[2]).all()


@pytest.mark.parametrize("t", [F32, BF16], ids=lambda t: TYPE_NAMES[t])
def test_write_strides_and_stray_rows(hl, dev, t):
    """Rows inside a fused projection, at an offset that no vector load takes; rows before the first and behind the last
    sequence are not read (they hold NaN); a row at a negative position is left out."""
    import torch

    dim, block, heads = 96, 16, 3
    rng = np.random.default_rng(7)
    cache = Cache(12, 1, heads, dim, block)
    cache.fill(rng)
    gpu = OnGpu(hl, dev, cache)
    lens, starts = np.array([18, 3, 33]), np.array([2, 6, 11, 20], dtype=np.int32)  # 4, 5 (two before position 0), 9 rows
    tables = tables_for(rng, lens, block, 12, 4, stray=99)
    row = 2 * heads * dim + 5
    x = rng.standard_normal((25, row))
    x[:2], x[20:] = np.nan, np.nan
    x[6:8] = np.inf
    xd, xx = to_type(x, t, dev)
    k, v = xx[:, 1:1 + heads * dim].reshape(25, heads, dim), xx[:, 1 + heads * dim:1 + 2 * heads * dim].reshape(25, heads, dim)
    status = torch.full((1,), 77, dtype=torch.int32, device=dev)
    hl.kv_write(t, gpu.cache, 0, gpu.batch(tables, lens, starts, 25, max_rows=1), xd[:, 1:], xd[:, 1 + heads * dim:], k_stride=row, v_stride=row,
                status=status)
    write_ref(cache, 0, tables, lens, starts, k, v)
    same_pool(gpu, cache)
    assert status.item() == 0


def test_write_and_read_bad_pages(hl, dev):
    """Ids out of range and tokens past the table are left out and reported; the rest of the batch is written."""
    import torch

    dim, block, heads = 64, 16, 2
    rng = np.random.default_rng(11)
    cache = Cache(6, 1, heads, dim, block)
    cache.fill(rng)
    gpu = OnGpu(hl, dev, cache)
    tables = np.array([[0, 6], [-1, 1], [2, 3]], dtype=np.int32)
    lens, starts = np.array([20, 30, 40]), batch([20, 30, 40])  # the last one is longer than its table
    k, kx = to_type(rng.standard_normal((90, heads, dim)), F32, dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    b = gpu.batch(tables, lens, starts)
    hl.kv_write(F32, gpu.cache, 0, b, k, k, status=status)
    write_ref(cache, 0, tables, lens, starts, kx, kx)
    same_pool(gpu, cache)
    assert status.item() == hl.STATUS_BAD_INDEX
    out = torch.full((91, heads, dim), 5.0, device=dev)
    hl.kv_read(gpu.cache, 0, b, out, None, status=status, status_keep=True)
    got = out.cpu().numpy()
    bad = np.isnan(got).all((1, 2))
    assert np.array_equal(np.flatnonzero(bad), np.r_[16:20, 20:36, 82:90])
    assert np.all(got[90] == 5.0) and np.isfinite(got[~bad]).all()
    assert status.item() == hl.STATUS_BAD_INDEX
    hl.kv_read(gpu.cache, 0, gpu.batch(tables[2:], lens[2:] - 20, batch([20])), out, None, status=status)
    assert status.item() == 0


@pytest.mark.parametrize("dim,block", [(64, 16), (96, 128), (256, 32)])
def test_read(hl, dev, dim, block):
    import torch

    heads, rng = 3, np.random.default_rng(dim)
    cache = Cache(20, 2, heads, dim, block)
    cache.fill(rng)
    gpu = OnGpu(hl, dev, cache)
    lens, rows = np.array([2 * block + 3, 0, 5, block]), np.array([block + 9, 2, 8, 1])  # two, and three rows before position 0
    tables = tables_for(rng, lens, block, 20, 3)
    starts = batch(rows) + 1
    k = torch.full((int(starts[-1]) + 1, heads, dim), 9.0, device=dev)
    v = torch.full((heads, int(starts[-1]) + 1, dim), 9.0, device=dev)  # [head][row][dim]
    hl.kv_read(gpu.cache, 1, gpu.batch(tables, lens, starts, len(k)), k, v, v_stride=dim, v_head_stride=len(k) * dim)
    k, v = k.cpu().numpy(), v.cpu().numpy().transpose(1, 0, 2)
    for s, (n, r) in enumerate(zip(lens, rows)):
        kk, vv = (x.transpose(1, 0, 2).astype(np.float32) for x in cache.tokens(tables[s], n, 1))
        pad = np.zeros((max(r - n, 0), heads, dim), dtype=np.float32)
        assert np.array_equal(k[starts[s]:starts[s + 1]], np.concatenate([pad, kk[max(n - r, 0):]]))
        assert np.array_equal(v[starts[s]:starts[s + 1]], np.concatenate([pad, vv[max(n - r, 0):]]))
    for x in (k, v):
        assert np.all(x[0] == 9.0) and np.all(x[-1] == 9.0)


def test_far_pages(hl, dev):
    """Pages whose bytes lie past 4 GiB of the pool."""
    import torch

    dim, block, heads, layers = 256, 128, 8, 16
    cache = Cache(2, layers, heads, dim, block)
    per = cache.bytes.shape[1]
    n_pages = (5 << 30) // per + 1
    pool = torch.zeros((n_pages, per), dtype=torch.uint8, device=dev)
    rng = np.random.default_rng(1)
    k, kx = to_type(rng.standard_normal((150, heads, dim)), BF16, dev)
    v, vx = to_type(rng.standard_normal((150, heads, dim)), BF16, dev)
    far = np.array([[n_pages - 1, n_pages - 2]], dtype=np.int32)
    c = hl.KvCache(pool, n_pages, layers, heads, dim, block)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    b = hl.KvBatch(ints(far), 2, ints([150]), ints([0, 150]), 1, 150)
    hl.kv_write(BF16, c, 15, b, k, v)
    write_ref(cache, 15, np.array([[1, 0]], dtype=np.int32), np.array([150]), batch([150]), kx, vx)
    got = Cache(*cache.geometry)
    got.bytes[:] = pool[-2:].cpu().numpy()
    assert np.array_equal(got.bytes, cache.bytes)
    assert not pool[:-2].any()
