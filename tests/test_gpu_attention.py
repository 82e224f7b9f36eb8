"""ATTENTION over the 8-bit paged cache on the GPU against the definition in 64 bits."""
import numpy as np
import pytest

from kv_helpers import BF16, F16, F32, TYPE_NAMES, Cache, attention_bound, attention_ref, batch, tables_for, to_type
from test_gpu_kv_cache import OnGpu

pytestmark = pytest.mark.gpu


def setup(hl, dev, rng, lens, heads_kv, dim, block, layers=1, spare=3, clean=False):
    """A filled cache, its tables and its copy on the GPU, where every byte that no token owns is a code of -128 or a
    scale of NaN: pages of no sequence, and tokens behind a sequence's end."""
    lens = np.asarray(lens)
    n_pages = int(sum(-(-n // block) for n in lens)) + spare
    cache = Cache(n_pages, layers, heads_kv, dim, block)
    cache.fill(rng)
    tables = tables_for(rng, lens, block, n_pages, max(1, int(max(-(-n // block) for n in lens))), stray=n_pages + 5)
    if not clean:
        used = set()
        scales = cache.scales.copy()
        for s, n in enumerate(lens):
            used |= set(tables[s, :-(-n // block)].tolist())
            if n % block:
                for layer in range(layers):
                    cache.k_codes(tables[s, n // block], layer)[:, n % block:] = -128
                    cache.v_codes(tables[s, n // block], layer)[:, :, n % block:] = -128
        scales[[p for p in range(n_pages) if p not in used]] = np.nan
        cache.set_scales(scales)
    return cache, tables, OnGpu(hl, dev, cache)


def run(hl, dev, gpu, cache, tables, lens, rows, t, heads, q, layer=0, window=0, scale=0.0, starts=None, n_rows=None, **kw):
    """The kernel's out, checked against the definition; q: [row, head, dim]."""
    import torch

    starts = batch(rows) if starts is None else starts
    qd, qx = to_type(q, t, dev)
    out = torch.full_like(qd, 5.0)
    status = torch.full((1,), 77, dtype=torch.int32, device=dev)
    hl.attention(t, gpu.cache, layer, gpu.batch(tables, lens, starts, len(q) if n_rows is None else n_rows, **kw), qd, out, heads, window=window,
                 scale=scale, status=status)
    got = out.double().cpu().numpy()
    assert status.item() == 0
    check(t, got, cache, layer, tables, lens, starts, qx, window, scale or None)
    return got


def check(t, got, cache, layer, tables, lens, starts, qx, window, scale):
    want, weight, reach = attention_ref(cache, layer, tables, lens, starts, qx, window, scale)
    vmax = float(np.nan_to_num(cache.scales[:, layer, 1]).max()) * 127
    tol = attention_bound(t, cache.dim, int(max(lens, default=0)), want, weight, reach, vmax)
    mine = slice(int(starts[0]), int(starts[-1]))
    if t == F16:  # values past its largest number, 65504, round to infinity
        over = np.abs(want) + tol >= 65504
        assert np.all(np.sign(got[over]) == np.sign(want[over])) and np.all(np.abs(got[over]) >= 65504 - 2 * tol[over])
        got, want = np.where(over, 0, got), np.where(over, 0, want)
    err = np.abs(got - want)[mine]
    assert np.all(err <= tol[mine]), f"{err.max()} of {np.abs(want).max()}, {(err / tol[mine]).max()} times the bound, {np.isnan(got[mine]).sum()} NaN"
    assert np.all(got[:mine.start] == 5.0) and np.all(got[mine.stop:] == 5.0)  # rows of no sequence


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=lambda t: TYPE_NAMES[t])
@pytest.mark.parametrize("dim,block,kv,group", [(64, 16, 2, 4), (96, 32, 1, 7), (128, 64, 2, 1), (192, 128, 1, 5), (256, 16, 4, 6), (128, 16, 1, 20)])
def test_one_row_each(hl, dev, t, dim, block, kv, group):
    """The decode form: a token per sequence, lengths around the step of 64, the pages and zero."""
    print("[case] attention step", TYPE_NAMES[t], dim, block, kv, group, flush=True)
    rng = np.random.default_rng(dim + block + t)
    lens = np.array([1, 2, 15, 16, 17, 63, 64, 65, 128, 129, 300, 777])
    cache, tables, gpu = setup(hl, dev, rng, lens, kv, dim, block, layers=2)
    q = rng.standard_normal((len(lens), kv * group, dim)) * 2
    run(hl, dev, gpu, cache, tables, lens, np.ones(len(lens), int), t, kv * group, q, layer=1, max_rows=1)


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=lambda t: TYPE_NAMES[t])
@pytest.mark.parametrize("dim,block,kv,group,window", [(64, 16, 2, 3, 0), (128, 32, 1, 4, 33), (96, 16, 2, 2, 1), (256, 64, 1, 6, 100), (192, 16, 1, 1, 0),
                                                       (128, 64, 2, 8, 0)])
def test_ragged_rows(hl, dev, t, dim, block, kv, group, window):
    """Verify steps, chunks and prompts in one batch: rows that see nothing (more rows than tokens), sequences without
    rows, windows that begin inside a page."""
    print("[case] attention ragged", TYPE_NAMES[t], dim, block, kv, group, window, flush=True)
    rng = np.random.default_rng(dim + block + t + window)
    lens, rows = np.array([70, 0, 5, 131, 16, 200, 1, 0]), np.array([70, 0, 8, 4, 1, 37, 1, 3])
    cache, tables, gpu = setup(hl, dev, rng, lens, kv, dim, block)
    q = rng.standard_normal((int(rows.sum()), kv * group, dim)) * 3
    got = run(hl, dev, gpu, cache, tables, lens, rows, t, kv * group, q, window=window)
    starts = batch(rows)
    assert np.all(got[starts[2]:starts[2] + 3] == 0) and np.all(got[starts[7]:] == 0)


@pytest.mark.parametrize("t", [F32, BF16], ids=lambda t: TYPE_NAMES[t])
@pytest.mark.parametrize("dim,rows,length,window", [(128, 1, 20011, 0), (256, 3, 9000, 0), (64, 1, 30000, 5000), (128, 150, 3001, 0), (256, 260, 700, 0),
                                                    (96, 90, 1500, 200)])
def test_long(hl, dev, t, dim, rows, length, window):
    """Long caches, split over workgroups; long chunks."""
    print("[case] attention long", TYPE_NAMES[t], dim, rows, length, window, flush=True)
    rng = np.random.default_rng(length)
    lens = np.array([length, 40])
    cache, tables, gpu = setup(hl, dev, rng, lens, 1, dim, 32)
    q = rng.standard_normal((rows + 1, 3, dim)) * 2
    run(hl, dev, gpu, cache, tables, lens, np.array([rows, 1]), t, 3, q, window=window)


@pytest.mark.parametrize("t", [F32, BF16], ids=lambda t: TYPE_NAMES[t])
@pytest.mark.parametrize("seqs", [64, 65, 129, 300])
def test_many_sequences(hl, dev, t, seqs):
    """More sequences than a wave has lanes, empty ones among them, long ones split over several workgroups."""
    print("[case] attention", TYPE_NAMES[t], seqs, "sequences", flush=True)
    rng = np.random.default_rng(seqs)
    rows, lens = rng.integers(0, 3, seqs), rng.integers(0, 40, seqs)
    lens[rng.integers(0, seqs, 4)] = 1500
    lens = np.maximum(lens, rows)
    cache, tables, gpu = setup(hl, dev, rng, lens, 2, 64, 32)
    q = rng.standard_normal((int(rows.sum()), 6, 64))
    run(hl, dev, gpu, cache, tables, lens, rows, t, 6, q, max_rows=2, max_kv=1500)
    run(hl, dev, gpu, cache, tables, lens, rows, t, 6, q)


def test_launch_hints_are_only_hints(hl, dev):
    """max_rows and max_kv smaller than the truth: the same values."""
    rng = np.random.default_rng(2)
    lens, rows = np.array([500, 90]), np.array([75, 2])
    cache, tables, gpu = setup(hl, dev, rng, lens, 2, 64, 16)
    q = rng.standard_normal((77, 4, 64))
    run(hl, dev, gpu, cache, tables, lens, rows, F32, 4, q, max_rows=1, max_kv=64)
    run(hl, dev, gpu, cache, tables, lens, rows, F32, 4, q, max_rows=3, max_kv=130)


@pytest.mark.parametrize("rows", [1, 3, 40, 200])
def test_strides_and_stray_rows(hl, dev, rows):
    """q inside a row-fused projection at an odd offset, out as [head][row][dim]; rows of no sequence stay."""
    import torch

    rng = np.random.default_rng(rows)
    dim, kv, heads = 64, 2, 6
    lens = np.array([rows + 30, rows])
    cache, tables, gpu = setup(hl, dev, rng, lens, kv, dim, 16)
    starts = np.array([2, 2 + rows, 2 + 2 * rows], dtype=np.int32)
    n = 2 * rows + 4
    wide = heads * dim + 7
    x = rng.standard_normal((n, wide))
    x[:2], x[2 + 2 * rows:] = np.nan, np.inf
    xd, xx = to_type(x, BF16, dev)
    out = torch.full((heads, n, dim), 5.0, dtype=torch.bfloat16, device=dev)
    hl.attention(BF16, gpu.cache, 0, gpu.batch(tables, lens, starts, n), xd[:, 3:], out, heads, q_stride=wide, out_stride=dim, out_head_stride=n * dim)
    got = out.double().cpu().numpy().transpose(1, 0, 2)
    check(BF16, got, cache, 0, tables, lens, starts, xx[:, 3:3 + heads * dim].reshape(n, heads, dim), 0, None)


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=lambda t: TYPE_NAMES[t])
@pytest.mark.parametrize("rows", [2, 160])
def test_wide_ranges(hl, dev, t, rows):
    """Blocks of V and K whose scales lie far apart, all-zero blocks, rows of q from tiny to large, a negative and a
    large scale on the scores."""
    rng = np.random.default_rng(rows)
    dim, block, kv, group = 64, 16, 2, 2
    lens = np.array([400, rows])
    cache, tables, gpu = setup(hl, dev, rng, lens, kv, dim, block, clean=True)
    s = cache.scales.copy()
    s[:, :, 1] *= 2.0 ** rng.integers(-30, 30, s[:, :, 1].shape)
    s[:, :, 0] *= 2.0 ** rng.integers(-6, 2, s[:, :, 0].shape)
    zero = rng.random(s.shape) < 0.2
    s[zero] = 0
    cache.codes[zero] = 0
    cache.set_scales(s)
    gpu = OnGpu(hl, dev, cache)
    q = rng.standard_normal((2 * rows, kv * group, dim)) * 2.0 ** rng.integers(-10, 2, (2 * rows, kv * group, 1))
    q[0, 0] = 0
    run(hl, dev, gpu, cache, tables, lens, np.array([rows, rows]), t, kv * group, q)
    run(hl, dev, gpu, cache, tables, lens, np.array([rows, rows]), t, kv * group, q, scale=-0.3)
    run(hl, dev, gpu, cache, tables, lens, np.array([rows, rows]), t, kv * group, q * 2, scale=1.0)


@pytest.mark.parametrize("rows", [1, 6, 100])
def test_not_finite(hl, dev, rows):
    """A row of q that is not finite is NaN and no other is; a NaN block reaches the rows that see it only; so does a page
    out of range, which is reported."""
    import torch

    rng = np.random.default_rng(rows)
    dim, block, heads = 128, 16, 2
    lens, counts = np.array([rows + 40, rows + 64, rows + 3]), np.array([rows] * 3)
    cache, tables, gpu = setup(hl, dev, rng, lens, 1, dim, block)
    cache.set_scales(np.where(np.arange(cache.n_pages)[:, None, None, None] == tables[1, 3], np.nan, cache.scales))  # tokens 48..63
    gpu = OnGpu(hl, dev, cache)
    q = rng.standard_normal((3 * rows, heads, dim)).astype(np.float32)
    q[0, 1, 5], q[rows - 1, 0, 0] = np.nan, np.inf
    bad = tables.copy()
    bad[2, 0] = cache.n_pages
    out, status = torch.full((3 * rows, heads, dim), 5.0, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    qd = torch.from_numpy(q).to(dev)
    hl.attention(F32, gpu.cache, 0, gpu.batch(bad, lens, batch(counts)), qd, out, heads, window=0, status=status)
    nan = out.isnan().cpu().numpy()
    want = np.zeros((3 * rows, heads), dtype=bool)
    want[0, 1] = want[rows - 1, 0] = True
    want[rows:] = True  # every row sees the NaN block, and the missing page
    assert np.array_equal(nan.all(2), want) and np.array_equal(nan.any(2), want)
    assert status.item() == hl.STATUS_BAD_INDEX
    # a window that ends before the NaN block begins sees none of it
    hl.attention(F32, gpu.cache, 0, gpu.batch(bad[1:2], lens[1:2], batch(counts[1:2])), qd[rows:2 * rows], out, heads, window=1, status=status)
    assert not out[:rows].isnan().any() and status.item() == 0


def test_lengths_past_the_table(hl, dev):
    """A length that the table has no room for: NaN and a status, after no more work than the table's."""
    import torch

    rng = np.random.default_rng(4)
    cache, tables, gpu = setup(hl, dev, rng, [64, 64, 64, 20], 1, 64, 16)
    q = torch.randn((5, 2, 64), device=dev)
    for window in (0, 7):
        out, status = torch.full_like(q, 5.0), torch.zeros(1, dtype=torch.int32, device=dev)
        hl.attention(F32, gpu.cache, 0, gpu.batch(tables, np.array([65, (1 << 31) - 1, 64, -5]), batch([1, 1, 2, 1])), q, out, 2, window=window, status=status)
        assert out[:2].isnan().all() and out[2:4].isfinite().all() and torch.all(out[4] == 0)
        assert status.item() == hl.STATUS_BAD_INDEX


@pytest.mark.parametrize("t,rows,length", [(F32, 1, 5000), (BF16, 1, 5000), (F32, 5, 3000), (BF16, 300, 900)])
def test_repeats_and_replays_bitwise(hl, dev, t, rows, length):
    """The same call twice, with its own workspace, and captured and replayed with other lengths between: bitwise the eager
    results."""
    import torch

    rng = np.random.default_rng(6)
    cache, tables, gpu = setup(hl, dev, rng, [length], 2, 128, 16, clean=True)
    heads = 8
    q, _ = to_type(rng.standard_normal((rows, heads, 128)), t, dev)
    b = gpu.batch(tables, np.array([length]), batch([rows]), max_rows=rows, max_kv=length)
    out, again = torch.empty_like(q), torch.empty_like(q)
    call = lambda o, **kw: hl.attention(t, gpu.cache, 0, b, q, o, heads, **kw)  # noqa: E731
    call(out)
    call(again)
    assert torch.equal(out, again)
    need = hl.attention_workspace(t, gpu.cache, 0, b, q, out, heads)
    ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device=dev)
    call(again, workspace=ws)
    assert torch.equal(out, again)
    small = torch.empty(max(need // 2 // 16 * 16, 16), dtype=torch.uint8, device=dev)
    call(again, workspace=small)  # fewer splits: within rounding
    assert torch.allclose(out.float(), again.float(), rtol=2.0 ** -6, atol=2.0 ** -8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(again)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(again)
    for n in (length, length - 100, rows, length):
        b.kv_lens.fill_(n)
        call(out)
        torch.cuda.synchronize()
        again.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, again)
    with torch.cuda.stream(s):
        hl.stream_release()


def test_capture_without_a_workspace(hl, dev):
    """The first call of a stream under capture, and two graphs with workspaces of their own replayed at once."""
    import torch

    rng = np.random.default_rng(8)
    cache, tables, gpu = setup(hl, dev, rng, [3000, 2000], 1, 64, 16)
    q, qx = to_type(rng.standard_normal((2, 4, 64)), F32, dev)
    lens, starts = np.array([3000, 2000]), batch([1, 1])
    b = gpu.batch(tables, lens, starts)
    outs = [torch.full_like(q, 5.0) for _ in range(3)]
    need = hl.attention_workspace(F32, gpu.cache, 0, b, q, outs[0], 4)
    assert need > 0
    torch.cuda.synchronize()
    graphs, streams, keep = [], [torch.cuda.Stream() for _ in range(3)], []
    for i, (s, o) in enumerate(zip(streams, outs)):
        g = torch.cuda.CUDAGraph()
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if i else None
        keep.append(ws)
        torch.cuda.synchronize()
        with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
            hl.attention(F32, gpu.cache, 0, b, q, o, 4, workspace=ws)
        graphs.append(g)
    for _ in range(5):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o in outs:
        check(F32, o.double().cpu().numpy(), cache, 0, tables, lens, starts, qx, 0, None)
    assert torch.equal(outs[1], outs[2])


def test_far_pages(hl, dev):
    """Pages whose bytes lie past 4 GiB of the pool."""
    import torch

    dim, block, heads, layers = 256, 128, 8, 16
    rng = np.random.default_rng(1)
    small = Cache(2, layers, heads, dim, block)
    small.fill(rng)
    n_pages = (5 << 30) // small.bytes.shape[1] + 2
    pool = torch.zeros((n_pages, small.bytes.shape[1]), dtype=torch.uint8, device=dev)
    pool[-2:] = torch.from_numpy(small.bytes).to(dev)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    c = hl.KvCache(pool, n_pages, layers, heads, dim, block)
    for rows in (1, 200):
        lens, starts = np.array([201]), batch([rows])
        q, qx = to_type(rng.standard_normal((rows, heads, dim)), BF16, dev)
        out = torch.empty_like(q)
        hl.attention(BF16, c, 15, hl.KvBatch(ints([[n_pages - 1, n_pages - 2]]), 2, ints([201]), ints([0, rows]), 1, rows), q, out, heads)
        check(BF16, out.double().cpu().numpy(), small, 15, np.array([[1, 0]]), lens, starts, qx, 0, None)
