"""Rows in 8 bits and their products on the GPU: codes are the exact nearest integers, sums are exact."""
import numpy as np
import pytest

from kv_helpers import BF16, F16, F32, TYPE_NAMES, to_type, torch_type
from layer_helpers import gemm_ref, padded, quantized

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("t", [F32, F16, BF16], ids=lambda t: TYPE_NAMES[t])


def check_rows(codes, scales, x):
    want_codes, want_scales = quantized(x)
    assert np.array_equal(scales, want_scales, equal_nan=True)
    assert np.array_equal(codes, want_codes)


@TYPES
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 15), (5, 16), (2, 17), (7, 100), (4, 513), (33, 1024), (2, 5120), (600, 3001), (3, 17408), (2, 131071), (1, 40000)])
def test_quantize_rows(hl, dev, t, rows, cols):
    import torch

    print("[case] quantize_rows", TYPE_NAMES[t], rows, cols, flush=True)
    rng = np.random.default_rng(rows + cols)
    x, xx = to_type(rng.standard_normal((rows, cols)) * np.exp(3 * rng.standard_normal((rows, 1))), t, dev)
    codes = torch.full((rows, padded(cols) + 16), 77, dtype=torch.int8, device=dev)
    scales = torch.full((rows,), 3.0, device=dev)
    hl.quantize_rows(t, x, codes, scales, rows, cols, codes_stride=padded(cols) + 16)
    got = codes.cpu().numpy()
    check_rows(got[:, :padded(cols)], scales.cpu().numpy(), xx)
    assert np.all(got[:, padded(cols):] == 77)  # what lies between rows is left alone


@TYPES
def test_quantize_rows_ties_and_edges(hl, dev, t):
    """Quotients on and beside a half, rows of zeros, of one value, of the smallest and largest values, and with values that are not finite."""
    import torch

    rng = np.random.default_rng(11)
    cols = 333
    rows = [np.zeros(cols), np.full(cols, -2.5), np.r_[127.0, np.arange(cols - 1) % 255 / 2 - 63.5], np.r_[127.0, rng.integers(-126, 126, cols - 1) + 0.5],
            np.r_[254.0, rng.integers(-250, 250, cols - 1)], np.full(cols, 2.0 ** -24), rng.standard_normal(cols) * 3e4, np.r_[np.zeros(cols - 1), 1.0]]
    if t != F16:
        rows += [rng.standard_normal(cols) * 2.0 ** -75, rng.standard_normal(cols) * 2.0 ** -90, rng.standard_normal(cols) * 2.0 ** 120, np.full(cols, 2.0 ** -73.01)]
    for bad in (np.nan, np.inf, -np.inf):
        row = rng.standard_normal(cols)
        row[rng.integers(cols)] = bad
        rows.append(row)
    x, xx = to_type(np.stack(rows), t, dev)
    n = len(rows)
    codes, scales = torch.empty(n, padded(cols), dtype=torch.int8, device=dev), torch.empty(n, device=dev)
    hl.quantize_rows(t, x, codes, scales, n, cols)
    check_rows(codes.cpu().numpy(), scales.cpu().numpy(), xx)
    # rows that begin on any element
    wide, wx = to_type(rng.standard_normal(1 + n * 335), t, dev)
    hl.quantize_rows(t, wide[1:], codes, scales, n, cols, x_stride=335)
    check_rows(codes.cpu().numpy(), scales.cpu().numpy(), wx[1:].reshape(n, 335)[:, :cols])


def test_quantize_many_rows(hl, dev):
    """More rows than a launch has."""
    import torch

    rows, cols = (1 << 21) + 5, 20
    x = torch.randn(rows, cols, device=dev, dtype=torch.float32, generator=torch.Generator(device=dev).manual_seed(1)).half()
    codes, scales = torch.empty(rows, 32, dtype=torch.int8, device=dev), torch.empty(rows, device=dev)
    hl.quantize_rows(F16, x, codes, scales, rows, cols)
    for at in (slice(0, 3), slice((1 << 21) - 2, rows)):
        check_rows(codes[at].cpu().numpy(), scales[at].cpu().numpy(), x[at].double().cpu().numpy())


def product(hl, dev, t, rows, cols, n_vec, rng, w_pad=0, x_pad=0, y_pad=0, lo=-127):
    import torch

    ws, xs = padded(cols) + w_pad, padded(cols) + x_pad
    w = rng.integers(lo, 128, (rows, ws)).astype(np.int8)
    x = rng.integers(lo, 128, (n_vec, xs)).astype(np.int8)
    x[:, cols:padded(cols)] = 0  # w's padding holds anything
    wsc, xsc = (np.exp(rng.standard_normal(n)).astype(np.float32) / 3e3 for n in (rows, n_vec))
    wd, xd, wsd, xsd = (torch.from_numpy(v).to(dev) for v in (w, x, wsc, xsc))
    y = torch.full((n_vec, rows + y_pad), 5.0, dtype=torch_type(t), device=dev)
    hl.gemm_i8(t, wd, wsd, xd, xsd, y, rows, cols, n_vec, w_stride=ws, x_stride=xs, y_stride=rows + y_pad)
    got = y.double().cpu().numpy()
    want, tol = gemm_ref(t, w, wsc, x, xsc, cols)
    err = np.abs(got[:, :rows] - want)
    assert np.all(err <= tol), f"{(err / tol).max()} of the tolerance at {np.unravel_index(np.argmax(err / tol), err.shape)}"
    assert np.all(got[:, rows:] == 5.0)
    return y, (wd, wsd, xd, xsd)


# one vector to many, tiles that end inside, steps of K that end inside
SHAPES = [(1, 1, 1), (16, 64, 1), (17, 63, 2), (40, 256, 16), (100, 1000, 17), (64, 5120, 31), (33, 272, 33), (300, 528, 64), (257, 129, 65), (130, 2064, 100),
          (500, 384, 129), (1000, 512, 250), (257, 640, 257), (600, 1040, 513), (2100, 144, 300), (64, 17408, 3), (256, 4096, 256), (513, 4112, 511)]


@TYPES
@pytest.mark.parametrize("rows,cols,n_vec", SHAPES)
def test_gemm_i8(hl, dev, t, rows, cols, n_vec):
    print("[case] gemm_i8", TYPE_NAMES[t], rows, cols, n_vec, flush=True)
    product(hl, dev, t, rows, cols, n_vec, np.random.default_rng(rows + cols + n_vec))


@pytest.mark.parametrize("rows,cols,n_vec", [(70, 300, 5), (70, 300, 70), (300, 300, 300), (515, 1100, 515)])
def test_gemm_i8_strides(hl, dev, rows, cols, n_vec):
    """Rows apart, codes of -128, y in rows of an odd length: what lies between stays."""
    print("[case] gemm_i8 strides", rows, cols, n_vec, flush=True)
    rng = np.random.default_rng(rows)
    for t in (F32, BF16):
        product(hl, dev, t, rows, cols, n_vec, rng, w_pad=48, x_pad=16, y_pad=3, lo=-128)


@pytest.mark.parametrize("rows,n_vec", [((1 << 21) + 40, 3), ((1 << 21) + 40, 17), (24, (1 << 16) + 100), (4500, 70)])
def test_gemm_i8_past_a_launch(hl, dev, rows, n_vec):
    """More channels or vectors than a launch takes: the ends of both, and the seams."""
    import torch

    print("[case] gemm_i8 past a launch", rows, n_vec, flush=True)
    g = torch.Generator(device=dev).manual_seed(3)
    cols = 24
    w, x = (torch.randint(-127, 128, (n, 32), dtype=torch.int8, device=dev, generator=g) for n in (rows, n_vec))
    x[:, cols:] = 0
    ws, xs = (torch.rand(n, device=dev, generator=g) for n in (rows, n_vec))
    y = torch.full((n_vec, rows), float("nan"), dtype=torch.bfloat16, device=dev)
    hl.gemm_i8(BF16, w, ws, x, xs, y, rows, cols, n_vec)
    want = torch.matmul(x.float(), w.float().t()).double() * (xs.double()[:, None] * ws.double())
    assert bool(((y.double() - want).abs() <= want.abs() * (2.0 ** -8 * 1.01 + 2.0 ** -22)).all())


def test_gemm_i8_largest_sums(hl, dev):
    """The longest rows of the largest codes: the sum takes all of 32 bits."""
    import torch

    cols, rows = 131071, 20
    for n_vec in (1, 40, 300):
        w = torch.full((rows, padded(cols)), -128, dtype=torch.int8, device=dev)
        x = torch.full((n_vec, padded(cols)), -128, dtype=torch.int8, device=dev)
        x[:, cols:] = 0
        x[::2] = 127
        x[::2, cols:] = 0
        ones = torch.ones(max(rows, n_vec), device=dev)
        y = torch.empty(n_vec, rows, device=dev)
        hl.gemm_i8(F32, w, ones, x, ones, y, rows, cols, n_vec)
        want = np.where(np.arange(n_vec) % 2 == 0, -128 * 127 * cols, 128 * 128 * cols).astype(np.float32)
        assert np.array_equal(y.cpu().numpy(), np.repeat(want[:, None], rows, 1))


@TYPES
def test_gemm_i8_rows_do_not_depend_on_the_call(hl, dev, t):
    """A row of y is bitwise the same alone and beside any number of others, whichever kernel runs."""
    import torch

    rows, cols, n_vec = 520, 1296, 700
    y, (w, ws, x, xs) = product(hl, dev, t, rows, cols, n_vec, np.random.default_rng(2))
    for n in (1, 3, 20, 60, 64, 65, 128, 200, 256, 300, 512):
        part = torch.empty(n, rows, dtype=y.dtype, device=dev)
        hl.gemm_i8(t, w, ws, x[7:], xs[7:], part, rows, cols, n)
        assert torch.equal(part, y[7:7 + n]), n


def test_gemm_i8_of_bad_rows(hl, dev):
    """A row with a value that is not finite is NaN in y, and only it; zero rows are zeros."""
    import torch

    rows, cols, n_vec = 90, 200, 70
    x = torch.randn(n_vec, cols, device=dev)
    x[3, 17] = float("inf")
    x[5] = 0
    w, ws = torch.randint(-127, 128, (rows, padded(cols)), dtype=torch.int8, device=dev), torch.rand(rows, device=dev)
    codes, scales, y = torch.empty(n_vec, padded(cols), dtype=torch.int8, device=dev), torch.empty(n_vec, device=dev), torch.empty(n_vec, rows, device=dev)
    hl.quantize_rows(F32, x, codes, scales, n_vec, cols)
    hl.gemm_i8(F32, w, ws, codes, scales, y, rows, cols, n_vec)
    assert bool(torch.isnan(y[3]).all()) and bool((y[5] == 0).all())
    y[3] = 0
    assert bool(torch.isfinite(y).all())


def test_projection_of_quantized_operands(hl, dev):
    """Both operands made by quantize_rows: the product is near the one of the values that they stand for, exactly near."""
    import torch

    rows, cols, n_vec = 300, 1001, 90
    rng = np.random.default_rng(8)
    (x, xx), (w, wx) = to_type(rng.standard_normal((n_vec, cols)), BF16, dev), to_type(rng.standard_normal((rows, cols)) * 0.02, F32, dev)
    xc, wc = (torch.empty(n, padded(cols), dtype=torch.int8, device=dev) for n in (n_vec, rows))
    xs, ws, y = torch.empty(n_vec, device=dev), torch.empty(rows, device=dev), torch.empty(n_vec, rows, device=dev)
    hl.quantize_rows(BF16, x, xc, xs, n_vec, cols)
    hl.quantize_rows(F32, w, wc, ws, rows, cols)
    hl.gemm_i8(F32, wc, ws, xc, xs, y, rows, cols, n_vec)
    (xq, xsq), (wq, wsq) = quantized(xx), quantized(wx)
    want, tol = gemm_ref(F32, wq, wsq, xq, xsq, cols)
    assert np.all(np.abs(y.double().cpu().numpy() - want) <= tol)


def test_gemm_i8_captured(hl, dev):
    """Both calls captured on a side stream and replayed with other inputs, eager work between."""
    import torch

    rows, cols, n_vec = 130, 600, 9
    g = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(n_vec, cols, device=dev, generator=g)
    w, ws = torch.randint(-127, 128, (rows, padded(cols)), dtype=torch.int8, device=dev, generator=g), torch.rand(rows, device=dev, generator=g)
    codes, scales, y = torch.empty(n_vec, padded(cols), dtype=torch.int8, device=dev), torch.empty(n_vec, device=dev), torch.empty(n_vec, rows, device=dev)

    def step(codes, scales, y):
        hl.quantize_rows(F32, x, codes, scales, n_vec, cols)
        hl.gemm_i8(F32, w, ws, codes, scales, y, rows, cols, n_vec)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step(codes, scales, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step(codes, scales, y)
    for _ in range(3):
        x.copy_(torch.randn(n_vec, cols, device=dev, generator=g))
        c2, s2, y2 = torch.empty_like(codes), torch.empty_like(scales), torch.empty_like(y)
        step(c2, s2, y2)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, y2) and torch.equal(codes, c2)


@TYPES
@pytest.mark.parametrize("rows,cols,stride", [(700, 90, 91), (513, 1000, 1000), (900, 2040, 2051), (600, 2048, 2048), (515, 4111, 4111)])
def test_quantize_rows_of_one_wave(hl, dev, t, rows, cols, stride):
    """Many narrow rows, a wave each, and the first sizes past that; rows of zeros and of one NaN among them."""
    import torch

    rng = np.random.default_rng(cols)
    x, xx = to_type(rng.standard_normal((rows, stride)) * np.exp(2 * rng.standard_normal((rows, 1))), t, dev)
    x[5], xx[5] = 0, 0
    x[rows - 2, cols - 1] = float("nan")
    xx[rows - 2, cols - 1] = np.nan
    codes, scales = torch.full((rows, padded(cols)), 77, dtype=torch.int8, device=dev), torch.full((rows,), 3.0, device=dev)
    hl.quantize_rows(t, x, codes, scales, rows, cols, x_stride=stride)
    check_rows(codes.cpu().numpy(), scales.cpu().numpy(), xx[:, :cols])
