"""The 8-bit product's kernels at the sizes that choose them: every shape of tiles over many steps of K, and the kernels for few vectors over
many pieces of it, against the exact sums. That the sizes choose these shapes is checked in test_layer_plans_host.py."""
import pytest

from kv_helpers import BF16, F16, F32, HALF_LEAST, HALF_STEP, TYPE_NAMES, U, torch_type
from layer_helpers import padded

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("t", [F32, F16, BF16], ids=lambda t: TYPE_NAMES[t])

# fragments of a wave along the channels and the vectors; channels, columns, vectors
SHAPES = [((8, 4), 14556, 1300, 772), ((8, 4), 14557, 1301, 771), ((7, 4), 16500, 1459, 607), ((6, 4), 20698, 1300, 393), ((5, 4), 16885, 1460, 389), ((8, 3), 12509, 1300, 782),
          ((7, 3), 10371, 1461, 769), ((6, 3), 16752, 1300, 193), ((4, 3), 16444, 1300, 131), ((4, 2), 12475, 1170, 133), ((3, 2), 16420, 1460, 65),
          ((2, 2), 8233, 1170, 65), ((4, 1), 511, 1170, 3261), ((3, 1), 16493, 1300, 17), ((2, 1), 8561, 1300, 17), ((1, 1), 60, 1461, 33), ((1, 1), 6143, 5119, 61)]
# channels and columns of the calls whose rows are compared, and their vectors
BESIDE, BATCHES = (16500, 1300), (1, 5, 16, 17, 32, 33, 65, 100, 131, 140, 193, 256, 300, 389, 500, 607, 700, 772)


def operands(dev, rows, cols, n_vec, seed):
    """Codes over their whole range, w's padding holding anything, scales of all sizes."""
    import torch

    g = torch.Generator(device=dev).manual_seed(seed)
    w, x = (torch.randint(-128, 128, (n, padded(cols)), dtype=torch.int8, device=dev, generator=g) for n in (rows, n_vec))
    x[:, cols:] = 0
    ws, xs = (torch.randn(n, device=dev, generator=g).exp() / 3e3 for n in (rows, n_vec))
    return w, ws, x, xs


def check(t, y, w, ws, x, xs, cols):
    """y against the sums in 64 bits, which are exact: as layer_helpers.gemm_ref, on the device."""
    import torch

    want = torch.matmul(x[:, :cols].double(), w[:, :cols].double().t()) * (xs.double()[:, None] * ws.double())
    off, tol = (y.double() - want).abs(), want.abs() * (3.01 * U + HALF_STEP[t] * 1.01) + HALF_LEAST[t] + 2.0 ** -148
    bad = ~(off <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {y.numel()}, {float((off / tol).max())} of the tolerance, first at {torch.nonzero(bad)[0].tolist()}"


def run(hl, dev, t, rows, cols, n_vec, operands, y_pad=0):
    import torch

    w, ws, x, xs = operands
    y = torch.full((n_vec, rows + y_pad), float("nan"), dtype=torch_type(t), device=dev)
    hl.gemm_i8(t, w, ws, x, xs, y, rows, cols, n_vec, y_stride=rows + y_pad)
    assert bool(torch.isnan(y[:, rows:]).all())
    return y[:, :rows]


@TYPES
@pytest.mark.parametrize("shape,rows,cols,n_vec", SHAPES, ids=lambda x: str(x).replace(" ", ""))
def test_tiles(hl, dev, t, shape, rows, cols, n_vec):
    print("[case] gemm_i8 tiles", TYPE_NAMES[t], shape, rows, cols, n_vec, flush=True)
    ops = operands(dev, rows, cols, n_vec, rows + cols)
    check(t, run(hl, dev, t, rows, cols, n_vec, ops), *ops, cols)
    # rows of y that begin anywhere are stored element by element
    check(t, run(hl, dev, t, rows, cols, n_vec, ops, y_pad=3), *ops, cols)


@TYPES
@pytest.mark.parametrize("rows", [100, 4096, 4097, 4500, 5120, 8191, 8200, 17408])
@pytest.mark.parametrize("cols,n_vec", [(3400, 1), (3391, 7), (5003, 16), (2048, 16)])
def test_few_vectors(hl, dev, t, rows, cols, n_vec):
    """One or two fragments of channels a workgroup, one to three workgroups a CU; a wave has many pieces of K, and what is left of it."""
    print("[case] gemm_i8 few", TYPE_NAMES[t], rows, cols, n_vec, flush=True)
    ops = operands(dev, rows, cols, n_vec, rows + cols)
    check(t, run(hl, dev, t, rows, cols, n_vec, ops), *ops, cols)


@TYPES
@pytest.mark.parametrize("rows,cols,n_vec", [(3000, 6500, 17), (4096, 5003, 32), (1000, 17408, 25)])
def test_two_fragments_of_vectors(hl, dev, t, rows, cols, n_vec):
    print("[case] gemm_i8 two fragments", TYPE_NAMES[t], rows, cols, n_vec, flush=True)
    ops = operands(dev, rows, cols, n_vec, rows + cols)
    check(t, run(hl, dev, t, rows, cols, n_vec, ops), *ops, cols)


@TYPES
def test_rows_are_the_same_in_every_shape(hl, dev, t):
    """A row of y is bitwise the same whichever kernel and shape of tiles makes it."""
    import torch

    rows, cols = BESIDE
    w, ws, x, xs = ops = operands(dev, rows, cols, max(BATCHES), 12)
    y = run(hl, dev, t, rows, cols, max(BATCHES), ops)
    check(t, y, *ops, cols)
    for n in BATCHES:
        for first in (0, max(BATCHES) - n):
            part = run(hl, dev, t, rows, cols, n, (w, ws, x[first:], xs[first:]))
            assert torch.equal(part, y[first:first + n]), (n, first)
