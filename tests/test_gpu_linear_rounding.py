"""Linear attention's outputs are rounded to their type once: products whose sums are exact in 32 bits come out as those sums, rounded."""
import pytest

from kv_helpers import BF16, F16, F32, TYPE_NAMES, torch_type

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("t", [F32, F16, BF16], ids=lambda t: TYPE_NAMES[t])
# rows of a sequence (steps, chunks, segments of chunks), heads, k_dim, v_dim: 64, 96 and 128 columns a workgroup
SHAPES = pytest.mark.parametrize("rows,heads,kd,vd", [(3, 4, 128, 128), (40, 4, 64, 128), (40, 4, 192, 96), (40, 144, 128, 128), (70, 144, 96, 128), (40, 72, 256, 256), (600, 144, 128, 128)])


def run(hl, dev, t, q, k, v, state, scale):
    """out of one sequence without decays; its state is updated in place."""
    import torch

    rows, heads, kd = q.shape
    out, ints = torch.full_like(v, 9.0), lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    batch = hl.LinearBatch(ints([0]), ints([0, rows]), 1, rows, rows)
    hl.linear_attention(t, hl.LinearState(state, 1, heads, kd, v.shape[-1]), batch, q, k, v, out, torch.zeros(heads, device=dev), heads, decay_per_head=True, scale=scale)
    return out


def picks(dev, t, rows, heads, kd):
    """q with a single 1 a row and head, and where it is."""
    import torch

    at = (torch.arange(rows, device=dev)[:, None] * 7 + torch.arange(heads, device=dev) * 5) % kd
    return torch.nn.functional.one_hot(at, kd).to(torch_type(t)), at


@TYPES
@SHAPES
def test_a_row_of_the_state(hl, dev, t, rows, heads, kd, vd):
    """k is zero, and q picks a row of the state: out is that row, each number rounded to the type once."""
    import torch

    g = torch.Generator(device=dev).manual_seed(rows + kd)
    state = torch.randn(1, heads, kd, vd, device=dev, generator=g)
    q, at = picks(dev, t, rows, heads, kd)
    v = torch.randn(rows, heads, vd, device=dev, generator=g).to(q.dtype)
    before = state.clone()
    out = run(hl, dev, t, q, torch.zeros_like(q), v, state, 1.0)
    want = before[0, torch.arange(heads, device=dev), at].to(q.dtype)
    assert torch.equal(out, want), f"{int((out != want).sum())} of {out.numel()}"
    assert torch.equal(state, before)


@TYPES
@SHAPES
def test_one_token_a_column(hl, dev, t, rows, heads, kd, vd):
    """Column c of v is 1 in row c alone, and q picks an element of k: out[i][c] is k[c]'s element times the scale, rounded to 32 bits, then to the
    type, for c <= i, and 0 behind."""
    import torch

    g = torch.Generator(device=dev).manual_seed(rows + kd)
    q, at = picks(dev, t, rows, heads, kd)
    k = torch.randn(rows, heads, kd, device=dev, generator=g).to(q.dtype)
    v = torch.zeros(rows, heads, vd, dtype=q.dtype, device=dev)
    n = min(rows, vd)
    v[torch.arange(n), :, torch.arange(n)] = 1
    scale = torch.tensor(0.5 ** 0.5)  # as it is held in 32 bits
    out = run(hl, dev, t, q, k, v, torch.zeros(1, heads, kd, vd, device=dev), float(scale))
    picked = k.float()[:n].permute(1, 2, 0)[torch.arange(heads, device=dev), at]  # [row, head, token]
    want = torch.zeros_like(out)
    want[..., :n] = (picked * scale.to(dev)).to(q.dtype) * (torch.arange(n, device=dev) <= torch.arange(rows, device=dev)[:, None])[:, None]
    assert torch.equal(out, want), f"{int((out != want).sum())} of {out.numel()}"
