"""PARTIAL_ROPE on the GPU against the rotation in 64 bits."""
import numpy as np
import pytest

from kv_helpers import BF16, F16, F32, HALF_LEAST, HALF_STEP, TYPE_NAMES, to_type

pytestmark = pytest.mark.gpu


def rope_ref(x, pos, freqs, rot, pairs, factor):
    """(rotated, |x| + |y| of each rotated element's pair) in 64 bits; x: [token, head, dim]."""
    angle = pos.astype(np.float64)[:, None] * freqs
    c, s = np.cos(angle)[:, None] * factor, np.sin(angle)[:, None] * factor
    i = np.arange(rot // 2)
    a, b = (i, i + rot // 2) if pairs == 0 else (2 * i, 2 * i + 1)
    out, reach = x.copy(), np.zeros_like(x)
    out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    reach[..., a] = reach[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return out, reach


def check(t, got, x, pos, freqs, rot, pairs, factor):
    want, reach = rope_ref(x, pos, freqs, rot, pairs, factor)
    # cos and sin: within 2 units of 2^-24 of the reduced angle's rounding and 2 of the functions', one for the
    # factor and one for each product and the sum; the angle itself is off by up to 2^-52 of its size in both
    angle = np.abs(pos.astype(np.float64)).max() * np.abs(freqs).max()  # in 64 bits: |-2^31| is no int32
    tol = reach * abs(factor) * (8 * 2.0 ** -24 + angle * 2.0 ** -51) + HALF_STEP[t] * np.abs(want) * 1.01 + HALF_LEAST[t] + 1e-37
    tol[reach == 0] = np.where(want[reach == 0] == x[reach == 0], 1e-45, 1)  # copied elements
    err = np.abs(got - want)
    assert np.all(err <= tol), f"{err.max()} at {np.unravel_index(np.argmax(err - tol), err.shape)}"
    same = np.arange(x.shape[-1]) >= rot
    assert np.array_equal(got[..., same], x[..., same])


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=lambda t: TYPE_NAMES[t])
@pytest.mark.parametrize("pairs", [0, 1])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot", [(1, 24, 4, 256, 64), (5, 3, 1, 96, 96), (33, 7, 2, 80, 20), (130, 8, 0, 128, 128),
                                                     (3, 1, 1, 70, 2), (2, 2, 1, 576, 512), (700, 5, 5, 64, 32)])
def test_rope(hl, dev, t, pairs, tokens, heads, kv, dim, rot):
    import torch

    print("[case] rope", TYPE_NAMES[t], pairs, tokens, heads, kv, dim, rot, flush=True)
    rng = np.random.default_rng(tokens + heads + rot + pairs)
    freqs, _ = hl.rope_freqs(rot, 1e6, scaling=hl.RopeScaling.NTK, scale=2.0)
    pos = rng.integers(0, 1 << 20, tokens).astype(np.int32)
    q, qx = to_type(rng.standard_normal((tokens, heads, dim)), t, dev)
    k, kx = to_type(rng.standard_normal((tokens, kv, dim)), t, dev)
    p, f = torch.from_numpy(pos).to(dev), torch.from_numpy(freqs).to(dev)
    qo, ko = torch.full_like(q, 7), torch.full_like(k, 7)
    hl.rope(t, p, f, tokens, dim, rot, q, qo, heads, k=k if kv else None, k_out=ko if kv else None, n_kv_heads=kv, pairs=pairs, factor=1.25)
    check(t, qo.double().cpu().numpy(), qx, pos, freqs, rot, pairs, 1.25)
    check(t, ko.double().cpu().numpy(), kx, pos, freqs, rot, pairs, 1.25)
    # in place, bitwise the same
    hl.rope(t, p, f, tokens, dim, rot, q, q, heads, k=k if kv else None, k_out=k if kv else None, n_kv_heads=kv, pairs=pairs, factor=1.25)
    assert torch.equal(q, qo) and torch.equal(k, ko)


@pytest.mark.parametrize("pairs", [0, 1])
@pytest.mark.parametrize("pos", [0, 1, -1, -12345, (1 << 20) + 3, (1 << 31) - 1, -(1 << 31)])
def test_rope_positions(hl, dev, pairs, pos):
    import torch

    dim = rot = 128
    freqs, _ = hl.rope_freqs(rot, 1e4)
    rng = np.random.default_rng(abs(pos) % 1000)
    q, qx = to_type(rng.standard_normal((1, 2, dim)), F32, dev)
    p = np.array([pos], dtype=np.int32)
    out = torch.empty_like(q)
    hl.rope(F32, torch.from_numpy(p).to(dev), torch.from_numpy(freqs).to(dev), 1, dim, rot, q, out, 2, pairs=pairs)
    check(F32, out.double().cpu().numpy(), qx, p, freqs, rot, pairs, 1.0)
    if pos == 0:
        assert torch.equal(out, q)


@pytest.mark.parametrize("t", [F32, BF16], ids=lambda t: TYPE_NAMES[t])
def test_rope_of_a_row_fused_projection(hl, dev, t):
    """q and k rotated in place where they lie side by side in the projection's rows, between v and padding that stay;
    and from [head][token][dim] to the dense layout, from an odd offset."""
    import torch

    tokens, heads, kv, dim, rot = 9, 6, 2, 64, 32
    row = (heads + 2 * kv) * dim + 3
    rng = np.random.default_rng(5)
    x, xx = to_type(rng.standard_normal((tokens, row)), t, dev)
    before = x.clone()
    freqs, _ = hl.rope_freqs(rot, 1e4)
    pos = np.arange(100, 100 + tokens, dtype=np.int32)
    p, f = torch.from_numpy(pos).to(dev), torch.from_numpy(freqs).to(dev)
    q, k = x[:, :heads * dim], x[:, heads * dim:]
    hl.rope(t, p, f, tokens, dim, rot, q, q, heads, k=k, k_out=k, n_kv_heads=kv, q_stride=row, q_out_stride=row, k_stride=row, k_out_stride=row)
    check(t, x[:, :heads * dim].double().cpu().numpy().reshape(tokens, heads, dim), xx[:, :heads * dim].reshape(tokens, heads, dim), pos, freqs, rot, 0, 1.0)
    kk = slice(heads * dim, (heads + kv) * dim)
    check(t, x[:, kk].double().cpu().numpy().reshape(tokens, kv, dim), xx[:, kk].reshape(tokens, kv, dim), pos, freqs, rot, 0, 1.0)
    assert torch.equal(x[:, (heads + kv) * dim:], before[:, (heads + kv) * dim:])

    y, yx = to_type(rng.standard_normal(1 + heads * tokens * dim), t, dev)
    out = torch.full((tokens + 1, heads, dim), 3.0, dtype=y.dtype, device=dev)
    hl.rope(t, p, f, tokens, dim, rot, y[1:], out, heads, q_stride=dim, q_head_stride=tokens * dim, pairs=1)
    want = yx[1:].reshape(heads, tokens, dim).transpose(1, 0, 2)
    check(t, out[:tokens].double().cpu().numpy(), np.ascontiguousarray(want), pos, freqs, rot, 1, 1.0)
    assert torch.all(out[tokens] == 3.0)


def test_rope_nothing(hl, dev):
    """No tokens, or no heads: nothing is read or written."""
    hl.rope(F32, 0, 0, 0, 128, 128, 0, 0, 4)
    hl.rope(F32, 0, 0, 5, 128, 128, 0, 0, 0)


@pytest.mark.parametrize("tokens,heads,kv", [((1 << 24) + 3, 1, 0), (2, 65535, 65535)])
def test_rope_sizes_past_a_grid(hl, dev, tokens, heads, kv):
    """More tokens than a launch's grid has threads for, more heads than it has rows."""
    import torch

    print("[case] rope past a grid", tokens, heads, kv, flush=True)
    g = torch.Generator(device=dev).manual_seed(5)
    q = torch.randn(tokens, heads, 2, device=dev, generator=g).half()
    k = torch.randn(tokens, kv, 2, device=dev, generator=g).half()
    pos = torch.randint(0, 1 << 16, (tokens,), device=dev, generator=g, dtype=torch.int32)
    freqs = torch.tensor([0.37], dtype=torch.float64, device=dev)
    qo, ko = torch.full_like(q, 7), torch.full_like(k, 7)
    hl.rope(F16, pos, freqs, tokens, 2, 2, q, qo, heads, k=k if kv else None, k_out=ko if kv else None, n_kv_heads=kv)
    angle = (pos.double() * 0.37)[:, None]
    for x, y in ((q, qo), (k, ko)):
        a, b = x[..., 0].double(), x[..., 1].double()
        c, s = angle.cos(), angle.sin()
        # as check() has it: the angle in 64 bits, sine and cosine and the products in 32, the result in 16
        reach = (a.abs() + b.abs()) * (8 * 2.0 ** -24 + 2.0 ** 16 * 0.37 * 2.0 ** -51) + HALF_LEAST[F16]
        for got, want in ((y[..., 0], a * c - b * s), (y[..., 1], b * c + a * s)):
            assert bool(((got.double() - want).abs() <= reach + want.abs() * HALF_STEP[F16] * 1.01).all())
