"""The heads' norms with the rotation on the GPU against the formula in 64 bits."""
import numpy as np
import pytest

from kv_helpers import BF16, F16, F32, TYPE_NAMES, to_type
from layer_helpers import norm_rope_ref

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("t", [F32, F16, BF16], ids=lambda t: TYPE_NAMES[t])


def check(t, got, x, w, eps, pos, freqs, rot, pairs, factor):
    want, tol = norm_rope_ref(t, x, w, eps, pos, freqs, rot, pairs, factor)
    err = np.abs(got - want)
    assert np.all(err <= tol), f"{(err / tol).max()} of the tolerance at {np.unravel_index(np.argmax(err / tol), err.shape)}"


@TYPES
@pytest.mark.parametrize("pairs", [0, 1])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot", [(1, 24, 4, 256, 64), (5, 3, 1, 96, 96), (33, 7, 2, 80, 20), (130, 8, 0, 128, 128), (3, 1, 1, 70, 2),
                                                     (2, 2, 1, 576, 512), (2, 1, 2, 1024, 512), (2, 3, 1, 1000, 40), (700, 5, 5, 64, 32), (9, 4, 1, 192, 96)])
def test_norm_rope(hl, dev, t, pairs, tokens, heads, kv, dim, rot):
    import torch

    print("[case] norm_rope", TYPE_NAMES[t], pairs, tokens, heads, kv, dim, rot, flush=True)
    rng = np.random.default_rng(tokens + heads + rot + pairs)
    freqs, _ = hl.rope_freqs(rot, 1e6, scaling=hl.RopeScaling.NTK, scale=2.0)
    pos = rng.integers(0, 1 << 20, tokens).astype(np.int32)
    q, qx = to_type(rng.standard_normal((tokens, heads, dim)) * 3, t, dev)
    k, kx = to_type(rng.standard_normal((tokens, kv, dim)) * 0.01, t, dev)
    qw, kw = ((1 + 0.3 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2))
    qwd, kwd, p, f = (torch.from_numpy(x).to(dev) for x in (qw, kw, pos, freqs))
    qo, ko = torch.full_like(q, 7), torch.full_like(k, 7)
    more = dict(q_norm=qwd, k=k if kv else None, n_kv_heads=kv, k_norm=kwd if kv else None, eps=1e-4, pairs=pairs, factor=1.25)
    hl.norm_rope(t, p, f, tokens, dim, rot, q, qo, heads, k_out=ko if kv else None, **more)
    check(t, qo.double().cpu().numpy(), qx, qw.astype(np.float64), 1e-4, pos, freqs, rot, pairs, 1.25)
    check(t, ko.double().cpu().numpy(), kx, kw.astype(np.float64), 1e-4, pos, freqs, rot, pairs, 1.25)
    # in place, bitwise the same
    hl.norm_rope(t, p, f, tokens, dim, rot, q, q, heads, k_out=k if kv else None, **more)
    assert torch.equal(q, qo) and torch.equal(k, ko)


@TYPES
def test_norm_of_one_part_only(hl, dev, t):
    """Without weights a part is rotated only, bitwise as rope does it."""
    import torch

    tokens, heads, kv, dim, rot = 17, 6, 2, 128, 64
    rng = np.random.default_rng(3)
    freqs = torch.from_numpy(hl.rope_freqs(rot, 1e4)[0]).to(dev)
    pos = torch.arange(50, 50 + tokens, dtype=torch.int32, device=dev)
    q, qx = to_type(rng.standard_normal((tokens, heads, dim)), t, dev)
    k, _ = to_type(rng.standard_normal((tokens, kv, dim)), t, dev)
    w = torch.from_numpy((1 + 0.1 * rng.standard_normal(dim)).astype(np.float32)).to(dev)
    qo, ko, q2, k2 = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q), torch.empty_like(k)
    hl.rope(t, pos, freqs, tokens, dim, rot, q, q2, heads, k=k, k_out=k2, n_kv_heads=kv)
    hl.norm_rope(t, pos, freqs, tokens, dim, rot, q, qo, heads, q_norm=w, k=k, k_out=ko, n_kv_heads=kv)
    assert torch.equal(ko, k2)
    check(t, qo.double().cpu().numpy(), qx, w.double().cpu().numpy(), 1e-6, pos.cpu().numpy(), freqs.cpu().numpy(), rot, 0, 1.0)
    hl.norm_rope(t, pos, freqs, tokens, dim, rot, q, qo, heads, k=k, k_out=ko, n_kv_heads=kv)
    assert torch.equal(qo, q2) and torch.equal(ko, k2)


@TYPES
def test_norm_rope_of_a_row_fused_projection(hl, dev, t):
    """q and k in place where they lie side by side in rows of any length; a head of zeros, and one with a NaN, which stays alone."""
    import torch

    tokens, heads, kv, dim, rot = 9, 6, 2, 64, 32
    row = (heads + 2 * kv) * dim + 3
    rng = np.random.default_rng(5)
    x, xx = to_type(rng.standard_normal((tokens, row)), t, dev)
    x[2, dim:2 * dim] = 0
    xx[2, dim:2 * dim] = 0
    x[4, 3 * dim + 5] = float("nan")
    before = x.clone()
    freqs, _ = hl.rope_freqs(rot, 1e4)
    pos = np.arange(100, 100 + tokens, dtype=np.int32)
    w = (1 + 0.1 * rng.standard_normal(dim)).astype(np.float32)
    p, f, wd = (torch.from_numpy(v).to(dev) for v in (pos, freqs, w))
    q, k = x[:, :heads * dim], x[:, heads * dim:]
    hl.norm_rope(t, p, f, tokens, dim, rot, q, q, heads, q_norm=wd, k=k, k_out=k, n_kv_heads=kv, k_norm=wd, q_stride=row, q_out_stride=row, k_stride=row,
                 k_out_stride=row)
    got = x.double().cpu().numpy()
    n = heads + kv
    got_heads, want_heads = got[:, :n * dim].reshape(tokens, n, dim).copy(), xx[:, :n * dim].reshape(tokens, n, dim).copy()
    assert np.all(np.isnan(got_heads[4, 3]))
    got_heads[4, 3] = want_heads[4, 3] = 0
    check(t, got_heads, want_heads, w.astype(np.float64), 1e-6, pos, freqs, rot, 0, 1.0)
    assert torch.equal(x[:, n * dim:], before[:, n * dim:])


@pytest.mark.parametrize("tokens,heads,kv", [((1 << 23) + 3, 1, 0), (2, 65535, 65535)])
def test_norm_rope_past_a_grid(hl, dev, tokens, heads, kv):
    import torch

    print("[case] norm_rope past a grid", tokens, heads, kv, flush=True)
    g = torch.Generator(device=dev).manual_seed(5)
    dim = 8
    q = torch.randn(tokens, heads, dim, device=dev, generator=g).half()
    k = torch.randn(tokens, kv, dim, device=dev, generator=g).half()
    pos = torch.randint(0, 1 << 16, (tokens,), device=dev, generator=g, dtype=torch.int32)
    freqs = torch.tensor([0.37, 0.1], dtype=torch.float64, device=dev)
    w = torch.ones(dim, device=dev)
    qo, ko = torch.full_like(q, 7), torch.full_like(k, 7)
    hl.norm_rope(F16, pos, freqs, tokens, dim, 4, q, qo, heads, q_norm=w, k=k if kv else None, k_out=ko if kv else None, n_kv_heads=kv, k_norm=w)
    for at in (slice(0, 2), slice(tokens - 2, tokens)):
        for x, y in ((q, qo), (k, ko)):
            if y.numel():
                check(F16, y[at].double().cpu().numpy(), x[at].double().cpu().numpy(), np.ones(dim), 1e-6, pos[at].cpu().numpy(), freqs.cpu().numpy(), 4, 0, 1.0)
    # every head was written
    for y in (qo, ko):
        assert not bool((y == 7).all(-1).any())


@TYPES
@pytest.mark.parametrize("pairs", [0, 1], ids=["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot", [(2051, 5, 2, 128, 128), (4099, 3, 0, 64, 32), (1025, 9, 4, 256, 64)])
def test_norm_rope_of_many_tokens(hl, dev, t, pairs, tokens, heads, kv, dim, rot):
    """Several tokens a workgroup, the last one's not all there."""
    import torch

    rng = np.random.default_rng(tokens)
    freqs, _ = hl.rope_freqs(rot, 1e4)
    pos = rng.integers(0, 5000, tokens).astype(np.int32)
    q, qx = to_type(rng.standard_normal((tokens, heads, dim)) * 2, t, dev)
    k, kx = to_type(rng.standard_normal((tokens, max(kv, 1), dim)), t, dev)
    qw, kw = ((1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2))
    qwd, kwd, p, f = (torch.from_numpy(x).to(dev) for x in (qw, kw, pos, freqs))
    qo, ko = torch.full_like(q, 7), torch.full_like(k, 7)
    hl.norm_rope(t, p, f, tokens, dim, rot, q, qo, heads, q_norm=qwd, k=k if kv else None, k_out=ko if kv else None, n_kv_heads=kv, k_norm=kwd, pairs=pairs)
    check(t, qo.double().cpu().numpy(), qx, qw.astype(np.float64), 1e-6, pos, freqs, rot, pairs, 1.0)
    if kv:
        check(t, ko.double().cpu().numpy(), kx, kw.astype(np.float64), 1e-6, pos, freqs, rot, pairs, 1.0)


def test_norm_rope_of_far_rows(hl, dev):
    """Rows whose offsets pass 32 bits of bytes and of elements, in place, on another stream than the current one."""
    import torch

    tokens, heads, dim, stride = 70, 2, 64, 1 << 26
    big = torch.empty(tokens * stride, dtype=torch.bfloat16, device=dev)
    rows = big.view(tokens, stride)[:, :heads * dim]
    rng = np.random.default_rng(9)
    x, xx = to_type(rng.standard_normal((tokens, heads * dim)), BF16, dev)
    rows.copy_(x)
    freqs, _ = hl.rope_freqs(dim, 1e4)
    pos = np.arange(tokens, dtype=np.int32)
    p, f, w = torch.from_numpy(pos).to(dev), torch.from_numpy(freqs).to(dev), torch.ones(dim, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    hl.norm_rope(BF16, p, f, tokens, dim, dim, big, big, heads, q_norm=w, q_stride=stride, q_out_stride=stride, stream=side.cuda_stream)
    side.synchronize()
    check(BF16, rows.double().cpu().numpy().reshape(tokens, heads, dim), xx.reshape(tokens, heads, dim), np.ones(dim), 1e-6, pos, freqs, dim, 0, 1.0)
