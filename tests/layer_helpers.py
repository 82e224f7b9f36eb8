"""8-bit rows and their products, the heads' norms with the rotation, and linear attention in plain numpy, in 64 bits: what the kernels
are compared with, and how far they may be off."""
from __future__ import annotations

import numpy as np

from kv_helpers import F32, HALF_LEAST, HALF_STEP, MIN_SCALE, U, nearest


def padded(cols):
    return -(-cols // 16) * 16


def quantized(x):
    """Codes (padded with zeros) and scales of rows of x (64 bits, values of at most 24 bits), as halo_mi_quantize_rows defines them."""
    rows, cols = x.shape
    codes = np.zeros((rows, padded(cols)), dtype=np.int8)
    top = np.abs(x).max(1)
    with np.errstate(all="ignore"):
        scales = (top / 127).astype(np.float32)  # 53 bits decide where 24 are kept: x / 127 is never within 2^-32 of a tie
        scales[scales < np.float32(MIN_SCALE)] = 0
        scales[~np.isfinite(top)] = np.nan
    for r in range(rows):
        if scales[r] > 0:
            codes[r, :cols] = nearest(x[r], float(scales[r]))
    return codes, scales


def gemm_ref(t, w, ws, x, xs, cols):
    """The product in 64 bits, and how far a result in type t may be off: three roundings to 24 bits (the scales' product, the sum, their
    product) and one to the type."""
    total = x[:, :cols].astype(np.int64) @ w[:, :cols].astype(np.int64).T
    want = total * (xs.astype(np.float64)[:, None] * ws.astype(np.float64))
    return want, np.abs(want) * (3.01 * U + HALF_STEP[t] * 1.01) + HALF_LEAST[t] + 2.0 ** -148


def norm_rope_ref(t, x, w, eps, pos, freqs, rot, pairs, factor):
    """Normed and rotated heads [token, head, dim] in 64 bits, and how far they may be off."""
    dim = x.shape[-1]
    mean = (x * x).sum(-1, keepdims=True) / dim
    y = x if w is None else x / np.sqrt(mean + eps) * w
    # the norm: the squares' sum is off by at most (dim + 1) units of 2^-24, half of that in the root; three more for 1 / dim and
    # eps, the root and the quotient (two), and two for the products
    off = 0.0 if w is None else ((dim + 1) / 2 + 6) * U
    angle = pos.astype(np.float64)[:, None] * freqs
    c, s = np.cos(angle)[:, None] * factor, np.sin(angle)[:, None] * factor
    i = np.arange(rot // 2)
    a, b = (i, i + rot // 2) if pairs == 0 else (2 * i, 2 * i + 1)
    out, reach = y.copy(), np.abs(y) * off
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    far = np.abs(angle).max() if angle.size else 0.0
    # the rotation: 8 units of the pair's reach (sine, cosine, factor, products, sum), and the angle's own 53 bits
    both = (np.abs(y[..., a]) + np.abs(y[..., b])) * abs(factor) * (off + 8 * U + far * 2.0 ** -51)
    reach[..., a] = reach[..., b] = both
    return out, reach + HALF_STEP[t] * np.abs(out) * 1.01 + HALF_LEAST[t] + 1e-37


def linear_ref(t, q, k, v, decay, state, scale):
    """One sequence, row by row: out [row, head, v_dim] and the state [head, k_dim, v_dim] in 64 bits, and how far both may be off.
    q, k: [row, head, k_dim]; decay: [row, head].

    `reach` runs along with the state as the sum of all terms' sizes, `off` as what the roundings of its steps add up to: a
    step multiplies by exp(g), whose argument is rounded (|g| units) and whose result is (2), rounds the product and the new term, and adds
    (4 in all); the chunked form has as many roundings per term in other places, its sums of up to 64 tokens among them. Decays under
    2^-126 may count as 0."""
    rows, heads, kd = q.shape
    state, reach = state.astype(np.float64).copy(), np.abs(state.astype(np.float64))
    off = np.zeros_like(state)
    out, far = np.zeros((rows, heads, v.shape[-1])), np.zeros((rows, heads, v.shape[-1]))
    # what a dot product over k_dim and up to 64 tokens rounds; 16-bit types: weights and states in two pieces of 8 bits
    c = (kd + 192) * U + (0.0 if t == F32 else 2.0 ** -15)
    with np.errstate(all="ignore"):
        for r in range(rows):
            g = np.maximum(decay[r].astype(np.float64), -1e4)[:, None, None]
            fade = np.exp(g)
            new = k[r][:, :, None] * v[r][:, None, :]
            off = fade * (off + (6 + np.abs(g)) * U * reach) + 2.0 ** -120 * reach
            state = fade * state + new
            reach = fade * reach + np.abs(new)
            off += 4 * U * reach
            out[r] = scale * np.einsum("hk,hkv->hv", q[r], state)
            far[r] = abs(scale) * np.einsum("hk,hkv->hv", np.abs(q[r]), off + c * reach)
        far += HALF_STEP[t] * np.abs(out) * 1.01 + HALF_LEAST[t] + 1e-37
        # the chunked form adds a chunk's terms to the state at once, 64 roundings
        return out, far, state, off + 64 * U * reach + 1e-37


def linear_ref_on(t, q, k, v, decay, state, scale):
    """linear_ref in torch, for states of many heads: tensors of 64 bits on one device. Multiplies and sums elements, no library product."""
    import torch

    rows, heads, kd = q.shape
    state, reach = state.clone(), state.abs()
    off = torch.zeros_like(state)
    out, far = torch.zeros_like(v), torch.zeros_like(v)
    c = (kd + 192) * U + (0.0 if t == F32 else 2.0 ** -15)
    g = decay.clamp(min=-1e4)  # NaN stays
    fades, grown = g.exp(), (6 + g.abs()) * U
    for r in range(rows):
        fade = fades[r, :, None, None]
        new = k[r, :, :, None] * v[r, :, None, :]
        off = fade * (off + grown[r, :, None, None] * reach) + 2.0 ** -120 * reach
        state = fade * state + new
        reach = fade * reach + new.abs()
        off += 4 * U * reach
        out[r] = scale * (q[r, :, :, None] * state).sum(1)
        far[r] = abs(scale) * (q[r, :, :, None].abs() * (off + c * reach)).sum(1)
    far += HALF_STEP[t] * out.abs() * 1.01 + HALF_LEAST[t] + 1e-37
    return out, far, state, off + 64 * U * reach + 1e-37


def tile_plan(shapes, rows, cols, n_vec):
    """The shape of tiles that gemm_i8 takes for many vectors, as k_gemm_i8.hip's plan_tiles chooses among `shapes` (fragments along the channels and
    the vectors, stages), with the tiles in both directions and what each has: (shape, tiles_n, tiles_t, each_n, each_t)."""
    cus, up = 256, lambda a, b: -(-a // b)
    best, least = None, 1e300
    for fn, ft, stages in shapes:
        tiles_t = up(n_vec, 64 * ft)
        each_t = up(n_vec, tiles_t)
        tiles_t = up(n_vec, each_t)
        few = up(rows, 32 * fn)
        stage = (up(32 * fn, 64) * 64 + 64 * ft) * 128
        beside = min(max(1, 160 * 1024 // (stages * stage)), up(few * tiles_t, cus))
        slots, products = cus * beside, 0.056 * fn * ft
        rounds = up(few * tiles_t, slots)

        def share(n):
            return up(up(rows, n), 8) * 8

        def loads(each_n):
            return 0.015 / 8 * (each_n + each_t) + 0.04 * (fn + ft) - 0.05

        each_n = share(few)
        if loads(each_n) > products:
            each_n = share(max(few, min(slots * rounds // tiles_t, up(rows, 8))))
        time = rounds * (2.0 + up(cols, 128) * beside * max(products, loads(each_n)))
        if time < least:
            least, best = time, ((fn, ft, stages), up(rows, each_n), tiles_t, each_n, each_t)
    return best
