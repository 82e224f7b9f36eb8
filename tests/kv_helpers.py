"""The 8-bit paged cache, its attention and its pages in plain numpy, in 64 bits: what the kernels are compared with."""
from __future__ import annotations

import math

import numpy as np

F32, F16, BF16 = 0, 1, 30
TYPE_NAMES = {F32: "f32", F16: "f16", BF16: "bf16"}
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}  # one rounding, relative
# ... and absolute, half the spacing of the smallest numbers: f16 values under 2^-14 are 2^-24 apart, so one rounding is
# off by up to 2^-25 there whatever its relative size
HALF_LEAST = {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134}
U = 2.0 ** -24
MIN_SCALE = 2.0 ** -80


def torch_type(t):
    import torch

    return {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}[t]


def to_type(x, t, dev):
    """x rounded to the type, on the device, and what it then holds, in 64 bits."""
    import torch

    y = torch.from_numpy(np.ascontiguousarray(x)).to(torch_type(t))
    return y.to(dev), y.double().numpy()


def page_bytes(layers, heads, dim, block):
    units = 2 * layers * heads
    return -(-(units * block * dim + 4 * units) // 128) * 128


class Cache:
    """The pool as numpy bytes, with views of its codes [page, layer, 2, head, block * dim] and scales [page, layer, 2, head]."""

    def __init__(self, n_pages, layers, heads, dim, block):
        self.geometry = (n_pages, layers, heads, dim, block)
        self.n_pages, self.layers, self.heads, self.dim, self.block = self.geometry
        self.bytes = np.zeros((n_pages, page_bytes(layers, heads, dim, block)), dtype=np.uint8)

    @property
    def codes(self):
        n = 2 * self.layers * self.heads * self.block * self.dim
        return self.bytes[:, :n].view(np.int8).reshape(self.n_pages, self.layers, 2, self.heads, -1)

    def scales_at(self):
        n = 2 * self.layers * self.heads * self.block * self.dim
        return n, n + 8 * self.layers * self.heads

    @property
    def scales(self):
        a, b = self.scales_at()
        return np.ascontiguousarray(self.bytes[:, a:b]).view(np.float32).reshape(self.n_pages, self.layers, 2, self.heads)

    def set_scales(self, s):
        a, b = self.scales_at()
        self.bytes[:, a:b] = np.ascontiguousarray(s, dtype=np.float32).reshape(self.n_pages, -1).view(np.uint8)

    def k_codes(self, page, layer):
        """[head, token, dim] of a page, a view."""
        return self.bytes_of(page, layer, 0).reshape(self.heads, self.block, self.dim)

    def v_codes(self, page, layer):
        """[head, dim, token] of a page, a view."""
        return self.bytes_of(page, layer, 1).reshape(self.heads, self.dim, self.block)

    def bytes_of(self, page, layer, which):
        n = self.heads * self.block * self.dim
        at = (2 * layer + which) * n
        return self.bytes[page, at:at + n].view(np.int8)

    def fill(self, rng, scale=3.5 / 127):
        """Codes and scales everywhere, as a model leaves them."""
        n = 2 * self.layers * self.heads * self.block * self.dim
        c = np.clip(np.rint(rng.standard_normal((self.n_pages, n)) * 34), -127, 127).astype(np.int8)
        self.bytes[:, :n] = c.view(np.uint8)
        self.set_scales(scale * np.exp(0.3 * rng.standard_normal((self.n_pages, self.layers, 2, self.heads))))

    def tokens(self, pages, n, layer):
        """K and V values [head, token, dim] in 64 bits of the first n tokens in `pages`."""
        k, v, s = [], [], self.scales.astype(np.float64)
        for p in pages[:-(-n // self.block)]:
            k.append(self.k_codes(p, layer) * s[p, layer, 0][:, None, None])
            v.append(self.v_codes(p, layer).transpose(0, 2, 1) * s[p, layer, 1][:, None, None])
        if not k:
            z = np.zeros((self.heads, 0, self.dim))
            return z, z
        return np.concatenate(k, 1)[:, :n], np.concatenate(v, 1)[:, :n]


def nearest(x, s):
    """The integers nearest to x / s, ties to even, exactly (x: 24-bit values or integers times one; s: 24 bits)."""
    r = np.rint(x / s)
    up, down = (2 * r + 1) * s, (2 * r - 1) * s
    odd = np.mod(r, 2) == 1
    r = np.where((2 * x > up) | ((2 * x == up) & odd), r + 1, r)
    return np.where((2 * x < down) | ((2 * x == down) & odd), r - 1, r)


def write_ref(cache, layer, tables, lens, starts, k, v):
    """KV_WRITE on the numpy cache; k, v: [row, head, dim] in 64 bits, holding values of at most 24 bits."""
    scales, block = cache.scales.copy(), cache.block
    for s in range(len(lens)):
        rows, n = starts[s + 1] - starts[s], lens[s]
        first = n - rows
        a = max(first, 0)
        for j in range(a // block, -(-n // block) if rows else 0):
            lo, hi = max(a, j * block), min(n, (j + 1) * block)
            if lo >= hi or j >= tables.shape[1] or not 0 <= tables[s, j] < cache.n_pages:
                continue
            page, off = tables[s, j], lo - j * block
            r0 = starts[s] + lo - first
            for which, x in ((0, k), (1, v)):
                for h in range(cache.heads):
                    val = x[r0:r0 + hi - lo, h]
                    old = float(scales[page, layer, which, h]) if off else 0.0
                    with np.errstate(all="ignore"):
                        fit = float(np.float32(np.abs(val).max()) / np.float32(127))
                    new = max(old, fit) if fit >= MIN_SCALE else old
                    if not np.isfinite(val).all() or math.isnan(old):
                        scales[page, layer, which, h] = np.nan
                        continue
                    scales[page, layer, which, h] = new
                    c = cache.k_codes(page, layer)[h] if which == 0 else cache.v_codes(page, layer)[h].T
                    if off and new > old > 0:
                        c[:off] = nearest(c[:off] * old, new)
                    c[off:off + hi - lo] = np.clip(nearest(val, new), -127, 127) if new > 0 else 0
    cache.set_scales(scales)


def attention_ref(cache, layer, tables, lens, starts, q, window=0, scale=None):
    """(out, sum of p |v|, largest score error unit) per row and head, in 64 bits. q: [row, head, dim]. The last
    two are what the error bounds are made of: sum_t p_t |v_t| / sum p, and scale * max_t sum_d |q_d k_td|."""
    n_rows, heads, dim = q.shape
    group = heads // cache.heads
    out, weight = np.zeros_like(q), np.zeros_like(q)
    reach = np.zeros((n_rows, heads))
    scale = 1 / math.sqrt(dim) if scale is None else scale
    for s in range(len(lens)):
        rows, n = starts[s + 1] - starts[s], lens[s]
        k, v = cache.tokens(tables[s], n, layer)
        for i in range(rows):
            pos = n - rows + i
            lo = max(pos - window + 1, 0) if window else 0
            if pos < 0:
                continue
            for h in range(heads):
                kk, vv, x = k[h // group, lo:pos + 1], v[h // group, lo:pos + 1], q[starts[s] + i, h]
                score = kk @ x * scale
                p = np.exp(score - score.max())
                p /= p.sum()
                out[starts[s] + i, h] = p @ vv
                weight[starts[s] + i, h] = p @ np.abs(vv)
                reach[starts[s] + i, h] = (np.abs(kk) @ np.abs(x)).max() * abs(scale)
    return out, weight, reach


def attention_bound(t, dim, tokens, out, weight, reach, vmax):
    """How far the kernel's out may be off.

    Scores: dim products summed in fp32 (dim U), q within 2^-22 for fp32 and exact for 16 bits, the two
    multiplications by scales and the logarithm's rounding (4 U) on values up to the score plus |log2 vs| < 32 and the
    shift by the maximum: (dim + 8) U + 2^-22 of reach, and 64 U at the level of the exponent.
    Weights: exp2 within 2 U, then 11 bits (2^-12 kept relative) or two pieces (2^-22). They are carried times 2^8 (two
    pieces: 2^14) of a reference that is at most the row's largest, and f16's smallest step is 2^-24: what is lost
    under its normal numbers is up to 2^-25 / 2^8 (2^-25 / 2^14) of the largest weight, for each token. Both sums have up to `tokens` terms: tokens U each. A relative error e of
    every weight moves the quotient by at most 2 e sum p |v|.
    """
    pieces = 2.0 ** -22 if t == F32 else 2.0 ** -12
    e = ((dim + 8) * U + (2.0 ** -22 if t == F32 else 0)) * reach[..., None] + 64 * U + pieces
    sums = 2 * (tokens + 16) * U
    return weight * (2 * e + sums) + tokens * (2.0 ** -38 if t == F32 else 2.0 ** -32) * vmax + HALF_STEP[t] * np.abs(out) * 1.01 + HALF_LEAST[t] + 1e-30


def batch(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


def tables_for(rng, lens, block, n_pages, width, stray=-1):
    """Distinct pages for each sequence, in no order; the rest of a row is `stray`."""
    ids, at = rng.permutation(n_pages), 0
    out = np.full((len(lens), width), stray, dtype=np.int32)
    for i, n in enumerate(lens):
        need = -(-n // block)
        out[i, :need] = ids[at:at + need]
        at += need
    assert at <= n_pages
    return out


class PagesModel:
    """Reference counts, lengths and tables as the library keeps them, one step at a time."""

    def __init__(self, n_pages, block, slots, width):
        self.block, self.width = block, width
        self.refs = [0] * n_pages
        self.lens = [0] * slots
        self.tables = [[-1] * width for _ in range(slots)]
        self.owner = list(range(n_pages))  # what each page's bytes are: the page they came from

    def need(self, n):
        return -(-n // self.block)

    def _grant(self, wants):
        free = [p for p, r in enumerate(self.refs) if r <= 0]
        given, at = [], 0
        for w in wants:
            given.append(free[at:at + w] if at + w <= len(free) else None if w else [])
            at += w
        return given

    def resize(self, slots, news):
        """Status bits of the call."""
        status, seen, todo = 0, set(), []
        for s, n in zip(slots, news):
            ok = 0 <= s < len(self.lens) and s not in seen and n >= 0
            seen.add(s)
            if not ok:
                status |= 8
            elif self.need(n) > self.width:
                status |= 16
            else:
                have, length = self.need(self.lens[s]), self.lens[s]
                cow = n > length and length % self.block and self.refs[self.tables[s][have - 1]] > 1
                todo.append((s, n, have, bool(cow), max(self.need(n) - have, 0) + bool(cow)))
        given = self._grant([t[4] for t in todo])
        drop = []
        for (s, n, have, cow, _), pages in zip(todo, given):
            if pages is None:
                status |= 16
                continue
            if cow:
                old = self.tables[s][have - 1]
                drop.append(old)
                self.owner[pages[0]] = self.owner[old]
            for i, p in enumerate(pages):
                self.tables[s][have - cow + i] = p
                self.refs[p] = 1
            for c in range(self.need(n), have):
                drop.append(self.tables[s][c])
                self.tables[s][c] = -1
            self.lens[s] = n
        for p in drop:
            self.refs[p] -= 1
        return status

    def fork(self, src, dst):
        status, seen, todo = 0, set(), []
        before = list(self.lens)
        for s, d in zip(src, dst):
            ok = 0 <= s < len(before) and 0 <= d < len(before) and s != d and d not in seen and before[d] == 0
            seen.add(d)
            if ok:
                todo.append((s, d, int(before[s] % self.block != 0)))
            else:
                status |= 8
        given = self._grant([t[2] for t in todo])
        for (s, d, part), pages in zip(todo, given):
            if pages is None:
                status |= 16
                continue
            full = before[s] // self.block
            for c in range(full):
                self.tables[d][c] = self.tables[s][c]
                self.refs[self.tables[s][c]] += 1
            if part:
                self.tables[d][full] = pages[0]
                self.refs[pages[0]] = 1
                self.owner[pages[0]] = self.owner[self.tables[s][full]]
            self.lens[d] = before[s]
        return status

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        moved = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        holes = [p for p in range(live) if self.refs[p] <= 0]
        place = dict(zip(moved, holes))
        for p, h in place.items():
            self.refs[h], self.refs[p] = self.refs[p], 0
            self.owner[h] = self.owner[p]
        for s, n in enumerate(self.lens):
            for c in range(self.need(n)):
                self.tables[s][c] = place.get(self.tables[s][c], self.tables[s][c])
        return live
