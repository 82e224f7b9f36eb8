"""Linear attention in chunks of 128 columns a workgroup, as models of many heads run it, against the recurrence in 64 bits: every head size and
type, whole and in segments, beside the states before and over them; prompts beside single rows; row starts that fall."""
import numpy as np
import pytest

from kv_helpers import BF16, F16, F32, TYPE_NAMES
from layer_helpers import linear_ref_on
from test_gpu_linear import Case

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("t", [F32, F16, BF16], ids=lambda t: TYPE_NAMES[t])


class Wide(Case):
    """A batch whose reference is computed on the device."""

    def want(self, fresh=(), scale=None):
        import torch

        group = self.heads // self.k_heads
        outs, states = {}, {}
        for i, n in enumerate(self.rows):
            if n == 0:
                continue
            at = slice(self.starts[i], self.starts[i] + n)
            s = np.zeros_like(self.sx[0]) if i in fresh else self.sx[self.slots[i]]
            d = np.broadcast_to(self.dx, (n, self.heads)) if self.per_head else self.dx[at]
            on = [torch.from_numpy(np.array(x, dtype=np.float64)).to(self.dev) for x in
                  (self.qx[at].repeat(group, 1), self.kx[at].repeat(group, 1), self.vx[at], d, s)]
            o, otol, s, stol = (x.cpu().numpy() for x in linear_ref_on(self.t, *on, self.kd ** -0.5 if scale is None else scale))
            outs[i], states[i] = (at, o, otol), (self.slots[i], s, stol)
        return outs, states

    def is_wide(self):
        """Whether the chunks take 128 columns a workgroup however the sequences are cut."""
        return self.vd % 128 == 0 and self.heads * (self.vd // 128) * len(self.rows) > 128 and max(self.rows) > 16


def both_ways(c, hl, **kw):
    """The states beside those before the call, then over them."""
    fresh = kw.get("fresh", ())
    lens = None if not fresh else [n + (i not in fresh) for i, n in enumerate(c.rows)]
    got = c.call(hl, lens=lens)
    c.check(got, **kw)
    assert np.array_equal(c.s.cpu().numpy(), c.sx)
    c.out.fill_(9.0)
    again = c.call(hl, lens=lens, in_place=True)
    c.check(again, in_place=True, **kw)
    return got, again


@TYPES
@pytest.mark.parametrize("vd", [128, 256])
@pytest.mark.parametrize("kd", [64, 96, 128, 192, 256])
def test_chunks(hl, dev, t, kd, vd):
    """Two chunks and a ragged one, a whole one and one row, less than one; every other call gives one decay a head."""
    print("[case] linear wide", TYPE_NAMES[t], kd, vd, flush=True)
    heads = 48 * 128 // vd
    c = Wide(dev, t, [70, 33, 17], heads, heads // 3, kd, vd, kd + vd, per_head=kd % 128 == 0, lead=1, tail=2)
    assert c.is_wide()
    (out, new), (out2, new2) = both_ways(c, hl, fresh=(1,))
    # bitwise the same in both places
    assert np.array_equal(out, out2) and all(np.array_equal(new[i], new2[i]) for i in c.slots)


@TYPES
@pytest.mark.parametrize("kd,vd", [(64, 128), (96, 128), (128, 128), (192, 128), (256, 128), (128, 256)])
def test_segments(hl, dev, t, kd, vd):
    """Two long sequences, cut, and a short one between them."""
    import torch

    print("[case] linear wide segments", TYPE_NAMES[t], kd, vd, flush=True)
    heads = 48 * 128 // vd
    c = Wide(dev, t, [700, 40, 1000], heads, heads // 3, kd, vd, kd)
    assert c.is_wide()
    state = hl.LinearState(c.s, c.n_slots, heads, kd, vd, c.new)
    batch = hl.LinearBatch(c.ints(c.slots), c.ints(c.starts), 3, c.n, 1000)
    assert hl.linear_attention_workspace(t, state, batch, c.q, c.k, c.v, c.out, c.d, heads // 3) >= 3 * heads * (kd * vd + 1) * 4
    (out, new), (out2, new2) = both_ways(c, hl)
    assert np.array_equal(out, out2) and all(np.array_equal(new[i], new2[i]) for i in c.slots)


@TYPES
@pytest.mark.parametrize("kd", [128, 256])
def test_rounded_lengths(hl, dev, t, kd):
    """Lengths of whole chunks and whole segments, the segments' remainders among them."""
    c = Wide(dev, t, [512, 32, 768], 48, 16, kd, 128, 3)
    assert c.is_wide()
    both_ways(c, hl, fresh=(0,))


@TYPES
def test_decays_at_the_edges(hl, dev, t):
    """No decay, a state that is emptied in the midst, decays far under the smallest number, strong ones beside weak ones, and growth."""
    def none(d):
        return np.zeros_like(d)

    def emptied(d):
        d = d.copy()
        d[len(d) // 2], d[len(d) - 2, 0], d[35, 5:9] = -np.inf, -np.inf, -np.inf
        return d

    def far(d):
        d = d.copy()
        d[::3], d[1::3] = -3e38, -90.0
        return d

    def apart(d):
        d = np.full_like(d, -1e-4)
        d[::7] = -60.0
        return d

    for way in (none, emptied, far, apart, lambda d: np.full_like(d, 0.01)):
        c = Wide(dev, t, [60, 100, 45], 48, 16, 128, 128, 23, decay=way)
        assert c.is_wide()
        c.dx = np.maximum(c.dx, -1e4)  # the reference's floor on decays
        c.check(c.call(hl))


@TYPES
@pytest.mark.parametrize("kd", [128, 256])
def test_values_that_are_not_finite_stay_behind(hl, dev, t, kd):
    """A bad value reaches its own row and later ones of its sequence only, and of v only its own column."""
    for which, bad, at in (("v", np.nan, 37), ("v", np.inf, 64), ("v", -np.inf, 99), ("k", np.nan, 70), ("q", np.inf, 32), ("d", np.nan, 51)):
        c = Wide(dev, t, [100, 33, 20], 48, 48, kd, 128, 31)
        assert c.is_wide()
        x = {"v": c.v, "k": c.k, "q": c.q, "d": c.d}[which]
        head, col = 41, 60
        if which == "d":
            x[at, head] = bad
        else:
            x[at, head, col] = bad
        out, new = c.call(hl)
        outs, states = c.want()
        for i in range(3):
            rows, o, otol = outs[i]
            slot, s, stol = states[i]
            good, kept = np.ones_like(o, bool), np.ones_like(s, bool)
            if i == 0:
                if which == "v":
                    good[at:, head, col], kept[head, :, col] = False, False
                elif which == "q":
                    good[at, head] = False
                else:
                    good[at:, head] = False
                    kept[head, col if which == "k" else slice(None)] = False
            err, serr = np.abs(out[rows] - o), np.abs(new[slot] - s)
            assert np.all(err[good] <= otol[good]), (which, bad, i, np.argwhere(good & ~(err <= otol))[0])
            assert np.all(serr[kept] <= stol[kept]), (which, bad, i)
            assert not np.isfinite(out[rows][~good]).any() and not np.isfinite(new[slot][~kept]).any(), (which, bad, i)


@TYPES
def test_prompts_beside_single_rows(hl, dev, t):
    """A serving step's batch: two prompts among sequences of one row and of none, some of which begin."""
    rows = [1] * 9 + [300] + [1, 0, 1, 1, 0, 1] + [130] + [1] * 9
    c = Wide(dev, t, rows, 24, 8, 64, 128, 47)
    assert c.is_wide()
    both_ways(c, hl, fresh=(3, 9, 20))


@TYPES
def test_falling_row_starts_are_computed(hl, dev, t):
    """Row starts that fall and pass the end are cut: the first sequence has no rows, the second has what is left."""
    c = Wide(dev, t, [80, 3], 2, 1, 64, 64, 17, n_slots=6)
    n = c.n
    c.starts, c.slots = np.array([40, 30, 1 << 30], dtype=np.int32), np.array([1, 2], dtype=np.int32)
    got = c.call(hl, max_rows=n)
    c.rows = [0, n - 30]
    c.check(got)


@TYPES
@pytest.mark.parametrize("heads,kd,vd", [(4, 64, 64), (48, 128, 128)])
def test_falling_row_starts_that_count_rows_twice(hl, dev, t, heads, kd, vd):
    """The same rows are two sequences', in two slots: the workspace has room for one's states between segments, and the other runs uncut. Nothing
    is written past the workspace."""
    import torch

    n = 1300
    c = Wide(dev, t, [n], heads, heads // 2, kd, vd, 19, n_slots=5)
    c.starts, c.slots, c.rows = np.array([0, n, 0, n], dtype=np.int32), np.array([3, 0, 1], dtype=np.int32), [n, 0, n]
    for in_place in (False, True):
        state = hl.LinearState(c.s, c.n_slots, heads, kd, vd, None if in_place else c.new)
        batch = hl.LinearBatch(c.ints(c.slots), c.ints(c.starts), 3, n, n)
        need = hl.linear_attention_workspace(t, state, batch, c.q, c.k, c.v, c.out, c.d, heads // 2)
        assert need > 0
        ws = torch.full((need + 4096,), 85, dtype=torch.uint8, device=dev)
        c.out.fill_(9.0)
        # both begin, so that both give the same rows
        got = c.call(hl, lens=[n, 1, n], in_place=in_place, max_rows=n, workspace=ws, workspace_bytes=need)
        c.check(got, fresh=(0, 2), in_place=in_place)
        assert bool((ws[need:] == 85).all())


def test_repeats_bitwise(hl, dev):
    """The same prompts again and again, other calls between: every bit the same, on this stream and on another."""
    import torch

    heads, kh, kd, vd, lens = 48, 16, 128, 128, [1501, 90, 2100]
    rows, ints = sum(lens), lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    g = torch.Generator(device=dev).manual_seed(8)

    def call():
        q, k, v = (torch.randn(rows, h, d, device=dev, generator=g).bfloat16() for h, d in ((kh, kd), (kh, kd), (heads, vd)))
        state = torch.randn(3, heads, kd, vd, device=dev, generator=g)
        new, out = torch.empty_like(state), torch.empty_like(v)
        batch = hl.LinearBatch(ints([1, 2, 0]), ints(np.concatenate([[0], np.cumsum(lens)]).tolist()), 3, rows, max(lens))
        return (BF16, hl.LinearState(state, 3, heads, kd, vd, new), batch, q, k, v, out, -0.05 * torch.rand(rows, heads, device=dev, generator=g), kh), new, out

    (one, new, out), (other, _, _) = call(), call()
    hl.linear_attention(*one)
    first = new.clone(), out.clone()
    side = torch.cuda.Stream()
    for i in range(6):
        new.zero_()
        out.zero_()
        hl.linear_attention(*other)
        torch.cuda.synchronize()
        hl.linear_attention(*one, stream=side.cuda_stream if i % 2 else None)
        torch.cuda.synchronize()
        assert torch.equal(new, first[0]) and torch.equal(out, first[1])


@pytest.mark.parametrize("t", [F32, BF16], ids=lambda t: TYPE_NAMES[t])
@pytest.mark.parametrize("heads", [2, 48], ids=["narrow", "wide"])
def test_large_values(hl, dev, t, heads):
    """States, and their products with q, near 2^70, under decays that the chunks take late: a column of the state has a deviation of
    2^69 / sqrt(128) times sqrt(1 / (1 - e^-0.14)), 2^67, which scale times a sum over 128 values of q keeps; a hundred thousand outputs pass 4 of it."""
    c = Wide(dev, t, [300, 90, 120], heads, 2, 128, 128, 29, decay=lambda d: np.full_like(d, -0.07))
    c.k *= 2.0 ** 30
    c.v *= 2.0 ** 39
    c.kx, c.vx = c.kx * 2.0 ** 30, c.vx * 2.0 ** 39
    c.s *= 2.0 ** 66
    c.sx = c.sx * np.float32(2.0 ** 66)
    out, new = got = c.call(hl)
    assert 2.0 ** 68 < np.abs(out).max() < 2.0 ** 72
    c.check(got)
