"""Linear attention on the GPU against the recurrence in 64 bits, row by row."""
import math

import numpy as np
import pytest

from kv_helpers import BF16, F16, F32, TYPE_NAMES, to_type, torch_type
from layer_helpers import linear_ref

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("t", [F32, F16, BF16], ids=lambda t: TYPE_NAMES[t])


class Case:
    """A batch's operands on the device and in numpy; states of all slots, the ones of no sequence among them."""

    def __init__(self, dev, t, rows, heads, k_heads, kd, vd, seed, n_slots=None, per_head=False, lead=0, tail=0, decay=None):
        import torch

        self.t, self.dev, self.rows, self.heads, self.k_heads, self.kd, self.vd, self.per_head = t, dev, rows, heads, k_heads, kd, vd, per_head
        self.rng = rng = np.random.default_rng(seed)
        n = lead + sum(rows) + tail
        self.n, self.lead = n, lead
        self.q, self.qx = to_type(rng.standard_normal((n, k_heads, kd)), t, dev)
        self.k, self.kx = to_type(rng.standard_normal((n, k_heads, kd)) / math.sqrt(kd), t, dev)
        self.v, self.vx = to_type(rng.standard_normal((n, heads, vd)), t, dev)
        rate = np.exp(rng.uniform(math.log(1e-3), math.log(2.0), heads))
        d = -rate if per_head else -rate * rng.uniform(0, 1.5, (n, heads))
        self.dx = (d if decay is None else decay(d)).astype(np.float32)
        self.d = torch.from_numpy(self.dx).to(dev)
        self.n_slots = len(rows) + 2 if n_slots is None else n_slots
        self.sx = rng.standard_normal((self.n_slots, heads, kd, vd)).astype(np.float32)
        self.s = torch.from_numpy(self.sx).to(dev)
        self.slots = rng.permutation(self.n_slots)[:len(rows)].astype(np.int32)
        self.starts = np.cumsum([lead] + list(rows)).astype(np.int32)
        self.out = torch.full((n, heads, vd), 9.0, dtype=torch_type(t), device=dev)
        self.new = torch.full_like(self.s, 4.0)

    def ints(self, x):
        import torch

        return torch.tensor(np.asarray(x), dtype=torch.int32, device=self.dev)

    def call(self, hl, lens=None, in_place=False, max_rows=None, **kw):
        state = hl.LinearState(self.s, self.n_slots, self.heads, self.kd, self.vd, None if in_place else self.new)
        batch = hl.LinearBatch(self.ints(self.slots), self.ints(self.starts), len(self.rows), self.n, max(self.rows) if max_rows is None else max_rows,
                               None if lens is None else self.ints(lens))
        kw = {"decay_per_head": self.per_head, **kw}
        hl.linear_attention(self.t, state, batch, self.q, self.k, self.v, self.out, self.d, self.k_heads, **kw)
        return self.out.double().cpu().numpy(), (self.s if in_place else self.new).double().cpu().numpy()

    def want(self, fresh=(), scale=None):
        """(out, its tolerance, states, their tolerance, which slots) of the batch."""
        group = self.heads // self.k_heads
        outs, states = {}, {}
        for i, n in enumerate(self.rows):
            if n == 0:
                continue
            at = slice(self.starts[i], self.starts[i] + n)
            s = np.zeros_like(self.sx[0]) if i in fresh else self.sx[self.slots[i]]
            d = np.broadcast_to(self.dx, (n, self.heads)) if self.per_head else self.dx[at]
            o, otol, s, stol = linear_ref(self.t, self.qx[at].repeat(group, 1), self.kx[at].repeat(group, 1), self.vx[at], d, s,
                                          self.kd ** -0.5 if scale is None else scale)
            outs[i], states[i] = (at, o, otol), (self.slots[i], s, stol)
        return outs, states

    def check(self, got, fresh=(), scale=None, in_place=False, skip=()):
        out, new = got
        outs, states = self.want(fresh, scale)
        touched_rows, touched = np.zeros(self.n, bool), np.zeros(self.n_slots, bool)
        for i in outs:
            at, o, otol = outs[i]
            slot, s, stol = states[i]
            touched_rows[at] = True
            if i in skip:
                continue
            touched[slot] = True
            for name, g, w, tol in (("out", out[at], o, otol), ("state", new[slot], s, stol)):
                err = np.abs(g - w)
                bad = ~(err <= tol) & ~(np.isnan(w) & np.isnan(g))
                assert not bad.any(), f"{name} of sequence {i}: {np.nanmax(err / tol)} of the tolerance, first at {np.argwhere(bad)[0]}"
        assert np.all(out[~touched_rows] == 9.0)
        assert np.array_equal(new[~touched], (self.sx if in_place else np.full_like(self.sx, 4.0))[~touched])


# rows of the sequences, heads, heads of q and k, k_dim, v_dim
BATCHES = [([1], 4, 2, 128, 128), ([1, 1, 1, 1, 1], 6, 2, 64, 96), ([4, 4, 2], 3, 3, 128, 64), ([0, 1, 0, 7, 0], 2, 1, 96, 256), ([16, 17], 2, 2, 256, 128),
           ([63, 64, 65], 2, 1, 128, 128), ([33], 5, 5, 192, 64), ([200], 4, 1, 64, 64), ([127, 1, 0, 300], 3, 1, 128, 192), ([129, 260], 2, 2, 96, 96),
           ([513], 1, 1, 256, 256), ([1000], 2, 1, 128, 128), ([95, 31, 160], 2, 1, 64, 256), ([70, 140], 2, 2, 192, 192), ([350], 2, 1, 256, 96)]


@TYPES
@pytest.mark.parametrize("rows,heads,k_heads,kd,vd", BATCHES, ids=lambda x: str(x).replace(" ", ""))
def test_linear(hl, dev, t, rows, heads, k_heads, kd, vd):
    print("[case] linear", TYPE_NAMES[t], rows, heads, k_heads, kd, vd, flush=True)
    c = Case(dev, t, rows, heads, k_heads, kd, vd, sum(rows) + kd)
    got = c.call(hl)
    c.check(got)
    assert np.array_equal(c.s.cpu().numpy(), c.sx)  # the states before the call are kept
    # in place, and a host that does not know the longest sequence
    c.check(c.call(hl, in_place=True, max_rows=0), in_place=True)


@TYPES
@pytest.mark.parametrize("rows", [[3, 1, 2], [100, 1, 65, 130]], ids=str)
def test_decay_per_head_and_sequences_that_begin(hl, dev, t, rows):
    """One decay a head; where seq_lens says that a sequence begins, its slot's bytes do not matter."""
    c = Case(dev, t, rows, 4, 2, 128, 64, 77, per_head=True, lead=3, tail=5)
    lens = [rows[0], rows[1] + 1, *rows[2:]]
    fresh = {0, *range(2, len(rows))}
    for i in fresh:
        c.s[int(c.slots[i])] = float("nan")
        c.sx[c.slots[i]] = np.nan
    c.check(c.call(hl, lens=lens), fresh=fresh)


@TYPES
def test_more_rows_than_the_host_says(hl, dev, t):
    c = Case(dev, t, [150, 3, 40], 2, 1, 128, 128, 5)
    c.check(c.call(hl, max_rows=1))
    c = Case(dev, t, [150, 3, 40], 2, 1, 128, 128, 6)
    c.check(c.call(hl, max_rows=30))


@TYPES
@pytest.mark.parametrize("rows", [[5], [230]], ids=str)
def test_decays_at_the_edges(hl, dev, t, rows):
    """No decay at all, a state that is emptied in the midst, decays far under the smallest number, and growth."""
    for way in range(4):
        def decay(d):
            d = d.copy()
            if way == 0:
                d[:] = 0
            elif way == 1:
                d[len(d) // 2] = -np.inf
                d[len(d) - 2, 0] = -np.inf
            elif way == 2:
                d[::3] = -3e38
                d[1::3] = -90.0
            else:
                d[:] = 0.01
            return d

        c = Case(dev, t, rows, 2, 1, 64, 64, 9 + way, decay=decay)
        if way == 1:
            # the reference's floor on decays stands for -inf
            c.dx[np.isinf(c.dx)] = -1e4
        if way == 2:
            c.dx = np.maximum(c.dx, -1e4)
        c.check(c.call(hl))


@TYPES
def test_long_far_decays_keep_their_differences(hl, dev, t):
    """Strong decays early must not cost the weak ones behind them their precision."""
    def decay(d):
        d = np.full_like(d, -1e-4)
        d[::7] = -60.0
        return d

    c = Case(dev, t, [300], 2, 2, 128, 64, 21, decay=decay)
    c.check(c.call(hl))


@TYPES
@pytest.mark.parametrize("rows,at", [([6], 3), ([200], 70), ([200], 64), ([200], 199), ([400], 130)], ids=str)
def test_values_that_are_not_finite_stay_behind(hl, dev, t, rows, at):
    """A bad value reaches its own row and later ones only, and of v only its own column."""
    for which, bad in (("v", np.nan), ("v", np.inf), ("k", np.nan), ("q", np.inf), ("d", np.nan)):
        c = Case(dev, t, rows, 3, 3, 64, 64, 31)
        x = {"v": c.v, "k": c.k, "q": c.q, "d": c.d}[which]
        if which == "d":
            x[at, 1] = bad
        else:
            x[at, 1, 20] = bad
        out, new = c.call(hl)
        outs, states = c.want()
        _, o, otol = outs[0]
        slot, s, stol = states[0]
        good, kept = np.ones_like(o, bool), np.ones_like(s, bool)
        if which == "v":
            good[at:, 1, 20], kept[1, :, 20] = False, False
        elif which == "q":
            good[at, 1] = False
        else:
            good[at:, 1], kept[1] = False, False
        err, serr = np.abs(out - o), np.abs(new[slot] - s)
        assert np.all(err[good] <= otol[good]), (which, bad, np.argwhere(good & ~(err <= otol))[0])
        assert not np.isfinite(out[~good]).any(), (which, bad)
        if which == "k":
            # k's own row of the state is bad, the others hold
            kept[1] = True
            kept[1, 20] = False
        if which != "q":
            assert not np.isfinite(new[slot][~kept]).any()
        assert np.all(serr[kept] <= stol[kept]), (which, bad)


@TYPES
def test_slots_out_of_range_and_named_twice(hl, dev, t):
    import torch

    for rows in ([1, 2, 1, 3], [70, 90, 1, 66]):
        c = Case(dev, t, rows, 2, 1, 128, 64, 13, n_slots=5)
        c.slots = np.array([2, 5, 2, -1], dtype=np.int32)
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        got = c.call(hl, status=status)
        assert int(status) == hl.STATUS_BAD_INDEX
        c.sx = np.concatenate([c.sx, np.zeros_like(c.sx[:1])])  # what the reference reads in the place of slot 5
        outs, _ = c.want()
        for i in (1, 2, 3):
            assert np.isnan(got[0][outs[i][0]]).all()
        c.sx = c.sx[:5]
        good = Case.check
        c.slots = np.array([2, 0, 0, 0], dtype=np.int32)
        good(c, got, skip=(1, 2, 3))
        # a call without faults clears the word, unless it is kept
        c.slots = np.array([2, 1, 0, 3], dtype=np.int32)
        c.call(hl, status=status, status_keep=True)
        assert int(status) == hl.STATUS_BAD_INDEX
        c.check(c.call(hl, status=status))
        assert int(status) == 0
        # a sequence without rows has no slot
        c.rows, c.starts, c.slots = [0, sum(rows)], np.array([0, 0, sum(rows)], dtype=np.int32), np.array([4, 4], dtype=np.int32)
        c.new.fill_(4.0)
        c.check(c.call(hl, status=status))
        assert int(status) == 0


@TYPES
def test_row_starts_out_of_order(hl, dev, t):
    """Falling or far row starts are cut; nothing outside the operands is touched."""
    c = Case(dev, t, [80, 3], 2, 1, 64, 64, 17, n_slots=6)
    c.starts, c.slots = np.array([40, 30, 1 << 30], dtype=np.int32), np.array([1, 2], dtype=np.int32)
    out, _ = c.call(hl)
    assert np.all(out[:30] == 9.0) and np.isfinite(out).all()


@TYPES
@pytest.mark.parametrize("rows", [[2, 1], [130, 20]], ids=str)
def test_row_fused_operands(hl, dev, t, rows):
    """q, k, v and out side by side in rows of an odd length, from an odd offset, with heads apart; decays in wider rows; the scale given."""
    import torch

    heads, kh, kd, vd = 4, 2, 64, 96
    c = Case(dev, t, rows, heads, kh, kd, vd, 41, lead=2)
    row = 2 * kh * kd + heads * (vd + 5) + heads * vd + 7
    wide = torch.full((c.n * row + 1,), 9.0, dtype=torch_type(t), device=dev)[1:].view(c.n, row)
    at = np.cumsum([0, kh * kd, kh * kd, heads * (vd + 5)])
    wide[:, :at[1]] = c.q.flatten(1)
    wide[:, at[1]:at[2]] = c.k.flatten(1)
    wide[:, at[2]:at[3]].unflatten(1, (heads, vd + 5))[..., :vd] = c.v
    before = wide.clone()
    decays = torch.full((c.n, heads + 3), float("nan"), device=dev)
    decays[:, :heads] = c.d
    state = hl.LinearState(c.s, c.n_slots, heads, kd, vd, c.new)
    batch = hl.LinearBatch(c.ints(c.slots), c.ints(c.starts), len(rows), c.n, max(rows))
    hl.linear_attention(t, state, batch, wide, wide[:, at[1]:], wide[:, at[2]:], wide[:, at[3]:], decays, kh, scale=0.75, decay_stride=heads + 3,
                        q_stride=row, k_stride=row, v_stride=row, v_head_stride=vd + 5, out_stride=row)
    end = at[3] + heads * vd
    out = wide[:, at[3]:end].unflatten(1, (heads, vd)).double().cpu().numpy()
    c.check((out, c.new.double().cpu().numpy()), scale=0.75)
    assert torch.equal(wide[:, :at[3]], before[:, :at[3]]) and torch.equal(wide[:, end:], before[:, end:])


@TYPES
def test_chunks_follow_steps(hl, dev, t):
    """A prompt at once, in pieces and row by row: the same sequence within the tolerances, and every run of the same call bitwise the same."""
    c = Case(dev, t, [150], 2, 1, 128, 128, 51)
    whole = c.call(hl)
    c.check(whole)
    again = c.call(hl)
    assert np.array_equal(whole[0], again[0]) and np.array_equal(whole[1], again[1])
    import torch

    for sizes in ([100, 50], [1] * 10 + [70] + [2] * 35):
        c.out.fill_(9.0)
        s, at = c.s.clone(), 0
        for n in sizes:
            state = hl.LinearState(s, c.n_slots, 2, 128, 128)
            batch = hl.LinearBatch(c.ints(c.slots), c.ints([at, at + n]), 1, c.n, n)
            hl.linear_attention(t, state, batch, c.q, c.k, c.v, c.out, c.d, 1)
            at += n
        new = torch.full_like(s, 4.0)
        new[int(c.slots[0])] = s[int(c.slots[0])]
        c.check((c.out.double().cpu().numpy(), new.double().cpu().numpy()))


@TYPES
@pytest.mark.parametrize("rows", [[3000], [1500, 20, 700]], ids=str)
def test_workspace(hl, dev, t, rows):
    """Long sequences with the stream's workspace, with one of the caller's, with a small one and with none."""
    import torch

    c = Case(dev, t, rows, 2, 1, 128, 64, 61)
    c.check(c.call(hl))
    state = hl.LinearState(c.s, c.n_slots, 2, 128, 64, c.new)
    batch = hl.LinearBatch(c.ints(c.slots), c.ints(c.starts), len(rows), c.n, max(rows))
    need = hl.linear_attention_workspace(t, state, batch, c.q, c.k, c.v, c.out, c.d, 1)
    for size in (need, need // 3, 16):
        size = max(size // 16 * 16, 16)
        ws = torch.full((size + 64,), 85, dtype=torch.uint8, device=dev)
        c.out.fill_(9.0)
        c.new.fill_(4.0)
        c.check(c.call(hl, workspace=ws, workspace_bytes=size))
        assert bool((ws[size:] == 85).all())


def test_captured_steps_and_prompts(hl, dev):
    """A decode step and a prompt captured whole, with workspaces of their own, and replayed with other rows, slots and lengths."""
    import torch

    for rows, other, max_rows in (([1, 1, 1], [1, 0, 1], 1), ([200, 100, 400], [400, 7, 90], 400)):
        c = Case(dev, BF16, rows, 2, 1, 128, 128, 71, tail=max(0, sum(other) - sum(rows)), n_slots=6)
        slots, starts = c.ints(c.slots), c.ints(c.starts)
        state = hl.LinearState(c.s, c.n_slots, 2, 128, 128, c.new)
        batch = hl.LinearBatch(slots, starts, 3, c.n, max_rows)
        need = hl.linear_attention_workspace(BF16, state, batch, c.q, c.k, c.v, c.out, c.d, 1)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)

        def run():
            hl.linear_attention(BF16, state, batch, c.q, c.k, c.v, c.out, c.d, 1, workspace=ws)

        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            run()
        for i in range(3):
            c.rows = rows if i % 2 == 0 else other
            c.starts = np.cumsum([0, *c.rows]).astype(np.int32)
            c.slots = np.roll(c.slots, i)
            slots.copy_(c.ints(c.slots))
            starts.copy_(c.ints(c.starts))
            c.out.fill_(9.0)
            c.new.fill_(4.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            c.check((c.out.double().cpu().numpy(), c.new.double().cpu().numpy()))


def test_many_sequences_and_far_slots(hl, dev):
    """Hundreds of sequences, and a pool whose far slots lie past 32 bits of bytes."""
    import torch

    seqs, heads, kd, vd = 700, 2, 64, 64
    n_slots = (1 << 32) // (4 * heads * kd * vd) + 800
    s = torch.empty(n_slots, heads, kd, vd, device=dev)
    c = Case(dev, BF16, [1] * seqs, heads, 1, kd, vd, 81, n_slots=seqs + 2)
    far = n_slots - c.n_slots
    s[far:] = c.s
    state = hl.LinearState(s, n_slots, heads, kd, vd)
    batch = hl.LinearBatch(c.ints(c.slots + far), c.ints(c.starts), seqs, c.n, 1)
    hl.linear_attention(BF16, state, batch, c.q, c.k, c.v, c.out, c.d, 1)
    c.check((c.out.double().cpu().numpy(), s[far:].double().cpu().numpy()), in_place=True)


@pytest.mark.parametrize("t, heads", [(F32, 64), (BF16, 40)], ids=["f32", "bf16"])
def test_long_sequences_in_place(hl, dev, t, heads):
    """The last segment of a sequence writes over the state that the first one begins with: in place is bitwise what it is beside it, with more
    segments than the GPU holds at once and without any."""
    import torch

    kh, kd, vd, lens = heads // 8, 128, 128, [2600, 300, 3300]
    rows, dt = sum(lens), torch.float32 if t == F32 else torch.bfloat16
    g = torch.Generator(device=dev).manual_seed(5)
    q, k, v = (torch.randn(rows, h, d, device=dev, generator=g).to(dt) for h, d in ((kh, kd), (kh, kd), (heads, vd)))
    decay = -0.02 * torch.rand(rows, heads, device=dev, generator=g)
    first = torch.randn(3, heads, kd, vd, device=dev, generator=g)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    batch = hl.LinearBatch(ints([2, 0, 1]), ints(np.concatenate([[0], np.cumsum(lens)]).tolist()), 3, rows, max(lens))
    out, new = torch.empty_like(v), torch.empty_like(first)
    beside = hl.LinearState(first, 3, heads, kd, vd, new)
    # one workspace for both: the stream's own may be smaller, and sequences cut elsewhere round elsewhere
    need = hl.linear_attention_workspace(t, beside, batch, q, k, v, out, decay, kh)
    assert need > 0
    space = torch.empty(need, dtype=torch.uint8, device=dev)
    hl.linear_attention(t, beside, batch, q, k, v, out, decay, kh, workspace=space, workspace_bytes=need)
    for _ in range(3):
        state, again = first.clone(), torch.empty_like(out)
        hl.linear_attention(t, hl.LinearState(state, 3, heads, kd, vd), batch, q, k, v, again, decay, kh, workspace=space, workspace_bytes=need)
        assert torch.equal(again, out) and torch.equal(state, new)


def test_replayed_in_place(hl, dev):
    """A batch of prompts, cut into segments, captured in place and replayed: every replay goes on from the states of the one before, as eager
    calls do."""
    import torch

    heads, kh, kd, vd, lens = 8, 4, 128, 128, [1500, 40, 2100]
    rows = sum(lens)
    g = torch.Generator(device=dev).manual_seed(6)
    q, k, v = (torch.randn(rows, h, d, device=dev, generator=g).bfloat16() for h, d in ((kh, kd), (kh, kd), (heads, vd)))
    decay = -0.05 * torch.rand(rows, heads, device=dev, generator=g)
    first = torch.randn(4, heads, kd, vd, device=dev, generator=g)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    batch = hl.LinearBatch(ints([3, 0, 1]), ints(np.concatenate([[0], np.cumsum(lens)]).tolist()), 3, rows, max(lens))
    state, out = first.clone(), torch.zeros_like(v)
    pool = hl.LinearState(state, 4, heads, kd, vd)
    need = hl.linear_attention_workspace(BF16, pool, batch, q, k, v, out, decay, kh)
    assert need > 0
    space = torch.empty(need, dtype=torch.uint8, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hl.linear_attention(BF16, pool, batch, q, k, v, out, decay, kh, workspace=space, workspace_bytes=need)
    eager, beside = first.clone(), torch.zeros_like(v)
    for _ in range(4):
        graph.replay()
        hl.linear_attention(BF16, hl.LinearState(eager, 4, heads, kd, vd), batch, q, k, v, beside, decay, kh, workspace=space, workspace_bytes=need)
        assert torch.equal(out, beside) and torch.equal(state, eager)
    assert torch.equal(state[2], first[2])


def test_two_streams_at_once(hl, dev):
    """Calls on two streams, each with its stream's workspace, do not meet: bitwise what they give one after the other."""
    import torch

    heads, kh, kd, vd, rows = 8, 8, 128, 128, 3000
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    sides, calls = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for seed in (1, 2):
        g = torch.Generator(device=dev).manual_seed(seed)
        q, k, v = (torch.randn(rows, heads, 128, device=dev, generator=g).bfloat16() for _ in range(3))
        decay = -0.05 * torch.rand(rows, heads, device=dev, generator=g)
        state = torch.randn(1, heads, kd, vd, device=dev, generator=g)
        new, out = torch.empty_like(state), torch.empty_like(v)
        args = (BF16, hl.LinearState(state, 1, heads, kd, vd, new), hl.LinearBatch(ints([0]), ints([0, rows]), 1, rows, rows), q, k, v, out, decay, kh)
        calls.append((args, new, out))
    want = []
    for (args, new, out), side in zip(calls, sides):
        torch.cuda.synchronize()
        hl.linear_attention(*args, stream=side.cuda_stream)
        torch.cuda.synchronize()
        want.append((new.clone(), out.clone()))
        new.zero_()
        out.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for (args, _, _), side in zip(calls, sides):
            hl.linear_attention(*args, stream=side.cuda_stream)
    torch.cuda.synchronize()
    for (_, new, out), (n, o) in zip(calls, want):
        assert torch.equal(new, n) and torch.equal(out, o)


@pytest.mark.parametrize("rows", [8, 70], ids=["steps", "chunks"])
def test_far_rows(hl, dev, rows):
    """Rows as far apart as they may be, their offsets past 32 bits."""
    import torch

    stride, kd, vd = 1 << 24, 64, 64
    far = [torch.empty(rows * stride, dtype=torch.float32, device=dev) for _ in range(2)]
    c = Case(dev, F32, [rows], 2, 2, kd, vd, 91)
    view = lambda b, at, x: b.view(rows, stride)[:, at:at + 128].copy_(x.reshape(rows, 128)) if x is not None else b.view(rows, stride)[:, at:at + 128]
    view(far[0], 0, c.q), view(far[0], 200, c.k), view(far[0], 1000, c.v)
    state = hl.LinearState(c.s, c.n_slots, 2, kd, vd, c.new)
    batch = hl.LinearBatch(c.ints(c.slots), c.ints(c.starts), 1, rows, rows)
    hl.linear_attention(F32, state, batch, far[0], far[0][200:], far[0][1000:], far[1], c.d, 2, q_stride=stride, k_stride=stride, v_stride=stride, out_stride=stride)
    c.check((view(far[1], 0, None).double().cpu().numpy().reshape(rows, 2, vd), c.new.double().cpu().numpy()))


@TYPES
@pytest.mark.parametrize("kd,vd", [(64, 96), (96, 64), (128, 128), (192, 192), (256, 64)])
def test_rows_between_steps_and_chunks(hl, dev, t, kd, vd):
    """The row counts where a call goes over from row after row to chunks, for each type and head size."""
    for n in (2, 3, 6, 7, 8, 9, 15, 16, 17):
        print("[case] linear between", TYPE_NAMES[t], kd, vd, n, flush=True)
        c = Case(dev, t, [n, 1, n - 1, 0], 3, 1, kd, vd, 7 * n)
        c.check(c.call(hl))
