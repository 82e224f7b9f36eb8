"""A decoder layer's step through the 8-bit projections, the heads' norms with the rotation, linear attention and the output projection, as
they are used together: prompts, then single tokens, eager and captured."""
import numpy as np
import pytest

from kv_helpers import BF16, F32, HALF_STEP, TYPE_NAMES, torch_type
from layer_helpers import gemm_ref, linear_ref, norm_rope_ref, quantized

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KH, DIM, ROT, SLOTS = 320, 4, 2, 64, 32, 4
QKV = (2 * KH + HEADS) * DIM


class Layer:
    def __init__(self, hl, dev, t, n):
        import torch

        self.hl, self.t, self.dev, self.n = hl, t, dev, n
        rng = np.random.default_rng(6)
        put = lambda x: torch.from_numpy(x).to(dev)  # noqa: E731
        self.w, self.ws = quantized((rng.standard_normal((QKV, HIDDEN)) / np.sqrt(HIDDEN)).astype(np.float32).astype(np.float64))
        self.o, self.os = quantized((rng.standard_normal((HIDDEN, HEADS * DIM)) / 16).astype(np.float32).astype(np.float64))
        self.wd, self.wsd, self.od, self.osd = map(put, (self.w, self.ws, self.o, self.os))
        self.norms = (1 + 0.2 * rng.standard_normal((2, DIM))).astype(np.float32)
        self.normd = put(self.norms)
        self.freqs = hl.rope_freqs(ROT, 1e4)[0]
        self.freqd = put(self.freqs)
        self.decay = -rng.uniform(0.01, 0.3, HEADS).astype(np.float32)
        self.decayd = put(self.decay)
        self.state = torch.zeros(SLOTS, HEADS, DIM, DIM, device=dev)
        empty = lambda *s, dt=torch_type(t): torch.zeros(*s, dtype=dt, device=dev)  # noqa: E731
        self.x, self.qkv, self.att, self.y = empty(n, HIDDEN), empty(n, QKV), empty(n, HEADS * DIM), empty(n, HIDDEN)
        self.codes, self.scales = empty(n, HIDDEN, dt=torch.int8), empty(n, dt=torch.float32)
        self.codes2, self.scales2 = empty(n, HEADS * DIM, dt=torch.int8), empty(n, dt=torch.float32)
        self.pos, self.slots, self.starts = (empty(k, dt=torch.int32) for k in (n, 2, 3))

    def run(self, rows):
        hl, t, n = self.hl, self.t, sum(rows)
        hl.quantize_rows(t, self.x, self.codes, self.scales, n, HIDDEN)
        hl.gemm_i8(t, self.wd, self.wsd, self.codes, self.scales, self.qkv, QKV, HIDDEN, n)
        q, k, v = self.qkv, self.qkv[:, KH * DIM:], self.qkv[:, 2 * KH * DIM:]
        row = dict(q_stride=QKV, k_stride=QKV)
        hl.norm_rope(t, self.pos, self.freqd, n, DIM, ROT, q, q, KH, q_norm=self.normd[0], k=k, k_out=k, n_kv_heads=KH, k_norm=self.normd[1], q_out_stride=QKV,
                     k_out_stride=QKV, **row)
        hl.linear_attention(t, hl.LinearState(self.state, SLOTS, HEADS, DIM, DIM), hl.LinearBatch(self.slots, self.starts, 2, n, max(rows)), q, k, v, self.att,
                            self.decayd, KH, decay_per_head=True, v_stride=QKV, **row)
        hl.quantize_rows(t, self.att, self.codes2, self.scales2, n, HEADS * DIM)
        hl.gemm_i8(t, self.od, self.osd, self.codes2, self.scales2, self.y, HIDDEN, HEADS * DIM, n)

    def check(self, rows, pos, before):
        """Every call's outputs against its own formula on the inputs that it had."""
        n, num = sum(rows), lambda x: x.double().cpu().numpy()  # noqa: E731
        near = lambda got, want, tol: np.testing.assert_array_less(np.abs(got - want), tol + 1e-30)  # noqa: E731
        c, s = quantized(num(self.x[:n]))
        assert np.array_equal(self.codes[:n].cpu().numpy(), c) and np.array_equal(self.scales[:n].cpu().numpy(), s)
        want, tol = gemm_ref(self.t, self.w, self.ws, c, s, HIDDEN)
        got = num(self.qkv[:n])
        v = slice(2 * KH * DIM, QKV)
        near(got[:, v], want[:, v], tol[:, v])
        # q and k were normed in place: the formula runs on the product that the device rounded to the type
        import torch

        rounded = torch.from_numpy(want).to(torch_type(self.t)).double().numpy()
        for i in range(2):
            heads = slice(i * KH * DIM, (i + 1) * KH * DIM)
            x = rounded[:, heads].reshape(n, KH, DIM)
            w, tol = norm_rope_ref(self.t, x, self.norms[i].astype(np.float64), 1e-6, pos, self.freqs, ROT, 0, 1.0)
            # a product that rounds to the type's neighbour is a whole step away, and turns into its pair; the norm halves nothing of it
            step = 2.02 * HALF_STEP[self.t] + 2.0 ** -20
            scale = np.abs(self.norms[i]).max() / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)
            near(got[:, heads].reshape(n, KH, DIM), w, tol + 2 * step * scale * np.abs(x).max(-1, keepdims=True) * 1.5)
        q, k = (got[:, i * KH * DIM:(i + 1) * KH * DIM].reshape(n, KH, DIM).repeat(HEADS // KH, 1) for i in range(2))
        att, at, state = num(self.att[:n]), 0, num(self.state)
        for i, m in enumerate(rows):
            r = slice(at, at + m)
            o, otol, st, stol = linear_ref(self.t, q[r], k[r], got[r, v].reshape(m, HEADS, DIM), np.broadcast_to(self.decay, (m, HEADS)),
                                           before[int(self.slots[i])], DIM ** -0.5)
            near(att[r].reshape(m, HEADS, DIM), o, otol)
            near(state[int(self.slots[i])], st, stol)
            at += m
        c, s = quantized(att)
        want, tol = gemm_ref(self.t, self.o, self.os, c, s, HEADS * DIM)
        near(num(self.y[:n]), want, tol)


@pytest.mark.parametrize("t", [F32, BF16], ids=lambda t: TYPE_NAMES[t])
def test_layer(hl, dev, t):
    import torch

    layer = Layer(hl, dev, t, 150)
    g = torch.Generator(device=dev).manual_seed(9)
    layer.slots.copy_(torch.tensor([3, 1]))

    def inputs(rows, first):
        n = sum(rows)
        layer.x[:n] = torch.randn(n, HIDDEN, device=dev, generator=g)
        pos = np.concatenate([np.arange(f, f + m) for f, m in zip(first, rows)]).astype(np.int32)
        layer.pos[:n] = torch.from_numpy(pos).to(dev)
        layer.starts.copy_(torch.tensor([0, rows[0], n]))
        return pos

    lens = [110, 40]
    pos = inputs(lens, [0, 0])
    before = layer.state.double().cpu().numpy()
    layer.run(lens)
    layer.check(lens, pos, before)
    # single tokens, eager on a side stream, then the step captured there and replayed
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = None
    for i in range(4):
        pos = inputs([1, 1], lens)
        before = layer.state.double().cpu().numpy()
        torch.cuda.synchronize()
        if i == 0:
            with torch.cuda.stream(s):
                layer.run([1, 1])
        else:
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=s):
                    layer.run([1, 1])
            graph.replay()
        torch.cuda.synchronize()
        layer.check([1, 1], pos, before)
        lens = [n + 1 for n in lens]
