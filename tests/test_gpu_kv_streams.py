"""A decode step captured whole and replayed, and two threads that serve at once on streams of their own."""
import threading

import numpy as np
import pytest

from kv_helpers import BF16, F32, TYPE_NAMES, batch, torch_type

pytestmark = pytest.mark.gpu

PAGES, LAYERS, KV, GROUP, DIM, BLOCK, SLOTS, WIDTH = 200, 2, 2, 4, 128, 16, 3, 40
HEADS = KV * GROUP


class Server:
    """Three sequences, the buffers of their decode step, and the step: every length is on the device."""

    def __init__(self, hl, dev, t, seed):
        import torch

        self.hl, self.t, self.dev = hl, t, dev
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        self.pool = torch.zeros(PAGES, hl.kv_page_bytes(LAYERS, KV, DIM, BLOCK), dtype=torch.uint8, device=dev)
        self.state = hl.KvState(ints([0] * PAGES), ints([0] * SLOTS), ints([[-1] * WIDTH] * SLOTS), SLOTS, WIDTH)
        self.cache = hl.KvCache(self.pool, PAGES, LAYERS, KV, DIM, BLOCK)
        self.slots, self.lens, self.status = ints([0, 1, 2]), ints([0] * SLOTS), ints([0])
        self.freqs = torch.from_numpy(hl.rope_freqs(DIM, 1e4)[0]).to(dev)
        self.rng = torch.Generator(device=dev).manual_seed(seed)
        self.q, self.k, self.v, self.out = (torch.zeros(SLOTS, h, DIM, dtype=torch_type(t), device=dev) for h in (HEADS, KV, KV, HEADS))
        self.batch = hl.KvBatch(self.state.tables, WIDTH, self.lens, ints(batch([1] * SLOTS).tolist()), SLOTS, SLOTS, 1)
        self.prefill([300, 15, 511])

    def prefill(self, lens):
        import torch

        hl, n = self.hl, sum(lens)
        self.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        hl.kv_resize(self.cache, self.state, self.slots, self.lens, SLOTS, status=self.status)
        starts = torch.from_numpy(batch(lens)).to(self.dev)
        k, v = (torch.randn(n, KV, DIM, device=self.dev, generator=self.rng).to(torch_type(self.t)) for _ in range(2))
        b = hl.KvBatch(self.state.tables, WIDTH, self.lens, starts, SLOTS, n)
        for layer in range(LAYERS):
            hl.kv_write(self.t, self.cache, layer, b, k, v, status=self.status, status_keep=True)

    def inputs(self):
        import torch

        for x in (self.q, self.k, self.v):
            x.copy_(torch.randn(x.shape, device=self.dev, generator=self.rng))

    def step(self):
        hl = self.hl
        self.lens.add_(1)
        hl.kv_resize(self.cache, self.state, self.slots, self.lens, SLOTS, status=self.status, status_keep=True)
        hl.rope(self.t, self.lens, self.freqs, SLOTS, DIM, DIM, self.q, self.q, HEADS, k=self.k, k_out=self.k, n_kv_heads=KV)
        for layer in range(LAYERS):
            hl.kv_write(self.t, self.cache, layer, self.batch, self.k, self.v, status=self.status, status_keep=True)
            hl.attention(self.t, self.cache, layer, self.batch, self.q, self.out, HEADS, status=self.status, status_keep=True)
            self.q.add_(self.out)

    def same_as(self, other):
        import torch

        return all(torch.equal(x, y) for x, y in ((self.out, other.out), (self.pool, other.pool), (self.lens, other.lens),
                                                  (self.state.tables, other.state.tables), (self.state.refs, other.state.refs)))


@pytest.mark.parametrize("t", [F32, BF16], ids=lambda t: TYPE_NAMES[t])
def test_captured_decode(hl, dev, t):
    """One graph, replayed while the sequences grow over pages: bitwise the eager steps, every replay."""
    import torch

    print("[case] captured decode", TYPE_NAMES[t], flush=True)
    eager, captured = Server(hl, dev, t, 1), Server(hl, dev, t, 1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        captured.inputs()
        captured.step()  # the stream has its workspace now
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            captured.step()
    eager.inputs()
    eager.step()
    torch.cuda.synchronize()
    assert eager.same_as(captured)
    for _ in range(20):
        for x in (eager, captured):
            x.inputs()
        eager.step()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert eager.same_as(captured)
    assert eager.status.item() == 0 and captured.status.item() == 0
    assert captured.lens.tolist() == [321, 36, 532]
    with torch.cuda.stream(s):
        hl.stream_release()


def test_two_threads(hl, dev):
    """Two threads, each with a stream, a cache and a server of its own: what each would have got alone."""
    import torch

    print("[case] two threads", flush=True)
    kinds = [(F32, 3), (BF16, 4)]

    def serve(t, seed):
        x = Server(hl, dev, t, seed)
        for _ in range(15):
            x.inputs()
            x.step()
        return x

    alone = [serve(*k) for k in kinds]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                got[i] = serve(*kinds[i])
                s.synchronize()
                hl.stream_release()
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for x, y in zip(alone, got):
        assert x.same_as(y)
