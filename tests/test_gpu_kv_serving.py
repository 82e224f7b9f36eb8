"""Rotary positions, the cache's pages, its writes and the attention over it as a server runs them together."""
import numpy as np
import pytest

from kv_helpers import BF16, F32, TYPE_NAMES, Cache, attention_bound, attention_ref, batch, to_type, write_ref
from test_gpu_rope import rope_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [F32, BF16], ids=lambda t: TYPE_NAMES[t])
def test_serve(hl, dev, t):
    """Prompts, decode steps, a verify step that is taken back in part, forks that go their own ways, freed slots and a
    packed pool: at every step the attention's values over what the cache then holds, and what it holds."""
    import torch

    rng = np.random.default_rng(9)
    n_pages, layers, kv, group, dim, block, rot, slots, width = 60, 2, 2, 3, 64, 16, 32, 6, 12
    heads = kv * group
    cache = Cache(n_pages, layers, kv, dim, block)  # what the pages should hold, by their numbers on the GPU
    pool = torch.from_numpy(cache.bytes.copy()).to(dev)
    ints = lambda x: torch.tensor(np.asarray(x, dtype=np.int32).copy(), device=dev)  # noqa: E731
    refs, lens, tables = ints(np.zeros(n_pages)), ints(np.zeros(slots)), ints(np.full((slots, width), -1))
    c, state = hl.KvCache(pool, n_pages, layers, kv, dim, block), hl.KvState(refs, lens, tables, slots, width)
    status = ints([0])
    freqs_h, _ = hl.rope_freqs(rot, 1e4)
    freqs = torch.from_numpy(freqs_h).to(dev)
    now = np.zeros(slots, dtype=np.int64)

    def resize(which, news):
        hl.kv_resize(c, state, ints(which), ints(news), len(which), status=status)
        now[which] = news

    def held():
        """The cache as the GPU holds it."""
        got = Cache(n_pages, layers, kv, dim, block)
        got.bytes[:] = pool.cpu().numpy()
        return got

    def step(which, rows):
        """`rows` new tokens of each slot through both layers."""
        resize(which, now[which] + rows)
        starts, n = batch([rows] * len(which)), rows * len(which)
        table = tables[torch.tensor(which, device=dev)].contiguous()
        b = hl.KvBatch(table, width, ints(now[which]), ints(starts), len(which), n, rows, int(now.max()))
        pos = np.concatenate([np.arange(now[s] - rows, now[s]) for s in which]).astype(np.int32)
        for layer in range(layers):
            q, qx = to_type(rng.standard_normal((n, heads, dim)), t, dev)
            k, kx = to_type(rng.standard_normal((n, kv, dim)), t, dev)
            v, vx = to_type(rng.standard_normal((n, kv, dim)), t, dev)
            hl.rope(t, ints(pos), freqs, n, dim, rot, q, q, heads, k=k, k_out=k, n_kv_heads=kv)
            for got, x in ((q, qx), (k, kx)):
                want, reach = rope_ref(x, pos, freqs_h, rot, 0, 1.0)
                assert np.abs(got.double().cpu().numpy() - want).max() <= np.abs(reach).max() * (2.0 ** -8 if t == BF16 else 2.0 ** -20)
            before = held()
            hl.kv_write(t, c, layer, b, k, v, status=status, status_keep=True)
            table_h = table.cpu().numpy()
            write_ref(before, layer, table_h, now[which], starts, k.double().cpu().numpy(), v.double().cpu().numpy())
            assert np.array_equal(held().bytes, before.bytes)
            out = torch.empty_like(q)
            hl.attention(t, c, layer, b, q, out, heads, status=status, status_keep=True)
            want, weight, reach = attention_ref(before, layer, table_h, now[which], starts, q.double().cpu().numpy())
            tol = attention_bound(t, dim, int(now.max()), want, weight, reach, float(before.scales.max()) * 127)
            assert np.all(np.abs(out.double().cpu().numpy() - want) <= tol)
        assert status.item() == 0

    step([0, 3], 37)
    step([1], 16)
    for _ in range(3):
        step([0, 1, 3], 1)
    step([0, 3], 4)
    resize([0], [now[0] - 3])  # three of the four drafts were wrong
    step([0, 1, 3], 1)
    hl.kv_fork(c, state, ints([0, 0, 3]), ints([2, 4, 5]), 3, status=status)
    now[[2, 4, 5]] = now[[0, 0, 3]]
    step([0, 2, 4, 5], 2)
    resize([4, 2], [now[4] - 12, now[2] - 12])  # into pages that slot 0 holds too
    step([4, 2], 3)
    resize([0, 3], [0, 0])
    hl.kv_compact(c, state)
    live = int((refs > 0).sum())
    assert torch.all(refs[:live] > 0) and not torch.any(refs[live:])
    step([1, 2, 4, 5], 5)
    step([0], 90)
    resize(list(range(slots)), [0] * slots)
    assert not torch.any(refs)
