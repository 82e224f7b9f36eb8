"""The pages' owner on the GPU against a model of it in Python: counts, lengths, tables and the pages' bytes."""
import numpy as np
import pytest

from kv_helpers import PagesModel

pytestmark = pytest.mark.gpu

GEOMETRY = dict(layers=2, heads=1, dim=64, block=16)  # 4.1 KB a page; the big ones below


class Owner:
    """The state on the GPU beside its model; every page's bytes begin as its own number's."""

    def __init__(self, hl, dev, n_pages, slots, width, layers=2, heads=1, dim=64, block=16, stride=0):
        import torch

        self.hl, self.dev, self.torch = hl, dev, torch
        self.model = PagesModel(n_pages, block, slots, width)
        per = hl.kv_page_bytes(layers, heads, dim, block)
        self.pool = torch.arange(n_pages, dtype=torch.int32, device=dev)[:, None].repeat(1, per // 4).contiguous()
        self.pool ^= torch.arange(per // 4, dtype=torch.int32, device=dev) << 12
        self.first = self.pool.clone()
        self.stride = stride or width
        self.refs = torch.zeros(n_pages, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(slots, dtype=torch.int32, device=dev)
        self.tables = torch.full((slots, self.stride), -1, dtype=torch.int32, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self.cache = hl.KvCache(self.pool, n_pages, layers, heads, dim, block)
        self.state = hl.KvState(self.refs, self.lens, self.tables, slots, width, stride)

    def ints(self, x):
        return self.torch.tensor(list(x), dtype=self.torch.int32, device=self.dev)

    def resize(self, slots, news):
        self.hl.kv_resize(self.cache, self.state, self.ints(slots), self.ints(news), len(slots), status=self.status)
        self.same(self.model.resize(slots, news))

    def fork(self, src, dst):
        self.hl.kv_fork(self.cache, self.state, self.ints(src), self.ints(dst), len(src), status=self.status)
        self.same(self.model.fork(src, dst))

    def compact(self):
        live = self.torch.zeros(1, dtype=self.torch.int32, device=self.dev)
        self.hl.kv_compact(self.cache, self.state, live=live)
        assert live.item() == self.model.compact()
        self.same(None)

    def same(self, status):
        m = self.model
        if status is not None:
            assert self.status.item() == status
        assert self.lens.tolist() == m.lens
        assert self.tables[:, :m.width].tolist() == m.tables
        assert self.torch.all(self.tables[:, m.width:] == -1)
        assert self.refs.tolist() == m.refs
        assert self.torch.equal(self.pool, self.first[self.torch.tensor(m.owner, device=self.dev)])


def test_resize(hl, dev):
    o = Owner(hl, dev, 20, 6, 5, stride=7)
    o.resize([2, 0, 5], [33, 16, 1])
    o.resize([0, 2, 1, 5], [17, 32, 0, 16])  # grows a page, drops one, stays empty, stays in its page
    o.resize([3, 4], [80, 16])
    o.resize([2, 5, 3], [0, 0, 15])  # freed pages serve from the next call on
    o.resize([1, 2], [48, 5])
    o.resize([0, 1, 2, 3, 4, 5], [0] * 6)
    assert o.refs.sum().item() == 0


def test_resize_refusals_on_the_device(hl, dev):
    """Slots out of range, named twice, negative lengths and lengths past the table leave everything else as it should be;
    when the pages run out, later entries that need some get none and others still do."""
    o = Owner(hl, dev, 8, 5, 4)
    o.resize([0, 9, -1, 0, 1], [20, 16, 16, 64, 30])
    o.resize([2, 3, 1], [65, -3, 31])
    o.resize([2, 3, 0, 1, 4], [64, 16, 3, 40, 1])  # 4 pages are free: 2 takes them, 3 gets none, 0 shrinks
    o.resize([3], [16])
    o.resize([4, 1], [40, 10])


def test_fork_and_copy_on_write(hl, dev):
    o = Owner(hl, dev, 24, 8, 6)
    o.resize([0, 1], [37, 32])
    o.fork([0, 0, 1, 5], [2, 3, 4, 6])  # two forks of a slot, one without a partial page, one of an empty slot
    o.resize([2, 0, 4], [38, 48, 33])
    o.resize([4, 2], [20, 30])  # back into pages that the source holds too
    o.resize([4, 2, 0, 3], [21, 33, 60, 37])  # grown behind shared tokens: copies
    o.fork([2], [7])
    o.resize([7, 2], [40, 40])
    o.resize(list(range(8)), [0] * 8)
    assert o.refs.sum().item() == 0


def test_fork_refusals_on_the_device(hl, dev):
    o = Owner(hl, dev, 6, 6, 4)
    o.resize([0, 1], [20, 40])
    o.fork([0, 0, 8, 0, 1, 1], [0, 9, 2, 1, 2, 2])  # itself, out of range (twice), not empty; 1 -> 2; 2 named twice
    o.fork([0, 1], [3, 4])  # no page is free
    assert o.status.item() == hl.STATUS_KV_FULL
    o.resize([2, 1], [0, 16])
    o.fork([0, 1, 0], [3, 4, 5])


def test_compact(hl, dev):
    o = Owner(hl, dev, 40, 7, 6)
    o.resize(range(7), [30, 96, 17, 5, 64, 33, 80])
    o.resize([1, 3, 5], [0, 0, 0])
    o.fork([4, 0], [1, 3])
    o.compact()
    o.compact()  # packed already
    o.resize([1, 4, 0], [70, 0, 31])
    o.compact()
    o.resize(range(7), [0] * 7)
    o.compact()


def test_many_slots_and_pages(hl, dev):
    """Lists of 1024 and more pages than the deciding workgroup looks at in a step."""
    slots = 1030
    o = Owner(hl, dev, 9001, slots, 40)
    rng = np.random.default_rng(0)
    for _ in range(3):
        order = rng.permutation(slots)[:1024].tolist()
        o.resize(order, rng.integers(0, 200, 1024).tolist())
    empty = [s for s in range(slots) if o.model.lens[s] == 0]
    full = [s for s in range(slots) if o.model.lens[s]]
    o.fork([full[i % 5] for i in range(len(empty))], empty)
    o.compact()
    assert o.model.refs[0] and not o.model.refs[-1]


def test_long_growth_and_large_pages(hl, dev):
    """One slot takes thousands of pages at once, and pages of 1.06 MB move."""
    o = Owner(hl, dev, 6000, 3, 5000)
    o.resize([1, 0], [16 * 4500 - 3, 100])
    o.resize([1, 2], [200, 40])
    o.compact()
    o = Owner(hl, dev, 40, 6, 4, layers=8, heads=4, dim=128, block=128)
    o.resize(range(4), [300, 129, 511, 1])
    o.fork([0, 2], [4, 5])
    o.resize([0, 2], [0, 0])
    o.compact()


@pytest.mark.parametrize("entries", [0, 1, 9])
def test_copy_pages(hl, dev, entries):
    o = Owner(hl, dev, 30, 1, 1, layers=3, heads=2, dim=96, block=32)
    src, dst = [3, 3, 29, 7, 30, -1, 5, 0, 1][:entries], [0 + 10, 11, 12, 13, 14, 15, 31, 16, 17][:entries]
    hl.kv_copy_pages(o.cache, o.ints(src), o.ints(dst), entries, status=o.status)
    bad = 0
    for s, d in zip(src, dst):
        if 0 <= s < 30 and 0 <= d < 30:
            o.model.owner[d] = s
        else:
            bad = hl.STATUS_BAD_INDEX
    o.same(bad)


def test_stray_ids_in_tables(hl, dev):
    """An id in a table that is no page is passed over and reported: nothing outside the pool or the counts is touched."""
    o = Owner(hl, dev, 10, 3, 4)
    o.resize([0], [40])
    o.tables[0, 0] = 10
    o.tables[0, 2] = -7
    hl.kv_fork(o.cache, o.state, o.ints([0]), o.ints([1]), 1, status=o.status)
    assert o.status.item() == hl.STATUS_BAD_INDEX
    assert o.tables[1].tolist() == [10, 1, 3, -1] and o.refs.tolist() == [1, 2, 1, 1, 0, 0, 0, 0, 0, 0]
    hl.kv_resize(o.cache, o.state, o.ints([0, 1]), o.ints([0, 41]), 2, status=o.status)
    assert o.status.item() == hl.STATUS_BAD_INDEX
    assert o.tables[0].tolist() == [-1] * 4 and o.refs.tolist() == [1, 1, 1, 1, 0, 0, 0, 0, 0, 0]
    hl.kv_compact(o.cache, o.state)
    assert o.tables[1].tolist() == [10, 1, 3, -1]
    assert o.torch.equal(o.pool, o.first)


def test_captured_growth(hl, dev):
    """A captured resize follows the lists' and the state's values at each replay, on a stream of its own."""
    import torch

    s = torch.cuda.Stream()
    o = Owner(hl, dev, 60, 3, 10)
    slots, news = o.ints([0, 1, 2]), o.ints([0, 0, 0])
    torch.cuda.synchronize()  # the pool was made on another stream
    with torch.cuda.stream(s):
        hl.kv_resize(o.cache, o.state, slots, news, 3, status=o.status)  # the stream's workspace
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            news += 7
            hl.kv_resize(o.cache, o.state, slots, news, 3, status=o.status)
            hl.kv_compact(o.cache, o.state)
    lens = [0, 0, 0]
    for step in range(6):
        if step == 3:
            with torch.cuda.stream(s):
                news -= 15
            lens = [n - 15 for n in lens]
        g.replay()
        s.synchronize()
        torch.cuda.synchronize()
        lens = [n + 7 for n in lens]
        status = o.model.resize([0, 1, 2], lens)
        o.model.compact()
        o.same(status)
    with torch.cuda.stream(s):
        hl.stream_release()
