"""Ids out of range in the tables of the pages' owner: an entry that would copy such a page, or write behind its tokens, is
left as it is; nothing gets a page whose bytes are another sequence's."""
import pytest

from test_gpu_kv_pages import Owner

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stray", [-7, 10, 1 << 30])
def test_fork_of_a_stray_last_page(hl, dev, stray):
    """The source's last page is not full and is none: its entry takes no page and sets no length, the others go on."""
    o = Owner(hl, dev, 10, 5, 4)
    o.resize([0, 1], [40, 20])  # pages 0 1 2 and 3 4
    o.tables[0, 2] = stray
    hl.kv_fork(o.cache, o.state, o.ints([0, 1]), o.ints([2, 3]), 2, status=o.status)
    assert o.status.item() == hl.STATUS_BAD_INDEX
    assert o.lens.tolist() == [40, 20, 0, 20, 0]
    assert o.tables.tolist() == [[0, 1, stray, -1], [3, 4, -1, -1], [-1] * 4, [3, 5, -1, -1], [-1] * 4]
    assert o.refs.tolist() == [1, 1, 1, 2, 1, 1, 0, 0, 0, 0]
    assert o.torch.equal(o.pool[5], o.first[4]) and o.torch.equal(o.pool[6:], o.first[6:])


@pytest.mark.parametrize("stray", [-7, 10, 1 << 30])
def test_growth_behind_a_stray_last_page(hl, dev, stray):
    """A slot whose last page is not full and is none does not grow; it shrinks, and frees what it holds."""
    o = Owner(hl, dev, 10, 4, 4)
    o.resize([0, 1], [40, 20])
    o.tables[0, 2] = stray
    hl.kv_resize(o.cache, o.state, o.ints([0, 1, 2]), o.ints([60, 33, 5]), 3, status=o.status)
    assert o.status.item() == hl.STATUS_BAD_INDEX
    assert o.lens.tolist() == [40, 33, 5, 0]
    assert o.tables.tolist() == [[0, 1, stray, -1], [3, 4, 5, -1], [6, -1, -1, -1], [-1] * 4]
    assert o.refs.tolist() == [1] * 7 + [0] * 3
    hl.kv_resize(o.cache, o.state, o.ints([0]), o.ints([47]), 1, status=o.status)  # inside the page
    assert o.status.item() == hl.STATUS_BAD_INDEX and o.lens[0].item() == 40
    hl.kv_resize(o.cache, o.state, o.ints([0]), o.ints([32]), 1, status=o.status)
    assert o.status.item() == hl.STATUS_BAD_INDEX and o.lens[0].item() == 32 and o.tables[0].tolist() == [0, 1, -1, -1]
    hl.kv_resize(o.cache, o.state, o.ints([0]), o.ints([64]), 1, status=o.status)
    assert o.status.item() == 0 and o.tables[0].tolist() == [0, 1, 7, 8]  # page 2 is held still: its id was lost, not its count
    assert o.torch.equal(o.pool, o.first)


def test_stray_whole_pages(hl, dev):
    """Among whole pages: shared as they are, given back as -1, counted by neither."""
    o = Owner(hl, dev, 10, 3, 4)
    o.resize([0], [40])
    o.tables[0, 0] = 10
    hl.kv_fork(o.cache, o.state, o.ints([0]), o.ints([1]), 1, status=o.status)
    assert o.status.item() == hl.STATUS_BAD_INDEX
    assert o.tables[1].tolist() == [10, 1, 3, -1] and o.lens.tolist() == [40, 40, 0]
    assert o.refs.tolist() == [1, 2, 1, 1, 0, 0, 0, 0, 0, 0]
    assert o.torch.equal(o.pool[3], o.first[2])
    hl.kv_resize(o.cache, o.state, o.ints([0, 1]), o.ints([0, 41]), 2, status=o.status)
    assert o.status.item() == hl.STATUS_BAD_INDEX
    assert o.tables[0].tolist() == [-1] * 4 and o.tables[1].tolist() == [10, 1, 3, -1]
    assert o.refs.tolist() == [1, 1, 0, 1, 0, 0, 0, 0, 0, 0]
