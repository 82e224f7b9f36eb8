"""Page calls that are refused for want of scratch memory leave the status word alone, and a call without entries needs none.
No GPU calls."""
import pytest

from test_kv_host import A, B, D, E, F, _cache, refused


@pytest.mark.parametrize("name", ["kv_resize", "kv_fork"])
def test_scratch_memory(hl, name):
    """A pool whose pages do not fit the scratch memory: refused before the status word is cleared (which, with no GPU here, would
    be what fails); without entries there is nothing to do."""
    call = getattr(hl, name)
    far = dict(refs=1 << 44, lens=1 << 45, tables=1 << 46, n_slots=4, table_width=4)
    big = _cache(hl, pages=9_000_000, layers=1, heads=1, dim=64)
    assert "too many pages" in refused(hl, hl.ErrorCode.Unsupported, call, big, hl.KvState(**far), 1 << 47, 1 << 48, 3, status=1 << 49, stream=0)
    call(big, hl.KvState(**far), 0, 0, 0, stream=0)
    call(_cache(hl, pool=A), hl.KvState(B, B + 0x1000, B + 0x2000, 4, 4), D, E, 0, stream=0)
    refused(hl, hl.ErrorCode.Kernel, call, _cache(hl, pool=A), hl.KvState(B, B + 0x1000, B + 0x2000, 4, 4), D, E, 0, status=F + 2, stream=0)
