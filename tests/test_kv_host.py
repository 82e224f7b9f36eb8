"""Attention over the 8-bit cache on the host: the rotary frequencies, the page geometry, and the calls that are refused
before anything is enqueued. No GPU calls."""
import ctypes
import math

import numpy as np
import pytest

from kv_helpers import BF16, F16, F32, page_bytes


def test_page_bytes(hl):
    for layers, heads, dim, block in [(1, 1, 64, 16), (16, 4, 256, 16), (2, 8, 128, 64), (3, 5, 96, 128), (64, 8, 192, 32)]:
        assert hl.kv_page_bytes(layers, heads, dim, block) == page_bytes(layers, heads, dim, block)
    for bad in [(0, 1, 64, 16), (1, 0, 64, 16), (1, 1, 80, 16), (1, 1, 512, 16), (1, 1, 64, 8), (1, 1, 64, 48), (1, 1, 64, 256),
                (4096, 1024, 256, 128)]:
        assert hl.kv_page_bytes(*bad) == 0


@pytest.mark.parametrize("rot", [2, 64, 128, 510])
def test_rope_freqs(hl, rot):
    i = np.arange(rot // 2)
    plain = 1e7 ** (-2 * i / rot)
    near = lambda a, b: np.testing.assert_allclose(a, b, rtol=1e-14)  # noqa: E731  (pow within an ulp or two)
    f, m = hl.rope_freqs(rot, 1e7)
    near(f, plain)
    assert m == 1.0
    f, m = hl.rope_freqs(rot, 1e7, scaling=hl.RopeScaling.LINEAR, scale=4.0)
    near(f, plain / 4)
    assert m == 1.0
    f, m = hl.rope_freqs(rot, 1e7, scaling=hl.RopeScaling.NTK, scale=4.0)
    near(f, plain if rot == 2 else (1e7 * 4.0 ** (rot / (rot - 2))) ** (-2 * i / rot))
    f, m = hl.rope_freqs(rot, 1e7, scaling=hl.RopeScaling.YARN, scale=8.0, context=4096)
    assert m == np.float32(0.1 * math.log(8.0) + 1)
    turns = plain * 4096 / (2 * math.pi)
    # a pair that turns clearly more than 32 times keeps its frequency, one that turns clearly less than once is divided
    pair = math.log(1e7) * 2 / rot  # a pair's step in the logarithm of its turns
    near(f[np.log(turns) > math.log(32) + pair], plain[np.log(turns) > math.log(32) + pair])
    near(f[np.log(turns) < -pair], plain[np.log(turns) < -pair] / 8)
    assert np.all(f <= plain * (1 + 1e-14)) and np.all(f >= plain / 8 * (1 - 1e-14))
    f, m = hl.rope_freqs(rot, 1e7, scaling=hl.RopeScaling.YARN, scale=1.0, context=4096)
    near(f, plain)
    assert m == 1.0


def refused(hl, code, call, *args, **kw):
    with pytest.raises(hl.HaloError) as e:
        call(*args, **kw)
    assert e.value.code == code, e.value
    return str(e.value)


def test_rope_freqs_refusals(hl):
    K, U, C = hl.ErrorCode.Kernel, hl.ErrorCode.Unsupported, hl.ErrorCode.Config
    refused(hl, U, hl.rope_freqs, 3)
    refused(hl, U, hl.rope_freqs, 0)
    refused(hl, U, hl.rope_freqs, 514)
    refused(hl, K, hl.rope_freqs, 64, 0.5)
    refused(hl, K, hl.rope_freqs, 64, math.inf)
    refused(hl, C, hl.rope_freqs, 64, 1e4, scaling=9)
    refused(hl, K, hl.rope_freqs, 64, 1e4, scaling=hl.RopeScaling.LINEAR, scale=0.5)
    refused(hl, K, hl.rope_freqs, 64, 1e4, scaling=hl.RopeScaling.NTK, scale=math.nan)
    refused(hl, K, hl.rope_freqs, 64, 1e4, scaling=hl.RopeScaling.YARN, scale=2.0)
    refused(hl, K, hl.rope_freqs, 64, 1e4, scaling=hl.RopeScaling.YARN, scale=2.0, context=4096, beta_slow=40.0)


# Addresses that no call reaches: every call below is refused on the host.
A, B, C_, D, E, F = (0x10000000 * i for i in range(1, 7))


def test_rope_refusals(hl):
    K, U, C = hl.ErrorCode.Kernel, hl.ErrorCode.Unsupported, hl.ErrorCode.Config

    def call(t=F32, pos=A, freqs=B, n=8, dim=128, rot=128, q=C_, q_out=D, heads=4, **kw):
        hl.rope(t, pos, freqs, n, dim, rot, q, q_out, heads, stream=0, **kw)

    refused(hl, U, call, t=12)
    refused(hl, C, call, pairs=2)
    refused(hl, K, call, rot=3)
    refused(hl, K, call, rot=0)
    refused(hl, K, call, rot=130)
    refused(hl, K, call, dim=1024, rot=514)
    refused(hl, U, call, dim=0, rot=0)
    refused(hl, K, call, q=0)
    refused(hl, K, call, q_out=0)
    refused(hl, K, call, pos=0)
    refused(hl, K, call, freqs=0)
    refused(hl, K, call, freqs=B + 4)
    refused(hl, K, call, pos=A + 2)
    refused(hl, K, call, q=C_ + 2)
    refused(hl, K, call, t=BF16, q_out=D + 1)
    refused(hl, K, call, q_stride=100)
    refused(hl, K, call, q_head_stride=100)
    refused(hl, K, call, q_stride=1 << 41)
    refused(hl, K, call, factor=math.nan)
    refused(hl, K, call, q_out=C_ + 512)  # overlaps its input, not in place
    refused(hl, K, call, q_out=C_, q_out_stride=1024)  # in place with another stride
    refused(hl, K, call, q_out=A)  # over the positions
    refused(hl, K, call, q_out=B)
    refused(hl, K, call, k=E, k_out=D, n_kv_heads=2)  # over q's output
    refused(hl, K, call, k=E, k_out=C_, n_kv_heads=2)  # over q's input
    refused(hl, K, call, k=D + 4 * 128 * 3, k_out=E, n_kv_heads=2, q_out_stride=1024, k_stride=1024)  # one head shared in each row
    refused(hl, U, call, heads=70000)


def _cache(hl, pool=A, pages=10, layers=2, heads=2, dim=128, block=16):
    return hl.KvCache(pool, pages, layers, heads, dim, block)


def _batch(hl, tables=B, width=4, lens=B + 0x1000, starts=B + 0x2000, seqs=2, rows=3, **kw):
    return hl.KvBatch(tables, width, lens, starts, seqs, rows, **kw)


def _batched_calls(hl):
    return {
        "write": lambda c, l, b, **kw: hl.kv_write(kw.pop("t", F32), c, l, b, kw.pop("x", D), kw.pop("y", E), stream=0, **kw),
        "read": lambda c, l, b, **kw: hl.kv_read(c, l, b, kw.pop("x", D), kw.pop("y", E), stream=0, **kw),
        "attention": lambda c, l, b, **kw: hl.attention(kw.pop("t", F32), c, l, b, kw.pop("x", D), kw.pop("y", E), kw.pop("heads", 4),
                                                        stream=0, **kw),
    }


@pytest.mark.parametrize("name", ["write", "read", "attention"])
def test_batched_refusals(hl, name):
    K, U = hl.ErrorCode.Kernel, hl.ErrorCode.Unsupported
    f = _batched_calls(hl)[name]
    for bad in [dict(dim=80), dict(block=8), dict(layers=0), dict(heads=0)]:
        refused(hl, U, f, _cache(hl, **bad), 0, _batch(hl))
    refused(hl, K, f, _cache(hl, pages=0), 0, _batch(hl))
    refused(hl, K, f, _cache(hl, pool=0), 0, _batch(hl))
    refused(hl, K, f, _cache(hl, pool=A + 8), 0, _batch(hl))
    refused(hl, K, f, _cache(hl), 2, _batch(hl))
    refused(hl, K, f, _cache(hl), 0, _batch(hl, width=0))
    refused(hl, K, f, _cache(hl), 0, _batch(hl, width=1 << 28))
    refused(hl, K, f, _cache(hl), 0, _batch(hl, table_stride=3))
    refused(hl, K, f, _cache(hl), 0, _batch(hl, tables=0))
    refused(hl, K, f, _cache(hl), 0, _batch(hl, lens=B + 2))
    refused(hl, K, f, _cache(hl), 0, _batch(hl, starts=0))
    refused(hl, U, f, _cache(hl), 0, _batch(hl, seqs=70000))
    refused(hl, K, f, _cache(hl), 0, _batch(hl, rows=1 << 31))
    refused(hl, K, f, _cache(hl), 0, _batch(hl), x=D + 1)
    refused(hl, K, f, _cache(hl), 0, _batch(hl), status=F + 2)
    refused(hl, K, f, _cache(hl), 0, _batch(hl), status=A + 64)
    refused(hl, K, f, _cache(hl), 0, _batch(hl), y=A + 4096)  # over the pool
    if name != "read":
        refused(hl, U, f, _cache(hl), 0, _batch(hl), t=8)
        refused(hl, K, f, _cache(hl), 0, _batch(hl), x=0)
        refused(hl, K, f, _cache(hl), 0, _batch(hl), y=0)
    if name != "write":
        refused(hl, K, f, _cache(hl), 0, _batch(hl), y=B + 16)  # out over the tables
        refused(hl, K, f, _cache(hl), 0, _batch(hl), y=D + 64)  # out over q, or v over k
    if name == "attention":
        refused(hl, K, f, _cache(hl), 0, _batch(hl), heads=3)
        refused(hl, K, f, _cache(hl), 0, _batch(hl), heads=0)
        refused(hl, K, f, _cache(hl), 0, _batch(hl), scale=math.inf)
        refused(hl, K, f, _cache(hl), 0, _batch(hl), scale=math.nan)
        refused(hl, K, f, _cache(hl), 0, _batch(hl), workspace=F + 4, workspace_bytes=1 << 20)
        refused(hl, K, f, _cache(hl), 0, _batch(hl), workspace=E, workspace_bytes=1 << 20)
        refused(hl, K, f, _cache(hl), 0, _batch(hl), q_stride=511)
        refused(hl, K, f, _cache(hl), 0, _batch(hl), out_head_stride=64)
        assert hl.attention_workspace(F32, _cache(hl, heads=3), 0, _batch(hl), D, E, 4) == 0


def test_tensors_must_be_on_the_gpu(hl):
    import torch

    x = torch.zeros(4096)
    refused(hl, hl.ErrorCode.Kernel, hl.kv_read, _cache(hl, pool=x), 0, _batch(hl), D, E, stream=0)
    refused(hl, hl.ErrorCode.Kernel, hl.rope, F32, x, B, 8, 128, 128, C_, D, 4, stream=0)


def test_page_refusals(hl):
    K, U = hl.ErrorCode.Kernel, hl.ErrorCode.Unsupported
    st = lambda refs=B, lens=B + 0x1000, tables=B + 0x2000, slots=4, width=4, **kw: hl.KvState(refs, lens, tables, slots, width, **kw)  # noqa: E731
    resize = lambda c, s, x=D, y=E, n=3, **kw: hl.kv_resize(c, s, x, y, n, stream=0, **kw)  # noqa: E731
    fork = lambda c, s, x=D, y=E, n=3, **kw: hl.kv_fork(c, s, x, y, n, stream=0, **kw)  # noqa: E731
    compact = lambda c, s, **kw: hl.kv_compact(c, s, stream=0, **kw)  # noqa: E731
    for f in (resize, fork, compact):
        refused(hl, U, f, _cache(hl, dim=100), st())
        refused(hl, K, f, _cache(hl, pool=0), st())
        refused(hl, K, f, _cache(hl), st(refs=0))
        refused(hl, K, f, _cache(hl), st(lens=B + 0x1001))
        refused(hl, K, f, _cache(hl), st(tables=0))
        refused(hl, K, f, _cache(hl), st(slots=0))
        refused(hl, K, f, _cache(hl), st(width=0))
        refused(hl, K, f, _cache(hl), st(width=4, table_stride=3))
        refused(hl, K, f, _cache(hl), st(lens=B + 4))  # over refs
        refused(hl, K, f, _cache(hl), st(tables=A + 256))  # in the pool
    for f in (resize, fork):
        refused(hl, U, f, _cache(hl), st(), n=hl.KV_LIST_MAX + 1)
        refused(hl, U, f, _cache(hl, pages=1 << 23, layers=1, heads=1, dim=64), st(refs=1 << 44, lens=1 << 45, tables=1 << 46, width=1 << 23), n=1024)
        refused(hl, K, f, _cache(hl), st(), x=0)
        refused(hl, K, f, _cache(hl), st(), y=E + 2)
        refused(hl, K, f, _cache(hl), st(), x=B + 0x1004)
        for word in (B + 8, B + 0x1004, B + 0x2010, A + 4096, D + 4, E + 8, F + 2):  # on refs, lens, tables, the pool, a list
            refused(hl, K, f, _cache(hl), st(), status=word)
        refused(hl, K, f, _cache(hl), st(slots=1 << 30, table_stride=1 << 40))
    refused(hl, U, compact, _cache(hl, pages=1 << 24, layers=1, heads=1, dim=64), st(refs=1 << 44, lens=1 << 45, tables=1 << 46))
    for word in (B, B + 0x1004, B + 0x2010, A + 4096, F + 1):
        refused(hl, K, compact, _cache(hl), st(), live=word)
    copy = lambda c, x=D, y=E, n=3, **kw: hl.kv_copy_pages(c, x, y, n, stream=0, **kw)  # noqa: E731
    refused(hl, U, copy, _cache(hl, block=24))
    refused(hl, K, copy, _cache(hl), x=0)
    refused(hl, K, copy, _cache(hl), y=A)
    refused(hl, K, copy, _cache(hl), status=D + 8)


def test_null_params(hl):
    lib = hl.lib()
    for name in ("halo_mi_rope", "halo_mi_kv_write", "halo_mi_kv_read", "halo_mi_attention"):
        assert getattr(lib, name)(None, None) == hl.ErrorCode.Kernel
    assert lib.halo_mi_attention_workspace(None) == 0
    assert lib.halo_mi_kv_compact(None, None, None, None) == hl.ErrorCode.Kernel
    assert lib.halo_mi_kv_copy_pages(None, None, None, 0, None, 0, None) == hl.ErrorCode.Kernel
    assert lib.halo_mi_rope_freqs(64, ctypes.c_double(1e4), None, None, None) == hl.ErrorCode.Kernel


def test_kinds_of_numbers(hl):
    """Any integer kind serves; one that does not fit its member, or is none, is refused and not wrapped."""
    import numpy as np

    K = hl.ErrorCode.Kernel
    call = lambda n=0, dim=128, **kw: hl.rope(F32, A, B, n, dim, 64, C_, D, 4, stream=0, **kw)  # noqa: E731
    call(np.int64(0), np.uint8(128), q_stride=np.int32(512), factor=np.float64(1.5))
    for bad in (-1, 1 << 32, 1.5, "3", None):
        refused(hl, K, call, n=bad)
    refused(hl, K, call, q_stride=-512)
    refused(hl, K, call, q_stride=1 << 64)
    refused(hl, K, call, factor=1e39)
    empty = _batch(hl, seqs=np.int64(0), rows=np.int32(0))
    for name, f in _batched_calls(hl).items():
        f(_cache(hl, pages=np.int64(10)), np.int16(1), empty)
        refused(hl, K, f, _cache(hl, pages=-1), 0, empty)
        refused(hl, K, f, _cache(hl), -1, empty)
        refused(hl, K, f, _cache(hl), 0, _batch(hl, rows=-3))
        refused(hl, K, f, _cache(hl), 0, _batch(hl, table_stride=-1))
