"""Operands that lie side by side in rows of one buffer are apart, and those that share an element are not. No GPU calls: the
batches have no sequences, so that a call with nothing against it returns before a launch."""
import pytest

from kv_helpers import BF16, F32
from test_kv_host import B, D, _cache, refused

ROW = 2 * 128  # elements of a token's heads in K or V


def batch(hl):
    return hl.KvBatch(B, 4, B + 0x1000, B + 0x2000, 0, 3)


def test_read_side_by_side(hl):
    read = lambda k, v, ks, vs, **kw: hl.kv_read(_cache(hl), 0, batch(hl), k, v, k_stride=ks, v_stride=vs, stream=0, **kw)  # noqa: E731
    read(D, D + 4 * ROW, 2 * ROW, 2 * ROW)
    read(D + 4 * ROW, D, 2 * ROW, 2 * ROW)
    read(D, D + 4 * (ROW + 7), 2 * ROW + 7, 2 * ROW + 7)
    for k, v, ks, vs in [(D, D + 4 * (ROW - 1), 2 * ROW, 2 * ROW), (D, D + 4 * (ROW + 1), 2 * ROW, 2 * ROW), (D, D, 2 * ROW, 2 * ROW),
                         (D, D + 4 * ROW, 2 * ROW, 3 * ROW), (D, D + 4 * ROW, 0, 0), (D, D + 4 * 128, 2 * ROW, 2 * ROW)]:
        refused(hl, hl.ErrorCode.Kernel, read, k, v, ks, vs)


@pytest.mark.parametrize("t,size", [(F32, 4), (BF16, 2)])
def test_attention_side_by_side(hl, t, size):
    q = 4 * 128
    call = lambda x, y, xs, ys: hl.attention(t, _cache(hl), 0, batch(hl), x, y, 4, q_stride=xs, out_stride=ys, stream=0)  # noqa: E731
    call(D, D + size * q, 2 * q, 2 * q)
    call(D + size * q, D, 2 * q, 2 * q)
    call(D + size * ROW, D + size * (ROW + q), 2 * q + ROW, 2 * q + ROW)
    for x, y, xs, ys in [(D, D + size * (q - 1), 2 * q, 2 * q), (D, D + size * q, 2 * q, 2 * q + 8), (D, D, 2 * q, 2 * q), (D, D + size * q, 0, 0)]:
        refused(hl, hl.ErrorCode.Kernel, call, x, y, xs, ys)
