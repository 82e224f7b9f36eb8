"""8-bit integer products, norms with rotation and linear attention on the host: the calls that are refused before anything is
enqueued, and those that have nothing to do. No GPU calls."""
import math

import pytest

from kv_helpers import BF16, F16, F32
from test_kv_host import refused

# Addresses that no call reaches: every call below is refused on the host or has nothing to do.
A, B, C, D, E, F, G, H, I, J = (0x10000000000 * i for i in range(1, 11))


def test_norm_rope_refusals(hl):
    K, U, Cf = hl.ErrorCode.Kernel, hl.ErrorCode.Unsupported, hl.ErrorCode.Config

    def call(t=F32, pos=A, freqs=B, n=8, dim=128, rot=128, q=C, q_out=D, heads=4, q_norm=E, **kw):
        hl.norm_rope(t, pos, freqs, n, dim, rot, q, q_out, heads, q_norm=q_norm, stream=0, **kw)

    refused(hl, U, call, t=12)
    refused(hl, Cf, call, pairs=2)
    refused(hl, K, call, rot=3)
    refused(hl, K, call, rot=130)
    refused(hl, U, call, dim=0, rot=0)
    refused(hl, K, call, q=0)
    refused(hl, K, call, q_out=0)
    refused(hl, K, call, pos=0)
    refused(hl, K, call, freqs=B + 4)
    refused(hl, K, call, q_norm=E + 2)
    refused(hl, K, call, q_out=C + 512)
    refused(hl, K, call, q_norm=D)  # an output over the weights
    refused(hl, K, call, q_norm=D + 4 * 8 * 4 * 128 - 4)
    refused(hl, K, call, k=F, k_out=G, n_kv_heads=2, k_norm=D + 64)  # q's output over k's weights
    refused(hl, K, call, k=F, k_out=G, n_kv_heads=2, k_norm=G)
    refused(hl, K, call, k=F, k_out=D, n_kv_heads=2)
    refused(hl, U, call, heads=70000)
    for eps in (math.nan, math.inf, -1e-6):
        refused(hl, K, call, eps=eps)
    refused(hl, K, call, n=-1)
    refused(hl, K, call, n=1 << 31)
    call(n=0)
    call(heads=0)


def test_quantize_rows_refusals(hl):
    K, U = hl.ErrorCode.Kernel, hl.ErrorCode.Unsupported

    def call(t=F32, x=A, codes=B, scales=C, rows=8, cols=100, **kw):
        hl.quantize_rows(t, x, codes, scales, rows, cols, stream=0, **kw)

    refused(hl, U, call, t=2)
    refused(hl, U, call, cols=0)
    refused(hl, U, call, cols=131072)
    refused(hl, K, call, rows=1 << 31)
    refused(hl, K, call, rows=-1)
    refused(hl, K, call, rows=1 << 32)
    refused(hl, K, call, x=0)
    refused(hl, K, call, codes=0)
    refused(hl, K, call, scales=0)
    refused(hl, K, call, x=A + 2)
    refused(hl, K, call, t=F16, x=A + 1)
    refused(hl, K, call, codes=B + 8)
    refused(hl, K, call, scales=C + 2)
    refused(hl, K, call, x_stride=99)
    refused(hl, K, call, x_stride=-100)
    refused(hl, K, call, codes_stride=100)
    refused(hl, K, call, codes_stride=96)
    refused(hl, K, call, codes_stride=(1 << 20) + 16)
    refused(hl, K, call, codes=A + 4 * 700)  # inside x
    refused(hl, K, call, scales=B + 7 * 112 + 108)  # inside the last row's padding
    refused(hl, K, call, scales=A)
    call(rows=0)


def test_gemm_i8_refusals(hl):
    K, U = hl.ErrorCode.Kernel, hl.ErrorCode.Unsupported

    def call(t=F32, w=A, ws=B, x=C, xs=D, y=E, rows=8, cols=100, n_vec=3, **kw):
        hl.gemm_i8(t, w, ws, x, xs, y, rows, cols, n_vec, stream=0, **kw)

    refused(hl, U, call, t=8)
    refused(hl, U, call, cols=0)
    refused(hl, U, call, cols=131072)
    refused(hl, K, call, rows=1 << 31)
    refused(hl, K, call, n_vec=1 << 31)
    refused(hl, K, call, n_vec=-1)
    for name in ("w", "ws", "x", "xs", "y"):
        refused(hl, K, call, **{name: 0})
    refused(hl, K, call, w=A + 8)
    refused(hl, K, call, x=C + 4)
    refused(hl, K, call, ws=B + 1)
    refused(hl, K, call, xs=D + 2)
    refused(hl, K, call, y=E + 2)
    refused(hl, K, call, t=BF16, y=E + 1)
    refused(hl, K, call, w_stride=100)
    refused(hl, K, call, w_stride=96)
    refused(hl, K, call, x_stride=120)
    refused(hl, K, call, x_stride=1 << 21)
    refused(hl, K, call, y_stride=7)
    refused(hl, K, call, y=A)
    refused(hl, K, call, y=C + 2 * 112 + 108)  # x's last padding
    refused(hl, K, call, y=B)
    refused(hl, K, call, y=D)
    call(rows=0)
    call(n_vec=0)


def test_linear_attention_refusals(hl):
    K, U = hl.ErrorCode.Kernel, hl.ErrorCode.Unsupported

    def call(t=F32, state=A, new=None, n_slots=3, heads=4, k_heads=2, kd=64, vd=128, slots=B, starts=B + 0x1000, lens=None, seqs=2, rows=5,
             q=C, k=D, v=E, out=F, decay=G, **kw):
        s = hl.LinearState(state, n_slots, heads, kd, vd, new)
        b = hl.LinearBatch(slots, starts, seqs, rows, 0, lens)
        hl.linear_attention(t, s, b, q, k, v, out, decay, k_heads, stream=0, **kw)

    refused(hl, U, call, t=9)
    refused(hl, U, call, kd=80)
    refused(hl, U, call, vd=512)
    refused(hl, U, call, seqs=65536)
    refused(hl, K, call, rows=1 << 31)
    refused(hl, K, call, heads=5)
    refused(hl, K, call, heads=0)
    refused(hl, K, call, k_heads=0)
    refused(hl, K, call, heads=5000, k_heads=5000)
    refused(hl, K, call, n_slots=0)
    refused(hl, K, call, n_slots=1 << 31)
    for name in ("state", "slots", "starts", "q", "k", "v", "out", "decay"):
        refused(hl, K, call, **{name: 0})
    for bad in ({"state": A + 8}, {"new": H + 8}, {"slots": B + 2}, {"starts": B + 2}, {"lens": B + 1}, {"decay": G + 2}, {"q": C + 2}):
        refused(hl, K, call, **bad)
    for scale in (math.nan, math.inf):
        refused(hl, K, call, scale=scale)
    refused(hl, K, call, decay_stride=3)
    refused(hl, K, call, decay_stride=4, decay_per_head=True)
    refused(hl, K, call, q_stride=100)
    refused(hl, K, call, v_head_stride=64)
    for name in ("q_stride", "k_stride", "v_stride"):  # a chunk's rows are addressed with 32 bits
        refused(hl, U, call, **{name: (1 << 24) + 1})
    slot = 4 * 4 * 64 * 128
    refused(hl, K, call, out=A + 3 * slot - 4)  # over the states
    refused(hl, K, call, out=C)
    refused(hl, K, call, out=D)
    refused(hl, K, call, out=E)
    refused(hl, K, call, out=G)
    refused(hl, K, call, out=B)
    refused(hl, K, call, new=A + slot)  # the new states over the old ones, not in place
    refused(hl, K, call, new=C)
    refused(hl, K, call, new=G - 3 * slot + 16)
    refused(hl, K, call, new=H, out=H + 3 * slot - 4)
    refused(hl, K, call, new=H, lens=H)
    refused(hl, K, call, workspace=I + 8, workspace_bytes=1 << 20)
    refused(hl, K, call, workspace=A, workspace_bytes=1 << 20)
    refused(hl, K, call, workspace=F, workspace_bytes=1 << 20)
    refused(hl, K, call, status=J + 2)
    refused(hl, K, call, status=F)
    refused(hl, K, call, status=A)
    call(rows=0)
    call(seqs=0)


def test_lists_of_another_type(hl):
    import torch

    s = hl.LinearState(A, 3, 4, 64, 64)
    for bad in (torch.zeros(2, dtype=torch.int64), torch.zeros(2)):
        with pytest.raises(hl.HaloError):
            hl.linear_attention(F32, s, hl.LinearBatch(bad, B, 2, 5), C, D, E, F, G, 2, stream=0)
    with pytest.raises(hl.HaloError):
        hl.gemm_i8(F32, torch.zeros(16, dtype=torch.uint8), B, C, D, E, 1, 16, 1, stream=0)
    with pytest.raises(hl.HaloError):
        hl.quantize_rows(F32, torch.zeros(16, dtype=torch.float64), B, C, 1, 16, stream=0)
