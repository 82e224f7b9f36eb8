"""Tensors of another type than an operand of the paged cache's calls has are refused: int64 lists, as torch makes them by
default, would be read as pairs of int32. No GPU calls: a tensor of the right type is refused for where it is."""
import pytest
import torch

from kv_helpers import BF16, F16, F32, torch_type

A, B, C, D, E, F = (0x10000000 * i for i in range(1, 7))


def cache(hl, pool=A):
    return hl.KvCache(pool, 10, 2, 2, 128, 16)


def batch(hl, **kw):
    x = dict(tables=B, table_width=4, kv_lens=B + 0x1000, row_starts=B + 0x2000, n_seqs=2, n_rows=3)
    return hl.KvBatch(**{**x, **kw})


def state(hl, **kw):
    x = dict(refs=B, lens=B + 0x1000, tables=B + 0x2000, n_slots=4, table_width=4)
    return hl.KvState(**{**x, **kw})


INTS, WORDS = (torch.int32,), (torch.int32, torch.uint32)


def operands(hl):
    """(name, allowed types, a call with a tensor of a given type in its place) of every operand that has a type."""
    out = []

    def add(name, kinds, call):
        out.append((name, kinds, call))

    for t in (F32, F16, BF16):
        own = (torch_type(t),)
        for at in ("q", "q_out", "k", "k_out"):
            add(f"rope {at} {t}", own, lambda x, t=t, at=at: hl.rope(t, A, B, 8, 128, 128, stream=0, n_heads=4, n_kv_heads=2, **{
                **dict(q=C, q_out=C, k=D, k_out=D), at: x}))
        add(f"write k {t}", own, lambda x, t=t: hl.kv_write(t, cache(hl), 0, batch(hl), x, E, stream=0))
        add(f"write v {t}", own, lambda x, t=t: hl.kv_write(t, cache(hl), 0, batch(hl), D, x, stream=0))
        add(f"attention q {t}", own, lambda x, t=t: hl.attention(t, cache(hl), 0, batch(hl), x, E, 4, stream=0))
        add(f"attention out {t}", own, lambda x, t=t: hl.attention(t, cache(hl), 0, batch(hl), D, x, 4, stream=0))
    add("rope positions", INTS, lambda x: hl.rope(F32, x, B, 8, 128, 128, C, C, 4, stream=0))
    add("rope freqs", (torch.float64,), lambda x: hl.rope(F32, A, x, 8, 128, 128, C, C, 4, stream=0))
    add("read k", (torch.float32,), lambda x: hl.kv_read(cache(hl), 0, batch(hl), x, E, stream=0))
    add("read v", (torch.float32,), lambda x: hl.kv_read(cache(hl), 0, batch(hl), D, x, stream=0))
    calls = {"write": lambda b, **kw: hl.kv_write(F32, cache(hl), 0, b, D, E, stream=0, **kw),
             "read": lambda b, **kw: hl.kv_read(cache(hl), 0, b, D, E, stream=0, **kw),
             "attention": lambda b, **kw: hl.attention(F32, cache(hl), 0, b, D, E, 4, stream=0, **kw)}
    for name, f in calls.items():
        for at in ("tables", "kv_lens", "row_starts"):
            add(f"{name} {at}", INTS, lambda x, f=f, at=at: f(batch(hl, **{at: x})))
        add(f"{name} status", WORDS, lambda x, f=f: f(batch(hl), status=x))
    pages = {"resize": hl.kv_resize, "fork": hl.kv_fork}
    for name, f in pages.items():
        for at in ("refs", "lens", "tables"):
            add(f"{name} {at}", INTS, lambda x, f=f, at=at: f(cache(hl), state(hl, **{at: x}), D, E, 3, stream=0))
        add(f"{name} first list", INTS, lambda x, f=f: f(cache(hl), state(hl), x, E, 3, stream=0))
        add(f"{name} second list", INTS, lambda x, f=f: f(cache(hl), state(hl), D, x, 3, stream=0))
        add(f"{name} status", WORDS, lambda x, f=f: f(cache(hl), state(hl), D, E, 3, status=x, stream=0))
    for at in ("refs", "lens", "tables"):
        add(f"compact {at}", INTS, lambda x, at=at: hl.kv_compact(cache(hl), state(hl, **{at: x}), stream=0))
    add("compact live", WORDS, lambda x: hl.kv_compact(cache(hl), state(hl), live=x, stream=0))
    add("copy src", INTS, lambda x: hl.kv_copy_pages(cache(hl), x, E, 3, stream=0))
    add("copy dst", INTS, lambda x: hl.kv_copy_pages(cache(hl), D, x, 3, stream=0))
    add("copy status", WORDS, lambda x: hl.kv_copy_pages(cache(hl), D, E, 3, status=x, stream=0))
    return out


KINDS = (torch.int64, torch.int32, torch.uint32, torch.int16, torch.uint8, torch.float64, torch.float32, torch.float16, torch.bfloat16)


def test_types_of_tensors(hl):
    for name, kinds, call in operands(hl):
        for kind in KINDS:
            with pytest.raises(hl.HaloError) as e:
                call(torch.zeros(4096, dtype=kind))
            assert e.value.code == hl.ErrorCode.Kernel, name
            want = "not on the current GPU" if kind in kinds else f"an operand is {kind}, not "
            assert want in str(e.value), f"{name} as {kind}: {e.value}"


def test_a_pool_has_no_type(hl):
    for kind in KINDS:
        with pytest.raises(hl.HaloError, match="not on the current GPU"):
            hl.kv_read(cache(hl, torch.zeros(4096, dtype=kind)), 0, batch(hl), D, E, stream=0)
        with pytest.raises(hl.HaloError, match="not on the current GPU"):
            hl.attention(F32, cache(hl), 0, batch(hl), D, E, 4, workspace=torch.zeros(4096, dtype=kind), stream=0)
