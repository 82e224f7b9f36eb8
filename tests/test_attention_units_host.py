"""How attention over few rows deals its units to workgroups (halo_amd/csrc/k_attention.hip: wave_scan, find_run, the walk of
k_attention_few, k_attention_few_join), restated in Python integers of 32 bits: row starts that do not fall give every
unit once; starts that fall, whose sums pass 32 bits, keep every index in range. No GPU."""
import random

import pytest

MOST = 0x7FFFFFFF
MASK = 0xFFFFFFFF


def capped(a, b):
    return min((a + b) & MASK, MOST)


def wrapped(a, b):
    return (a + b) & MASK


class OutOfRange(Exception):
    pass


def scan(v, add):
    out, off = list(v), 1
    while off < len(v):
        out = [add(x, out[i - off]) if i >= off else x for i, x in enumerate(out)]
        off *= 2
    return out


def total_of(units, add):
    t = 0
    for s0 in range(0, len(units), 64):
        t = add(t, scan(units[s0:s0 + 64], add)[-1])
    return t


def find_run(units, workgroups, i, add):
    total = total_of(units, add)
    per = max(1, (total + workgroups - 1) // workgroups)
    first = min(i * per, total)
    last, before, seq = min(first + per, total), 0, 0
    for s0 in range(0, len(units), 64):
        sums = scan(units[s0:s0 + 64], add)
        hit = [k for k, x in enumerate(sums) if (before + x) & MASK > first]
        if hit:
            before += sums[hit[0] - 1] if hit[0] else 0
            return first, last, s0 + hit[0], before
        before = (before + sums[-1]) & MASK
    return first, last, seq, before


def segments(units, workgroups, i, add, limit=5000):
    """(sequence, first unit in it, units, whole) of workgroup i; at most `limit` of them."""
    u, last, seq, before = find_run(units, workgroups, i, add)
    out = []
    while u < last and len(out) < limit:
        while u >= (before + units[seq]) & MASK:
            before = (before + units[seq]) & MASK
            seq += 1
            if seq >= len(units):
                raise OutOfRange("past the last sequence")
        n = min(units[seq] - (u - before), last - u)
        if n <= 0:
            raise OutOfRange("no units")
        out.append((seq, u - before, n))
        u += n
    return out


def join_parts(units, workgroups, seq, add, check):
    """The workgroups whose parts the join of a sequence adds (one tile and head: a segment is a sequence)."""
    total, before = 0, 0
    for s0 in range(0, len(units), 64):
        sums = scan(units[s0:s0 + 64], add)
        if s0 <= seq < s0 + 64:
            before = add(total, sums[seq - s0 - 1] if seq > s0 else 0)
        total = add(total, sums[-1])
    per = max(1, (total + workgroups - 1) // workgroups)
    w0, w1 = before // per, ((before + units[seq] - 1) & MASK) // per
    if check and w1 >= workgroups:
        return []
    if w1 >= workgroups or w0 > w1:
        raise OutOfRange("past the workspace")
    return list(range(w0, w1 + 1))


@pytest.mark.parametrize("seed", range(20))
def test_every_unit_once(seed):
    rng = random.Random(seed)
    units = [rng.choice((0, 1, 2, rng.randint(0, 400))) for _ in range(rng.choice((1, 5, 63, 64, 65, 130, 200)))]
    workgroups = rng.choice((1, 7, 256, 768))
    seen = [[0] * n for n in units]
    who = [set() for _ in units]
    for i in range(workgroups):
        for seq, at, n in segments(units, workgroups, i, capped):
            who[seq].add(i)
            for k in range(at, at + n):
                seen[seq][k] += 1
    assert all(x == 1 for s in seen for x in s)
    for seq, n in enumerate(units):
        if n:
            assert set(join_parts(units, workgroups, seq, capped, True)) == who[seq]


# sequences' units as starts that fall give them: each is under 2^31 by the plan, together far past 2^32
FALLING = [
    [MOST, 0, MOST, 0, MOST, 0],
    [1 << 30, 0] * 40,
    [(1 << 31) - 5, 7, 1 << 20] * 50,
    [3, MOST - 1, 4, MOST - 7] * 20,
    [1 << 22] * 1500,
    [1 << 25, 3] * 70,
]


@pytest.mark.parametrize("units", FALLING, ids=range(len(FALLING)))
def test_sums_past_32_bits_stay_in_range(units):
    for workgroups in (1, 200, 768):
        for i in range(0, workgroups, max(1, workgroups // 20)):
            for seq, at, n in segments(units, workgroups, i, capped, 300):
                assert 0 <= seq < len(units) and 0 <= at and at + n <= units[seq]
        for seq, n in enumerate(units):
            if n:
                assert all(w < workgroups for w in join_parts(units, workgroups, seq, capped, True))


def test_wrapped_sums_leave_the_range():
    """What the cap is for: with sums that wrap, some index does not stay in range."""
    found = 0
    for units in FALLING:
        try:
            for i in range(768):
                segments(units, 768, i, wrapped, 300)
            for seq, n in enumerate(units):
                if n:
                    join_parts(units, 768, seq, wrapped, False)
        except OutOfRange:
            found += 1
    assert found > len(FALLING) // 2
