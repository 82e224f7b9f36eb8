"""The operators around an 8-bit paged cache, as cases that can be timed and compared.

Between a layer's q / k / v projections and its output projection a serving program rotates q and k by their positions,
writes k and v into the sequences' pages in 8 bits, and attends over them; between steps it gives sequences pages, forks
them and packs the pool. Each case is one such call. `run` computes it in plain torch operations, or, where `own` is
true, through halo_amd's public functions.

The pool is n_pages records of page_bytes bytes. A page holds block_tokens tokens of every layer: K codes
[layer][0][head][token][dim] and V codes [layer][1][head][dim][token] (int8), then their scales [layer][2][head] (fp32):
the value of a code c is c * scale. A sequence's table row lists its pages in order.
"""
import math

import torch

own = False

TYPES = {"F32": (torch.float32, 0), "F16": (torch.float16, 1), "BF16": (torch.bfloat16, 30)}
TINY = 2.0 ** -80  # a block whose largest value is below 127 times this is held as zeros
MOST = {"bytes": 4e8, "flops": 3.2e11}  # a drawn case's work at most


def listed():
    return [
        # one token of one sequence through the hybrid model's attention heads, a quarter of each head rotated: latency
        {"name": "rope_f32_half_1", "kind": "rope", "type": "F32", "pairs": "half", "scaling": "none", "tokens": 1, "heads": 24,
         "kv_heads": 4, "dim": 256, "rot": 64, "theta": 1e7, "factor": 1.0, "pos": 20000},
        # a long prompt's ragged end in a context stretched four times: adjacent pairs, the whole head
        {"name": "rope_bf16_inter_6133", "kind": "rope", "type": "BF16", "pairs": "interleaved", "scaling": "yarn", "tokens": 6133,
         "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "theta": 1e4, "factor": 4.0, "pos": 1000},
        # a serving step: each of 61 sequences writes its newest token, pages half full
        {"name": "write_f32_61x1", "kind": "write", "type": "F32", "seqs": 61, "rows_lo": 1, "rows_hi": 1, "kv_lo": 3, "kv_hi": 900,
         "kv_heads": 4, "dim": 256, "block": 16, "layers": 2},
        # prompts of several sequences in one batch
        {"name": "write_bf16_ragged", "kind": "write", "type": "BF16", "seqs": 7, "rows_lo": 201, "rows_hi": 2100, "kv_lo": 201,
         "kv_hi": 2600, "kv_heads": 8, "dim": 128, "block": 64, "layers": 2},
        # one user at a short context
        {"name": "attn_f32_1x777", "kind": "attn", "type": "F32", "seqs": 1, "rows_lo": 1, "rows_hi": 1, "kv_lo": 777, "kv_hi": 777,
         "heads": 24, "kv_heads": 4, "dim": 256, "block": 16, "layers": 2, "window": 0},
        # a full serving batch of ragged sequences
        {"name": "attn_bf16_48_ragged", "kind": "attn", "type": "BF16", "seqs": 48, "rows_lo": 1, "rows_hi": 1, "kv_lo": 61,
         "kv_hi": 8100, "heads": 32, "kv_heads": 8, "dim": 128, "block": 16, "layers": 2, "window": 0},
        # one user at a very long context
        {"name": "attn_f32_1x131000", "kind": "attn", "type": "F32", "seqs": 1, "rows_lo": 1, "rows_hi": 1, "kv_lo": 131000,
         "kv_hi": 131000, "heads": 24, "kv_heads": 4, "dim": 256, "block": 64, "layers": 1, "window": 0},
        # the verify step of speculative decoding, four tokens a sequence, over a sliding window
        {"name": "attn_f16_verify_window", "kind": "attn", "type": "F16", "seqs": 8, "rows_lo": 4, "rows_hi": 4, "kv_lo": 900,
         "kv_hi": 6000, "heads": 24, "kv_heads": 4, "dim": 256, "block": 32, "layers": 2, "window": 2048},
        # a prefill chunk of 256 rows far into a document
        {"name": "attn_f32_chunk256", "kind": "attn", "type": "F32", "seqs": 1, "rows_lo": 256, "rows_hi": 256, "kv_lo": 16300,
         "kv_hi": 16300, "heads": 24, "kv_heads": 4, "dim": 256, "block": 16, "layers": 2, "window": 0},
        # whole prompts, ragged: the largest work
        {"name": "attn_bf16_prompts", "kind": "attn", "type": "BF16", "seqs": 3, "rows_lo": 700, "rows_hi": 5000, "kv_lo": 700,
         "kv_hi": 5000, "heads": 32, "kv_heads": 8, "dim": 128, "block": 64, "layers": 1, "window": 0},
        # eight sequences branch eightfold, and every branch takes room for its next token
        {"name": "branch_8x8", "kind": "branch", "seqs": 8, "ways": 8, "kv_lo": 100, "kv_hi": 1500, "pages": 1300, "kv_heads": 4,
         "dim": 256, "block": 16, "layers": 8},
        # the pool after many sequences came and went: the live pages move to its front
        {"name": "compact_1500", "kind": "compact", "seqs": 40, "kv_lo": 20, "kv_hi": 700, "pages": 1500, "kv_heads": 4, "dim": 256,
         "block": 16, "layers": 8},
    ]


def log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    case = draw_any(rng)
    while any(work(case)[k] > MOST[k] for k in MOST):
        for name in ("tokens", "rows_lo", "rows_hi", "kv_lo", "kv_hi"):
            if name in case:
                case[name] = max(1, case[name] * 3 // 4)
    return case


def draw_any(rng):
    kind = rng.choice(("rope", "write", "write", "attn", "attn", "attn", "attn", "branch", "compact"))
    dim = rng.choice((64, 96, 128, 128, 192, 256))
    kv_heads = rng.choice((1, 2, 4, 8, 5))
    heads = kv_heads * rng.choice((1, 2, 4, 6, 7, 8))
    block = rng.choice((16, 16, 32, 64, 128))
    t = rng.choice(sorted(TYPES))
    if kind == "rope":
        return {"kind": kind, "type": t, "pairs": rng.choice(("half", "interleaved")), "scaling": rng.choice(("none", "linear", "ntk", "yarn")),
                "tokens": log_int(rng, 1, 6000), "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": dim // rng.choice((1, 1, 2, 4)) // 2 * 2,
                "theta": rng.choice((1e4, 5e5, 1e7)), "factor": rng.choice((1.0, 2.0, 4.0, 8.0)), "pos": log_int(rng, 1, 1 << 20)}
    if kind == "write":
        seqs = log_int(rng, 1, 64)
        lo = log_int(rng, 1, max(1, 6000 // seqs))
        hi = log_int(rng, lo, max(lo, 12000 // seqs))
        if rng.random() < 0.4:
            lo = hi = rng.choice((1, 1, 2, 5))
        return {"kind": kind, "type": t, "seqs": seqs, "rows_lo": lo, "rows_hi": hi, "kv_lo": lo, "kv_hi": hi + rng.randint(0, 600),
                "kv_heads": kv_heads, "dim": dim, "block": block, "layers": rng.randint(1, 3)}
    if kind == "attn":
        way = rng.choice(("step", "step", "verify", "chunk", "prompt"))
        window = rng.choice((0, 0, 0, log_int(rng, 16, 4096)))
        if way == "prompt":
            seqs = rng.randint(1, 4)
            lo = log_int(rng, 16, 1500)
            hi = kv_hi = log_int(rng, lo, 3600)
            kv_lo = lo
        else:
            seqs = 1 if way == "chunk" else log_int(rng, 1, 48)
            lo, hi = {"step": (1, 1), "verify": (rng.randint(2, 4), rng.randint(4, 8)), "chunk": (rng.randint(33, 300),) * 2}[way]
            kv_lo = hi + log_int(rng, 1, 4000)
            kv_hi = log_int(rng, kv_lo, max(kv_lo, min(120000, 160000 // seqs) if way == "step" else min(20000, 80000 // seqs)))
        return {"kind": kind, "type": t, "seqs": seqs, "rows_lo": lo, "rows_hi": hi, "kv_lo": kv_lo, "kv_hi": kv_hi, "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "block": block, "layers": rng.randint(1, 2), "window": window}
    kv_hi = rng.randint(30, 1000)
    seqs, kv_lo = rng.randint(2, 24), rng.randint(1, 30)
    case = {"kind": kind, "seqs": seqs, "kv_lo": kv_lo, "kv_hi": kv_hi, "kv_heads": rng.choice((1, 2, 4)), "dim": dim, "block": block,
            "layers": rng.randint(1, 8)}
    if kind == "branch":
        case["ways"] = rng.randint(1, 6)
    live = sum(-(-n // block) for n in lengths(seqs, kv_lo, kv_hi)) + 3 * seqs * case.get("ways", 0)
    case["pages"] = live + rng.randint(1, 200)
    return case


def lengths(n, lo, hi):
    """n lengths spread over [lo, hi], the last one hi."""
    return [lo + int((hi - lo) * ((i + 1) * 0.6180339887498949 % 1.0)) for i in range(n - 1)] + [hi]


def shapes(case):
    """Rows and cached tokens (these rows among them) of each sequence."""
    rows = lengths(case["seqs"], case["rows_lo"], case["rows_hi"])
    return rows, [max(r, n) for r, n in zip(rows, lengths(case["seqs"], case["kv_lo"], case["kv_hi"]))]


def page_bytes(case):
    units = 2 * case["layers"] * case["kv_heads"]
    return -(-(units * case["block"] * case["dim"] + 4 * units) // 128) * 128


def work(case):
    kind = case["kind"]
    if kind == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        size = TYPES[case["type"]][0].itemsize
        return {"bytes": 2 * n * case["dim"] * size + 4 * case["tokens"] + 4 * case["rot"], "flops": 3 * n * case["rot"]}
    block = case["block"]
    if kind in ("branch", "compact"):
        kv = lengths(case["seqs"], case["kv_lo"], case["kv_hi"])
        ints = 4 * (case["pages"] + sum(-(-n // block) for n in kv))
        if kind == "branch":
            part = sum(n % block > 0 for n in kv)
            return {"bytes": part * (1 + case["ways"]) * page_bytes(case) + ints, "flops": 0}
        live = sum(-(-n // block) for n in kv)
        return {"bytes": 2 * (live * (case["pages"] - live) // case["pages"]) * page_bytes(case) + ints, "flops": 0}
    rows, kv = shapes(case)
    size, unit = TYPES[case["type"]][0].itemsize, case["kv_heads"] * case["dim"]
    if kind == "write":
        back = sum(read_rows(case))
        return {"bytes": sum(rows) * unit * 2 * (size + 1) + back * unit * 2 * 5, "flops": sum(rows) * unit * 4}
    w = case["window"] or 1 << 40
    seen = sum(min(n, w + r - 1) for r, n in zip(rows, kv))
    pairs = sum(sum(min(n - r + i + 1, w) for i in range(r)) for r, n in zip(rows, kv))
    return {"bytes": 2 * sum(rows) * case["heads"] * case["dim"] * size + 2 * seen * unit + 8 * case["kv_heads"] * (seen // block),
            "flops": 4 * pairs * case["heads"] * case["dim"]}


def generator(seed, *more):
    k = seed
    for v in more:
        k = (k * 1000003 + v + 1) % (1 << 62)
    return torch.Generator(device="cuda").manual_seed(k)


def normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


# ---- the cache -----------------------------------------------------------------------------------------------------


def codes_of(case, pool):
    """The codes as [page, layer, 2, head, block * dim], a view of the pool."""
    lay, h, n = case["layers"], case["kv_heads"], case["block"] * case["dim"]
    return pool[:, :2 * lay * h * n].unflatten(1, (lay, 2, h, n))


def scales_of(case, pool):
    """The scales as [page, layer, 2, head], a view of the pool."""
    lay, h = case["layers"], case["kv_heads"]
    at = 2 * lay * h * case["block"] * case["dim"]
    return pool[:, at:at + 8 * lay * h].view(torch.float32).unflatten(1, (lay, 2, h))


def filled_pool(case, n_pages, seed):
    """Codes as a normal distribution leaves them, some channels of K larger; scales of a block's maximum near 3.5."""
    g = generator(seed, 1)
    lay, h, block, dim = case["layers"], case["kv_heads"], case["block"], case["dim"]
    pool = torch.zeros((n_pages, page_bytes(case)), dtype=torch.int8, device="cuda")
    loud = 1 + 2 * (torch.rand(dim, generator=g, device="cuda") < 0.04)
    c = codes_of(case, pool)
    for layer in range(lay):
        k = normal(g, n_pages, h, block, dim).mul_(34).mul_(loud)
        c[:, layer, 0] = k.round_().clamp_(-127, 127).to(torch.int8).flatten(2)
        c[:, layer, 1] = normal(g, n_pages, h, dim * block).mul_(34).round_().clamp_(-127, 127).to(torch.int8)
    scales_of(case, pool).copy_((0.2 * normal(g, n_pages, lay, 2, h)).exp_().mul_(3.5 / 127))
    return pool


def shuffled_tables(lens, block, n_pages, width, seed):
    """Pages of the sequences, in no order; entries past a sequence's end are -1."""
    ids = torch.randperm(n_pages, generator=generator(seed, 2), device="cuda").to(torch.int32).tolist()
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for i, n in enumerate(lens):
        k = -(-n // block)
        table[i, :k] = torch.tensor(ids[at:at + k], dtype=torch.int32)
        at += k
    return table.cuda()


def read_rows(case):
    """How many of each sequence's last tokens are read back: from the start of the first page that the rows touch."""
    rows, kv = shapes(case)
    return [n - (n - r) // case["block"] * case["block"] for r, n in zip(rows, kv)]


def starts(rows):
    return torch.tensor([0] + rows, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


def batch_of(case, rows, kv, width):
    return {"lens": torch.tensor(kv, dtype=torch.int32, device="cuda"), "starts": starts(rows), "seqs": case["seqs"], "rows": sum(rows),
            "max_rows": max(rows), "max_kv": max(kv), "width": width}


# ---- states --------------------------------------------------------------------------------------------------------


def rope_table(case):
    """Radians per position of each pair, in 64 bits, and the factor on the rotated values."""
    rot, theta, f = case["rot"], case["theta"], case["factor"]
    i = torch.arange(rot // 2, dtype=torch.float64)
    if case["scaling"] == "ntk" and rot > 2:
        theta = theta * f ** (rot / (rot - 2))
    base = theta ** (-2 * i / rot)
    if case["scaling"] == "linear":
        return base / f, 1.0
    if case["scaling"] != "yarn" or f <= 1:
        return base, 1.0
    at = lambda turns: rot * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return base / f * ramp + base * (1 - ramp), 0.1 * math.log(f) + 1


def prepare(case, seed):
    kind, g = case["kind"], generator(seed, 0)
    if kind == "rope":
        dt = TYPES[case["type"]][0]
        freqs, factor = rope_table(case)
        q, k = (normal(g, case["tokens"], n, case["dim"]).to(dt) for n in (case["heads"], case["kv_heads"]))
        first = int(torch.randint(0, case["pos"] + 1, (1,), generator=g, device="cuda"))
        return {"case": case, "q": q, "k": k, "pos": torch.arange(first, first + case["tokens"], dtype=torch.int32, device="cuda"),
                "freqs": freqs.cuda(), "factor": factor, "q_out": torch.empty_like(q), "k_out": torch.empty_like(k)}
    if kind in ("branch", "compact"):
        return prepare_pages(case, seed, g)
    rows, kv = shapes(case)
    need = sum(-(-n // case["block"]) for n in kv)
    width = max(-(-n // case["block"]) for n in kv) + 1
    pool = filled_pool(case, need + 5, seed)
    state = {"case": case, "pool": pool, "tables": shuffled_tables(kv, case["block"], need + 5, width, seed),
             "batch": batch_of(case, rows, kv, width), "layer": case["layers"] - 1}
    dt = TYPES[case["type"]][0]
    if kind == "attn":
        # a head's scores spread over about two, and differ from head to head
        sharp = 1 + torch.rand(case["heads"], 1, generator=g, device="cuda")
        state["q"] = (normal(g, sum(rows), case["heads"], case["dim"]) * sharp).to(dt)
        state["out"] = torch.empty_like(state["q"])
        return state
    back = read_rows(case)
    state["back"] = batch_of(case, back, kv, width)
    for name in ("k", "v"):
        loud = 1 + 2 * (torch.rand(case["dim"], generator=g, device="cuda") < 0.04)
        state[name] = (normal(g, sum(rows), case["kv_heads"], case["dim"]) * (loud if name == "k" else 1)).to(dt)
        state[name + "_out"] = torch.empty((sum(back), case["kv_heads"], case["dim"]), device="cuda")
    return state


def prepare_pages(case, seed, g):
    """The pool's bytes, and as it was before the call: reference counts, lengths and tables."""
    kv = lengths(case["seqs"], case["kv_lo"], case["kv_hi"])
    ways = case.get("ways", 0)
    slots, width = case["seqs"] * (1 + ways), max(-(-n // case["block"]) for n in kv) + 1
    pool = torch.randint(-128, 128, (case["pages"], page_bytes(case)), generator=g, device="cuda", dtype=torch.int8)
    tables = torch.full((slots, width), -1, dtype=torch.int32, device="cuda")
    tables[:case["seqs"]] = shuffled_tables(kv, case["block"], case["pages"], width, seed)
    lens = torch.tensor(kv + [0] * (slots - len(kv)), dtype=torch.int32, device="cuda")
    refs = torch.zeros(case["pages"], dtype=torch.int32, device="cuda")
    refs[tables[tables >= 0].long()] = 1
    before = torch.cat([refs, lens, tables.flatten()])
    state = {"case": case, "pool": pool, "before": before, "now": before.clone(), "slots": slots, "width": width}
    if ways:
        state["src"] = torch.arange(case["seqs"], dtype=torch.int32, device="cuda").repeat_interleave(ways)
        state["dst"] = torch.arange(case["seqs"], slots, dtype=torch.int32, device="cuda")
        state["grown"] = (lens[:case["seqs"]] + 1).repeat_interleave(ways)
    return state


def page_state(state):
    """Reference counts, lengths and tables, set back to what they were before the call: views of state["now"]."""
    n, slots, width = state["case"]["pages"], state["slots"], state["width"]
    now = state["now"].copy_(state["before"])
    return now[:n], now[n:n + slots], now[n + slots:].view(slots, width)


# ---- the operators in plain torch ------------------------------------------------------------------------------------


def rotate(x, cos, sin, rot, pairs):
    y, x32 = x.clone(), x.float()
    if pairs == "half":
        a, b = x32[..., :rot // 2], x32[..., rot // 2:rot]
        y[..., :rot] = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)
    else:
        a, b = x32[..., 0:rot:2], x32[..., 1:rot:2]
        y[..., :rot] = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2).to(x.dtype)
    return y


def plain_rope(s):
    case = s["case"]
    angle = s["pos"].double()[:, None, None] * s["freqs"]
    cos, sin = (angle.cos() * s["factor"]).float(), (angle.sin() * s["factor"]).float()
    return [rotate(x, cos, sin, case["rot"], case["pairs"]) for x in (s["q"], s["k"])]


def row_places(b):
    """Sequence and position of each row of a batch: its rows are a sequence's last tokens."""
    r = torch.arange(b["rows"], device="cuda")
    seq = torch.searchsorted(b["starts"][1:].long(), r, right=True)
    return seq, b["lens"][seq].long() - b["starts"][seq + 1].long() + r


def plain_write(s):
    case, layer, block, dim = s["case"], s["layer"], s["case"]["block"], s["case"]["dim"]
    codes, scales = codes_of(case, s["pool"])[:, layer], scales_of(case, s["pool"])[:, layer]
    seq, pos = row_places(s["batch"])
    page, off = s["tables"][seq, pos // block].long(), pos % block
    pages, at = torch.unique(page, return_inverse=True)
    x = torch.stack([s["k"], s["v"]], 1).float()  # [row, 2, head, dim]
    top = x.abs().amax(-1)
    amax = torch.zeros((len(pages),) + top.shape[1:], device="cuda").scatter_reduce_(0, at[:, None, None].expand_as(top), top, "amax")
    first = torch.full((len(pages),), block, device="cuda").scatter_reduce_(0, at, off, "amin")
    old = torch.where(first[:, None, None] > 0, scales[pages], 0.0)
    fit = (amax.double() / 127).float()
    new = torch.maximum(old, torch.where(fit < TINY, 0.0, fit))
    # the tokens that the page holds already: their codes in the new scale, K [head, token, dim] and V [head, dim, token]
    held = codes[pages].double() * old.double()[..., None]
    held = torch.where(new[..., None] > 0, (held / new.double()[..., None]).round(), 0.0).clamp(-127, 127)
    k, v = held[:, 0].unflatten(-1, (block, dim)), held[:, 1].unflatten(-1, (dim, block))
    c = torch.where(new[at][..., None] > 0, x.double() / new[at].double()[..., None], 0.0).round().clamp(-127, 127)
    k[at, :, off], v[at, :, :, off] = c[:, 0], c[:, 1]
    codes[pages] = torch.stack([k.flatten(2), v.flatten(2)], 1).to(torch.int8)
    scales[pages] = new
    return plain_read(s, s["back"])


def plain_read(s, b):
    case, layer, block, dim = s["case"], s["layer"], s["case"]["block"], s["case"]["dim"]
    codes, scales = codes_of(case, s["pool"])[:, layer], scales_of(case, s["pool"])[:, layer]
    seq, pos = row_places(b)
    page, off = s["tables"][seq, pos // block].long(), pos % block
    k = codes[:, 0].unflatten(-1, (block, dim))[page, :, off].float() * scales[page, 0][..., None]
    v = codes[:, 1].unflatten(-1, (dim, block))[page, :, :, off].float() * scales[page, 1][..., None]
    return [k, v]


def plain_attention(s):
    case, b, layer, block, dim = s["case"], s["batch"], s["layer"], s["case"]["block"], s["case"]["dim"]
    h, group, n, top = case["kv_heads"], case["heads"] // case["kv_heads"], b["seqs"], b["max_rows"]
    codes, scales = codes_of(case, s["pool"])[:, layer], scales_of(case, s["pool"])[:, layer]
    pages = s["tables"][:, :b["width"] - 1].long().clamp(min=0)  # [seq, page]
    k, v = (codes[pages, j].float() * scales[pages, j][..., None] for j in (0, 1))
    k = k.unflatten(-1, (block, dim)).transpose(1, 2).flatten(2, 3)  # [seq, head, token, dim]
    v = v.unflatten(-1, (dim, block)).permute(0, 2, 1, 4, 3).flatten(2, 3)
    seq, pos = row_places(b)
    row = pos - (b["lens"][seq].long() - (b["starts"][seq + 1] - b["starts"][seq]).long())
    q = torch.zeros((n, top, case["heads"], dim), device="cuda")
    q[seq, row] = s["q"].float()
    q = q.view(n, top, h, group, dim).permute(0, 2, 1, 3, 4).reshape(n, h, top * group, dim)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(dim ** -0.5).view(n, h, top, group, -1)
    count = (b["starts"][1:] - b["starts"][:-1]).long()
    last = (b["lens"].long() - count)[:, None] + torch.arange(top, device="cuda")
    token = torch.arange(score.shape[-1], device="cuda")
    hidden = (token > last[..., None]) | (token >= b["lens"][:, None, None])
    if case["window"]:
        hidden |= token <= last[..., None] - case["window"]
    score.masked_fill_(hidden[:, None, :, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = score.sum(-1)
    out = torch.matmul(score.view(n, h, top * group, -1), v).view(n, h, top, group, dim) / total.clamp(min=1e-30)[..., None]
    return out.permute(0, 2, 1, 3, 4).reshape(n, top, case["heads"], dim)[seq, row].to(s["q"].dtype)


def plain_branch(s):
    refs, lens, tables = page_state(s)
    pool, block, src, dst = s["pool"], s["case"]["block"], s["src"].long(), s["dst"].long()
    column = torch.arange(s["width"], device="cuda")
    # fork: whole pages are shared, a page that is not full is copied into a free one, lowest first
    full, part = (lens[src] // block).long(), lens[src] % block > 0
    free = torch.nonzero(refs == 0).flatten()
    fresh = free[part.long().cumsum(0) - 1]
    row = tables[src].long()
    old = row.gather(1, full[:, None]).flatten()
    new = torch.where(column < full[:, None], row, torch.where((column == full[:, None]) & part[:, None], fresh[:, None], -1))
    pool[fresh[part]] = pool[old[part]]
    tables[dst] = new.int()
    lens[dst] = lens[src]
    held = new[new >= 0]
    refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    # room for one more token each
    have, want = -(-lens[dst] // block), -(-s["grown"] // block)
    takes = (column >= have[:, None]) & (column < want[:, None])
    free = torch.nonzero(refs == 0).flatten()[:int(takes.sum())]
    new = tables[dst]
    new[takes] = free.int()
    tables[dst] = new
    refs[free] = 1
    lens[dst] = s["grown"]
    return [pool, refs, lens, tables]


def plain_compact(s):
    refs, lens, tables = page_state(s)
    live = refs > 0
    n = int(live.sum())
    place = torch.arange(len(refs), device="cuda")
    src, dst = place[live & (place >= n)], place[~live & (place < n)]
    s["pool"][dst] = s["pool"][src]
    where = place.clone()
    where[src] = dst
    used = torch.arange(s["width"], device="cuda") < -(-lens // s["case"]["block"])[:, None]
    tables.copy_(torch.where(used, where[tables.clamp(min=0).long()].int(), tables))
    refs[dst] = refs[src]
    refs[src] = 0
    return [s["pool"][:n], refs, lens, tables]


PLAIN = {"rope": plain_rope, "write": plain_write, "attn": plain_attention, "branch": plain_branch, "compact": plain_compact}


# ---- the same through halo_amd -----------------------------------------------------------------------------------------


def cache_of(hl, s):
    case = s["case"]
    return hl.KvCache(s["pool"], len(s["pool"]), case["layers"], case["kv_heads"], case["dim"], case["block"])


def batch_call(hl, s, b):
    return hl.KvBatch(s["tables"], b["width"], b["lens"], b["starts"], b["seqs"], b["rows"], b["max_rows"], b["max_kv"])


def own_rope(hl, s):
    case = s["case"]
    pairs = hl.RopePairs.HALF if case["pairs"] == "half" else hl.RopePairs.INTERLEAVED
    hl.rope(TYPES[case["type"]][1], s["pos"], s["freqs"], case["tokens"], case["dim"], case["rot"], s["q"], s["q_out"], case["heads"],
            k=s["k"], k_out=s["k_out"], n_kv_heads=case["kv_heads"], pairs=pairs, factor=s["factor"])
    return [s["q_out"], s["k_out"]]


def own_write(hl, s):
    cache = cache_of(hl, s)
    hl.kv_write(TYPES[s["case"]["type"]][1], cache, s["layer"], batch_call(hl, s, s["batch"]), s["k"], s["v"])
    hl.kv_read(cache, s["layer"], batch_call(hl, s, s["back"]), s["k_out"], s["v_out"])
    return [s["k_out"], s["v_out"]]


def own_attention(hl, s):
    case = s["case"]
    hl.attention(TYPES[case["type"]][1], cache_of(hl, s), s["layer"], batch_call(hl, s, s["batch"]), s["q"], s["out"], case["heads"],
                 window=case["window"])
    return s["out"]


def own_branch(hl, s):
    refs, lens, tables = page_state(s)
    cache, state = cache_of(hl, s), hl.KvState(refs, lens, tables, s["slots"], s["width"])
    hl.kv_fork(cache, state, s["src"], s["dst"], len(s["src"]))
    hl.kv_resize(cache, state, s["dst"], s["grown"], len(s["dst"]))
    return [s["pool"], refs, lens, tables]


def own_compact(hl, s):
    refs, lens, tables = page_state(s)
    hl.kv_compact(cache_of(hl, s), hl.KvState(refs, lens, tables, s["slots"], s["width"]))
    n = sum(-(-n // s["case"]["block"]) for n in lengths(s["case"]["seqs"], s["case"]["kv_lo"], s["case"]["kv_hi"]))
    return [s["pool"][:n], refs, lens, tables]


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return PLAIN[kind](state)
    import halo_amd as hl

    return {"rope": own_rope, "write": own_write, "attn": own_attention, "branch": own_branch, "compact": own_compact}[kind](hl, state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------


def exact(case, seed):
    kind = case["kind"]
    if kind in ("branch", "compact"):
        return None
    s = prepare(case, seed)
    if kind == "rope":
        return exact_rope(s)
    rows, kv = shapes(case)
    return exact_write(s, rows, kv) if kind == "write" else exact_attention(s, rows, kv)


def exact_rope(s):
    case, out = s["case"], []
    turn = torch.polar(torch.full_like(s["freqs"], s["factor"])[None].expand(case["tokens"], -1), s["pos"].double()[:, None] * s["freqs"])
    half, rot = case["rot"] // 2, case["rot"]
    pick = torch.arange(rot, device="cuda").view(2, half) if case["pairs"] == "half" else torch.arange(rot, device="cuda").view(half, 2).t()
    for x in (s["q"], s["k"]):
        y = x.double()
        z = torch.complex(y[..., pick[0]], y[..., pick[1]]) * turn[:, None]
        y[..., pick[0]], y[..., pick[1]] = z.real, z.imag
        out.append(y)
    return out


def sequence(s, i, n, j):
    """K (j = 0) or V (j = 1) codes [head, token, dim] of sequence i's first n tokens, and each token's scale [head, token]."""
    case, block, dim = s["case"], s["case"]["block"], s["case"]["dim"]
    pages = s["tables"][i, :-(-n // block)].long()
    c = codes_of(case, s["pool"])[pages, s["layer"], j]
    c = c.unflatten(-1, (block, dim)) if j == 0 else c.unflatten(-1, (dim, block)).transpose(2, 3)
    sc = scales_of(case, s["pool"])[pages, s["layer"], j].double()
    return c.transpose(0, 1).flatten(1, 2)[:, :n].double(), sc.t().repeat_interleave(block, 1)[:, :n]


def exact_write(s, rows, kv):
    case, block, outs = s["case"], s["case"]["block"], ([], [])
    at = 0
    for i, (r, n) in enumerate(zip(rows, kv)):
        begin = (n - r) // block * block
        for j, name in enumerate(("k", "v")):
            fresh = s[name][at:at + r].double().transpose(0, 1)  # [head, row, dim]
            for lo in range(begin, n, block):
                a, b = max(lo, n - r), min(lo + block, n)
                x = fresh[:, a - (n - r):b - (n - r)]
                want = (x.abs().amax((1, 2)) / 127).float().double()
                want[want < TINY] = 0
                if a > lo:
                    c, sc = sequence(s, i, a, j)
                    want = torch.maximum(want, sc[:, lo])
                    x = torch.cat([c[:, lo:a] * sc[:, lo:a, None], x], 1)
                w = want[:, None, None]
                outs[j].append(torch.where(w > 0, (x / w).round().clamp(-127, 127) * w, 0.0).transpose(0, 1))
        at += r
    return [torch.cat(o) for o in outs]


def exact_attention(s, rows, kv):
    case, out, at = s["case"], [], 0
    group = case["heads"] // case["kv_heads"]
    for i, (r, n) in enumerate(zip(rows, kv)):
        (k, ks), (v, vs) = sequence(s, i, n, 0), sequence(s, i, n, 1)
        k, v = k * ks[..., None], v * vs[..., None]
        pos = torch.arange(n - r, n, device="cuda")[:, None]
        token = torch.arange(n, device="cuda")
        shown = (token <= pos) & ((token > pos - case["window"]) if case["window"] else True)
        o = torch.empty((r, case["heads"], case["dim"]), dtype=torch.float64, device="cuda")
        for head in range(case["heads"]):
            score = s["q"][at:at + r, head].double() @ k[head // group].t() / math.sqrt(case["dim"])
            p = torch.softmax(score.masked_fill_(~shown, -math.inf), -1)
            o[:, head] = p @ v[head // group]
        out.append(o)
        at += r
    return torch.cat(out)
