"""The operators of a decoder layer with 8-bit integer projections and linear attention, as cases that can be timed and compared.

Three kinds of call: a projection over 8-bit integers (each row of x is quantized with a scale of its own, then multiplied with
weights that have a scale for each output channel), the norms of q's and k's heads with the position rotation in the same
pass, and linear attention with a decay for each head, whose sequences keep a state from call to call. Each case is one
such call, or for a projection the two calls that it takes. `run` computes it in plain torch operations, or, where `own`
is true, through halo_amd's public functions.

Rows of 8-bit codes begin on 16 bytes: a row of `cols` codes is followed by zeros up to the next multiple of 16.
"""
import math

import torch

own = False

TYPES = {"F32": (torch.float32, 0), "F16": (torch.float16, 1), "BF16": (torch.bfloat16, 30)}
TINY = 2.0 ** -80  # a row whose largest value is below 127 times this is held as zeros
MOST = {"bytes": 6e8, "flops": 7.1e11}  # a drawn case's work at most


def listed():
    return [
        # one token through the hybrid model's attention heads, a quarter of each head rotated: latency
        {"name": "norm_rope_f32_1", "kind": "norm_rope", "type": "F32", "pairs": "half", "tokens": 1, "heads": 24, "kv_heads": 4, "dim": 256,
         "rot": 64, "theta": 1e7, "pos": 20000},
        # a long prompt's ragged end, whole heads in adjacent pairs
        {"name": "norm_rope_bf16_6133", "kind": "norm_rope", "type": "BF16", "pairs": "interleaved", "tokens": 6133, "heads": 32, "kv_heads": 8,
         "dim": 128, "rot": 128, "theta": 1e4, "pos": 1000},
        # one token of one user through a feed-forward block's first projection
        {"name": "i8_bf16_1", "kind": "i8", "type": "BF16", "out": "BF16", "n_vec": 1, "rows": 17408, "cols": 5120},
        # the verify step of speculative decoding through its second one
        {"name": "i8_f32_5", "kind": "i8", "type": "F32", "out": "F32", "n_vec": 5, "rows": 5120, "cols": 17408},
        # a serving step of 61 sequences through q's projection
        {"name": "i8_bf16_61", "kind": "i8", "type": "BF16", "out": "BF16", "n_vec": 61, "rows": 6144, "cols": 5120},
        # a prefill chunk
        {"name": "i8_f16_509", "kind": "i8", "type": "F16", "out": "F16", "n_vec": 509, "rows": 17408, "cols": 5120},
        # a whole batch of prompts: the largest work
        {"name": "i8_bf16_3990", "kind": "i8", "type": "BF16", "out": "BF16", "n_vec": 3990, "rows": 17408, "cols": 5120},
        # one token of one sequence through the hybrid model's linear heads: latency
        {"name": "linear_f32_1", "kind": "linear", "type": "F32", "seqs": 1, "rows_lo": 1, "rows_hi": 1, "fresh": 0, "heads": 48, "k_heads": 16,
         "k_dim": 128, "v_dim": 128, "decay": "tokens"},
        # a full serving batch's step
        {"name": "linear_bf16_61x1", "kind": "linear", "type": "BF16", "seqs": 61, "rows_lo": 1, "rows_hi": 1, "fresh": 0, "heads": 48,
         "k_heads": 16, "k_dim": 128, "v_dim": 128, "decay": "tokens"},
        # a verify step, four tokens a sequence, decays fixed for each head
        {"name": "linear_f16_verify", "kind": "linear", "type": "F16", "seqs": 8, "rows_lo": 4, "rows_hi": 4, "fresh": 0, "heads": 32,
         "k_heads": 32, "k_dim": 128, "v_dim": 128, "decay": "heads"},
        # a prefill chunk of 256 rows far into a document
        {"name": "linear_f32_chunk256", "kind": "linear", "type": "F32", "seqs": 1, "rows_lo": 256, "rows_hi": 256, "fresh": 0, "heads": 48,
         "k_heads": 16, "k_dim": 128, "v_dim": 128, "decay": "tokens"},
        # whole prompts, ragged, their states still empty
        {"name": "linear_bf16_prompts", "kind": "linear", "type": "BF16", "seqs": 4, "rows_lo": 601, "rows_hi": 5000, "fresh": 1, "heads": 48,
         "k_heads": 16, "k_dim": 128, "v_dim": 128, "decay": "tokens"},
    ]


def log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    case = draw_any(rng)
    while any(work(case)[k] > MOST[k] for k in MOST):
        for name in ("tokens", "n_vec", "rows", "rows_lo", "rows_hi"):
            if name in case:
                case[name] = max(1, case[name] * 3 // 4)
        if case["kind"] == "linear" and case["rows_hi"] == 1:
            case["seqs"] = max(1, case["seqs"] * 3 // 4)
    return case


def draw_any(rng):
    kind = rng.choice(("norm_rope", "i8", "i8", "i8", "linear", "linear", "linear"))
    t = rng.choice(sorted(TYPES))
    if kind == "norm_rope":
        dim, kv_heads = rng.choice((64, 80, 96, 128, 128, 192, 256)), rng.choice((1, 2, 4, 8, 5))
        return {"kind": kind, "type": t, "pairs": rng.choice(("half", "interleaved")), "tokens": log_int(rng, 1, 6000),
                "heads": kv_heads * rng.choice((1, 2, 4, 6, 7, 8)), "kv_heads": kv_heads, "dim": dim, "rot": dim // rng.choice((1, 1, 2, 4)) // 2 * 2,
                "theta": rng.choice((1e4, 5e5, 1e7)), "pos": log_int(rng, 1, 1 << 20)}
    if kind == "i8":
        return {"kind": kind, "type": t, "out": rng.choice(sorted(TYPES)), "n_vec": log_int(rng, 1, 4000), "rows": log_int(rng, 60, 24000),
                "cols": log_int(rng, 60, 24000)}
    way = rng.choice(("step", "verify", "chunk", "prompt", "prompt"))
    k_heads = rng.choice((1, 4, 8, 16, 5))
    seqs = {"step": log_int(rng, 1, 64), "verify": log_int(rng, 1, 32), "chunk": 1, "prompt": rng.randint(1, 5)}[way]
    lo, hi = {"step": (1, 1), "verify": (rng.randint(1, 4), rng.randint(4, 9)), "chunk": (rng.randint(20, 600),) * 2,
              "prompt": (log_int(rng, 16, 1500), 0)}[way]
    hi = hi or log_int(rng, lo, max(lo, 16000 // seqs))
    return {"kind": kind, "type": t, "seqs": seqs, "rows_lo": lo, "rows_hi": hi, "fresh": int(way == "prompt" and rng.random() < 0.6),
            "heads": k_heads * rng.choice((1, 2, 3, 4)), "k_heads": k_heads, "k_dim": rng.choice((64, 96, 128, 128, 192, 256)),
            "v_dim": rng.choice((64, 96, 128, 128, 192, 256)), "decay": rng.choice(("tokens", "tokens", "heads"))}


def lengths(n, lo, hi):
    """n lengths spread over [lo, hi], the last one hi."""
    return [lo + int((hi - lo) * ((i + 1) * 0.6180339887498949 % 1.0)) for i in range(n - 1)] + [hi]


def padded(cols):
    return -(-cols // 16) * 16


def work(case):
    kind, size = case["kind"], TYPES[case["type"]][0].itemsize
    if kind == "norm_rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["dim"] * size + 4 * case["tokens"] + 4 * case["rot"] + 8 * case["dim"], "flops": n * (4 * case["dim"] + 3 * case["rot"])}
    if kind == "i8":
        m, n, k = case["n_vec"], case["rows"], case["cols"]
        return {"bytes": m * k * size + n * k + 4 * n + m * n * TYPES[case["out"]][0].itemsize, "flops": 2 * m * n * k}
    rows, h, dk, dv = lengths(case["seqs"], case["rows_lo"], case["rows_hi"]), case["heads"], case["k_dim"], case["v_dim"]
    total = sum(rows)
    states = case["seqs"] * h * dk * dv * 4 * (1 if case["fresh"] else 2)
    decays = 4 * h * (total if case["decay"] == "tokens" else 1)
    # a token and head: its own product with the state and its own outer product
    return {"bytes": total * size * (2 * case["k_heads"] * dk + 2 * h * dv) + decays + states, "flops": 4 * total * h * dk * dv}


def generator(seed, *more):
    k = seed
    for v in more:
        k = (k * 1000003 + v + 1) % (1 << 62)
    return torch.Generator(device="cuda").manual_seed(k)


def normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def uniform(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


# ---- states --------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    return {"norm_rope": prepare_norm_rope, "i8": prepare_i8, "linear": prepare_linear}[case["kind"]](case, generator(seed, 0))


def prepare_norm_rope(case, g):
    """q and k as projections leave them, some dims larger; weights of the norms near 1."""
    dt, dim, rot = TYPES[case["type"]][0], case["dim"], case["rot"]
    q, k = ((normal(g, case["tokens"], n, dim) * (1 + 3 * (uniform(g, dim) < 0.04))).to(dt) for n in (case["heads"], case["kv_heads"]))
    first = int(torch.randint(0, case["pos"] + 1, (1,), generator=g, device="cuda"))
    freqs = case["theta"] ** (-2 * torch.arange(rot // 2, dtype=torch.float64) / rot)
    return {"case": case, "q": q, "k": k, "q_norm": 1 + 0.2 * normal(g, dim), "k_norm": 1 + 0.2 * normal(g, dim), "eps": 1e-6,
            "pos": torch.arange(first, first + case["tokens"], dtype=torch.int32, device="cuda"), "freqs": freqs.cuda(),
            "q_out": torch.empty_like(q), "k_out": torch.empty_like(k)}


def prepare_i8(case, g):
    """x with a few loud channels, as a norm leaves it; weights quantized by their rows when the model was loaded."""
    m, n, k = case["n_vec"], case["rows"], case["cols"]
    x = (normal(g, m, k) * (1 + 9 * (uniform(g, k) < 0.01))).to(TYPES[case["type"]][0])
    w = torch.zeros((n, padded(k)), dtype=torch.int8, device="cuda")
    w_scales = torch.empty(n, device="cuda")
    for a in range(0, n, 4096):
        part = normal(g, min(4096, n - a), k).mul_(0.02)
        w_scales[a:a + 4096] = part.abs().amax(1) / 127
        w[a:a + 4096, :k] = part.div_(w_scales[a:a + 4096, None]).round_().clamp_(-127, 127).to(torch.int8)
    # the program's own buffers between the two calls
    return {"case": case, "x": x, "w": w, "w_scales": w_scales, "codes": torch.empty((m, padded(k)), dtype=torch.int8, device="cuda"),
            "scales": torch.empty(m, device="cuda"), "y": torch.empty((m, n), dtype=TYPES[case["out"]][0], device="cuda")}


def prepare_linear(case, g):
    """Keys of length about 1, decays that differ from head to head, from hardly any to a forgetful one; states in shuffled slots."""
    dt, h, hk, dk, dv = TYPES[case["type"]][0], case["heads"], case["k_heads"], case["k_dim"], case["v_dim"]
    rows = lengths(case["seqs"], case["rows_lo"], case["rows_hi"])
    total, slots = sum(rows), case["seqs"] + 2
    rate = torch.exp(math.log(1e-3) * uniform(g, h))
    if case["decay"] == "tokens":
        decay = -rate * torch.nn.functional.softplus(normal(g, total, h))
    else:
        decay = -rate
    held = rows if case["fresh"] else [n + 100 for n in rows]
    states = normal(g, slots, h, dk, dv)
    return {"case": case, "q": normal(g, total, hk, dk).to(dt), "k": (normal(g, total, hk, dk) * dk ** -0.5).to(dt), "v": normal(g, total, h, dv).to(dt),
            "decay": decay, "out": torch.empty((total, h, dv), dtype=dt, device="cuda"), "states": states, "new_states": states.clone(),
            "slots": torch.randperm(slots, generator=g, device="cuda")[:case["seqs"]].to(torch.int32), "rows": rows,
            "starts": torch.tensor([0] + rows, dtype=torch.int32).cumsum(0).to(torch.int32).cuda(),
            "lens": torch.tensor(held, dtype=torch.int32, device="cuda")}


# ---- the operators in plain torch ------------------------------------------------------------------------------------


def plain_norm_rope(s):
    case, rot, outs = s["case"], s["case"]["rot"], []
    angle = s["pos"].double()[:, None, None] * s["freqs"]
    cos, sin = angle.cos().float(), angle.sin().float()
    for x, w in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
        y = x.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + s["eps"]) * w
        if case["pairs"] == "half":
            a, b = y[..., :rot // 2], y[..., rot // 2:rot]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = y[..., 0:rot:2], y[..., 1:rot:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        outs.append(torch.cat([turned, y[..., rot:]], -1).to(x.dtype))
    return outs


def plain_i8(s):
    x, k = s["x"].double(), s["case"]["cols"]
    scale = (x.abs().amax(1) / 127).float()
    scale = torch.where(scale < TINY, 0.0, scale)
    codes = torch.where(scale[:, None] > 0, x / scale[:, None].double(), 0.0).round().clamp(-127, 127).float()
    total = torch.zeros((len(x), len(s["w"])), dtype=torch.int32, device="cuda")
    for a in range(0, k, 1024):  # sums of 1024 products are exact in 32-bit floats
        b = min(a + 1024, k)
        total += torch.matmul(codes[:, a:b], s["w"][:, a:b].float().t()).to(torch.int32)
    return (total.double() * scale[:, None].double() * s["w_scales"].double()).to(TYPES[s["case"]["out"]][0])


def plain_linear(s):
    case, step = s["case"], 64
    n, h, hk, dk, dv = case["seqs"], case["heads"], case["k_heads"], case["k_dim"], case["v_dim"]
    top = -(-max(s["rows"]) // step) * step if max(s["rows"]) > step else max(s["rows"])
    step = min(step, top)
    row = torch.arange(len(s["q"]), device="cuda")
    seq = torch.searchsorted(s["starts"][1:].long(), row, right=True)
    at = row - s["starts"][seq].long()

    def spread(x, width):  # [seq, head, row, width], zeros behind a sequence's end
        y = torch.zeros((n, top, x.shape[1], width), device="cuda")
        y[seq, at] = x.float().view(len(x), -1, width)
        return y.transpose(1, 2)

    q = spread(s["q"], dk).repeat_interleave(h // hk, 1)
    k = spread(s["k"], dk).repeat_interleave(h // hk, 1)
    v = spread(s["v"], dv)
    g = spread(s["decay"].expand(len(row), h)[..., None], 1)[..., 0].double()
    state = s["states"][s["slots"].long()]
    if case["fresh"]:
        state = torch.zeros_like(state)
    out = torch.empty((n, h, top, dv), device="cuda")
    causal = torch.ones((step, step), device="cuda").tril()
    for a in range(0, top, step):
        qc, kc, vc = (x[:, :, a:a + step].contiguous() for x in (q, k, v))
        b = g[:, :, a:a + step].cumsum(2)
        fade = (b[..., :, None] - b[..., None, :]).clamp(max=0.0).float().exp() * causal
        score = torch.matmul(qc, kc.transpose(2, 3).contiguous()) * fade
        out[:, :, a:a + step] = torch.matmul(score, vc) + torch.matmul(qc * b.float().exp()[..., None], state)
        left = kc * (b[:, :, -1:] - b).float().exp()[..., None]
        state = state * b[:, :, -1].float().exp()[..., None, None] + torch.matmul(left.transpose(2, 3).contiguous(), vc)
    states = s["states"].clone()
    states[s["slots"].long()] = state
    return [(out.transpose(1, 2)[seq, at] * dk ** -0.5).to(s["q"].dtype), states]


PLAIN = {"norm_rope": plain_norm_rope, "i8": plain_i8, "linear": plain_linear}


# ---- the same through halo_amd -----------------------------------------------------------------------------------------


def own_norm_rope(hl, s):
    case = s["case"]
    pairs = hl.RopePairs.HALF if case["pairs"] == "half" else hl.RopePairs.INTERLEAVED
    hl.norm_rope(TYPES[case["type"]][1], s["pos"], s["freqs"], case["tokens"], case["dim"], case["rot"], s["q"], s["q_out"], case["heads"],
                 q_norm=s["q_norm"], k=s["k"], k_out=s["k_out"], n_kv_heads=case["kv_heads"], k_norm=s["k_norm"], eps=s["eps"], pairs=pairs)
    return [s["q_out"], s["k_out"]]


def own_i8(hl, s):
    case = s["case"]
    hl.quantize_rows(TYPES[case["type"]][1], s["x"], s["codes"], s["scales"], case["n_vec"], case["cols"])
    hl.gemm_i8(TYPES[case["out"]][1], s["w"], s["w_scales"], s["codes"], s["scales"], s["y"], case["rows"], case["cols"], case["n_vec"])
    return s["y"]


def own_linear(hl, s):
    case = s["case"]
    state = hl.LinearState(s["states"], len(s["states"]), case["heads"], case["k_dim"], case["v_dim"], s["new_states"])
    batch = hl.LinearBatch(s["slots"], s["starts"], case["seqs"], sum(s["rows"]), max(s["rows"]), s["lens"])
    hl.linear_attention(TYPES[case["type"]][1], state, batch, s["q"], s["k"], s["v"], s["out"], s["decay"], case["k_heads"],
                        decay_per_head=case["decay"] == "heads")
    return [s["out"], s["new_states"]]


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return PLAIN[kind](state)
    import halo_amd as hl

    return {"norm_rope": own_norm_rope, "i8": own_i8, "linear": own_linear}[kind](hl, state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------


def exact(case, seed):
    return {"norm_rope": exact_norm_rope, "i8": exact_i8, "linear": exact_linear}[case["kind"]](prepare(case, seed))


def exact_norm_rope(s):
    case, out = s["case"], []
    turn = torch.polar(torch.ones_like(s["freqs"])[None].expand(case["tokens"], -1), s["pos"].double()[:, None] * s["freqs"])
    half, rot = case["rot"] // 2, case["rot"]
    pick = torch.arange(rot, device="cuda").view(2, half) if case["pairs"] == "half" else torch.arange(rot, device="cuda").view(half, 2).t()
    for x, w in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
        y = x.double()
        y = y / (y.square().sum(-1, keepdim=True) / case["dim"] + s["eps"]).sqrt() * w.double()
        z = torch.complex(y[..., pick[0]], y[..., pick[1]]) * turn[:, None]
        y[..., pick[0]], y[..., pick[1]] = z.real, z.imag
        out.append(y)
    return out


def exact_i8(s):
    """The codes are the nearest integers to x over its row's scale, which is held in 32 bits: a part of the definition."""
    x = s["x"].double()
    scale = (x.abs().amax(1, keepdim=True) / 127).float().double()
    codes = torch.round(x / scale.clamp(min=1e-300))
    w = s["w"][:, :s["case"]["cols"]].double() * s["w_scales"].double()[:, None]
    return torch.matmul(codes * scale, w.t().contiguous())


def exact_linear(s):
    """Token by token: the state fades, takes k's and v's outer product and is read with q."""
    case, group = s["case"], s["case"]["heads"] // s["case"]["k_heads"]
    states, out = s["states"].double(), torch.empty(s["out"].shape, dtype=torch.float64, device="cuda")
    fade = s["decay"].double().exp().expand(len(out), case["heads"])
    first = 0
    for slot, rows in zip(s["slots"].tolist(), s["rows"]):
        state = torch.zeros_like(states[slot]) if case["fresh"] else states[slot].clone()
        for r in range(first, first + rows):
            q, k = (x[r].double().repeat_interleave(group, 0)[..., None] for x in (s["q"], s["k"]))
            state.mul_(fade[r, :, None, None]).addcmul_(k, s["v"][r].double()[:, None])
            out[r] = (state * q).sum(1)
        states[slot] = state
        first += rows
    return [out * case["k_dim"] ** -0.5, states]
