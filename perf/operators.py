"""Operators of serving over a paged cache, each in a plain form and as a user calls it, for timing and comparison.

listed() names the representative cases, draw() takes more from the same ranges.  prepare() makes what a program has in hand
before the call, run() is one pass, work() what a pass cannot do without, exact() the same results in 64 bits from the definition.

Kinds:
  rotate   rotary positions on the query and key heads of fused rows [q | k | v]: adjacent pairs or halves, part of the head,
           plain or YaRN-scaled tables, forward or transposed (the gradient)
  cache    new keys (rotated on the way) and values quantised into an 8-bit paged cache as they are written, and read back
  attend   attention of every sequence's new tokens over its paged cache, bf16 or 8-bit, causal, optionally in a sliding window

The paged cache: pool [page][keys, values][kv head][64 positions][D]; an 8-bit pool has a bf16 scale per position beside it,
[page][keys, values][kv head][64], and stands for the values bf16(number * scale).
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
PAGE = 64
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def listed():
    return [
        # one token of each of eight conversations: latency
        {"name": "rotate_step_8", "kind": "rotate", "dtype": "bf16", "tokens": 8, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "layout": "half",
         "inverse": False, "factor": 0.0, "table": 4096},
        # a long prompt, half of each head rotated, frequencies scaled for a longer context
        {"name": "rotate_prompt_8192", "kind": "rotate", "dtype": "bf16", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 64, "layout": "half",
         "inverse": False, "factor": 4.0, "table": 16384},
        # gradients of a rotation in fp32, adjacent pairs, an odd number of rows
        {"name": "rotate_back_1999", "kind": "rotate", "dtype": "f32", "tokens": 1999, "heads": 16, "kv_heads": 16, "dim": 64, "rot": 64, "layout": "adjacent",
         "inverse": True, "factor": 0.0, "table": 4096},
        # the new token of 64 conversations enters the cache
        {"name": "cache_step_64", "kind": "cache", "seqs": 64, "new": 1, "new_high": 1, "past": 500, "past_high": 8000, "kv_heads": 8, "dim": 128, "rot": 128,
         "layout": "half"},
        # prompts of four sequences enter the cache of a model without grouped heads
        {"name": "cache_prompts_4", "kind": "cache", "seqs": 4, "new": 1500, "new_high": 2500, "past": 0, "past_high": 0, "kv_heads": 32, "dim": 128, "rot": 64,
         "layout": "adjacent"},
        # interactive generation over a bf16 cache
        {"name": "decode_1_4096", "kind": "attend", "bits": 16, "seqs": 1, "new": 1, "new_high": 1, "past": 4095, "past_high": 4095, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 0},
        # a portion of a long prompt: what earlier portions left is in the cache
        {"name": "chunk_512_of_8192", "kind": "attend", "bits": 16, "seqs": 1, "new": 512, "new_high": 512, "past": 7680, "past_high": 7680, "heads": 32, "kv_heads": 8,
         "dim": 128, "window": 0},
        # a whole prompt, nothing in the cache before it
        {"name": "prompt_4096", "kind": "attend", "bits": 16, "seqs": 1, "new": 4096, "new_high": 4096, "past": 0, "past_high": 0, "heads": 32, "kv_heads": 32, "dim": 128,
         "window": 0},
        # continuous batching: single tokens beside portions of prompts, ragged contexts
        {"name": "mixed_16", "kind": "attend", "bits": 16, "seqs": 16, "new": 1, "new_high": 256, "past": 200, "past_high": 3900, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 0},
        # 64 conversations over an 8-bit cache
        {"name": "q8_decode_64", "kind": "attend", "bits": 8, "seqs": 64, "new": 1, "new_high": 1, "past": 511, "past_high": 8191, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 0},
        # a portion of a prompt over an 8-bit cache
        {"name": "q8_chunk_1000_of_9000", "kind": "attend", "bits": 8, "seqs": 1, "new": 1000, "new_high": 1000, "past": 8000, "past_high": 8000, "heads": 32, "kv_heads": 8,
         "dim": 128, "window": 0},
        # heads of 64 in a sliding window, a few tokens of each sequence (drafts being verified)
        {"name": "q8_window_drafts_12", "kind": "attend", "bits": 8, "seqs": 12, "new": 2, "new_high": 9, "past": 300, "past_high": 5000, "heads": 16, "kv_heads": 4, "dim": 64,
         "window": 1024},
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rotate", "cache", "attend", "attend", "attend"])
    dim = rng.choice([64, 128, 128])
    if kind == "rotate":
        kv = rng.choice([1, 2, 4, 8, 16])
        rot = rng.choice([dim, dim, dim // 2, dim // 4, 2 * rng.randint(1, dim // 2)])
        return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f32"]), "tokens": _log(rng, 1, 8192), "heads": kv * rng.randint(1, 32 // kv), "kv_heads": kv, "dim": dim,
                "rot": rot, "layout": rng.choice(["half", "adjacent"]), "inverse": rng.random() < 0.4, "factor": rng.choice([0.0, 4.0, 16.0]), "table": _log(rng, 512, 65536)}
    seqs = _log(rng, 1, 64)
    if kind == "cache":
        new = _log(rng, 1, max(1, 8192 // seqs))
        past = rng.choice([0, _log(rng, 1, 8000)])
        return {"kind": kind, "seqs": seqs, "new": max(1, new // rng.randint(1, 8)), "new_high": new, "past": past, "past_high": past * rng.randint(1, 3),
                "kv_heads": rng.choice([1, 2, 4, 8, 16, 32]), "dim": dim, "rot": rng.choice([0, dim, dim // 2, 2 * rng.randint(1, dim // 2)]),
                "layout": rng.choice(["half", "adjacent"])}
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([g for g in (1, 2, 3, 4, 5, 6, 7, 8, 16) if g * kv <= 32])
    new = rng.choice([1, _log(rng, 1, 16), _log(rng, 1, max(1, 4096 // seqs))])
    past = rng.choice([0, _log(rng, 1, 8000), _log(rng, 256, 12000)])
    low = max(0, past // rng.randint(1, 16))
    while seqs > 1 and (seqs * heads * new * (past + new) > 1 << 28 or seqs * (past + new) * kv * dim > 1 << 28):
        seqs = (seqs + 1) // 2
    return {"kind": kind, "bits": rng.choice([8, 16]), "seqs": seqs, "new": max(1, new // rng.randint(1, 8)), "new_high": new, "past": low, "past_high": past, "heads": heads,
            "kv_heads": kv, "dim": dim, "window": rng.choice([0, 0, _log(rng, 16, 4096)])}


# ---- sizes ------------------------------------------------------------------------------------------------------------
def _spread(low, high, n):
    """n whole numbers from low to high in equal ratios."""
    if n == 1:
        return [high]
    return [min(high, max(low, int(round((low + 1) * ((high + 1) / (low + 1)) ** (i / (n - 1)) - 1)))) for i in range(n)]


def _lengths(case):
    """(new tokens, tokens already in the cache) of every sequence: long portions do not go with long contexts."""
    n = case["seqs"]
    new, past = _spread(case["new"], case["new_high"], n), _spread(case["past"], case["past_high"], n)
    step = next(k for k in (7, 5, 3, 11, 1) if math.gcd(k, n) == 1)
    return new, [past[(i * step + 1) % n] for i in range(n)]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(1000003 * (int(seed) + 1))


def _randn(g, shape, dtype=F32):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def _table(rot, length, factor=0.0, base=10000.0, original=4096.0, fast=32.0, slow=1.0):
    """(cos, sin) of every position and pair, angles in 64 bits; factor: YaRN scaling of the frequencies."""
    half = rot // 2
    i = torch.arange(half, dtype=F64, device=DEV)
    freq = base ** (-2.0 * i / rot)
    size = 1.0
    if factor:
        pair = lambda turns: rot * math.log(original / (2.0 * math.pi * turns)) / (2.0 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(pair(fast)), 0.0), min(math.ceil(pair(slow)), rot - 1.0)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        freq = freq / factor * ramp + freq * (1.0 - ramp)
        size = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(length, dtype=F64, device=DEV)[:, None] * freq
    return torch.stack([size * angle.cos(), size * angle.sin()], -1).to(F32).contiguous()


def _round_up_bf16(x):
    """The smallest bf16 number that is not below x > 0."""
    return ((x.to(F32).view(torch.int32) + 0xFFFF) & ~0xFFFF).view(F32)


def _quantise(x):
    """fp32 [..., D] -> (whole numbers, bf16 scales [...])."""
    most = x.abs().amax(-1)
    small = most < 2.0 ** -100
    scale = torch.where(small, torch.zeros_like(most), _round_up_bf16(most / 127.0))
    back = torch.where(small, torch.zeros_like(most), 1.0 / scale)
    return torch.round(x * back[..., None]).clamp(-127, 127), scale.to(BF16)


def prepare(case, seed):
    kind, g = case["kind"], _gen(seed)
    if kind == "rotate":
        T, D, Hq, Hk = case["tokens"], case["dim"], case["heads"], case["kv_heads"]
        dt = BF16 if case["dtype"] == "bf16" else F32
        rows = _randn(g, (T, (Hq + 2 * Hk) * D), dt)
        start = int(torch.randint(0, case["table"], (1,), generator=g, device=DEV))
        at = ((torch.arange(T, device=DEV) + start) % case["table"]).to(torch.int32)
        return {"case": case, "q": rows[:, :Hq * D], "k": rows[:, Hq * D:(Hq + Hk) * D], "at": at, "table": _table(case["rot"], case["table"], case["factor"]),
                "q_out": torch.empty(T, Hq * D, dtype=dt, device=DEV), "k_out": torch.empty(T, Hk * D, dtype=dt, device=DEV)}
    n, Hk, D = case["seqs"], case["kv_heads"], case["dim"]
    new, past = _lengths(case)
    T, ctx = sum(new), [a + b for a, b in zip(new, past)]
    pages = [-(-c // PAGE) for c in ctx]
    total, most = sum(pages), max(pages)
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)  # a pool in use hands its pages out in any order
    table, at = torch.zeros(n, most, dtype=torch.int32, device=DEV), 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    seq = np.repeat(np.arange(n), new)
    off = np.concatenate([np.arange(k) for k in new])
    where = lambda v: torch.from_numpy(np.asarray(v, np.int64)).to(DEV)  # noqa: E731
    state = {"case": case, "tokens": T, "table": table, "ctx": torch.tensor(ctx, dtype=torch.int32, device=DEV), "seq": where(seq), "off": where(off),
             "starts": torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=DEV),
             "pos": where(np.asarray(past)[seq] + off), "max_new": max(new), "max_ctx": max(ctx)}
    if kind == "cache":
        rows = _randn(g, (T, 2 * Hk * D), BF16)
        rows *= torch.rand(T, 1, generator=g, device=DEV).mul_(4).exp2_()  # (rows of different size)
        rot = case["rot"]
        return {**state, "k": rows[:, :Hk * D], "v": rows[:, Hk * D:], "rope": _table(rot, max(ctx)) if rot else None,
                "pool": torch.zeros(total, 2, Hk, PAGE, D, dtype=torch.int8, device=DEV), "scales": torch.zeros(total, 2, Hk, PAGE, dtype=BF16, device=DEV)}
    pool, scales = torch.empty(total, 2, Hk, PAGE, D, dtype=BF16 if case["bits"] == 16 else torch.int8, device=DEV), None
    if case["bits"] == 8:
        scales = torch.empty(total, 2, Hk, PAGE, dtype=BF16, device=DEV)
    for p0 in range(0, total, 512):
        x = _randn(g, pool[p0:p0 + 512].shape)
        if scales is None:
            pool[p0:p0 + 512] = x.to(BF16)
        else:
            whole, scales[p0:p0 + 512] = _quantise(x)
            pool[p0:p0 + 512] = whole.to(torch.int8)
    q = _randn(g, (T, case["heads"] * D), BF16)
    return {**state, "q": q, "pool": pool, "scales": scales, "out": torch.empty_like(q)}


# ---- one pass ---------------------------------------------------------------------------------------------------------
def _rotated(x, pairs, rot, layout, inverse):
    """x [T, H, D] with the rotation of pairs [T, rot / 2, 2] on its first components, in the type of x."""
    c, s = pairs[:, None, :, 0], pairs[:, None, :, 1]
    s = -s if inverse else s
    x1, x2 = (x[..., :rot:2], x[..., 1:rot:2]) if layout == "adjacent" else (x[..., :rot // 2], x[..., rot // 2:rot])
    y1, y2 = x1 * c - x2 * s, x2 * c + x1 * s
    head = torch.stack([y1, y2], -1).flatten(-2) if layout == "adjacent" else torch.cat([y1, y2], -1)
    return torch.cat([head, x[..., rot:]], -1)


def _plain_rotate(s):
    case = s["case"]
    pairs = s["table"][s["at"].long()]
    for x, y in ((s["q"], s["q_out"]), (s["k"], s["k_out"])):
        r = _rotated(x.to(F32).unflatten(1, (-1, case["dim"])), pairs, case["rot"], case["layout"], case["inverse"])
        y.copy_(r.flatten(1))
    return [s["q_out"], s["k_out"]]


def _plain_cache(s):
    case = s["case"]
    k, v = (s[n].to(F32).unflatten(1, (case["kv_heads"], case["dim"])) for n in "kv")
    if case["rot"]:
        k = _rotated(k, s["rope"][s["pos"]], case["rot"], case["layout"], False)
    page, at = s["table"][s["seq"], s["pos"] // PAGE].long(), s["pos"] % PAGE
    back = []
    for i, x in enumerate((k, v)):
        whole, scale = _quantise(x)
        s["pool"][page, i, :, at] = whole.to(torch.int8)
        s["scales"][page, i, :, at] = scale
        back.append((s["pool"][page, i, :, at].to(F32) * s["scales"][page, i, :, at].to(F32)[..., None]).to(BF16).flatten(1))
    return back


def _plain_attend(s):
    case = s["case"]
    n, Hq, Hk, D, N, C = case["seqs"], case["heads"], case["kv_heads"], case["dim"], s["max_new"], s["max_ctx"]
    pages = s["table"].long()
    kv = s["pool"][pages].to(F32)  # [n, P, 2, Hk, 64, D]
    if s["scales"] is not None:
        kv = (kv * s["scales"][pages].to(F32)[..., None]).to(BF16).to(F32)
    kv = kv.permute(2, 0, 3, 1, 4, 5).flatten(3, 4)[..., :C, :]
    # new tokens of every sequence at the end of N places
    row = (s["starts"][1:].long()[:, None] - N + torch.arange(N, device=DEV)).clamp_(0)
    q = s["q"].to(F32)[row].view(n, N, Hk, Hq // Hk, D).permute(0, 2, 3, 1, 4).reshape(n, Hk, -1, D)
    score = (q @ kv[0].transpose(-1, -2)).mul_(D ** -0.5).view(n, Hk, Hq // Hk, N, C)
    at = (s["ctx"].long()[:, None] - N + torch.arange(N, device=DEV))[:, :, None]
    key = torch.arange(C, device=DEV)
    seen = key <= at.clamp(min=0)
    if case["window"]:
        seen &= key > at.clamp(min=0) - case["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    o = (p.view(n, Hk, -1, C) @ kv[1]).view(n, Hk, Hq // Hk, N, D) / p.sum(-1, keepdim=True)
    new = (s["starts"][1:] - s["starts"][:-1]).long()
    o = o.permute(0, 3, 1, 2, 4)[s["seq"], N - new[s["seq"]] + s["off"]]
    s["out"].copy_(o.reshape(s["tokens"], -1))
    return s["out"]


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        return {"rotate": _plain_rotate, "cache": _plain_cache, "attend": _plain_attend}[kind](state)
    import jasmine_b200 as jb
    layout = jb.ROPE_HALF if case.get("layout") == "half" else jb.ROPE_ADJACENT
    if kind == "rotate":
        jb.rope_rotate(state["q"], state["k"], state["table"], case["heads"], case["kv_heads"], case["dim"], case["rot"], state["at"], layout=layout,
                       inverse=case["inverse"], q_out=state["q_out"], k_out=state["k_out"])
        return [state["q_out"], state["k_out"]]
    if kind == "cache":
        jb.kv_append_q8(state["pool"], state["scales"], state["table"], state["k"], state["v"], state["starts"], state["ctx"], case["kv_heads"], case["dim"],
                        rope=state["rope"], rot_dim=case["rot"], layout=layout)
        return list(jb.kv_read(state["pool"], state["table"], state["starts"], state["ctx"], state["tokens"], case["kv_heads"], case["dim"], scales=state["scales"]))
    return jb.attn_chunk(state["q"], state["pool"], state["table"], state["starts"], state["ctx"], case["heads"], case["kv_heads"], case["dim"], state["max_new"],
                         state["max_ctx"], scales=state["scales"], window=case["window"], out=state["out"])


def work(case):
    D, Hk = case["dim"], case["kv_heads"]
    if case["kind"] == "rotate":
        T, H = case["tokens"], case["heads"] + Hk
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": T * (2 * H * D * size + 4) + min(T, case["table"]) * case["rot"] * 4, "flops": 3 * T * H * case["rot"]}
    new, past = _lengths(case)
    T, ctx = sum(new), [a + b for a, b in zip(new, past)]
    if case["kind"] == "cache":
        written = T * Hk * 2 * (D + 2)
        return {"bytes": T * Hk * D * 8 + 2 * written + T * case["rot"] * 4, "flops": T * Hk * (2 * D * 4 + 3 * case["rot"])}
    Hq, w = case["heads"], case["window"] or 1 << 40
    keys = sum(min(c, w + a - 1) for a, c in zip(new, ctx))
    pairs = 0
    for a, b in zip(new, past):
        free = max(0, min(a, w - b))  # queries that see everything before them
        pairs += free * b + free * (free + 1) // 2 + (a - free) * w if a > free else a * b + a * (a + 1) // 2
    entry = 2 * D * 2 if case["bits"] == 16 else 2 * (D + 2)
    return {"bytes": 2 * T * Hq * D * 2 + keys * Hk * entry, "flops": 4 * D * Hq * pairs}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------
def _exact_rotation(x, table, pos, rot, layout, sign):
    x = x.clone()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if layout == "adjacent" else (i, i + rot // 2)
        c, s = table[pos, i, 0].double()[:, None], sign * table[pos, i, 1].double()[:, None]
        u, v = x[:, :, a].clone(), x[:, :, b].clone()
        x[:, :, a], x[:, :, b] = u * c - v * s, u * s + v * c
    return x


def exact(case, seed):
    s, D = prepare(case, seed), case["dim"]
    if case["kind"] == "rotate":
        sign = -1.0 if case["inverse"] else 1.0
        return [_exact_rotation(s[n].double().reshape(case["tokens"], -1, D), s["table"], s["at"].long(), case["rot"], case["layout"], sign).reshape(case["tokens"], -1)
                for n in "qk"]
    if case["kind"] == "cache":
        k, v = (s[n].double().reshape(s["tokens"], case["kv_heads"], D) for n in "kv")
        if case["rot"]:
            k = _exact_rotation(k, s["rope"], s["pos"], case["rot"], case["layout"], 1.0)
        found = []
        for x in (k, v):
            low = x.abs().max(-1, keepdim=True).values / 127
            # bf16 numbers have eight bits: steps of 2^-7 of the power of two below
            step = torch.exp2(torch.floor(torch.log2(low)) - 7)
            scale = torch.ceil(low / step) * step
            found.append((torch.round(x / scale) * scale).reshape(s["tokens"], -1))
        return found
    Hq, Hk = case["heads"], case["kv_heads"]
    out = torch.empty(s["tokens"], Hq * D, dtype=F64, device=DEV)
    new, past = _lengths(case)
    t = 0
    for b in range(case["seqs"]):
        c = new[b] + past[b]
        pages = s["table"][b, :-(-c // PAGE)].long()
        kv = s["pool"][pages].double()
        if s["scales"] is not None:
            kv = (kv * s["scales"][pages].double().unsqueeze(-1)).to(BF16).double()  # (whole number times bf16: one rounding)
        at = torch.arange(past[b], c, device=DEV).unsqueeze(1)
        key = torch.arange(c, device=DEV)
        hidden = (key > at) | (key <= at - (case["window"] or c + 1))
        for h in range(Hq):
            K, V = (kv[:, i, h // (Hq // Hk)].reshape(-1, D)[:c] for i in (0, 1))
            w = torch.softmax((s["q"][t:t + new[b], h * D:(h + 1) * D].double() @ K.T / math.sqrt(D)).masked_fill(hidden, -math.inf), -1)
            out[t:t + new[b], h * D:(h + 1) * D] = w @ V
        t += new[b]
    return out
