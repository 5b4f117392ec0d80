"""Calls of the paged 4-bit cache's operators at the sizes at which a serving loop makes them.

A page holds units of 16 tokens; a unit of one KV head is 2304 bytes, seen here as 1152 half-words:

    [0, 512)      K codes: token t, half-word W at 32 t + W
    [512, 1024)   V codes: token t, half-word W at 64 (t / 2) + 2 W + t % 2
    [1024, 1088)  K scales (bf16): token t, group g at 4 t + g
    [1088, 1152)  V scales, the same

Nibble n of half-word W is the code of dim 32 n + W plus 8; group g is dims 32 g .. 32 g + 31.  A group's scale is the
largest magnitude / 7, rounded to bf16 and held in [2^-17, 9344]; a code is the whole number next to value / scale.
"""
import math
import random

import torch

own = False

HD = 128
UNIT = 1152                 # half-words of 16 tokens of one KV head
S_MIN, S_MAX = 2.0 ** -17, 9344.0
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one chat of 500 tokens: what counts is the latency of a layer's attention
        {"name": "decode_b1_t500", "kind": "decode", "dtype": "fp16", "n_q": 32, "n_kv": 8, "page": 64, "batch": 1, "shortest": 500, "longest": 500},
        # a batch of long contexts with few KV heads
        {"name": "decode_b8_t32768", "kind": "decode", "dtype": "bf16", "n_q": 16, "n_kv": 2, "page": 64, "batch": 8, "shortest": 32740, "longest": 32768},
        # a serving batch in which every sequence has its own length, empty slots among them, in small pages
        {"name": "decode_b64_ragged", "kind": "decode", "dtype": "fp16", "n_q": 32, "n_kv": 8, "page": 16, "batch": 64, "shortest": 0, "longest": 9100},
        # one very long context
        {"name": "decode_b1_t131072", "kind": "decode", "dtype": "bf16", "n_q": 32, "n_kv": 8, "page": 64, "batch": 1, "shortest": 131072, "longest": 131072},
        # a whole prompt against the cache that it was just written to
        {"name": "prefill_t8192", "kind": "prefill", "dtype": "bf16", "n_q": 32, "n_kv": 8, "page": 64, "batch": 1, "shortest": 8192, "longest": 8192, "q_least": 8192, "q_most": 8192},
        # chunks of several prompts behind contexts of their own
        {"name": "prefill_chunks_b5", "kind": "prefill", "dtype": "fp16", "n_q": 16, "n_kv": 2, "page": 32, "batch": 5, "shortest": 700, "longest": 9100, "q_least": 33, "q_most": 700},
        # four drafted tokens per sequence to be verified
        {"name": "verify_b16_q4_t2047", "kind": "prefill", "dtype": "bf16", "n_q": 32, "n_kv": 8, "page": 64, "batch": 16, "shortest": 1500, "longest": 2047, "q_least": 4, "q_most": 4},
        # one new token of each sequence of a batch
        {"name": "append_b32", "kind": "append", "dtype": "fp16", "n_q": 32, "n_kv": 8, "page": 64, "tokens": 32, "padded": 0},
        # a prompt's keys and values
        {"name": "append_t16384", "kind": "append", "dtype": "bf16", "n_q": 32, "n_kv": 8, "page": 64, "tokens": 16384, "padded": 0},
        # a ragged chunk in a padded buffer
        {"name": "append_t777_padded", "kind": "append", "dtype": "fp16", "n_q": 16, "n_kv": 2, "page": 16, "tokens": 777, "padded": 23},
        # a layer's part of a decode step: the new token of every sequence, then its attention
        {"name": "step_b32_t1000", "kind": "step", "dtype": "bf16", "n_q": 32, "n_kv": 8, "page": 64, "batch": 32, "shortest": 400, "longest": 1600},
        {"name": "step_b4_t4099", "kind": "step", "dtype": "fp16", "n_q": 16, "n_kv": 2, "page": 32, "batch": 4, "shortest": 4099, "longest": 4099},
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    kind = rng.choice(["decode", "decode", "prefill", "prefill", "append", "step"])
    n_kv = rng.choice([1, 2, 4, 8])
    case = {"kind": kind, "dtype": rng.choice(["fp16", "bf16"]), "n_q": n_kv * rng.choice([1, 2, 4, 7, 8]), "n_kv": n_kv, "page": rng.choice([16, 32, 64, 128])}
    if kind == "append":
        case["tokens"] = spread(1, 16384)
        case["padded"] = rng.choice([0, spread(1, 100)])
        return case
    case["batch"] = spread(1, 128)
    case["longest"] = max(2, spread(1, max(2, 1_000_000 // (n_kv * case["batch"]))))
    if kind == "prefill":
        # logits of a padded batch in 32 bits stay below those of the largest listed case
        case["longest"] = min(case["longest"], 12000)
        most = max(1, min(case["longest"], 2_000_000_000 // (case["batch"] * case["n_q"] * case["longest"])))
        case["q_most"] = spread(1, most)
        case["q_least"] = spread(1, case["q_most"])
        case["shortest"] = spread(case["q_most"], case["longest"])
        return case
    case["shortest"] = rng.choice([case["longest"], spread(1, case["longest"])])
    return case


def lengths(case):
    """(tokens, queries) of each sequence, from the case alone."""
    b = case["batch"]
    rng = random.Random(7 * b + case["longest"])
    span = case["longest"] - case["shortest"]
    lens = [case["shortest"] + (rng.randrange(span + 1) if span else 0) for _ in range(b)]
    if b > 1:
        lens[0], lens[-1] = case["longest"], case["shortest"]
    if case["kind"] == "step":
        lens = [max(1, t) for t in lens]
    if case["kind"] != "prefill":
        return lens, [1] * b
    q = [rng.randint(case["q_least"], case["q_most"]) for _ in range(b)]
    q[0] = case["q_most"]
    return lens, q


# ---- the format, in plain operations ------------------------------------------------------------------------------


def quantise(x):
    """(..., 128) -> codes in 0 .. 15 of the same shape, scales (..., 4)."""
    x = x.float()
    groups = x.unflatten(-1, (4, 32))
    scale = (groups.abs().amax(-1) / 7).to(torch.bfloat16).float().clamp(S_MIN, S_MAX)
    codes = torch.round(groups / scale[..., None]).clamp(-7, 7) + 8
    return codes.flatten(-2).to(torch.int32), scale


def places(slots, page):
    """Page and half-word positions (of codes and scales, K and V) of tokens in their pages."""
    dev = slots.device
    off, w, g = slots % page, torch.arange(32, device=dev), torch.arange(4, device=dev)
    unit, t = (off // 16 * UNIT)[..., None], (off % 16)[..., None]
    return slots // page, unit + 32 * t + w, unit + 512 + 64 * (t // 2) + 2 * w + t % 2, unit + 1024 + 4 * t + g, unit + 1088 + 4 * t + g


def store(pages, slots, k, v):
    """Quantises k and v (tokens, heads, 128) into the pages."""
    page = pages.shape[2] // (2 * UNIT) * 16
    half = pages.view(torch.int16)
    number, k_at, v_at, ks_at, vs_at = places(slots, page)
    heads = torch.arange(pages.shape[1], device=pages.device)[:, None]
    for x, at, s_at in ((k, k_at, ks_at), (v, v_at, vs_at)):
        codes, scale = quantise(x)
        c = codes.unflatten(-1, (4, 32))
        words = c[..., 0, :] | c[..., 1, :] << 4 | c[..., 2, :] << 8 | c[..., 3, :] << 12
        half[number[:, None, None], heads, at[:, None, :]] = words.to(torch.int16)
        half[number[:, None, None], heads, s_at[:, None, :]] = scale.to(torch.bfloat16).view(torch.int16)


def values(pages, slots):
    """Keys and values (..., heads, 128) in 32 bits of the tokens at `slots` (...)."""
    page = pages.shape[2] // (2 * UNIT) * 16
    half = pages.view(torch.int16)
    number, k_at, v_at, ks_at, vs_at = places(slots, page)
    heads = torch.arange(pages.shape[1], device=pages.device)[:, None]
    found = []
    for at, s_at in ((k_at, ks_at), (v_at, vs_at)):
        words = half[number[..., None, None], heads, at[..., None, :]].to(torch.int32)
        codes = torch.stack([(words >> 4 * n & 15) - 8 for n in range(4)], -2)
        scale = half[number[..., None, None], heads, s_at[..., None, :]].view(torch.bfloat16).float()
        found.append((codes * scale[..., None]).flatten(-2))
    return found


def rotate(x, cos, sin, positions):
    """x (tokens, heads, 128): dims d and d + 64 turned by their token's angle."""
    c, s = cos[positions][:, None], sin[positions][:, None]
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


# ---- states ----------------------------------------------------------------------------------------------------------


def channels(gen, n_kv, dev):
    """Magnitudes of the keys' dims: they differ widely, and two pairs of dims stand out in each head."""
    m = torch.exp(torch.randn(n_kv, 64, generator=gen, device=dev))
    m[:, :2] *= 8
    return torch.cat([m, m], -1)


def tables(n, dev):
    angle = torch.arange(n, dtype=torch.float64, device=dev)[:, None] * 500000.0 ** (-torch.arange(64, dtype=torch.float64, device=dev) / 64)
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, n_q, n_kv, page = DTYPES[case["dtype"]], case["n_q"], case["n_kv"], case["page"]
    page_bytes = page // 16 * 2 * UNIT

    def noise(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    m = channels(gen, n_kv, dev)
    state = {"kind": case["kind"]}

    def new_tokens(n, positions, table):
        state["k"], state["v"] = (noise(n, n_kv, HD) * m).to(dtype), noise(n, n_kv, HD).to(dtype)
        state["q"] = noise(n, n_q, HD).to(dtype)
        state["cos"], state["sin"] = tables(table, dev)
        state["positions"] = positions

    if case["kind"] == "append":
        n, extra = case["tokens"], case["padded"]
        n_pages = -(-(n + 5) // page) + 1
        state["pages"] = torch.zeros(n_pages, n_kv, page_bytes, dtype=torch.uint8, device=dev)
        order = torch.randperm(n_pages, generator=gen, device=dev)
        at = torch.arange(n, device=dev) + 5
        slots = order[at // page] * page + at % page
        state["slots"] = torch.cat([slots, torch.full((extra,), -1, device=dev)])
        new_tokens(n + extra, torch.cat([at, torch.zeros(extra, dtype=torch.int64, device=dev)]), n + 5)
        return state

    lens, queries = lengths(case)
    b, width = len(lens), max(1, -(-max(lens) // page))
    n_pages = sum(-(-t // page) for t in lens) + 3
    order = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros(b, width, dtype=torch.int32)
    order_host, used = order.cpu(), 0
    for i, t in enumerate(lens):
        own_pages = -(-t // page)
        table[i, :own_pages] = order_host[used:used + own_pages]
        used += own_pages
    state["table"] = table.to(dev)
    state["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    pages = torch.zeros(n_pages, n_kv, page_bytes, dtype=torch.uint8, device=dev)
    everything = torch.arange(n_pages * page, device=dev)
    for part in everything.split(max(1, 262144 // n_kv)):
        store(pages, part, noise(part.numel(), n_kv, HD) * m, noise(part.numel(), n_kv, HD))
    state["pages"] = pages
    if case["kind"] == "step":
        last = torch.tensor([t - 1 for t in lens], device=dev)
        state["slots"] = state["table"][torch.arange(b, device=dev), last // page].long() * page + last % page
        new_tokens(b, last, max(lens))
    else:
        n = sum(queries)
        q = noise(n, n_q, HD) / m.repeat_interleave(n_q // n_kv, 0).clamp(min=0.5)
        state["q"] = q.to(dtype)
        if case["kind"] == "prefill":
            ends = [0]
            for x in queries:
                ends.append(ends[-1] + x)
            state["ends"] = torch.tensor(ends, dtype=torch.int32, device=dev)
            state["most_q"], state["most"] = max(queries), max(lens)
    return state


# ---- the operators ---------------------------------------------------------------------------------------------------


def plain_attention(q, pages, table, lens, first, most):
    """q (sequences, queries, heads, 128) in 32 bits; query i sees the tokens up to first + i of its sequence."""
    page = pages.shape[2] // (2 * UNIT) * 16
    at = torch.arange(most, device=q.device)
    k, v = values(pages, table[:, at // page].long() * page + at % page)
    b, n, n_q = q.shape[:3]
    group = n_q // k.shape[2]
    qg = q.unflatten(2, (k.shape[2], group)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    logits = qg @ k.permute(0, 2, 3, 1) / math.sqrt(HD)
    limit = torch.minimum(lens[:, None], first[:, None] + 1 + torch.arange(n, device=q.device))
    hidden = at >= limit[:, None, :, None]
    logits = logits.unflatten(2, (group, n)).masked_fill_(hidden[:, :, None], -math.inf)
    top = logits.amax(-1, keepdim=True).clamp(min=-3e38)
    p = logits.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ v.permute(0, 2, 1, 3)).unflatten(2, (group, n)) / total.clamp(min=1e-30)
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)


def run(state):
    kind = state["kind"]
    if own:
        import blockgtq_b200 as B
        if kind in ("append", "step"):
            q = B.paged_kv4_append(state["pages"], state["slots"], state["k"], state["v"], q=state["q"], cos=state["cos"], sin=state["sin"], positions=state["positions"])
            if kind == "append":
                k, v = B.paged_kv4_read(state["pages"], state["slots"])
                return {"q": q, "k": k, "v": v}
            return {"out": B.paged_kv4_decode_attention(q, state["pages"], state["table"], state["lens"])}
        if kind == "decode":
            out, lse = B.paged_kv4_decode_attention(state["q"], state["pages"], state["table"], state["lens"], return_lse=True)
            return {"out": out, "lse": lse}
        return {"out": B.paged_kv4_prefill_attention(state["q"], state["pages"], state["table"], state["lens"], state["ends"], max_q_len=state["most_q"], max_seq_len=state["most"])}

    pages, q = state["pages"], state["q"]
    if kind in ("append", "step"):
        slots, turn = state["slots"], (state["cos"], state["sin"], state["positions"])
        live = slots >= 0 if kind == "append" else slice(None)
        store(pages, slots[live], rotate(state["k"], *turn)[live], state["v"][live])
        q = rotate(q, *turn).to(q.dtype)
        if kind == "append":
            k, v = values(pages, slots.clamp(min=0))
            there = (slots >= 0)[:, None, None]
            return {"q": q, "k": (k * there).half(), "v": (v * there).half()}
    table, lens = state["table"], state["lens"].long()
    most = table.shape[1] * (pages.shape[2] // (2 * UNIT) * 16)
    if kind == "prefill":
        ends = state["ends"].long()
        counts, i = ends[1:] - ends[:-1], torch.arange(state["most_q"], device=q.device)
        there = i < counts[:, None]
        padded = torch.zeros(len(counts), state["most_q"], *q.shape[1:], device=q.device)
        padded[there] = q.float()
        return {"out": plain_attention(padded, pages, table, lens, lens - counts, min(most, state["most"]))[there].to(q.dtype)}
    out = plain_attention(q.float()[:, None], pages, table, lens, lens - 1, most)[:, 0].to(q.dtype)
    if kind == "step":
        return {"out": out}
    return {"out": out, "lse": plain_lse(q.float(), pages, table, lens, most)}


def plain_lse(q, pages, table, lens, most):
    """Natural logarithm of the sum of each row's exponentials: (sequences, heads)."""
    page = pages.shape[2] // (2 * UNIT) * 16
    at = torch.arange(most, device=q.device)
    k, _ = values(pages, table[:, at // page].long() * page + at % page)
    logits = q.unflatten(1, (k.shape[2], -1)) @ k.permute(0, 2, 3, 1) / math.sqrt(HD)
    logits = logits.masked_fill(at >= lens[:, None, None, None], -math.inf)
    top = logits.amax(-1, keepdim=True).clamp(min=-3e38)
    return ((logits - top).exp().sum(-1).log() + top[..., 0]).flatten(1)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------


def exact_values(pages, page, slots):
    """Keys and values of the tokens at `slots` (a list of whole numbers), taken apart byte by byte."""
    raw = pages.view(pages.shape[0], pages.shape[1], page // 16, 2 * UNIT)
    number, unit, t = slots // page, slots % page // 16, slots % 16
    rows = raw[number, :, unit]                                   # (tokens, heads, 2304)
    pick = torch.arange(slots.numel(), device=slots.device)
    k = rows[..., :1024].unflatten(-1, (16, 32, 2))[pick, :, t]
    v = rows[..., 1024:2048].unflatten(-1, (8, 32, 2, 2))[pick, :, t // 2][pick, :, :, t % 2]
    both = []
    for codes, first in ((k, 2048), (v, 2176)):
        low, high = codes[..., 0], codes[..., 1]
        code = torch.cat([low & 15, low >> 4, high & 15, high >> 4], -1).double() - 8
        scale = rows[..., first:first + 128].contiguous().view(torch.bfloat16).unflatten(-1, (16, 4))[pick, :, t].double()
        both.append(code * scale.repeat_interleave(32, -1))
    return both


def exact_quantised(x):
    """(tokens, heads, 128) in 64 bits -> the values that the cache then stands for."""
    g = x.unflatten(-1, (4, 32))
    scale = (g.abs().amax(-1, keepdim=True) / 7).to(torch.bfloat16).double().clamp(S_MIN, S_MAX)
    return (torch.round(g / scale).clamp(-7, 7) * scale).flatten(-2)


def exact_rotated(x, state):
    angle_cos, angle_sin = state["cos"].double()[state["positions"]], state["sin"].double()[state["positions"]]
    x = x.double()
    y = x * torch.cat([angle_cos, angle_cos], -1)[:, None]
    return y + torch.roll(x, 64, -1) * torch.cat([-angle_sin, angle_sin], -1)[:, None]


def exact(case, seed):
    state = prepare(case, seed)
    page, kind = case["page"], case["kind"]
    if kind == "append":
        there = (state["slots"] >= 0)[:, None, None]
        return {"q": exact_rotated(state["q"], state), "k": exact_quantised(exact_rotated(state["k"], state)) * there, "v": exact_quantised(state["v"].double()) * there}
    lens, queries = lengths(case)
    q = state["q"]
    if kind == "step":
        q = exact_rotated(q, state).to(q.dtype)
        new = [exact_quantised(exact_rotated(state["k"], state)), exact_quantised(state["v"].double())]
    outs, sums, row = [], [], 0
    group = case["n_q"] // case["n_kv"]
    for i, (t, n) in enumerate(zip(lens, queries)):
        mine = q[row:row + n].double()
        row += n
        at = torch.arange(t, device=q.device)
        out = torch.zeros(n, case["n_q"], HD, dtype=torch.float64, device=q.device)
        lse = torch.full((n, case["n_q"]), -math.inf, dtype=torch.float64, device=q.device)
        if t:
            k, v = exact_values(state["pages"], page, state["table"][i].long()[at // page] * page + at % page)
            if kind == "step":
                k[-1], v[-1] = new[0][i], new[1][i]
            seen = t - n + 1 + torch.arange(n, device=q.device)
            for h in range(case["n_q"]):
                for part in torch.arange(n, device=q.device).split(1024):
                    logits = mine[part, h] @ k[:, h // group].T / math.sqrt(HD)
                    logits = torch.where(at < seen[part, None], logits, -math.inf)
                    lse[part, h] = torch.logsumexp(logits, -1)
                    out[part, h] = torch.softmax(logits, -1) @ v[:, h // group]
        outs.append(out)
        sums.append(lse)
    out = torch.cat(outs)
    return {"out": out, "lse": torch.cat(sums)} if kind == "decode" else {"out": out}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def work(case):
    n_q, n_kv, kind = case["n_q"], case["n_kv"], case["kind"]
    if kind == "append":
        n = case["tokens"]
        # keys, values, queries and the tables' rows in; pages and queries out; the pages in again, their values out
        return {"bytes": n * (n_kv * (512 + 144 + 144 + 512) + n_q * 512 + 512), "flops": n * (3 * 64 * 2 * (n_q + n_kv) + 4 * 128 * n_kv * 2)}
    lens, queries = lengths(case)
    rows = sum(queries)
    seen = sum(n * t - n * (n - 1) // 2 for t, n in zip(lens, queries))
    total = {"bytes": sum(lens) * n_kv * 144 + rows * n_q * 512, "flops": 512 * n_q * seen}
    if kind == "step":
        total["bytes"] += rows * (n_kv * 512 + 512)
    return total
