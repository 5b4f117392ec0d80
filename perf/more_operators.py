"""Calls around the paged 4-bit cache at the sizes at which a serving loop makes them: attention whose logits are capped, biased by distance or
masked by a window and a prefix; appending tokens whose rotary positions have several axes; copying pages.

A page holds units of 16 tokens; a unit of one KV head is 2304 bytes, seen here as 1152 half-words:

    [0, 512)      K codes: token t, half-word W at 32 t + W
    [512, 1024)   V codes: token t, half-word W at 64 (t / 2) + 2 W + t % 2
    [1024, 1088)  K scales (bf16): token t, group g at 4 t + g
    [1088, 1152)  V scales, the same

Nibble n of half-word W is the code of dim 32 n + W plus 8; group g is dims 32 g .. 32 g + 31.  A group's scale is the
largest magnitude / 7, rounded to bf16 and held in [2^-17, 9344]; a code is the whole number next to value / scale.

The attentions' rows, at position p of their sequence, see token t if t lies in the sequence's prefix, or t <= p and t > p - window.  Their logits
are c tanh(x / c) - slope |p - t| with x = q . k / sqrt(128), c the cap, one slope per query head.
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
        # one chat of 500 tokens with capped logits: what counts is the latency of a layer's attention
        {"name": "decode_cap_b1_t500", "kind": "decode", "dtype": "fp16", "n_q": 32, "n_kv": 8, "page": 64, "batch": 1, "shortest": 500, "longest": 500, "cap": 50.0, "slopes": False, "window": 0, "prefix": 0},
        # a batch of long contexts in a layer with a window that keeps the first tokens
        {"name": "decode_window_b8_t32768", "kind": "decode", "dtype": "bf16", "n_q": 16, "n_kv": 2, "page": 64, "batch": 8, "shortest": 32740, "longest": 32768, "cap": 0.0, "slopes": False, "window": 4096, "prefix": 4},
        # a serving batch of many lengths, empty slots among them, whose positions are a bias by distance
        {"name": "decode_slopes_b64_ragged", "kind": "decode", "dtype": "fp16", "n_q": 32, "n_kv": 8, "page": 16, "batch": 64, "shortest": 0, "longest": 9100, "cap": 0.0, "slopes": True, "window": 0, "prefix": 0},
        # one very long context, capped
        {"name": "decode_cap_b1_t131072", "kind": "decode", "dtype": "bf16", "n_q": 32, "n_kv": 8, "page": 64, "batch": 1, "shortest": 131072, "longest": 131072, "cap": 30.0, "slopes": False, "window": 0, "prefix": 0},
        # a whole prompt in a layer with capped logits and a window
        {"name": "prefill_cap_window_t8192", "kind": "prefill", "dtype": "bf16", "n_q": 32, "n_kv": 8, "page": 64, "batch": 1, "shortest": 8192, "longest": 8192, "q_least": 8192, "q_most": 8192, "cap": 50.0, "slopes": False, "window": 2048, "prefix": 0},
        # prompts that begin with a picture, whose tokens all rows see
        {"name": "prefill_prefix_b5", "kind": "prefill", "dtype": "fp16", "n_q": 16, "n_kv": 2, "page": 32, "batch": 5, "shortest": 700, "longest": 9100, "q_least": 650, "q_most": 700, "cap": 0.0, "slopes": False, "window": 0, "prefix": 576},
        # four drafted tokens per sequence to be verified, with a bias by distance and a window
        {"name": "verify_slopes_b16_q4_t2047", "kind": "prefill", "dtype": "bf16", "n_q": 32, "n_kv": 8, "page": 64, "batch": 16, "shortest": 1500, "longest": 2047, "q_least": 4, "q_most": 4, "cap": 0.0, "slopes": True, "window": 1024, "prefix": 0},
        # one new token of each sequence of a batch, its position by time, height and width
        {"name": "append_axes_b32", "kind": "append", "dtype": "fp16", "n_q": 32, "n_kv": 8, "page": 64, "tokens": 32, "padded": 0, "sections": "16,24,24", "interleaved": False},
        # the frames of a video in front of a text
        {"name": "append_axes_t16384", "kind": "append", "dtype": "bf16", "n_q": 32, "n_kv": 8, "page": 64, "tokens": 16384, "padded": 0, "sections": "16,24,24", "interleaved": False},
        # a ragged chunk in a padded buffer, axes taking turns
        {"name": "append_axes_t777_padded", "kind": "append", "dtype": "fp16", "n_q": 16, "n_kv": 2, "page": 16, "tokens": 777, "padded": 23, "sections": "24,20,20", "interleaved": True},
        # beams that part: the last, half-filled page of each, in all layers
        {"name": "copy_fork_b32", "kind": "copy", "layers": 36, "n_kv": 2, "page": 64, "pool": 400, "pages": 32, "whole": False},
        # held pages moved to the front of the pool
        {"name": "copy_compact_p256", "kind": "copy", "layers": 32, "n_kv": 8, "page": 64, "pool": 512, "pages": 256, "whole": True},
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    kind = rng.choice(["decode", "decode", "prefill", "prefill", "append", "copy"])
    n_kv, page = rng.choice([1, 2, 4, 8]), rng.choice([16, 32, 64, 128])
    if kind == "copy":
        layers = spread(1, 36)
        pool = max(2, min(spread(2, 2000), 1_100_000_000 // (layers * n_kv * page * 144)))
        return {"kind": kind, "layers": layers, "n_kv": n_kv, "page": page, "pool": pool, "pages": spread(1, pool // 2), "whole": rng.random() < 0.5}
    case = {"kind": kind, "dtype": rng.choice(["fp16", "bf16"]), "n_q": n_kv * rng.choice([1, 2, 4, 7, 8]), "n_kv": n_kv, "page": page}
    if kind == "append":
        case["tokens"] = spread(1, 16384)
        case["padded"] = rng.choice([0, spread(1, 100)])
        a = rng.randint(1, 60)
        b = rng.randint(1, 63 - a)
        case["sections"], case["interleaved"] = rng.choice([("16,24,24", False), ("32,32", False), ("24,20,20", True), ("16,16,16,16", True), (f"{a},{b},{64 - a - b}", rng.random() < 0.5)])
        return case
    case["cap"] = rng.choice([0.0, 15.0, 30.0, 50.0])
    case["slopes"] = rng.random() < 0.4
    case["batch"] = spread(1, 128)
    case["longest"] = max(2, spread(1, max(2, 1_000_000 // (n_kv * case["batch"]))))
    if kind == "prefill":
        # logits of a padded batch in 32 bits stay below those of the largest listed case
        case["longest"] = min(case["longest"], 12000)
        most = max(1, min(case["longest"], 2_000_000_000 // (case["batch"] * case["n_q"] * case["longest"])))
        case["q_most"] = spread(1, most)
        case["q_least"] = spread(1, case["q_most"])
        case["shortest"] = spread(case["q_most"], case["longest"])
    else:
        case["shortest"] = rng.choice([case["longest"], spread(1, case["longest"])])
    case["window"] = rng.choice([0, spread(1, case["longest"])])
    case["prefix"] = rng.choice([0, 4, spread(1, case["longest"])])
    return case


def lengths(case):
    """(tokens, queries, prefix) of each sequence, from the case alone."""
    b = case["batch"]
    rng = random.Random(7 * b + case["longest"])
    span = case["longest"] - case["shortest"]
    lens = [case["shortest"] + (rng.randrange(span + 1) if span else 0) for _ in range(b)]
    if b > 1:
        lens[0], lens[-1] = case["longest"], case["shortest"]
    q = [1] * b
    if case["kind"] == "prefill":
        q = [rng.randint(case["q_least"], case["q_most"]) for _ in range(b)]
        q[0] = case["q_most"]
    # (sinks are as many everywhere; pictures are of several sizes, and some prompts have none)
    most = case["prefix"]
    prefix = [most if most <= 4 else rng.choice([0, most, rng.randint(1, most)]) for _ in range(b)]
    prefix[0] = most
    return lens, q, prefix


def axis_of(case):
    """Axis of each of the 64 rotated pairs."""
    sections = [int(x) for x in case["sections"].split(",")]
    if not case["interleaved"]:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while len(out) < 64:
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return out


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


def rotate(x, cos, sin, positions, axis):
    """x (tokens, heads, 128): dims d and d + 64 turned by the angle of their token's position along the pair's axis."""
    pair = torch.arange(64, device=x.device)
    at = positions[axis].T                                        # (tokens, 64)
    c, s = cos[at, pair][:, None], sin[at, pair][:, None]
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
    n_kv, page = case["n_kv"], case["page"]
    page_bytes = page // 16 * 2 * UNIT
    state = {"kind": case["kind"]}

    if case["kind"] == "copy":
        # what a page holds is bytes to this path
        state["pages"] = torch.randint(0, 256, (case["layers"], case["pool"], n_kv, page_bytes), generator=gen, device=dev, dtype=torch.uint8)
        rng = random.Random(seed)
        order = rng.sample(range(case["pool"]), 2 * case["pages"])
        state["src"], state["dst"] = order[:case["pages"]], order[case["pages"]:]
        state["n_tokens"] = None if case["whole"] else [rng.randint(1, page) for _ in state["src"]]
        return state

    dtype, n_q = DTYPES[case["dtype"]], case["n_q"]

    def noise(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    m = channels(gen, n_kv, dev)

    if case["kind"] == "append":
        n, extra = case["tokens"], case["padded"]
        n_pages = -(-(n + 5) // page) + 1
        state["pages"] = torch.zeros(n_pages, n_kv, page_bytes, dtype=torch.uint8, device=dev)
        order = torch.randperm(n_pages, generator=gen, device=dev)
        at = torch.arange(n, device=dev) + 5
        slots = order[at // page] * page + at % page
        state["slots"] = torch.cat([slots, torch.full((extra,), -1, device=dev)])
        state["k"], state["v"] = (noise(n + extra, n_kv, HD) * m).to(dtype), noise(n + extra, n_kv, HD).to(dtype)
        state["q"] = noise(n + extra, n_q, HD).to(dtype)
        axis = axis_of(case)
        # frames of 24 x 24 patches: the first axis counts frames, the others lie within one
        frame, i = 24 * 24, torch.arange(n, device=dev)
        along = [i // frame, i % frame // 24, i % 24, i % 7][:max(axis) + 1]
        state["positions"] = torch.cat([torch.stack(along) + 5, torch.zeros(len(along), extra, dtype=torch.int64, device=dev)], 1)
        state["cos"], state["sin"] = tables(max(40, n // frame + 10), dev)
        state["axis"] = torch.tensor(axis, device=dev)
        if own:
            import blockgtq_b200 as B
            state["axes"] = B.rope_axes([int(x) for x in case["sections"].split(",")], interleaved=case["interleaved"])
        return state

    lens, queries, prefix = lengths(case)
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
    n = sum(queries)
    # (queries that a cap is trained with have logits that reach it)
    q = noise(n, n_q, HD) / m.repeat_interleave(n_q // n_kv, 0).clamp(min=0.5) * (4 if case["cap"] else 1)
    state["q"] = q.to(dtype)
    if case["kind"] == "prefill":
        ends = [0]
        for x in queries:
            ends.append(ends[-1] + x)
        state["ends"] = torch.tensor(ends, dtype=torch.int32, device=dev)
        state["most_q"], state["most"] = max(queries), max(lens)
    state["cap"], state["window"] = case["cap"] or None, case["window"] or None
    # one slope per head, from 1/2 down to 1/256 in equal factors
    state["slopes"] = 2.0 ** (-8.0 * torch.arange(1, n_q + 1, device=dev) / n_q) if case["slopes"] else None
    state["prefix"] = torch.tensor(prefix, dtype=torch.int32, device=dev) if case["prefix"] else None
    state["most_prefix"] = case["prefix"] or None
    return state


# ---- the operators ---------------------------------------------------------------------------------------------------


def plain_attention(state, q, lens, first, most):
    """q (sequences, queries, heads, 128) in 32 bits; query i is at position first + i of its sequence.  Results, and the natural logarithms of the
    rows' sums of exponentials."""
    pages, table = state["pages"], state["table"]
    page = pages.shape[2] // (2 * UNIT) * 16
    at = torch.arange(most, device=q.device)
    k, v = values(pages, table[:, at // page].long() * page + at % page)
    n, n_kv = q.shape[1], k.shape[2]
    group = q.shape[2] // n_kv
    qg = q.unflatten(2, (n_kv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    logits = (qg @ k.permute(0, 2, 3, 1)).mul_(1 / math.sqrt(HD)).unflatten(2, (group, n))
    if state["cap"]:
        logits.div_(state["cap"]).tanh_().mul_(state["cap"])
    position = first[:, None] + torch.arange(n, device=q.device)
    ahead = at - position[:, :, None]
    if state["slopes"] is not None:
        for h in range(group):
            logits[:, :, h] -= state["slopes"].view(n_kv, group)[:, h, None, None] * ahead.abs()[:, None].float()
    seen = ahead <= 0
    if state["window"]:
        seen &= ahead > -state["window"]
    if state["prefix"] is not None:
        seen |= at < state["prefix"][:, None, None]
    seen &= at < lens[:, None, None]
    logits.masked_fill_(~seen[:, None, None], -math.inf)
    top = logits.amax(-1, keepdim=True).clamp(min=-3e38)
    p = logits.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ v.permute(0, 2, 1, 3)).unflatten(2, (group, n)) / total.clamp(min=1e-30)
    lse = (total.log() + top).masked_fill(total == 0, -math.inf)[..., 0]
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3), lse.permute(0, 3, 1, 2).flatten(2, 3)


def run(state):
    kind = state["kind"]
    if own:
        import blockgtq_b200 as B
        if kind == "copy":
            B.paged_kv4_copy(state["pages"], state["src"], state["dst"], n_tokens=state["n_tokens"])
            return {"pages": state["pages"]}
        if kind == "append":
            q = B.paged_kv4_append(state["pages"], state["slots"], state["k"], state["v"], q=state["q"], cos=state["cos"], sin=state["sin"], positions=state["positions"], axes=state["axes"])
            k, v = B.paged_kv4_read(state["pages"], state["slots"])
            return {"q": q, "k": k, "v": v}
        scores = {"softcap": state["cap"], "slopes": state["slopes"], "window": state["window"], "prefix_lens": state["prefix"], "max_prefix_len": state["most_prefix"]}
        if kind == "decode":
            out, lse = B.paged_kv4_decode_attention(state["q"], state["pages"], state["table"], state["lens"], return_lse=True, **scores)
            return {"out": out, "lse": lse}
        return {"out": B.paged_kv4_prefill_attention(state["q"], state["pages"], state["table"], state["lens"], state["ends"], max_q_len=state["most_q"], max_seq_len=state["most"], **scores)}

    pages = state["pages"]
    if kind == "copy":
        src, dst = (torch.tensor(x, device=pages.device) for x in (state["src"], state["dst"]))
        if state["n_tokens"] is None:
            pages[:, dst] = pages[:, src]
        else:
            # units that hold the pages' first tokens
            units = pages.shape[3] // (2 * UNIT)
            taken = torch.arange(units, device=pages.device) < (torch.tensor(state["n_tokens"], device=pages.device)[:, None] + 15) // 16
            unit = pages.unflatten(3, (units, 2 * UNIT))
            i, u = taken.nonzero(as_tuple=True)
            unit[:, dst[i], :, u] = unit[:, src[i], :, u]
        return {"pages": pages}
    q = state["q"]
    if kind == "append":
        slots, turn = state["slots"], (state["cos"], state["sin"], state["positions"], state["axis"])
        live = slots >= 0
        store(pages, slots[live], rotate(state["k"], *turn)[live], state["v"][live])
        q = rotate(q, *turn).to(q.dtype)
        k, v = values(pages, slots.clamp(min=0))
        there = (slots >= 0)[:, None, None]
        return {"q": q, "k": (k * there).half(), "v": (v * there).half()}
    lens = state["lens"].long()
    most = state["table"].shape[1] * (pages.shape[2] // (2 * UNIT) * 16)
    if kind == "prefill":
        ends = state["ends"].long()
        counts, i = ends[1:] - ends[:-1], torch.arange(state["most_q"], device=q.device)
        there = i < counts[:, None]
        padded = torch.zeros(len(counts), state["most_q"], *q.shape[1:], device=q.device)
        padded[there] = q.float()
        return {"out": plain_attention(state, padded, lens, lens - counts, min(most, state["most"]))[0][there].to(q.dtype)}
    out, lse = plain_attention(state, q.float()[:, None], lens, lens - 1, most)
    return {"out": out[:, 0].to(q.dtype), "lse": lse[:, 0]}


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


def exact_rotated(x, case, state):
    out = x.double().clone()
    for d, axis in enumerate(axis_of(case)):
        at = state["positions"][axis]
        c, s = state["cos"].double()[at, d][:, None], state["sin"].double()[at, d][:, None]
        a, b = x[..., d].double(), x[..., d + 64].double()
        out[..., d], out[..., d + 64] = c * a - s * b, s * a + c * b
    return out


def exact(case, seed):
    state = prepare(case, seed)
    page, kind = case["page"], case["kind"]
    if kind == "copy":
        before, after = state["pages"], state["pages"].clone()
        for i, (a, b) in enumerate(zip(state["src"], state["dst"])):
            n = before.shape[3] if case["whole"] else math.ceil(state["n_tokens"][i] / 16) * 2304
            after[:, b, :, :n] = before[:, a, :, :n]
        return {"pages": after}
    if kind == "append":
        there = (state["slots"] >= 0)[:, None, None]
        return {"q": exact_rotated(state["q"], case, state), "k": exact_quantised(exact_rotated(state["k"], case, state)) * there, "v": exact_quantised(state["v"].double()) * there}
    lens, queries, prefix = lengths(case)
    q = state["q"]
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
            for part in torch.arange(n, device=q.device).split(1024):
                distance = (t - n + part)[:, None] - at
                seen = distance >= 0
                if case["window"]:
                    seen = seen & (distance < case["window"])
                if case["prefix"]:
                    seen = seen | (at < prefix[i])
                for h in range(case["n_q"]):
                    logits = mine[part, h] @ k[:, h // group].T / math.sqrt(HD)
                    if case["cap"]:
                        logits = case["cap"] * torch.tanh(logits / case["cap"])
                    if case["slopes"]:
                        logits = logits - state["slopes"][h].double() * distance.abs()
                    logits = torch.where(seen, logits, -math.inf)
                    lse[part, h] = torch.logsumexp(logits, -1)
                    out[part, h] = torch.softmax(logits, -1) @ v[:, h // group]
        outs.append(out)
        sums.append(lse)
    out = torch.cat(outs)
    return {"out": out, "lse": torch.cat(sums)} if kind == "decode" else {"out": out}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def work(case):
    n_kv, kind = case["n_kv"], case["kind"]
    if kind == "copy":
        # half of a page on average where it is not whole
        units = case["page"] // 16
        return {"bytes": 2 * case["layers"] * case["pages"] * n_kv * 2304 * (units if case["whole"] else (units + 1) / 2), "flops": 0}
    n_q = case["n_q"]
    if kind == "append":
        n = case["tokens"]
        # keys, values, queries and the tables' rows in; pages and queries out; the pages in again, their values out
        return {"bytes": n * (n_kv * (512 + 144 + 144 + 512) + n_q * 512 + 512), "flops": n * (3 * 64 * 2 * (n_q + n_kv) + 4 * 128 * n_kv * 2)}
    held = pairs = 0
    for t, n, p in zip(*lengths(case)):
        p = min(p, t)
        window = case["window"] or t
        held += min(t, p + min(t, window + n - 1))                # tokens that some row sees
        for i in range(n):
            behind = t - n + i + 1                                # tokens up to the row's own
            first = max(0, behind - window)
            pairs += behind - first + min(p, first) + max(0, p - behind)
    rows = sum(lengths(case)[1])
    return {"bytes": held * n_kv * 144 + rows * n_q * 512, "flops": 512 * n_q * pairs}
