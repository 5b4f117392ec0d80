"""The paged 4-bit cache in plain operations: the quantiser in 32 bits (its steps are single IEEE operations, so results are equal bit
for bit), the page's bytes taken apart one by one, attention in 64 bits with a bound on what a kernel may be off by."""
import math

import torch

HD, UNIT_BYTES = 128, 2304
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def rotated(x, cos, sin, positions):
    """fp32, every product and sum rounded by itself."""
    c, s = cos[positions][:, None], sin[positions][:, None]
    a, b = x.float()[..., :64], x.float()[..., 64:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def quantised(x):
    """(..., 128) fp32 -> signed codes (..., 128) int64, scales (..., 4) bf16."""
    g = x.float().reshape(*x.shape[:-1], 4, 32)
    top = g.abs().amax(-1)
    scale = (top / 7).bfloat16().float()
    scale = torch.where(scale.isnan(), scale, scale.clamp(2.0 ** -17, 9344.0))
    codes = torch.round(g / scale[..., None]).clamp(-7, 7).nan_to_num(0.0)
    return codes.reshape(x.shape).long(), scale.bfloat16()


def unit_offsets(t):
    """Byte offsets inside a unit: K half-words, V half-words, K scales, V scales of token t."""
    W, g = torch.arange(32), torch.arange(4)
    return 64 * t + 2 * W, 1024 + 128 * (t // 2) + 4 * W + 2 * (t % 2), 2048 + 8 * t + 2 * g, 2176 + 8 * t + 2 * g


def write(pages, slot, k, v):
    """Stores one token's k, v (n_kv, 128) fp32 into pages (n_pages, n_kv, bytes) uint8 on the CPU."""
    page = pages.shape[2] // UNIT_BYTES * 16
    p, off = slot // page, slot % page
    base = off // 16 * UNIT_BYTES
    at = unit_offsets(off % 16)
    for x, word_at, scale_at in ((k, at[0], at[2]), (v, at[1], at[3])):
        codes, scale = quantised(x)
        n = (codes + 8).reshape(-1, 4, 32)
        words = n[:, 0] + 16 * n[:, 1] + 256 * n[:, 2] + 4096 * n[:, 3]
        bits = torch.where(scale.isnan(), 0x7FFF, scale.view(torch.int16).long() & 0xFFFF)        # (the NaN that conversions on the GPU give)
        for at_, val in ((word_at, words), (scale_at, bits)):
            pages[p][:, base + at_] = (val & 0xFF).to(torch.uint8)
            pages[p][:, base + at_ + 1] = (val >> 8).to(torch.uint8)


def read(pages, slots):
    """Values (n, n_kv, 128) in 64 bits and scales (n, n_kv, 4) of K and of V."""
    page = pages.shape[2] // UNIT_BYTES * 16
    ks, vs, kss, vss = [], [], [], []
    for slot in slots.tolist():
        p, off = slot // page, slot % page
        at = [x + off // 16 * UNIT_BYTES for x in unit_offsets(off % 16)]
        for word_at, scale_at, vals, scales in ((at[0], at[2], ks, kss), (at[1], at[3], vs, vss)):
            words = pages[p][:, word_at].long() + 256 * pages[p][:, word_at + 1].long()
            codes = torch.cat([(words >> 4 * n) % 16 - 8 for n in range(4)], -1)
            bits = pages[p][:, scale_at].long() + 256 * pages[p][:, scale_at + 1].long()
            s = torch.where(bits > 32767, bits - 65536, bits).to(torch.int16).view(torch.bfloat16).double()
            vals.append(codes.double() * s.repeat_interleave(32, -1))
            scales.append(s)
    def stack(x, w):
        return torch.stack(x) if x else torch.zeros(0, pages.shape[1], w, dtype=torch.float64)
    return stack(ks, HD), stack(vs, HD), stack(kss, 4), stack(vss, 4)


def attention(q, pages, slots, seen, scale):
    """q (n, n_q, 128) over the tokens at ``slots``, row i the first seen[i] of them.  Returns out and lse in 64 bits, and the bound
    of each against a result of q's type:

    a logit is a sum of four groups' fp32 products: operands exact, 32 terms of |q| * 15 * scale and a start of |q| * 8 * scale each, a
    term cut at 2^-24 of 64 |q| * scale where codes lie unnormalised: d = 2^-20 * scale * sum |q| 15 ks holds 16 such cuts per
    accumulation of 16 and the rounding of the groups' sums, with 2^-20 more for the base's change, the subtraction of the maximum (its
    magnitude times 2^-22) and the exponential.  Each weight is off by a factor within 1 +- 2 d of numerator and denominator; weights are
    rounded once more to fp16 (2^-11), their products accumulate in fp32 over at most n / 16 steps of magnitude 15 p vs at most, and the
    result is rounded to q's type."""
    k, v, ks, vs = read(pages, slots)
    n, n_q = q.shape[:2]
    gqa = n_q // pages.shape[1]
    k, v, ks, vs = (x.repeat_interleave(gqa, 1) for x in (k, v, ks, vs))
    qd = q.double().cpu()
    T = k.shape[0]
    out, lse = torch.zeros(n, n_q, HD, dtype=torch.float64), torch.full((n, n_q), -math.inf, dtype=torch.float64)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for i in range(n):
        m = max(0, min(T, int(seen[i])))
        if m == 0:
            continue
        logits = torch.einsum("hd,thd->ht", qd[i], k[:m]) * scale
        lse[i] = torch.logsumexp(logits, -1)
        p = torch.softmax(logits, -1)
        out[i] = torch.einsum("ht,thd->hd", p, v[:m])
        size = torch.einsum("hd,thd->ht", qd[i].abs(), ks[:m].repeat_interleave(32, -1)) * abs(scale) * 15
        d = size.amax(-1) * 2.0 ** -20 + logits.abs().amax(-1) * 2.0 ** -22 + 2.0 ** -20
        mean = torch.einsum("ht,thd->hd", p, v[:m].abs())
        wide = torch.einsum("ht,thd->hd", p, vs[:m].repeat_interleave(32, -1)) * 15
        steps = (m / 16 + 16) * 2.0 ** -23
        tol[i] = (2.0 ** -11 + 4 * d[:, None]) * mean + 2 * steps * wide + HALF[q.dtype] * out[i].abs() * 1.01 + 1e-7
        tol_lse[i] = 2 * d + lse[i].abs() * 2.0 ** -22 + 1e-6
    return out, lse, tol, tol_lse
