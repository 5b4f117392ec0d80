"""Attention over the paged 4-bit cache in 64 bits, with a bound on what a kernel may be off by that is derived from the kernels' arithmetic.

With 2^-24 the half step of fp32, 2^-11 that of fp16:

logit   operands are exact: codes, or codes x scale, are fp16 numbers, and queries are fp16 after a power of two (bf16 ones lose at most 2^-23 of the
        row's largest).  A product's step of 16 dims adds 16 terms to an accumulator; each of the 17 is cut at 2^-24 of the largest's magnitude M
        at worst: 17 x 2^-24 x M per step, M looked up for every step, in both orders that the kernels take the dims in (four groups
        of two steps that start at zero, whose sums are then scaled and added, four roundings each; or eight steps in one).  The change of base
        and the reference's subtraction: 2^-22 of the largest logit; the exponential 3e-6 of the weight.
weight  rounded to fp16, relative 2^-11, where it lies in fp16's normal range.  References lie so that a row's largest weight is at least 2^7: weights below 2^-21 of it
        are cut at 2^-25 / 2^7 = 2^-32 of the largest one.
sums    V's operands are exact.  A step of 16 tokens cuts 17 terms at 2^-24 of the largest at worst, which is no more than the sum of all p |v|, or of p x 2^-14
        where v lies below fp16's normal range; tokens / 16 steps and one for each time a reference moves or shares are merged, 16 at most.
result  one division and product in fp32, one rounding to q's type.
"""
import math

import torch

import paged_reference as R

STEPS_BY_GROUP = [[32 * g + 8 * c + 4 * half + i for c in range(4) for i in range(4)] for g in range(4) for half in range(2)]
STEPS_IN_ONE = [list(range(16 * k, 16 * k + 16)) for k in range(8)]


def logit_cut(q, k):
    """What a logit's products and sums may lose, before the scale: q (h, 128), k (t, h, 128) -> (h, t)."""
    x = torch.einsum("hd,thd->htd", q, k)
    group, one = torch.zeros(2, *x.shape[:2], dtype=torch.float64).unbind(0)
    acc = torch.zeros_like(group)
    whole, running = torch.zeros_like(group), torch.zeros_like(group)
    for i, dims in enumerate(STEPS_BY_GROUP):
        if i % 2 == 0:
            acc = torch.zeros_like(acc)
        part, before = x[..., dims], acc
        acc = acc + part.sum(-1)
        group += 17 * 2.0 ** -24 * torch.maximum(part.abs().amax(-1), torch.maximum(before.abs(), acc.abs()))
        if i % 2:
            running = running + acc
            group += 2.0 ** -24 * (2 * acc.abs() + 2 * running.abs())
    for dims in STEPS_IN_ONE:
        part, before = x[..., dims], whole
        whole = whole + part.sum(-1)
        one += 17 * 2.0 ** -24 * torch.maximum(part.abs().amax(-1), torch.maximum(before.abs(), whole.abs()))
    return torch.maximum(group, one)


def attention(q, pages, slots, seen, scale, apart=False):
    """q (n, n_q, 128) over the tokens at ``slots``, row i the first seen[i] of them -> out, lse in 64 bits and the bound of each.  ``apart``: keys
    are equal, and then their logits are too, or so far apart that one has no weight beside the other: what logits lose changes no weight."""
    k, v, _, _ = R.read(pages, slots)
    n, n_q = q.shape[:2]
    gqa = n_q // pages.shape[1]
    k, v = (x.repeat_interleave(gqa, 1) for x in (k, v))
    qd = q.double().cpu()
    T = k.shape[0]
    out, lse = torch.zeros(n, n_q, R.HD, dtype=torch.float64), torch.full((n, n_q), -math.inf, dtype=torch.float64)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for i in range(n):
        m = max(0, min(T, int(seen[i])))
        if m == 0:
            continue
        logits = torch.einsum("hd,thd->ht", qd[i], k[:m]) * scale
        lse[i] = torch.logsumexp(logits, -1)
        p = torch.softmax(logits, -1)
        out[i] = torch.einsum("ht,thd->hd", p, v[:m])
        d = (logit_cut(qd[i], k[:m]) * abs(scale)).amax(-1) + logits.abs().amax(-1) * 2.0 ** -22 + 3e-6
        if q.dtype == torch.bfloat16:
            d = d + abs(scale) * 2.0 ** -23 * qd[i].abs().amax(-1) * k[:m].abs().sum(-1).amax(0)
        mean = torch.einsum("ht,thd->hd", p, v[:m].abs())
        cuts = (m / 16 + 16) * 18 * 2.0 ** -24
        between = torch.full_like(d, 3e-6) if apart else d
        tol[i] = (2.0 ** -11 + 2 * between[:, None] + 2.0 ** -20 + cuts) * mean + cuts * 2.0 ** -14 + 2.0 ** -32 * v[:m].abs().sum(0) \
            + R.HALF[q.dtype] * out[i].abs() * 1.01 + 2.0 ** -25
        tol_lse[i] = d + lse[i].abs() * 2.0 ** -22 + (m / 16 + 32) * 2.0 ** -23 + 2.0 ** -20
    return out, lse, tol, tol_lse


def check(got, lse, ref, rows):
    out, want_lse, tol, tol_lse = ref
    g = got[rows].double().cpu()
    assert torch.isfinite(g).all()
    off = (g - out).abs()
    assert (off <= tol).all(), ((off / tol.clamp(min=1e-30)).max(), off.max())
    if lse is not None:
        l = lse[rows].double().cpu()
        assert torch.equal(l == -math.inf, want_lse == -math.inf)
        f = torch.isfinite(want_lse)
        assert ((l - want_lse).abs()[f] <= tol_lse[f]).all(), (l - want_lse).abs()[f].max()
