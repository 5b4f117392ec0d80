"""Attention over the paged 4-bit cache with capped, biased and masked logits, in 64 bits, with a bound on what a kernel may be off by.

The bound is tests/paged_bounds.py's, token by token, and for what a logit goes through on the way (2^-24 the half step of fp32):

cap     c tanh(u), u = x / c.  What the products lose passes with a factor of at most 1, the slope of tanh.  Up to |u| = 1/2 a polynomial (1.5e-8 of the result)
        in 9 steps of one rounding each: 2^-20 of the result.  Beyond: three roundings of u (times its place's slope, u / cosh(u)^2 <= 0.45), the exponential's
        2^-22 (times 2 z / (z + 1)^2 <= 1/2), the reciprocal's 2^-23, the sum's, the difference's and the last product's 2^-24: below 2^-21 c, 2^-20 c with the
        constants' roundings.
bias    the slope times log2 e (two roundings), the distance as a number (one, exact below 2^24), a fused product and sum: 2^-22 of the bias and 2^-24 of the sum.
base    a logit and the reference that it is taken from: 2^-22 of either.
"""
import math

import torch

import paged_bounds as W
import paged_reference as R

LOG2E = 1.0 / math.log(2.0)


def read(pages, slots):
    """Values (n, n_kv, 128) in 64 bits of K and of V at ``slots``, on the pages' device."""
    page = pages.shape[2] // R.UNIT_BYTES * 16
    slots = slots.to(pages.device)
    unit = pages.unflatten(2, (page // 16, R.UNIT_BYTES))[slots // page, :, slots % page // 16].long()        # (n, n_kv, 2304)
    found = []
    offsets = [torch.stack(x) for x in zip(*[R.unit_offsets(t) for t in range(16)])]
    for word_at, scale_at in ((offsets[0], offsets[2]), (offsets[1], offsets[3])):
        at = word_at.to(pages.device)[slots % 16][:, None].expand(-1, pages.shape[1], -1)
        words = unit.gather(2, at) + 256 * unit.gather(2, at + 1)
        codes = torch.cat([(words >> 4 * n) % 16 - 8 for n in range(4)], -1)
        at = scale_at.to(pages.device)[slots % 16][:, None].expand(-1, pages.shape[1], -1)
        bits = unit.gather(2, at) + 256 * unit.gather(2, at + 1)
        scale = torch.where(bits > 32767, bits - 65536, bits).to(torch.int16).view(torch.bfloat16).double()
        found.append(codes.double() * scale.repeat_interleave(32, -1))
    return found


def seen_by(t, n, row, window=None, prefix=0, causal=True):
    """Which of t tokens row ``row`` of n sees."""
    at, p = torch.arange(t), t - n + row
    seen = at <= p if causal else torch.ones(t, dtype=torch.bool)
    if window is not None:
        seen &= at > p - window
    return seen | (at < prefix)


def attention(q, pages, slots, rows=None, scale=1 / math.sqrt(R.HD), softcap=None, slopes=None, window=None, prefix=0, causal=True):
    """The n rows of q (n, n_q, 128), a sequence's last positions, over its tokens at ``slots`` -> out, lse in 64 bits and the bound of each, of the
    rows ``rows`` (default: all)."""
    k, v = read(pages, slots)
    n, n_q = q.shape[:2]
    gqa, t = n_q // pages.shape[1], len(slots)
    k, v = (x.repeat_interleave(gqa, 1) for x in (k, v))
    dev = pages.device
    rows = list(range(n)) if rows is None else rows
    out, lse = torch.zeros(len(rows), n_q, R.HD, dtype=torch.float64, device=dev), torch.full((len(rows), n_q), -math.inf, dtype=torch.float64, device=dev)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for i, row in enumerate(rows):
        seen = seen_by(t, n, row, window, prefix, causal).to(dev)
        m = int(seen.sum())
        if m == 0:
            continue
        ks, vs, qd = k[seen], v[seen], q[row].double().to(dev)
        distance = (torch.arange(t, device=dev)[seen] - (t - n + row)).abs().double()
        x = torch.einsum("hd,thd->ht", qd, ks) * scale
        d = W.logit_cut(qd.cpu(), ks.cpu()).to(dev) * abs(scale) + x.abs() * 2.0 ** -22
        if q.dtype == torch.bfloat16:
            d = d + abs(scale) * 2.0 ** -23 * qd.abs().amax(-1)[:, None] * ks.abs().sum(-1).T
        if softcap is not None:
            y = softcap * torch.tanh(x / softcap)
            d = d + 2.0 ** -20 * torch.where(x.abs() < softcap * (0.5 - 1e-6), y.abs(), softcap)
        else:
            y = x
        if slopes is not None:
            bias = slopes.double().to(dev)[:, None] * distance
            y = y - bias
            d = d + bias.abs() * 2.0 ** -22 + y.abs() * 2.0 ** -24
        top = y.amax(-1, keepdim=True)
        d = d + (y.abs() + top.abs()) * 2.0 ** -22 + 3e-6
        lse[i] = torch.logsumexp(y, -1)
        p = torch.softmax(y, -1)
        out[i] = torch.einsum("ht,thd->hd", p, vs)
        # (weights are off by exp(d): d where it is small, and where it is not the weights are none)
        pd = p * torch.expm1(d)
        mean, cuts = torch.einsum("ht,thd->hd", p, vs.abs()), (m / 16 + 32) * 18 * 2.0 ** -24
        tol[i] = (2.0 ** -11 + 2.0 ** -20 + cuts) * mean + torch.einsum("ht,thd->hd", pd, vs.abs()) + pd.sum(-1)[:, None] * mean + cuts * 2.0 ** -14 \
            + 2.0 ** -32 * vs.abs().sum(0) + R.HALF[q.dtype] * out[i].abs() * 1.01 + 2.0 ** -25
        tol_lse[i] = pd.sum(-1) + lse[i].abs() * 2.0 ** -22 + (m / 16 + 32) * 2.0 ** -23 + 2.0 ** -20
    return out.cpu(), lse.cpu(), tol.cpu(), tol_lse.cpu()
