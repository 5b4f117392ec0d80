"""GPU: biases by distance with slopes of any size: a row's own token has none, whatever the slope and wherever the row lies in a batch or a tile."""
import math

import pytest
import torch

import paged_bounds as W
import paged_scores as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I32 = dict(dtype=torch.int32, device=DEV)
FORMS = {"auto": 0, "split": 15, "cluster1": 1, "cluster8": 8, "tcgen05": 14}


@pytest.fixture(params=list(FORMS))
def form(request, monkeypatch):
    from blockgtq_b200 import paged
    monkeypatch.setattr(paged, "_FORM", FORMS[request.param])


def _pool(gen, t, page=16):
    from blockgtq_b200 import page_bytes, paged_kv4_append
    n = -(-t // page)
    pages, slots = torch.zeros(n, 1, page_bytes(page), dtype=torch.uint8, device=DEV), torch.arange(t)
    k, v = (torch.randn(t, 1, 128, generator=gen).half().to(DEV) for _ in range(2))
    paged_kv4_append(pages, slots.to(DEV), k, v)
    return pages, torch.arange(n, **I32)[None], slots


def _attend(q, pages, table, t, **kw):
    from blockgtq_b200 import paged_kv4_prefill_attention
    return paged_kv4_prefill_attention(q.to(DEV), pages, table, torch.tensor([t], **I32), torch.tensor([0, len(q)], **I32), return_lse=True, **kw)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cap", [None, 20.0])
@pytest.mark.parametrize("t,n", [(1, 1), (33, 1), (300, 5), (161, 161), (700, 90)])
@pytest.mark.parametrize("prefix", [0, 40])
def test_slopes_of_many_sizes(dtype, cap, t, n, prefix, form):
    """Within tests/paged_scores.py's bound, which gives a bias 2^-22 of itself: none at a row's own place."""
    gen = torch.Generator().manual_seed(t)
    pages, table, slots = _pool(gen, t)
    q = (torch.randn(n, 8, 128, generator=gen) * 2).to(dtype)
    for slopes in ([0.0, 0.7, 3.3, 11.1, 33.3, 123.4, 777.7, 0.01], [-0.3, 0.1, 1.7, 5.9, 20.3, 60.1, 250.7, 0.9]):
        slopes = torch.tensor(slopes)
        kw = dict(softcap=cap, slopes=slopes)
        out, lse = _attend(q, pages, table, t, **dict(kw, slopes=slopes.to(DEV)), **(dict(prefix_lens=torch.tensor([prefix], **I32)) if prefix else {}))
        rows = sorted({*range(min(n, 4)), *range(0, n, 13), n - 1})
        W.check(out, lse, S.attention(q, pages, slots, rows=rows, prefix=min(prefix, t), **kw), rows)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cap", [None, 20.0])
@pytest.mark.parametrize("t,n", [(33, 1), (300, 5), (161, 161)])
def test_a_slope_beside_which_nothing_counts(dtype, cap, t, n, form):
    """From 1e5 on a row's own token has all the weight: its logit is the row's sum, its value the result."""
    gen = torch.Generator().manual_seed(t)
    pages, table, slots = _pool(gen, t)
    q = torch.randn(n, 8, 128, generator=gen).to(dtype)
    slopes = torch.tensor([1e5, 1e9, 1e20, 1e30, 1e36, 1e37, 1e38, 3.4e38])
    out, lse = _attend(q, pages, table, t, softcap=cap, slopes=slopes.to(DEV))
    k, v = (x.cpu()[:, 0] for x in S.read(pages, slots))
    own = torch.arange(t - n, t)
    x = torch.einsum("nhd,nd->nh", q.double(), k[own]) / math.sqrt(128)
    y = x if cap is None else cap * torch.tanh(x / cap)
    # products lose 2^-20 of their terms, a cap 2^-20 of itself; a weight of one is exact, its value rounded once
    off = 2.0 ** -20 * (torch.einsum("nhd,nd->nh", q.double().abs(), k[own].abs()) / math.sqrt(128) + (cap or 0)) + 1e-5
    assert ((lse.double().cpu() - y).abs() <= off).all(), (lse.double().cpu() - y).abs().amax(0)
    want = v[own][:, None].expand(-1, 8, -1)
    assert ((out.double().cpu() - want).abs() <= (torch.finfo(dtype).eps / 2 + 2.0 ** -20) * want.abs() + 2.0 ** -25).all()


def test_a_slope_that_is_no_number_shows_in_its_head_only(form):
    gen = torch.Generator().manual_seed(5)
    pages, table, slots = _pool(gen, 150)
    q = torch.randn(20, 8, 128, generator=gen).half()
    slopes = torch.tensor([0.5, math.nan, 0.25, 0.1, 0.0, 1.0, math.nan, 2.0])
    out, lse = _attend(q, pages, table, 150, slopes=slopes.to(DEV))
    bad = slopes.isnan().to(DEV)
    assert out[:, bad].isnan().all() and not out[:, ~bad].isnan().any() and torch.isfinite(lse[:, ~bad]).all()
