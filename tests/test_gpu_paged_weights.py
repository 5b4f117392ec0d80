"""GPU: the paged cache's attentions where tokens' magnitudes lie far apart, in every form of the launch, against 64 bits within the
bound of tests/paged_bounds.py."""
import math

import pytest
import torch

import paged_bounds as W

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 1 / math.sqrt(128)
FORMS = {"auto": 0, "split": 15, "cluster1": 1, "cluster2": 2, "cluster8": 8, "tcgen05": 14}


@pytest.fixture(params=list(FORMS))
def form(request, monkeypatch):
    """The forms that the attention's launch has (the library chooses one by the call's shape)."""
    from blockgtq_b200 import paged
    monkeypatch.setattr(paged, "_FORM", FORMS[request.param])
    return request.param


def _pages(k, v, page=16):
    """One sequence's pages in order, its table and slots; k and v (t, n_kv, 128)."""
    from blockgtq_b200 import page_bytes, paged_kv4_append
    t, n_kv = k.shape[:2]
    width = -(-t // page)
    pages = torch.full((width, n_kv, page_bytes(page)), 255, dtype=torch.uint8, device=DEV)
    slots = torch.arange(t)
    paged_kv4_append(pages, slots.to(DEV), k.to(DEV), v.to(DEV))
    return pages, torch.arange(width, dtype=torch.int32)[None].to(DEV), slots


def _attend(q, pages, table, t, form, rows, scale=SCALE):
    """The last `rows` positions' queries; one row by the decode call but in the form that it has not."""
    from blockgtq_b200 import paged_kv4_decode_attention, paged_kv4_prefill_attention
    i32 = dict(dtype=torch.int32, device=DEV)
    lens = torch.tensor([t], **i32)
    if rows == 1 and form != "tcgen05":
        return paged_kv4_decode_attention(q.to(DEV), pages, table, lens, scale=scale, return_lse=True)
    return paged_kv4_prefill_attention(q.to(DEV), pages, table, lens, torch.tensor([0, rows], **i32), scale=scale, return_lse=True)


@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("size,above", [(0.05, 12), (0.01, 14)])
@pytest.mark.parametrize("every", [2000, 32])
def test_a_far_larger_value_does_not_cost_the_others_their_bits(size, above, every, rows, form):
    """Values of one size; among them, once or in every batch of a warp, a token whose third group is 65000 with hardly any weight, and behind it one
    of zeros whose weight is 2^above of the others'."""
    gen = torch.Generator().manual_seed(above)
    t, gqa = 2000, 4
    k = (0.01 * torch.randn(t, 1, 128, generator=gen)).half()
    v = (size * (1 + 0.3 * torch.randn(t, 1, 128, generator=gen))).half()
    c = above * math.log(2) / (128 * SCALE)                         # a key of c everywhere has that logit with a query of ones
    k[8::every], v[8::every, :, 64:96] = -8, 65000
    k[9::every], v[9::every] = c, 0
    pages, table, slots = _pages(k, v)
    q = (1 + 0.01 * torch.randn(rows, gqa, 128, generator=gen)).half()
    out, lse = _attend(q, pages, table, t, form, rows)
    W.check(out, lse, W.attention(q, pages.cpu(), slots, [t - rows + 1 + i for i in range(rows)], SCALE), slice(0, rows))


@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("first", [0, 100])
def test_pages_of_zeros_read_as_zeros(first, rows, form):
    """Tokens that nothing was stored for (scales of zero): logits and values of zero, in front of others or alone."""
    gen = torch.Generator().manual_seed(first)
    t = 300
    k, v = (torch.randn(t, 1, 128, generator=gen).half() for _ in range(2))
    pages, table, slots = _pages(k, v)
    empty = pages[:t // 16 if first == 0 else first // 16]
    empty.zero_()
    n = 280 if first == 0 else t
    q = torch.randn(rows, 4, 128, generator=gen).half()
    out, lse = _attend(q, pages, table, n, form, rows)
    if first == 0:
        assert not out.any()
    W.check(out, lse, W.attention(q, pages.cpu(), slots[:n], [n - rows + 1 + i for i in range(rows)], SCALE), slice(0, rows))


def test_values_of_every_magnitude(form):
    """Each group of each token's values has a magnitude of its own, from 2^-17 to 2^15."""
    gen = torch.Generator().manual_seed(3)
    t, rows = 700, 9
    k = torch.randn(t, 2, 128, generator=gen).half()
    size = 2.0 ** (32 * torch.rand(t, 2, 4, 1, generator=gen) - 17)
    v = (size * torch.rand(t, 2, 4, 32, generator=gen)).reshape(t, 2, 128).half()
    pages, table, slots = _pages(k, v)
    q = torch.randn(rows, 8, 128, generator=gen).half()
    out, lse = _attend(q, pages, table, t, form, rows)
    W.check(out, lse, W.attention(q, pages.cpu(), slots, [t - rows + 1 + i for i in range(rows)], SCALE), slice(0, rows))


@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("dtype,size", [(torch.float16, 1.0), (torch.float16, 2.0 ** 6), (torch.float16, 15000.0), (torch.bfloat16, 1e12), (torch.bfloat16, 1e28)])
def test_logits_of_any_magnitude(dtype, size, rows, form):
    """Keys of 9000 in size under queries of `size`: logits up to what fp32 holds.  Their steps are then larger than a weight's whole range."""
    gen = torch.Generator().manual_seed(77)
    t = 500
    one = 3000 * torch.randn(1, 2, 128, generator=gen)
    k = one.repeat(t, 1, 1)
    k[5:9], k[300] = -k[5:9], -k[300]                           # each head has its largest logit in many tokens, or in these
    v = torch.randn(t, 2, 128, generator=gen).to(dtype)
    pages, table, slots = _pages(k.to(dtype), v)
    q = (size * torch.randn(rows, 8, 128, generator=gen)).to(dtype)
    out, lse = _attend(q, pages, table, t, form, rows)
    W.check(out, lse, W.attention(q, pages.cpu(), slots, [t - rows + 1 + i for i in range(rows)], SCALE, apart=True), slice(0, rows))


def test_a_scale_whose_product_with_a_power_of_two_vanishes(form):
    """bf16 queries of 2^-130 are brought up by 2^140, which goes out of the scale again: of 1e-30 nothing is left, and every token weighs the same."""
    gen = torch.Generator().manual_seed(78)
    t, rows = 300, 5
    k, v = (torch.randn(t, 2, 128, generator=gen).bfloat16() for _ in range(2))
    pages, table, slots = _pages(k, v)
    q = (2.0 ** -130 * torch.randn(rows, 8, 128, generator=gen)).bfloat16()
    out, lse = _attend(q, pages, table, t, form, rows, scale=1e-30)
    W.check(out, lse, W.attention(q, pages.cpu(), slots, [t - rows + 1 + i for i in range(rows)], 1e-30), slice(0, rows))
