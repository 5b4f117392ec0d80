"""GPU: the paged 4-bit cache against plain operations: stored bytes bit for bit, attention against 64 bits within the bound that
tests/paged_reference.py derives."""
import math

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float16, torch.bfloat16]


def _tables(n):
    angle = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    return angle.cos().float(), angle.sin().float()


def _noise(gen, *shape):
    return torch.randn(*shape, generator=gen)


def _case(gen, n_kv, page, lens, spare=2, dtype=torch.float16):
    """Pages holding sequences of these lengths in shuffled order, everything else in them all ones (codes 7, scales NaN)."""
    from blockgtq_b200 import page_bytes, paged_kv4_append
    width = max(1, max(-(-t // page) for t in lens)) + 1
    n_pages = sum(-(-t // page) for t in lens) + spare
    order = torch.randperm(n_pages, generator=gen).tolist()
    table, slots = torch.full((len(lens), width), -7, dtype=torch.int32), []
    for b, t in enumerate(lens):
        for i in range(-(-t // page)):
            table[b, i] = order.pop()
        slots.append(torch.tensor([int(table[b, i // page]) * page + i % page for i in range(t)], dtype=torch.int64))
    pages = torch.full((n_pages, n_kv, page_bytes(page)), 255, dtype=torch.uint8, device=DEV)
    flat = torch.cat(slots)
    k = _noise(gen, len(flat), n_kv, 128) * torch.exp(_noise(gen, 1, n_kv, 128))
    v = _noise(gen, len(flat), n_kv, 128) * torch.exp(2 * _noise(gen, len(flat), 1, 1))
    paged_kv4_append(pages, flat.to(DEV), k.to(dtype).to(DEV), v.to(dtype).to(DEV))
    return pages, table, slots


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,n_kv,n_q,page,rope", [(1, 1, 1, 16, True), (3, 2, 14, 16, True), (37, 8, 32, 64, True), (64, 3, 3, 48, False), (258, 2, 4, 128, True)])
def test_append_stores_the_plain_quantisers_bytes(dtype, n, n_kv, n_q, page, rope):
    from blockgtq_b200 import page_bytes, paged_kv4_append, paged_kv4_read
    gen = torch.Generator().manual_seed(n)
    n_pages = -(-n // page) + 2
    slots = torch.randperm(n_pages * page, generator=gen)[:n]
    if n == 64:
        slots = torch.arange(n) + 5                       # neighbours, from an odd one on
    if n > 2:
        slots[1] = -1
    k, v, q = (_noise(gen, n, h, 128).to(dtype) for h in (n_kv, n_kv, n_q))
    if n > 30:
        k[2, 0, 32:64] = 0
        v[3, 0, :32] = 3.5
        v[3, 0, 5] = 7.0                                  # x / scale = 3.5: a tie, to the even code
        v[4, n_kv - 1, 7] = math.inf
        v[5, 0, 40] = math.nan
        k[6, 0] *= 1e-6
        k[7, 0] *= 3000
    cos, sin = _tables(300)
    positions = torch.randint(0, 300, (n,), generator=gen)
    background = torch.randint(0, 256, (n_pages, n_kv, page_bytes(page)), generator=gen, dtype=torch.uint8)
    want = background.clone()
    k_in = R.rotated(k, cos, sin, positions) if rope else k.float()
    for i in range(n):
        if slots[i] >= 0:
            R.write(want, int(slots[i]), k_in[i], v[i].float())
    pages = background.to(DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    extra = dict(q=q.to(DEV), cos=cos.to(DEV), sin=sin.to(DEV), positions=positions.to(DEV)) if rope else {}
    got_q = paged_kv4_append(pages, slots.to(DEV), k.to(DEV), v.to(DEV), status=status, **extra)
    assert (pages.cpu() != want).sum() == 0 and status.item() == 0
    if rope:
        assert torch.equal(got_q.cpu(), R.rotated(q, cos, sin, positions).to(dtype))
    else:
        assert got_q is None
    for t in (torch.float16, torch.float32, torch.bfloat16):
        gk, gv = paged_kv4_read(pages, slots.to(DEV), dtype=t)
        there = slots >= 0
        wk, wv, _, _ = R.read(want, slots[there])
        for g, w in ((gk, wk), (gv, wv)):
            assert g.dtype == t and not g.cpu()[~there].any()
            assert torch.equal(g.cpu()[there].nan_to_num(123.0), w.to(t).nan_to_num(123.0))


def test_append_takes_rows_of_any_stride_and_a_layer_of_a_pool():
    from blockgtq_b200 import page_bytes, paged_kv4_append
    gen = torch.Generator().manual_seed(5)
    n, n_kv, n_q = 9, 2, 4
    qkv = _noise(gen, n, n_q + 2 * n_kv, 128).half()
    cos, sin = _tables(50)
    wide = torch.cat([cos, sin], 1).to(DEV)
    pos, slots = torch.arange(n) + 20, torch.arange(n) + 3
    pool = torch.zeros(2, 3, n_kv, page_bytes(16), dtype=torch.uint8, device=DEV)
    dev = qkv.to(DEV)
    q, k, v = dev[:, :n_q], dev[:, n_q:n_q + n_kv], dev[:, n_q + n_kv:]
    got = paged_kv4_append(pool[1], slots.to(DEV), k, v, q=q, cos=wide[:, :64], sin=wide[:, 64:], positions=pos.to(DEV))
    odd = torch.zeros(n, n_kv, 131, dtype=torch.float16, device=DEV)[:, :, 3:]             # rows that no wide load can take
    odd.copy_(v)
    other = torch.zeros_like(pool)
    paged_kv4_append(other[1], slots.to(DEV), k.transpose(0, 1).contiguous().transpose(0, 1), odd, cos=wide[:, :64], sin=wide[:, 64:], positions=pos.to(DEV))
    want = torch.zeros(3, n_kv, page_bytes(16), dtype=torch.uint8)
    kr = R.rotated(qkv[:, n_q:n_q + n_kv], cos, sin, pos)
    for i in range(n):
        R.write(want, int(slots[i]), kr[i], qkv[i, n_q + n_kv:].float())
    assert torch.equal(pool[1].cpu(), want) and torch.equal(other[1].cpu(), want) and not pool[0].any()
    assert torch.equal(got.cpu(), R.rotated(qkv[:, :n_q], cos, sin, pos).half())


def test_slots_and_positions_out_of_range_are_reported_and_store_nothing():
    from blockgtq_b200 import page_bytes, paged_kv4_append, paged_kv4_read
    pages = torch.zeros(2, 1, page_bytes(16), dtype=torch.uint8, device=DEV)
    rows = torch.ones(1, 1, 128, dtype=torch.float16, device=DEV)
    cos, sin = (x.to(DEV) for x in _tables(4))
    def one(slot, position):
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        paged_kv4_append(pages, torch.tensor([slot], device=DEV), rows, rows, cos=cos, sin=sin, positions=torch.tensor([position], device=DEV), status=status)
        return status.item()
    assert one(32, 0) == 2 and one(1 << 40, 0) == 2 and not pages.any()
    assert one(-1, 99) == 0 and not pages.any()
    assert one(0, 4) == 2 and not pages[0, 0, :64].any()          # the key; the value has no angle
    assert one(0, 3) == 0 and pages[0, 0, :64].any()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    k, v = paged_kv4_read(pages, torch.tensor([32, 0], device=DEV), status=status)
    assert status.item() == 2 and not k[0].any() and k[1].any()


FORMS = {"auto": 0, "split": 15, "cluster1": 1, "cluster2": 2, "cluster8": 8}


@pytest.fixture(params=list(FORMS))
def form(request, monkeypatch):
    """The forms that the attention's launch has; the library chooses one by the call's shape."""
    from blockgtq_b200 import paged
    monkeypatch.setattr(paged, "_FORM", FORMS[request.param])


@pytest.fixture(params=[*FORMS, "tcgen05"])
def rows_form(request, monkeypatch):
    from blockgtq_b200 import paged
    monkeypatch.setattr(paged, "_FORM", (FORMS | {"tcgen05": 14})[request.param])


def _check(got, lse, ref, rows):
    out, want_lse, tol, tol_lse = ref
    g = got[rows].double().cpu()
    assert torch.isfinite(g).all()
    off = (g - out).abs()                                     # (a row that sees nothing has a bound of zero)
    assert (off <= tol).all(), ((off - tol).max(), off.max())
    if lse is not None:
        l = lse[rows].double().cpu()
        assert torch.equal(l == -math.inf, want_lse == -math.inf)
        f = torch.isfinite(want_lse)
        assert ((l - want_lse).abs()[f] <= tol_lse[f]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_kv,gqa,page,lens", [
    (1, 1, 16, [1]), (2, 4, 64, [0, 1, 15, 16, 17]), (2, 8, 16, [33, 0, 0, 300]), (1, 7, 48, [500, 31, 32]), (8, 2, 128, [257, 129]),
    (1, 3, 32, [2000]), (4, 1, 64, [63, 64, 65, 640])])
def test_decode_against_64_bits(dtype, n_kv, gqa, page, lens, form):
    from blockgtq_b200 import paged_kv4_decode_attention
    gen = torch.Generator().manual_seed(sum(lens) + gqa)
    pages, table, slots = _case(gen, n_kv, page, lens, dtype=dtype)
    q = (_noise(gen, len(lens), n_kv * gqa, 128) * 1.5).to(dtype)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out, lse = paged_kv4_decode_attention(q.to(DEV), pages, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), return_lse=True, status=status)
    assert status.item() == 0 and out.dtype == dtype
    host = pages.cpu()
    for b, t in enumerate(lens):
        _check(out, lse, R.attention(q[b:b + 1], host, slots[b], [t], 1 / math.sqrt(128)), slice(b, b + 1))


@pytest.mark.parametrize("magnitude", [1e-30, 1e-3, 3e3, 1e30])
def test_decode_of_bf16_queries_of_any_magnitude(magnitude):
    from blockgtq_b200 import paged_kv4_decode_attention
    gen = torch.Generator().manual_seed(3)
    pages, table, slots = _case(gen, 2, 16, [70])
    q = (_noise(gen, 1, 4, 128) * magnitude).bfloat16()
    scale = 0.1 / magnitude
    out, lse = paged_kv4_decode_attention(q.to(DEV), pages, table.to(DEV), torch.tensor([70], dtype=torch.int32, device=DEV), scale=scale, return_lse=True)
    _check(out, lse, R.attention(q, pages.cpu(), slots[0], [70], torch.tensor(scale).item()), slice(0, 1))


def test_decode_of_many_sequences_and_of_one_long_one_cut_between_ctas(form):
    from blockgtq_b200 import paged_kv4_decode_attention
    gen = torch.Generator().manual_seed(11)
    lens = [int(x) for x in torch.randint(0, 40, (700,), generator=gen)]
    lens[350] = 9000
    pages, table, slots = _case(gen, 1, 16, lens)
    q = _noise(gen, len(lens), 2, 128).half()
    out, lse = paged_kv4_decode_attention(q.to(DEV), pages, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), return_lse=True)
    host = pages.cpu()
    for b in [0, 1, 2, 3, 255, 256, 257, 349, 350, 351, 511, 512, 699]:
        _check(out, lse, R.attention(q[b:b + 1], host, slots[b], [lens[b]], 1 / math.sqrt(128)), slice(b, b + 1))


PREFILLS = [
    # n_kv, gqa, page, (tokens, queries) per sequence
    (1, 1, 16, [(1, 1)]), (2, 4, 64, [(5, 5), (70, 3), (16, 16)]), (1, 7, 32, [(40, 9), (0, 0), (33, 33)]), (2, 8, 16, [(130, 1), (131, 40)]),
    (1, 2, 128, [(300, 300)]), (2, 4, 32, [(900, 129), (257, 64)]), (1, 3, 16, [(5, 9), (0, 4), (20, 2)])]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_kv,gqa,page,seqs", PREFILLS)
def test_prefill_against_64_bits(dtype, n_kv, gqa, page, seqs, causal, rows_form):
    from blockgtq_b200 import paged_kv4_prefill_attention
    lens, counts = [t for t, _ in seqs], [n for _, n in seqs]
    gen = torch.Generator().manual_seed(sum(lens) + gqa)
    pages, table, slots = _case(gen, n_kv, page, lens, dtype=dtype)
    n, behind = sum(counts), 3
    q = (_noise(gen, n + behind, n_kv * gqa, 128) * 1.5).to(dtype)
    ends = [sum(counts[:i]) for i in range(len(counts) + 1)]
    out = torch.full((n + behind, n_kv * gqa, 128), 77.0, dtype=dtype, device=DEV)
    got, lse = paged_kv4_prefill_attention(q.to(DEV), pages, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
                                           torch.tensor(ends, dtype=torch.int32, device=DEV), max_q_len=max(counts), max_seq_len=max(lens),
                                           causal=causal, return_lse=True, out=out)
    assert got is out and (out[n:] == 77).all()
    host = pages.cpu()
    for b, (t, m) in enumerate(seqs):
        seen = [t - m + 1 + i if causal else t for i in range(m)]
        _check(out, lse, R.attention(q[ends[b]:ends[b + 1]], host, slots[b], seen, 1 / math.sqrt(128)), slice(ends[b], ends[b + 1]))


@pytest.mark.parametrize("bad", ["-1", "n", "1 << 30"])
def test_a_page_number_outside_the_pool_leaves_its_tokens_out(form, bad):
    from blockgtq_b200 import paged_kv4_decode_attention
    gen = torch.Generator().manual_seed(2)
    pages, table, slots = _case(gen, 1, 16, [40, 40])
    q = _noise(gen, 2, 2, 128).half()
    table[0, 1] = eval(bad, {"n": pages.shape[0]})
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out, lse = paged_kv4_decode_attention(q.to(DEV), pages, table.to(DEV), torch.tensor([40, 40], dtype=torch.int32, device=DEV), return_lse=True, status=status)
    assert status.item() == 4
    left = torch.cat([slots[0][:16], slots[0][32:]])
    _check(out, lse, R.attention(q[:1], pages.cpu(), left, [24], 1 / math.sqrt(128)), slice(0, 1))
    _check(out, lse, R.attention(q[1:], pages.cpu(), slots[1], [40], 1 / math.sqrt(128)), slice(1, 2))


def test_a_page_number_outside_the_pool_in_a_prefill(rows_form):
    from blockgtq_b200 import paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(2)
    pages, table, slots = _case(gen, 2, 16, [200, 150])
    q = _noise(gen, 100, 4, 128).half()
    table[0, 1], table[0, 9], table[0, 12] = -1, pages.shape[0], 1 << 30
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out, lse = paged_kv4_prefill_attention(q.to(DEV), pages, table.to(DEV), torch.tensor([200, 150], dtype=torch.int32, device=DEV),
                                           torch.tensor([0, 60, 100], dtype=torch.int32, device=DEV), return_lse=True, status=status)
    assert status.item() == 4
    keep = torch.tensor([i for i in range(200) if i // 16 not in (1, 9, 12)])
    seen = [int((keep < 141 + i).sum()) for i in range(60)]
    _check(out, lse, R.attention(q[:60], pages.cpu(), slots[0][keep], seen, 1 / math.sqrt(128)), slice(0, 60))
    _check(out, lse, R.attention(q[60:], pages.cpu(), slots[1], [111 + i for i in range(40)], 1 / math.sqrt(128)), slice(60, 100))


def test_more_rows_than_the_caller_said_are_attended_all_the_same(rows_form):
    from blockgtq_b200 import paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(17)
    lens, counts = [700, 90, 300], [40, 7, 1]
    pages, table, slots = _case(gen, 2, 16, lens)
    q = _noise(gen, sum(counts), 8, 128).half()
    ends = [0, 40, 47, 48]
    out, lse = paged_kv4_prefill_attention(q.to(DEV), pages, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
                                           torch.tensor(ends, dtype=torch.int32, device=DEV), max_q_len=2, return_lse=True)
    host = pages.cpu()
    for b, (t, m) in enumerate(zip(lens, counts)):
        _check(out, lse, R.attention(q[ends[b]:ends[b + 1]], host, slots[b], [t - m + 1 + i for i in range(m)], 1 / math.sqrt(128)), slice(ends[b], ends[b + 1]))


def test_a_length_beyond_the_table_is_held_to_it():
    from blockgtq_b200 import paged_kv4_decode_attention
    gen = torch.Generator().manual_seed(2)
    pages, table, slots = _case(gen, 1, 16, [32])
    q = _noise(gen, 1, 2, 128).half()
    for t in (33, 1 << 30, -5):
        n = torch.tensor([t], dtype=torch.int32, device=DEV)
        out, lse = paged_kv4_decode_attention(q.to(DEV), pages, table[:, :2].to(DEV), n, return_lse=True)
        _check(out, lse, R.attention(q, pages.cpu(), slots[0], [min(32, t)], 1 / math.sqrt(128)), slice(0, 1))
        out, lse = paged_kv4_decode_attention(q.to(DEV), pages, table.to(DEV), n, return_lse=True, max_seq_len=20)
        _check(out, lse, R.attention(q, pages.cpu(), slots[0], [min(20, t)], 1 / math.sqrt(128)), slice(0, 1))


def test_no_number_in_a_row_shows_and_in_a_hidden_place_does_not(form):
    from blockgtq_b200 import paged_kv4_append, paged_kv4_decode_attention, paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(9)
    pages, table, slots = _case(gen, 1, 16, [40])
    k, v = (_noise(gen, 1, 1, 128).half() for _ in range(2))
    v[0, 0, 33] = math.nan                                     # group 1 of V of token 39
    paged_kv4_append(pages, slots[0][39:].to(DEV), k.to(DEV), v.to(DEV))
    q = _noise(gen, 4, 2, 128).half().to(DEV)
    def run(t):
        return paged_kv4_decode_attention(q[:1], pages, table.to(DEV), torch.tensor([t], dtype=torch.int32, device=DEV))
    assert torch.isfinite(run(39)).all()
    nan = run(40).isnan()[0]
    assert nan[:, 32:64].all() and not nan[:, :32].any() and not nan[:, 64:].any()
    k[0, 0, 0] = math.nan
    paged_kv4_append(pages, slots[0][39:].to(DEV), k.to(DEV), torch.zeros_like(v).to(DEV))
    assert run(40).isnan().all() and torch.isfinite(run(39)).all()


def test_no_number_in_a_prefill_shows_in_the_rows_that_see_it(rows_form):
    from blockgtq_b200 import paged_kv4_append, paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(9)
    pages, table, slots = _case(gen, 1, 16, [300])
    k, v = (_noise(gen, 2, 1, 128).half() for _ in range(2))
    v[0, 0, 33] = math.nan                                     # group 1 of V of token 251
    k[1, 0, 100] = math.nan                                    # K of token 280
    paged_kv4_append(pages, slots[0][[251, 280]].to(DEV), k.to(DEV), v.to(DEV))
    q = _noise(gen, 70, 2, 128).half().to(DEV)
    out, lse = paged_kv4_prefill_attention(q, pages, table.to(DEV), torch.tensor([300], dtype=torch.int32, device=DEV),
                                           torch.tensor([0, 70], dtype=torch.int32, device=DEV), return_lse=True)
    first = 300 - 70                                           # position of row 0
    nan = out.isnan()
    assert not nan[:251 - first].any() and nan[280 - first:].all() and nan[251 - first:, :, 32:64].all()
    assert not nan[251 - first:280 - first, :, :32].any() and not nan[251 - first:280 - first, :, 64:].any()
    assert torch.isfinite(lse[:280 - first]).all() and lse[280 - first:].isnan().all()


def test_a_key_that_is_no_number_shows_wherever_it_lies_in_a_tile(rows_form):
    from blockgtq_b200 import paged_kv4_append, paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(23)
    pages, table, slots = _case(gen, 1, 16, [160] * 40)
    k, v = _noise(gen, 40, 1, 128).half(), _noise(gen, 40, 1, 128).half()
    k[:, 0, 5] = math.nan
    at = [100 + i for i in range(40)]                          # of sequence i
    paged_kv4_append(pages, torch.stack([slots[i][t] for i, t in enumerate(at)]).to(DEV), k.to(DEV), v.to(DEV))
    q = _noise(gen, 40 * 80, 1, 128).half().to(DEV)
    out = paged_kv4_prefill_attention(q, pages, table.to(DEV), torch.full((40,), 160, dtype=torch.int32, device=DEV),
                                      torch.arange(0, 41 * 80, 80, dtype=torch.int32, device=DEV), max_q_len=80).view(40, 80, 128)
    for i, t in enumerate(at):
        assert torch.isfinite(out[i, :t - 80]).all() and out[i, t - 80:].isnan().all(), i


def test_a_prefill_whose_blocks_are_cut_between_ctas():
    """Few blocks with long contexts beside many short ones, rows that see nothing, and a query of a layer's strided projection."""
    from blockgtq_b200 import paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(29)
    seqs = [(3000, 70), (1, 1), (0, 40), (5, 90), (129, 129)] + [(40 + i, 20) for i in range(30)]
    lens, counts = [t for t, _ in seqs], [n for _, n in seqs]
    pages, table, slots = _case(gen, 2, 64, lens)
    ends = [sum(counts[:i]) for i in range(len(counts) + 1)]
    q = _noise(gen, ends[-1], 10, 128).half()
    out, lse = paged_kv4_prefill_attention(q.to(DEV)[:, 1:7], pages, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
                                           torch.tensor(ends, dtype=torch.int32, device=DEV), return_lse=True)
    host = pages.cpu()
    for b, (t, m) in enumerate(seqs):
        if b < 8 or b == len(seqs) - 1:
            _check(out, lse, R.attention(q[ends[b]:ends[b + 1], 1:7], host, slots[b], [t - m + 1 + i for i in range(m)], 1 / math.sqrt(128)),
                   slice(ends[b], ends[b + 1]))


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scales_of_any_sign(scale, rows_form):
    from blockgtq_b200 import paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(19)
    pages, table, slots = _case(gen, 1, 16, [150])
    q = _noise(gen, 60, 3, 128).half()
    out, lse = paged_kv4_prefill_attention(q.to(DEV), pages, table.to(DEV), torch.tensor([150], dtype=torch.int32, device=DEV),
                                           torch.tensor([0, 60], dtype=torch.int32, device=DEV), return_lse=True, scale=scale)
    _check(out, lse, R.attention(q, pages.cpu(), slots[0], [91 + i for i in range(60)], scale), slice(0, 60))


def test_steps_of_the_cache_from_prompt_to_decode_on_another_stream():
    """Prompts, chunks behind them and single tokens through PagedKV4Cache, sequences coming and going, against 64 bits."""
    from blockgtq_b200 import PagedKV4Cache
    gen = torch.Generator().manual_seed(21)
    L, n_q, n_kv = 2, 4, 2
    cache = PagedKV4Cache(L, n_q, n_kv, n_pages=40, max_seq_len=200, page_size=16, device=DEV)
    cos, sin = _tables(200)
    rope = (cos.to(DEV), sin.to(DEV))
    a, b = cache.add_sequence(), cache.add_sequence()
    stream = torch.cuda.Stream(DEV)
    def step(seqs, counts):
        n = sum(counts)
        cache.begin_step(seqs, counts)
        for layer in range(L):
            q, k, v = (_noise(gen, n, h, 128).half() for h in (n_q, n_kv, n_kv))
            out = cache.append_and_attend(layer, q.to(DEV), k.to(DEV), v.to(DEV), rope=rope)
            at, host = 0, cache.pages[layer].cpu()
            positions = torch.cat([torch.arange(cache.seq_len(s) - c, cache.seq_len(s)) for s, c in zip(seqs, counts)])
            qr = R.rotated(q, cos, sin, positions).half()
            for s, c in zip(seqs, counts):
                t = cache.seq_len(s)
                slots = torch.tensor([cache._seqs[s][1][i // 16] * 16 + i % 16 for i in range(t)])
                _check(out, None, R.attention(qr[at:at + c], host, slots, [t - c + 1 + i for i in range(c)], 1 / math.sqrt(128)), slice(at, at + c))
                at += c
        cache.check_status()
    with torch.cuda.stream(stream):
        step([a, b], [37, 5])
        step([b, a], [1, 1])
        step([a], [20])
        cache.free_sequence(a)
        c = cache.add_sequence()
        step([c, b], [50, 4])
        step([b, c], [1, 1])
    torch.cuda.current_stream().wait_stream(stream)


def test_a_captured_step_follows_the_lengths():
    from blockgtq_b200 import paged_kv4_append, paged_kv4_decode_attention
    gen = torch.Generator().manual_seed(31)
    lens = [60, 7, 0]
    pages, table, slots = _case(gen, 2, 16, [t + 20 for t in lens])
    table, table_dev = table, table.to(DEV)
    cos, sin = _tables(200)
    rope = dict(cos=cos.to(DEV), sin=sin.to(DEV))
    q, k, v = (torch.zeros(3, h, 128, dtype=torch.float16, device=DEV) for h in (8, 2, 2))
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    slot, pos = torch.zeros(3, dtype=torch.int64, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    def layer():
        qr = paged_kv4_append(pages, slot, k, v, q=q, positions=pos, **rope)
        return paged_kv4_decode_attention(qr, pages, table_dev, n, return_lse=True)
    slot.fill_(-1)
    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = layer()
    for i in range(3):
        fresh = [_noise(gen, 3, h, 128).half() for h in (8, 2, 2)]
        for x, y in zip((q, k, v), fresh):
            x.copy_(y)
        pos.copy_(torch.tensor([t + i for t in lens]))
        slot.copy_(torch.tensor([int(slots[b][t + i]) for b, t in enumerate(lens)]))
        n.copy_(torch.tensor([t + i + 1 for t in lens], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        host, qr = pages.cpu(), R.rotated(fresh[0], cos, sin, pos.cpu()).half()
        for b, t in enumerate(lens):
            _check(out, lse, R.attention(qr[b:b + 1], host, slots[b], [t + i + 1], 1 / math.sqrt(128)), slice(b, b + 1))


def test_results_do_not_change_from_call_to_call():
    from blockgtq_b200 import paged_kv4_decode_attention
    gen = torch.Generator().manual_seed(41)
    lens = [1500, 3, 900]
    pages, table, _ = _case(gen, 2, 16, lens)
    q = _noise(gen, 3, 8, 128).half().to(DEV)
    args = (q, pages, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))
    first = paged_kv4_decode_attention(*args)
    for _ in range(5):
        assert torch.equal(first, paged_kv4_decode_attention(*args))


@pytest.mark.parametrize("dtype", TYPES)
def test_one_token_with_all_the_weight_gives_its_values_as_they_are(dtype, form):
    """Its weight times its scale is exact, the sum over its weight is code x scale within a few steps of fp32.  That product has 11 bits: fp16
    holds it, so fp16 is equal.  bf16 rounds it, from a sum that may lie 2^-22 beside a tie: within half a step and that.
    In the second sequence the other tokens' logits lie at least 40 (in powers of two) below it."""
    from blockgtq_b200 import paged_kv4_append, paged_kv4_decode_attention, paged_kv4_read
    gen = torch.Generator().manual_seed(5)
    pages, table, slots = _case(gen, 2, 16, [1, 70], dtype=dtype)
    v = _noise(gen, 70, 2, 128).to(dtype)
    k = torch.full((70, 2, 128), -7.0).to(dtype)
    k[37] = 7.0
    paged_kv4_append(pages, slots[1].to(DEV), k.to(DEV), v.to(DEV))
    paged_kv4_append(pages, slots[0].to(DEV), k[:1].to(DEV), v[5:6].to(DEV))
    q = torch.ones(2, 14, 128).to(dtype).to(DEV)
    out = paged_kv4_decode_attention(q, pages, table.to(DEV), torch.tensor([1, 70], dtype=torch.int32, device=DEV))
    for b, t in ((0, 0), (1, 37)):
        want = paged_kv4_read(pages, slots[b][t:t + 1].to(DEV), dtype=torch.float16)[1][0].double().repeat_interleave(7, 0)
        slack = 0 if dtype == torch.float16 else 2 ** -8 + 2 ** -20
        assert bool(((out[b].double() - want).abs() <= slack * want.abs()).all())


@pytest.mark.parametrize("n", [6, 5000])
def test_a_token_without_an_angle_is_not_stored_at_all(n):
    from blockgtq_b200 import page_bytes, paged_kv4_append
    gen = torch.Generator().manual_seed(n)
    n_pages = n // 64 + 1
    k, v = (_noise(gen, n, 4, 128).half().to(DEV) for _ in range(2))
    cos, sin = (x.to(DEV) for x in _tables(n))
    slots, pos = torch.arange(n, device=DEV), torch.arange(n, device=DEV)
    bad = torch.tensor([1, n - 2], device=DEV)
    pos[bad] = torch.tensor([n, -1], device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got, want = (torch.zeros(n_pages, 4, page_bytes(64), dtype=torch.uint8, device=DEV) for _ in range(2))
    paged_kv4_append(got, slots, k, v, cos=cos, sin=sin, positions=pos, status=status)
    assert status.item() == 2
    status.zero_()
    slots[bad] = -1
    paged_kv4_append(want, slots, k, v, cos=cos, sin=sin, positions=pos, status=status)
    assert status.item() == 0 and torch.equal(got, want)


def test_tables_of_any_stride(rows_form):
    from blockgtq_b200 import paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(8)
    pages, table, slots = _case(gen, 2, 16, [70, 33])
    q = _noise(gen, 20, 8, 128).half()
    i32 = dict(dtype=torch.int32, device=DEV)
    lens, cu = torch.tensor([70, 9, 33, 9], **i32)[::2], torch.tensor([0, 9, 12, 9, 20, 9], **i32)[::2]
    wide = torch.zeros(2, table.shape[1] + 3, **i32)
    wide[:, 2:-1] = table
    for tab in (wide[:, 2:-1], table.to(DEV).t().contiguous().t()):
        out, lse = paged_kv4_prefill_attention(q.to(DEV), pages, tab, lens, cu, return_lse=True)
        for b, (a, z, t) in enumerate([(0, 12, 70), (12, 20, 33)]):
            _check(out, lse, R.attention(q[a:z], pages.cpu(), slots[b], [t - z + a + 1 + i for i in range(z - a)], 1 / math.sqrt(128)), slice(a, z))


def test_pages_behind_four_gigabytes(rows_form):
    """A pool of 5 GB whose heads are 2.4 GB apart: pages on both sides of 2^32 bytes."""
    from blockgtq_b200 import page_bytes, paged_kv4_append, paged_kv4_prefill_attention, paged_kv4_read
    gen = torch.Generator().manual_seed(9)
    n_pages, t = 1 << 20, 150
    pages = torch.empty(2, n_pages, page_bytes(16), dtype=torch.uint8, device=DEV).transpose(0, 1)
    order = [n_pages - 1 - 97 * i for i in range(5)] + [3 * i for i in range(5)]
    slots = torch.tensor([order[i // 16] * 16 + i % 16 for i in range(t)])
    k, v, q = (_noise(gen, t, h, 128).half() for h in (2, 2, 4))
    paged_kv4_append(pages, slots.to(DEV), k.to(DEV), v.to(DEV))
    small = torch.zeros(10, 2, page_bytes(16), dtype=torch.uint8)
    for i, p in enumerate(order):
        small[i] = pages[p].cpu()
    here = torch.arange(t)
    ref = R.attention(q[:20], small, here, [t - 19 + i for i in range(20)], 1 / math.sqrt(128))
    i32 = dict(dtype=torch.int32, device=DEV)
    out, lse = paged_kv4_prefill_attention(q[:20].to(DEV), pages, torch.tensor([order], **i32), torch.tensor([t], **i32), torch.tensor([0, 20], **i32), return_lse=True)
    _check(out, lse, ref, slice(0, 20))
    for far, near in zip(paged_kv4_read(pages, slots.to(DEV)), paged_kv4_read(small.to(DEV), here.to(DEV))):
        assert torch.equal(far, near)


def test_two_graphs_of_one_pool_of_memory(rows_form):
    """Their workspaces may be the same memory: replayed in turn, each gives its own results."""
    from blockgtq_b200 import paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(12)
    pages, table, slots = _case(gen, 2, 16, [900, 300])
    i32 = dict(dtype=torch.int32, device=DEV)
    cases, graphs, pool = [(0, 900, 40), (1, 300, 290)], [], None
    for b, t, n in cases:
        q = _noise(gen, n, 4, 128).half()
        args = (q.to(DEV), pages, table[b:b + 1].to(DEV), torch.tensor([t], **i32), torch.tensor([0, n], **i32))
        paged_kv4_prefill_attention(*args)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            out = paged_kv4_prefill_attention(*args)
        pool = g.pool()
        want = R.attention(q, pages.cpu(), slots[b], [t - n + 1 + i for i in range(n)], 1 / math.sqrt(128))
        graphs.append((g, out, args, want, n))
    for which in (0, 1, 1, 0, 1, 0):
        g, out, _, want, n = graphs[which]
        g.replay()
        torch.cuda.synchronize()
        _check(out, None, want, slice(0, n))


@pytest.mark.parametrize("form", [1, 8, 14, 15])
def test_the_library_reads_no_further_than_the_table(form):
    """Lengths and max_tokens beyond the table's width: a row of it is not left."""
    from blockgtq_b200 import _lib
    gen = torch.Generator().manual_seed(14)
    pages, table, slots = _case(gen, 2, 16, [48, 48])
    i32 = dict(dtype=torch.int32, device=DEV)
    wide = torch.full((2, 40), -1, **i32)                 # what lies behind a row would be reported
    wide[:, :3] = table[:, :3].to(DEV)
    q = _noise(gen, 10, 4, 128).half()
    qd, out, status = q.to(DEV), torch.zeros(10, 4, 128, dtype=torch.float16, device=DEV), torch.zeros(1, **i32)
    lens, cu = torch.tensor([400, 48], **i32), torch.tensor([0, 6, 10], **i32)
    flags, lib = _lib.PAGED_CAUSAL | form << _lib.PAGED_FORM_SHIFT, _lib.lib()
    need = lib.bgtq_paged_workspace_bytes(2, 10, 4, 2, 6, 500, flags)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    rc = lib.bgtq_paged_attend(qd.data_ptr(), 512, 128, pages.data_ptr(), pages.stride(0), pages.stride(1), pages.shape[0], 16, wide.data_ptr(), 40, 3,
                               lens.data_ptr(), cu.data_ptr(), 2, 10, 4, 2, 6, 500, 1 / math.sqrt(128), flags, ws.data_ptr(), need, out.data_ptr(), 512, 128,
                               0, status.data_ptr(), _lib.stream_ptr(torch.device(DEV)))
    torch.cuda.synchronize()
    assert rc == 0 and status.item() == 0
    for b, (a, z) in enumerate([(0, 6), (6, 10)]):
        _check(out, None, R.attention(q[a:z], pages.cpu(), slots[b], [48 - z + a + 1 + i for i in range(z - a)], 1 / math.sqrt(128)), slice(a, z))


@pytest.mark.parametrize("n_kv,lens", [(3, [70001, 41, 33000, 0, 12345]), (1, [120000])])
def test_long_sequences_whose_shares_end_inside_a_round(n_kv, lens, monkeypatch):
    """Shares of odd numbers of batches, and more partials of a triple than are merged in one pass."""
    from blockgtq_b200 import paged, paged_kv4_decode_attention
    monkeypatch.setattr(paged, "_FORM", FORMS["split"])
    gen = torch.Generator().manual_seed(len(lens))
    pages, table, slots = _case(gen, n_kv, 64, lens)
    q = (_noise(gen, len(lens), n_kv, 128) * 3).half()
    out, lse = paged_kv4_decode_attention(q.to(DEV), pages, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), return_lse=True)
    host = pages.cpu()
    for b, t in enumerate(lens):
        _check(out, lse, R.attention(q[b:b + 1], host, slots[b], [t], 1 / math.sqrt(128)), slice(b, b + 1))


def test_calls_on_two_streams_at_once():
    from blockgtq_b200 import paged_kv4_decode_attention, paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(51)
    i32 = dict(dtype=torch.int32, device=DEV)
    lens = [5000, 17, 2600]
    pages, table, _ = _case(gen, 2, 16, lens)
    q, rows = (_noise(gen, n, 8, 128).half().to(DEV) for n in (3, 900))
    args = pages, table.to(DEV), torch.tensor(lens, **i32)
    cu = torch.tensor([0, 400, 417, 900], **i32)
    want = paged_kv4_decode_attention(q, *args), paged_kv4_prefill_attention(rows, *args, cu)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(DEV) for _ in range(2)], ([], [])
    for _ in range(10):
        with torch.cuda.stream(streams[0]):
            got[0].append(paged_kv4_decode_attention(q, *args))
        with torch.cuda.stream(streams[1]):
            got[1].append(paged_kv4_prefill_attention(rows, *args, cu))
    torch.cuda.synchronize()
    for results, w in zip(got, want):
        assert all(torch.equal(r, w) for r in results)
