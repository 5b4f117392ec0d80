"""GPU: attention over the paged cache with capped logits, biases by distance, windows and prefixes, against 64 bits."""
import math

import pytest
import torch

import paged_bounds as W
import paged_scores as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I32 = dict(dtype=torch.int32, device=DEV)
FORMS = {"auto": 0, "split": 15, "cluster1": 1, "cluster2": 2, "cluster8": 8}
TYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(params=list(FORMS))
def form(request, monkeypatch):
    """The forms that the attention's launch has; the library chooses one by the call's shape."""
    from blockgtq_b200 import paged
    monkeypatch.setattr(paged, "_FORM", FORMS[request.param])


@pytest.fixture(params=[*FORMS, "tcgen05"])
def rows_form(request, monkeypatch):
    from blockgtq_b200 import paged
    monkeypatch.setattr(paged, "_FORM", (FORMS | {"tcgen05": 14})[request.param])


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
        at = torch.arange(t)
        slots.append(table[b].long()[at // page] * page + at % page)
    pages = torch.full((n_pages, n_kv, page_bytes(page)), 255, dtype=torch.uint8, device=DEV)
    flat = torch.cat(slots)
    k = _noise(gen, len(flat), n_kv, 128) * torch.exp(_noise(gen, 1, n_kv, 128))
    v = _noise(gen, len(flat), n_kv, 128) * torch.exp(2 * _noise(gen, len(flat), 1, 1))
    paged_kv4_append(pages, flat.to(DEV), k.to(dtype).to(DEV), v.to(dtype).to(DEV))
    return pages, table, slots


def _slopes(n_q):
    return 2.0 ** (-8.0 * torch.arange(1, n_q + 1) / n_q)


# what each layer does beside plain attention; prefixes are per sequence, taken in turn
SCORES = {
    "cap": dict(softcap=30.0),
    "low cap": dict(softcap=1.5),
    "slopes": dict(slopes=True),
    "window": dict(window=40),
    "one token": dict(window=1),
    "sinks": dict(window=200, prefix=(4, 4, 4)),
    "prefix": dict(prefix=(70, 0, 1000)),
    "all": dict(softcap=5.0, slopes=True, window=100, prefix=(33, 5, 0)),
    "wide": dict(window=1 << 31, slopes=True),
}


def _arguments(scores, lens, n_q, longest=None):
    """Keywords of the call, and of the definition for sequence b."""
    slopes = _slopes(n_q) if scores.get("slopes") else None
    prefix = [scores["prefix"][b % 3] for b in range(len(lens))] if "prefix" in scores else None
    call = dict(softcap=scores.get("softcap"), window=scores.get("window"), slopes=None if slopes is None else slopes.to(DEV),
                prefix_lens=None if prefix is None else torch.tensor(prefix, **I32), max_prefix_len=longest)
    def of(b):
        p = 0 if prefix is None else min(prefix[b], lens[b], prefix[b] if longest is None else longest)
        return dict(softcap=scores.get("softcap"), window=scores.get("window"), slopes=slopes, prefix=p)
    return call, of


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scores", list(SCORES))
@pytest.mark.parametrize("n_kv,gqa,page,lens", [(2, 4, 16, [1, 0, 33, 700]), (1, 8, 64, [2500, 64]), (8, 1, 32, [31, 300, 32, 1])])
def test_decode_against_64_bits(dtype, scores, n_kv, gqa, page, lens, form):
    from blockgtq_b200 import paged_kv4_decode_attention
    gen = torch.Generator().manual_seed(len(lens))
    pages, table, slots = _case(gen, n_kv, page, lens, dtype=dtype)
    q = (_noise(gen, len(lens), n_kv * gqa, 128) * 2).to(dtype)
    call, of = _arguments(SCORES[scores], lens, n_kv * gqa)
    status = torch.zeros(1, **I32)
    out, lse = paged_kv4_decode_attention(q.to(DEV), pages, table.to(DEV), torch.tensor(lens, **I32), return_lse=True, status=status, **call)
    assert status.item() == 0
    for b in range(len(lens)):
        W.check(out, lse, S.attention(q[b:b + 1], pages, slots[b], **of(b)), slice(b, b + 1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scores,causal", [(s, c) for s in SCORES for c in (True, False) if c or "window" not in SCORES[s]])       # (windows are causal)
@pytest.mark.parametrize("n_kv,gqa,page,seqs", [(2, 4, 16, [(1, 1), (40, 3), (33, 0), (700, 2)]), (1, 8, 64, [(400, 130), (5, 9), (1100, 1)]),
                                                (2, 3, 32, [(333, 300), (0, 4), (129, 129)])])
def test_prefill_against_64_bits(dtype, scores, causal, n_kv, gqa, page, seqs, rows_form):
    """(tokens, queries) of each sequence; queries beyond the tokens see what a row in front of the sequence sees: the prefix."""
    from blockgtq_b200 import paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(len(seqs))
    lens, counts = [t for t, _ in seqs], [n for _, n in seqs]
    pages, table, slots = _case(gen, n_kv, page, lens, dtype=dtype)
    n = sum(counts)
    q = (_noise(gen, n + 2, n_kv * gqa, 128) * 2).to(dtype)
    ends = [0]
    for c in counts:
        ends.append(ends[-1] + c)
    call, of = _arguments(SCORES[scores], lens, n_kv * gqa)
    status, before = torch.zeros(1, **I32), torch.full(q.shape, 7.0, dtype=dtype, device=DEV)
    out, lse = paged_kv4_prefill_attention(q.to(DEV), pages, table.to(DEV), torch.tensor(lens, **I32), torch.tensor(ends, **I32), max_q_len=max(counts),
                                           causal=causal, return_lse=True, status=status, out=before, **call)
    assert status.item() == 0 and (out[n:] == 7.0).all()
    for b, (t, c) in enumerate(seqs):
        rows = sorted({*range(min(c, 3)), *range(0, c, 37), *range(max(0, c - 3), c)})
        if rows:
            ref = S.attention(q[ends[b]:ends[b + 1]], pages, slots[b], rows=rows, causal=causal, **of(b))
            W.check(out, lse, ref, [ends[b] + r for r in rows])


@pytest.mark.parametrize("window,prefix,longest", [(1000, 4, None), (1000, 4, 4), (1000, 1300, 64), (257, 0, None), (4096, 4, 4), (64, 4095, None)])
def test_a_window_over_long_sequences(window, prefix, longest, form):
    """Batches between the prefix and the window are not in the list of work: shares, merging and ragged starts."""
    from blockgtq_b200 import paged_kv4_decode_attention
    gen = torch.Generator().manual_seed(window)
    lens = [5000, 0, 4097, 12000, 999, 1000, 1001, 8224, 37]
    pages, table, slots = _case(gen, 2, 32, lens)
    q = _noise(gen, len(lens), 8, 128).half()
    scores = dict(window=window, prefix=(prefix,) * 3) if prefix else dict(window=window)
    call, of = _arguments(scores, lens, 8, longest)
    out, lse = paged_kv4_decode_attention(q.to(DEV), pages, table.to(DEV), torch.tensor(lens, **I32), return_lse=True, **call)
    for b in range(len(lens)):
        W.check(out, lse, S.attention(q[b:b + 1], pages, slots[b], **of(b)), slice(b, b + 1))


@pytest.mark.parametrize("scores", ["sinks", "all", "cap"])
def test_more_sequences_than_a_warp_looks_over(scores, form):
    from blockgtq_b200 import paged_kv4_decode_attention
    gen = torch.Generator().manual_seed(17)
    lens = [(37 * i) % 400 for i in range(150)]
    pages, table, slots = _case(gen, 1, 16, lens)
    q = _noise(gen, len(lens), 4, 128).half()
    call, of = _arguments(SCORES[scores], lens, 4)
    out, lse = paged_kv4_decode_attention(q.to(DEV), pages, table.to(DEV), torch.tensor(lens, **I32), return_lse=True, **call)
    for b in range(0, 150, 7):
        W.check(out, lse, S.attention(q[b:b + 1], pages, slots[b], **of(b)), slice(b, b + 1))


@pytest.mark.parametrize("scores", ["cap", "sinks", "all", "prefix", "slopes"])
def test_a_long_prefill_whose_blocks_are_cut_between_ctas(scores, monkeypatch):
    from blockgtq_b200 import paged, paged_kv4_prefill_attention
    monkeypatch.setattr(paged, "_FORM", 14)
    gen = torch.Generator().manual_seed(23)
    lens, counts = [5000, 2300], [1500, 2300]
    pages, table, slots = _case(gen, 2, 64, lens)
    q = _noise(gen, sum(counts), 8, 128).half()
    call, of = _arguments(SCORES[scores], lens, 8)
    ends = [0, 1500, 3800]
    out, lse = paged_kv4_prefill_attention(q.to(DEV), pages, table.to(DEV), torch.tensor(lens, **I32), torch.tensor(ends, **I32), return_lse=True, **call)
    for b in range(2):
        rows = sorted({0, 1, 63, 64, 255, 256, 700, 1024, 1337, counts[b] - 1})
        W.check(out, lse, S.attention(q[ends[b]:ends[b + 1]], pages, slots[b], rows=rows, **of(b)), [ends[b] + r for r in rows])


@pytest.mark.parametrize("where,seen", [(3, True), (50, False), (99, False), (100, True), (139, True)])
@pytest.mark.parametrize("what", ["k", "v"])
def test_no_number_shows_in_the_rows_that_see_it_only(where, seen, what, rows_form):
    """140 tokens, a window of 40, a prefix of 4: the last row sees tokens 0 to 3 and 100 to 139."""
    from blockgtq_b200 import paged_kv4_append, paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(where)
    pages, table, slots = _case(gen, 1, 16, [140])
    k, v = (_noise(gen, 1, 1, 128).half() for _ in range(2))
    (k if what == "k" else v)[0, 0, 70] = math.nan
    paged_kv4_append(pages, slots[0][where:where + 1].to(DEV), k.to(DEV), v.to(DEV))
    for n in (1, 3, 90):
        q = _noise(gen, n, 8, 128).half().to(DEV)
        args = (pages, table.to(DEV), torch.tensor([140], **I32), torch.tensor([0, n], **I32))
        for extra in (dict(softcap=30.0), dict(), dict(slopes=_slopes(8).to(DEV))):
            out = paged_kv4_prefill_attention(q, *args, window=40, prefix_lens=torch.tensor([4], **I32), **extra)
            for row in range(n):
                hit = bool(S.seen_by(140, n, row, 40, 4)[where])
                if row == n - 1:
                    assert hit == seen
                got = out[row].isnan()
                if what == "k":
                    assert got.all() if hit else not got.any()
                else:
                    assert got[:, 64:96].all() == hit and not got[:, :64].any() and not got[:, 96:].any()
                    assert hit or not got.any()


def test_a_cap_of_any_size_and_logits_beyond_it(rows_form):
    from blockgtq_b200 import paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(2)
    pages, table, slots = _case(gen, 1, 16, [200])
    args = (pages, table.to(DEV), torch.tensor([200], **I32), torch.tensor([0, 5], **I32))
    for dtype, scale in ((torch.float16, 0.1), (torch.bfloat16, 0.1), (torch.float16, 100.0), (torch.float16, -3.0), (torch.float16, 0.0)):
        q = _noise(gen, 5, 4, 128).to(dtype)
        for cap in (2.0 ** -64, 1e-3, 1.0, 60.0, 1e4, 2.0 ** 64):
            out, lse = paged_kv4_prefill_attention(q.to(DEV), *args, scale=scale, return_lse=True, softcap=cap)
            W.check(out, lse, S.attention(q, pages, slots[0], scale=scale, softcap=cap), slice(0, 5))
    # queries of every magnitude, and keys of zeros: logits are none of fp32's, or nothing at all
    from blockgtq_b200 import paged_kv4_append
    zero = torch.zeros(40, 1, 128, dtype=torch.float16, device=DEV)
    paged_kv4_append(pages, slots[0][20:60].to(DEV), zero, zero)
    for scale in (1e30, 1.0, 1e-30):
        for cap in (2.0 ** -64, 1.0, 2.0 ** 64):
            for top in (3e38, 1.0, 1e-38):
                q = (_noise(gen, 5, 4, 128).sign() * top).bfloat16()
                q[1] = 0
                out, lse = paged_kv4_prefill_attention(q.to(DEV), *args, scale=scale, return_lse=True, softcap=cap)
                k, v = (x.cpu() for x in S.read(pages, slots[0]))
                y = cap * torch.tanh(torch.einsum("nhd,td->nht", q.double(), k[:, 0]) * scale / cap)
                for row in range(5):
                    # a logit is off by 2^-20 of its terms' magnitudes, and the sum by what its largest ones are
                    want = torch.logsumexp(y[row, :, :196 + row], -1)
                    size = torch.einsum("hd,td->ht", q[row].double().abs(), k[:196 + row, 0].abs()) * scale
                    off = 2.0 ** -20 * (torch.minimum(size, torch.tensor(cap, dtype=torch.float64)).amax(-1) + want.abs() + 1) + 1e-5
                    assert torch.isfinite(out[row]).all() and ((lse[row].double().cpu() - want).abs() <= off).all(), (scale, cap, top, row)
    # logits far beyond fp32's range end at the cap
    q = torch.full((5, 4, 128), 3e38, dtype=torch.bfloat16)
    out, lse = paged_kv4_prefill_attention(q.to(DEV), *args, return_lse=True, softcap=20.0)
    assert torch.isfinite(out).all() and (lse <= 20.0 + math.log(200) + 1e-3).all()


def _near(got, p, v, off):
    """got (h, 128) fp16 is p (h, t) times v (t, 128), each logit off by off (h,): weights and results are rounded to fp16, sums cut as in tests/paged_bounds.py."""
    room = (2 * off[:, None] + 2.0 ** -10 + (len(v) / 16 + 32) * 18 * 2.0 ** -24) * (p @ v.abs()) + 2.0 ** -32 * v.abs().sum(0) + 2.0 ** -25
    assert ((got - p @ v).abs() <= room).all(), ((got - p @ v).abs() / room).max()


@pytest.mark.parametrize("cap", [2.0 ** 64, 1e9, 1e6, 50.0, None])
@pytest.mark.parametrize("scale", [1e-38, 1.0, 2.0 ** 20, 2.0 ** 24, 2.0 ** 30])
def test_logits_that_grow_along_a_sequence(cap, scale, rows_form):
    """Keys k_t = (1 + t / 64) k in steps that 4 bits hold: references follow, whatever the size of a step in fp32, and the weights stay finite and at most one.
    Row i sees the tokens of its window; where one logit is far above the others, its value is the result."""
    from blockgtq_b200 import page_bytes, paged_kv4_append, paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(3)
    t, n = 700, 300
    pages, slots = torch.zeros(44, 1, page_bytes(16), dtype=torch.uint8, device=DEV), torch.arange(t, device=DEV)
    k = torch.zeros(t, 1, 128)
    k[:, 0, 0] = 7.0 * (1 + torch.arange(t) // 64)                        # one code, bf16 scales: exact
    v = _noise(gen, t, 1, 128)
    paged_kv4_append(pages, slots, k.half().to(DEV), v.half().to(DEV))
    q = torch.zeros(n, 4, 128)
    q[:, :, 0] = torch.tensor([1.0, 2.0, -1.0, 0.5])
    for window in (None, 90):
        out, lse = paged_kv4_prefill_attention(q.half().to(DEV), pages, torch.arange(44, **I32)[None], torch.tensor([t], **I32), torch.tensor([0, n], **I32), scale=scale,
                                               return_lse=True, softcap=cap, window=window)
        ks, vs = (x.cpu()[:, 0] for x in S.read(pages, slots))
        for row in (0, 1, 63, 64, 150, 299):
            seen = S.seen_by(t, n, row, window)
            x = torch.einsum("hd,td->ht", q[row].double(), ks[seen]) * scale
            y = x if cap is None else cap * torch.tanh(x / cap)
            want = torch.logsumexp(y, -1)
            # products are exact here: a cap's 2^-20, its base's and the reference's 2^-22, the sum's
            off = 2.0 ** -20 * (y.abs().amax(-1) + want.abs()) + 1e-5
            assert ((lse[row].double().cpu() - want).abs() <= off).all(), (row, lse[row], want)
            got = out[row].double().cpu()
            assert torch.isfinite(got).all() and (got.abs() <= vs[seen].abs().amax(0) * 1.01).all()
            few = off < 1e-3
            _near(got[few], torch.softmax(y, -1)[few], vs[seen], off[few])


def test_scores_that_change_nothing_change_no_bit(rows_form):
    from blockgtq_b200 import paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(8)
    pages, table, _ = _case(gen, 2, 32, [300, 77])
    q = _noise(gen, 60, 8, 128).half().to(DEV)
    args = (pages, table.to(DEV), torch.tensor([300, 77], **I32), torch.tensor([0, 50, 60], **I32))
    want = paged_kv4_prefill_attention(q, *args)
    assert torch.equal(paged_kv4_prefill_attention(q, *args, window=400), want)
    assert torch.equal(paged_kv4_prefill_attention(q, *args, prefix_lens=torch.tensor([9, 9], **I32), max_prefix_len=0), want)
    # a prefix that every row sees anyhow
    near = paged_kv4_prefill_attention(q, *args, prefix_lens=torch.tensor([100, -3], **I32))
    assert (near - want).abs().max() <= 2.0 ** -9 * want.abs().max()


def test_tensors_of_any_layout_and_counted_launches(rows_form):
    from blockgtq_b200 import _lib, paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(11)
    pages, table, slots = _case(gen, 2, 16, [90, 333])
    q = _noise(gen, 20, 8, 128).half()
    call, of = _arguments(SCORES["all"], [90, 333], 8)
    args = (pages, table.to(DEV), torch.tensor([90, 333], **I32), torch.tensor([0, 7, 20], **I32))
    before = _lib.launches
    want = paged_kv4_prefill_attention(q.to(DEV), *args, **call)
    made = _lib.launches - before
    odd = torch.zeros(20, 8, 129, dtype=torch.float16, device=DEV)[:, :, 1:]
    odd.copy_(q)
    wide = dict(call, slopes=call["slopes"].repeat_interleave(2)[::2], prefix_lens=call["prefix_lens"].repeat_interleave(3)[::3])
    assert torch.equal(paged_kv4_prefill_attention(odd, *args, **wide), want)
    assert _lib.launches - before == 2 * made
    for b, (lo, hi) in enumerate(((0, 7), (7, 20))):
        W.check(want, None, S.attention(q[lo:hi], pages, slots[b], **of(b)), slice(lo, hi))


def test_pages_in_front_of_the_window_need_not_be_there(form):
    """Their numbers in the table are those of no page, and nothing is reported."""
    from blockgtq_b200 import paged_kv4_decode_attention
    gen = torch.Generator().manual_seed(31)
    pages, table, slots = _case(gen, 2, 16, [3000])
    q = _noise(gen, 1, 8, 128).half()
    want = S.attention(q, pages, slots[0], window=500, prefix=20)
    table[0, 4:150] = 1 << 30                                    # tokens 64 to 2399; the window's first batch begins at 2496
    status = torch.zeros(1, **I32)
    out, lse = paged_kv4_decode_attention(q.to(DEV), pages, table.to(DEV), torch.tensor([3000], **I32), return_lse=True, status=status, window=500,
                                          prefix_lens=torch.tensor([20], **I32))
    assert status.item() == 0
    W.check(out, lse, want, slice(0, 1))


@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("rows", [1, 5])
def test_pages_that_no_row_sees_a_token_of(page, rows, rows_form):
    """Wherever the window begins in a page, a batch or a tile: what is hidden as a whole has no number, all else is read."""
    from blockgtq_b200 import paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(page)
    pages, table, slots = _case(gen, 1, page, [500])
    q = _noise(gen, rows, 4, 128).half()
    for window in (1, 15, 16, 17, 31, 33, 47, 100, 127, 129, 200, 333):
        for prefix in (0, 1, 16, 40):
            status, part = torch.zeros(1, **I32), table.clone()
            first = 500 - rows + 1 - window                      # the first row's window
            for i in range(500 // page + 1):
                if i * page >= prefix and (i + 1) * page <= first:
                    part[0, i] = -1
            kw = dict(window=window, prefix_lens=torch.tensor([prefix], **I32))
            args = torch.tensor([500], **I32), torch.tensor([0, rows], **I32)
            want = paged_kv4_prefill_attention(q.to(DEV), pages, table.to(DEV), *args, **kw)
            got = paged_kv4_prefill_attention(q.to(DEV), pages, part.to(DEV), *args, status=status, **kw)
            assert status.item() == 0 and torch.equal(got, want)


@pytest.mark.parametrize("scores", ["window", "sinks", "all"])
@pytest.mark.parametrize("longest", [None, 50])
def test_a_window_far_into_long_sequences_needs_little_room(scores, longest, monkeypatch):
    """The workspace holds the tiles of prefixes and windows, one behind the other: rows of sequences far longer, wherever their windows begin in a tile."""
    from blockgtq_b200 import _lib, paged, paged_kv4_prefill_attention
    monkeypatch.setattr(paged, "_FORM", 14)
    gen = torch.Generator().manual_seed(53)
    lens, counts = [9000, 4096, 130, 5003, 0, 6400], [70, 1, 130, 300, 3, 64]
    pages, table, slots = _case(gen, 1, 64, lens)
    q = _noise(gen, sum(counts), 4, 128).half()
    call, of = _arguments(SCORES[scores], lens, 4, longest)
    ends = [0]
    for c in counts:
        ends.append(ends[-1] + c)
    status = torch.zeros(1, **I32)
    out, lse = paged_kv4_prefill_attention(q.to(DEV), pages, table.to(DEV), torch.tensor(lens, **I32), torch.tensor(ends, **I32), return_lse=True, status=status, **call)
    assert status.item() == 0
    for b, c in enumerate(counts):
        rows = sorted({0, c // 2, c - 1})
        W.check(out, lse, S.attention(q[ends[b]:ends[b + 1]], pages, slots[b], rows=rows, **of(b)), [ends[b] + r for r in rows])
    def room(window):
        sc = _lib.PagedScores(None, None, 0.0, window, 0, 0)
        return _lib.lib().bgtq_paged_scored_workspace_bytes(2, 512, 32, 8, 256, 131072, _lib.PAGED_CAUSAL | 14 << 8, sc)
    assert room(4096) < room(0) / 10


def test_a_captured_call_follows_lengths_prefixes_and_slopes(rows_form):
    from blockgtq_b200 import paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(41)
    pages, table, slots = _case(gen, 1, 16, [400, 260])
    q = _noise(gen, 30, 4, 128).half()
    lens, cu, prefix, slopes = torch.tensor([300, 100], **I32), torch.tensor([0, 4, 30], **I32), torch.tensor([0, 9], **I32), torch.zeros(4, device=DEV)
    dev_q, dev_table = q.to(DEV), table.to(DEV)
    def call():
        return paged_kv4_prefill_attention(dev_q, pages, dev_table, lens, cu, return_lse=True, softcap=9.0, window=64, prefix_lens=prefix, slopes=slopes)
    call()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream(DEV)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out, lse = call()
    for (a, b), p, s in (((300, 100), (0, 9), 0.0), ((400, 260), (77, 260), 0.3), ((5, 33), (0, 0), 1.0)):
        lens.copy_(torch.tensor([a, b], **I32))
        prefix.copy_(torch.tensor(p, **I32))
        slopes.fill_(s)
        graph.replay()
        for i, (t, lo, hi) in enumerate(((a, 0, 4), (b, 4, 30))):
            ref = S.attention(q[lo:hi], pages, slots[i][:t], softcap=9.0, window=64, prefix=min(p[i], t), slopes=torch.full((4,), s))
            W.check(out, lse, ref, slice(lo, hi))


@pytest.mark.parametrize("scores", ["window", "sinks", "all", "slopes"])
def test_more_rows_and_longer_sequences_than_the_caller_said(scores, rows_form):
    """max_q_len and max_prefix_len choose the launch; lengths are held to max_seq_len, prefixes to max_prefix_len."""
    from blockgtq_b200 import paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(19)
    pages, table, slots = _case(gen, 2, 16, [600, 90])
    q = _noise(gen, 130, 8, 128).half()
    call, of = _arguments(SCORES[scores], [500, 90], 8, 20 if "prefix" in SCORES[scores] else None)
    out, lse = paged_kv4_prefill_attention(q.to(DEV), pages, table.to(DEV), torch.tensor([600, 90], **I32), torch.tensor([0, 100, 130], **I32), max_q_len=2, max_seq_len=500,
                                           return_lse=True, **call)
    for b, (lo, hi, t) in enumerate(((0, 100, 500), (100, 130, 90))):
        rows = [0, 1, 17, hi - lo - 1]
        given = of(b)
        given["prefix"] = min(given["prefix"], 20) if "prefix" in SCORES[scores] else 0
        W.check(out, lse, S.attention(q[lo:hi], pages, slots[b][:t], rows=rows, **given), [lo + r for r in rows])


@pytest.mark.parametrize("bad", [-1, 1 << 30, 9999])
def test_a_page_number_outside_the_pool_leaves_its_tokens_out(bad, rows_form):
    """Told in the status where a row's window or prefix has them, and not else."""
    from blockgtq_b200 import paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(29)
    pages, table, slots = _case(gen, 1, 16, [900])
    q = _noise(gen, 3, 4, 128).half()
    for page, told in ((50, True), (0, True), (20, False)):      # tokens 800 .., 0 .., 320 ..
        broken, status = table.clone(), torch.zeros(1, **I32)
        broken[0, page] = bad
        out, lse = paged_kv4_prefill_attention(q.to(DEV), pages, broken.to(DEV), torch.tensor([900], **I32), torch.tensor([0, 3], **I32), return_lse=True, softcap=20.0,
                                               window=200, prefix_lens=torch.tensor([10], **I32), status=status)
        assert status.item() == (4 if told else 0)
        k, v = (x.cpu()[:, 0] for x in S.read(pages, slots[0]))
        for row in range(3):
            seen = S.seen_by(900, 3, row, 200, 10)
            seen[16 * page:16 * page + 16] = False
            y = 20 * torch.tanh(torch.einsum("hd,td->ht", q[row].double(), k[seen]) / math.sqrt(128) / 20)
            # products lose 2^-20 of their terms, a cap 2^-20 of itself
            off = 2.0 ** -20 * (torch.einsum("hd,td->ht", q[row].double().abs(), k[seen].abs()).amax(-1) / math.sqrt(128) + 20) + 1e-5
            assert ((lse[row].double().cpu() - torch.logsumexp(y, -1)).abs() <= off + 1e-5).all()
            _near(out[row].double().cpu(), torch.softmax(y, -1), v[seen], off)


def test_calls_on_two_streams_at_once():
    from blockgtq_b200 import paged_kv4_decode_attention, paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(37)
    pages, table, _ = _case(gen, 2, 16, [1500, 700, 30])
    args = (pages, table.to(DEV), torch.tensor([1500, 700, 30], **I32))
    q, few = _noise(gen, 400, 8, 128).half().to(DEV), _noise(gen, 3, 8, 128).half().to(DEV)
    cu = torch.tensor([0, 300, 380, 400], **I32)
    kinds = [_arguments(SCORES[k], [1500, 700, 30], 8)[0] for k in ("all", "cap", "sinks", "slopes", "prefix")]
    calls = [lambda kw=kw: paged_kv4_prefill_attention(q, *args, cu, **kw) for kw in kinds] + [lambda kw=kw: paged_kv4_decode_attention(few, *args, **kw) for kw in kinds]
    want = [c() for c in calls]
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for c in calls:
            for s, results in zip(streams, got):
                with torch.cuda.stream(s):
                    results.append(c())
    torch.cuda.synchronize()
    for results in got:
        assert all(torch.equal(r, want[i % len(want)]) for i, r in enumerate(results))


def test_two_graphs_of_one_pool_of_memory(rows_form):
    """Their workspaces may be the same memory: replayed one behind the other, each answers as it did."""
    from blockgtq_b200 import paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(43)
    pages, table, _ = _case(gen, 1, 16, [800, 300])
    args = (pages, table.to(DEV), torch.tensor([800, 300], **I32))
    cases = []
    for n, kind in ((40, "all"), (12, "cap")):
        q = _noise(gen, n, 8, 128).half().to(DEV)
        kw = _arguments(SCORES[kind], [800, 300], 8)[0]
        cases.append((q, torch.tensor([0, n // 2, n], **I32), kw))
    want = [paged_kv4_prefill_attention(q, *args, cu, **kw).clone() for q, cu, kw in cases]
    torch.cuda.synchronize()
    pool, graphs, outs = None, [], []
    for q, cu, kw in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(paged_kv4_prefill_attention(q, *args, cu, **kw))
        pool = g.pool()
        graphs.append(g)
    for i in (0, 1, 0, 0, 1):
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i], want[i])
