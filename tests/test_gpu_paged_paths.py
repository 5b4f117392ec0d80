"""GPU: the paged cache's attentions on their rarer ways: tiles that pass one workspace, more sequences and blocks than a plan's pass takes, groups of
every size.  Against 64 bits within the bound of tests/paged_bounds.py."""
import math

import pytest
import torch

import paged_bounds as W

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 1 / math.sqrt(128)
I32 = dict(dtype=torch.int32, device=DEV)


def _sequences(gen, n_kv, page, lens, width=None, dtype=torch.float16):
    """Pages in shuffled order, tables of `width` columns (those behind a sequence name no page), slots."""
    from blockgtq_b200 import page_bytes, paged_kv4_append
    need = [-(-t // page) for t in lens]
    width = max(1, *need) if width is None else width
    order = torch.randperm(sum(need) + 1, generator=gen).tolist()
    table, slots = torch.full((len(lens), width), -9, dtype=torch.int32), []
    for b, t in enumerate(lens):
        for i in range(need[b]):
            table[b, i] = order.pop()
        at = torch.arange(t)
        slots.append(table[b].long()[at // page] * page + at % page)
    pages = torch.full((sum(need) + 1, n_kv, page_bytes(page)), 255, dtype=torch.uint8, device=DEV)
    flat = torch.cat(slots)
    k, v = (torch.randn(len(flat), n_kv, 128, generator=gen).to(dtype).to(DEV) for _ in range(2))
    paged_kv4_append(pages, flat.to(DEV), k, v)
    return pages, table.to(DEV), slots


def _prefill(gen, pages, table, lens, counts, n_q, dtype=torch.float16, **kw):
    from blockgtq_b200 import paged_kv4_prefill_attention
    ends = [sum(counts[:i]) for i in range(len(counts) + 1)]
    q = torch.randn(ends[-1], n_q, 128, generator=gen).to(dtype)
    status = torch.zeros(1, **I32)
    out, lse = paged_kv4_prefill_attention(q.to(DEV), pages, table, torch.tensor(lens, **I32), torch.tensor(ends, **I32), return_lse=True, status=status, **kw)
    assert status.item() == 0
    return q, ends, out, lse


def _check_sequences(which, q, ends, out, lse, pages, slots, lens, counts, causal=True):
    host = pages.cpu()
    for b in which:
        t, m = lens[b], counts[b]
        seen = [t - m + 1 + i if causal else t for i in range(m)]
        W.check(out, lse, W.attention(q[ends[b]:ends[b + 1]], host, slots[b], seen, SCALE), slice(ends[b], ends[b + 1]))


# tokens a table holds, KV heads, sequences: a tile of 128 tokens is 64 KB, and 2 GiB of them are a launch's
@pytest.mark.parametrize("held,n_kv,lens,counts", [
    (1 << 18, 2, [40, 300, 0, 129, 17, 700, 1, 128, 260, 65, 33], [40, 70, 3, 9, 17, 150, 1, 128, 10, 0, 33]),      # 8 sequences, then 3
    (1 << 21, 3, [200, 150], [90, 150]),                                                                            # 2 heads, then 1, of each sequence
    ((1 << 22) + 128, 2, [140], [60]),                                                                              # more for one head
])
@pytest.mark.parametrize("causal", [True, False])
def test_tiles_of_more_than_one_workspace(held, n_kv, lens, counts, causal, monkeypatch):
    from blockgtq_b200 import _lib, paged
    monkeypatch.setattr(paged, "_FORM", 14)
    gen = torch.Generator().manual_seed(n_kv)
    pages, table, slots = _sequences(gen, n_kv, 128, lens, width=held // 128)
    before = _lib.launches
    q, ends, out, lse = _prefill(gen, pages, table, lens, counts, 4 * n_kv, causal=causal)
    assert _lib.launches - before == 3 * {2: 2, 3: 4}[n_kv]
    _check_sequences(range(len(lens)), q, ends, out, lse, pages, slots, lens, counts, causal)


@pytest.mark.parametrize("form", [0, 14, 15])
def test_more_sequences_than_a_plan_takes_at_once(form, monkeypatch):
    from blockgtq_b200 import paged
    monkeypatch.setattr(paged, "_FORM", form)
    gen = torch.Generator().manual_seed(600)
    lens = [int(x) for x in torch.randint(1, 60, (600,), generator=gen)]
    counts = [min(t, int(x)) for t, x in zip(lens, torch.randint(0, 30, (600,), generator=gen))]
    lens[300], counts[300], lens[512], counts[512], lens[7], counts[7] = 900, 200, 0, 4, 3, 9
    pages, table, slots = _sequences(gen, 1, 16, lens)
    q, ends, out, lse = _prefill(gen, pages, table, lens, counts, 2)
    _check_sequences([0, 1, 7, 8, 255, 256, 257, 299, 300, 301, 511, 512, 513, 598, 599], q, ends, out, lse, pages, slots, lens, counts)


def test_more_blocks_than_a_plan_takes_at_once(monkeypatch):
    from blockgtq_b200 import paged
    monkeypatch.setattr(paged, "_FORM", 14)
    gen = torch.Generator().manual_seed(601)
    lens, counts = [300, 9000, 40], [300, 9000, 40]                     # 9000 rows of 8 heads: 282 blocks
    pages, table, slots = _sequences(gen, 1, 64, lens)
    q, ends, out, lse = _prefill(gen, pages, table, lens, counts, 8)
    _check_sequences([0, 2], q, ends, out, lse, pages, slots, lens, counts)
    host = pages.cpu()
    for i in (0, 1, 31, 32, 4095, 8191, 8192, 8223, 8224, 8999):
        row = ends[1] + i
        W.check(out, lse, W.attention(q[row:row + 1], host, slots[1][:i + 1], [i + 1], SCALE), slice(row, row + 1))


FORMS = {"auto": 0, "split": 15, "cluster1": 1, "cluster2": 2, "cluster4": 4, "cluster8": 8, "tcgen05": 14}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gqa", range(1, 9))
@pytest.mark.parametrize("form", list(FORMS))
def test_groups_of_every_size(form, gqa, dtype, monkeypatch):
    from blockgtq_b200 import paged
    monkeypatch.setattr(paged, "_FORM", FORMS[form])
    gen = torch.Generator().manual_seed(10 * gqa)
    lens, counts = [290, 61, 1000], [83, 61, 2]
    pages, table, slots = _sequences(gen, 2, 48, lens, dtype=dtype)
    q, ends, out, lse = _prefill(gen, pages, table, lens, counts, 2 * gqa, dtype)
    _check_sequences(range(3), q, ends, out, lse, pages, slots, lens, counts)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", ["auto", "split", "cluster1", "cluster8"])
def test_decode_within_the_bound_of_its_arithmetic(form, dtype, monkeypatch):
    from blockgtq_b200 import paged, paged_kv4_decode_attention
    monkeypatch.setattr(paged, "_FORM", FORMS[form])
    gen = torch.Generator().manual_seed(4)
    lens = [1, 17, 0, 300, 2500, 33]
    pages, table, slots = _sequences(gen, 2, 32, lens, dtype=dtype)
    q = (2 * torch.randn(len(lens), 12, 128, generator=gen)).to(dtype)
    out, lse = paged_kv4_decode_attention(q.to(DEV), pages, table, torch.tensor(lens, **I32), return_lse=True)
    host = pages.cpu()
    for b, t in enumerate(lens):
        W.check(out, lse, W.attention(q[b:b + 1], host, slots[b], [t], SCALE), slice(b, b + 1))
