"""GPU: calls of the paged cache's operators as a program makes them: results in buffers of its own, other streams, counted launches."""
import math

import pytest
import torch

import paged_bounds as W

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I32 = dict(dtype=torch.int32, device=DEV)


def _sequence(gen, t, n_kv=2, page=16):
    """Pages in order that hold t random tokens, their table and slots."""
    from blockgtq_b200 import page_bytes, paged_kv4_append
    width = -(-t // page)
    pages = torch.zeros(width, n_kv, page_bytes(page), dtype=torch.uint8, device=DEV)
    k, v = (torch.randn(t, n_kv, 128, generator=gen).half().to(DEV) for _ in range(2))
    slots = torch.arange(t)
    paged_kv4_append(pages, slots.to(DEV), k, v)
    return pages, torch.arange(width, **I32)[None], slots


@pytest.mark.parametrize("rows", [6, 100])
def test_a_result_in_other_columns_of_the_queries_buffer(rows):
    from blockgtq_b200 import paged_kv4_prefill_attention
    gen = torch.Generator().manual_seed(rows)
    pages, table, _ = _sequence(gen, 300)
    buffer = torch.randn(rows, 12, 128, generator=gen).half().to(DEV)
    q, out, rest = buffer[:, 4:8], buffer[:, 8:], buffer[:, :4].clone()
    args = (pages, table, torch.tensor([300], **I32), torch.tensor([0, rows], **I32))
    want, before = paged_kv4_prefill_attention(q, *args), q.clone()
    assert paged_kv4_prefill_attention(q, *args, out=out) is out
    assert torch.equal(out, want) and torch.equal(q, before) and torch.equal(buffer[:, :4], rest)
    outer = torch.empty(4, rows, 128, dtype=torch.float16, device=DEV).transpose(0, 1)
    assert torch.equal(paged_kv4_prefill_attention(q, *args, out=outer), want)
    wide = torch.zeros(rows + 1, 4, 128, dtype=torch.float16, device=DEV)
    for bad in (buffer[:, 6:10], buffer[:, 4:8], wide.as_strided((rows, 4, 128), (128, 128, 1))):
        with pytest.raises(ValueError, match="of its own"):
            paged_kv4_prefill_attention(q, *args, out=bad)
    with pytest.raises(ValueError, match="of its own"):
        paged_kv4_prefill_attention(wide[1:], *args, out=wide[:-1])


def test_a_step_on_another_stream_keeps_what_it_reads():
    """The step's slots, table and lengths belong to the stream that began it; the layers run late, on another."""
    from blockgtq_b200 import PagedKV4Cache
    gen = torch.Generator().manual_seed(61)
    caches = [PagedKV4Cache(1, 4, 2, n_pages=40, max_seq_len=200, page_size=16, device=DEV) for _ in range(2)]
    tokens = [[torch.randn(n, h, 128, generator=gen).half().to(DEV) for h in (4, 2, 2)] for n in (50, 2, 2, 2)]
    side, got = torch.cuda.Stream(DEV), ([], [])
    torch.cuda.synchronize()
    for cache, results, late in zip(caches, got, (False, True)):
        a, b = cache.add_sequence(), cache.add_sequence()
        for rows, counts in zip(tokens, ([30, 20], [1, 1], [1, 1], [1, 1])):
            cache.begin_step([a, b], counts)
            if late:
                with torch.cuda.stream(side):
                    torch.cuda._sleep(20_000_000)
                    results.append(cache.append_and_attend(0, *rows))
            else:
                results.append(cache.append_and_attend(0, *rows))
            cache.free_sequence(cache.add_sequence())
            junk = [torch.full((1 << k,), 7, **I32) for k in range(3, 9)]         # takes what has been given back
            del junk
        torch.cuda.synchronize()
        cache.check_status()
    assert all(torch.equal(x, y) for x, y in zip(*got))
    assert torch.equal(caches[0].pages, caches[1].pages)


def test_a_step_is_not_captured():
    """Replayed behind its step, the graph would store tokens in pages that are another sequence's by then."""
    from blockgtq_b200 import PagedKV4Cache
    cache = PagedKV4Cache(1, 4, 2, n_pages=4, max_seq_len=60, page_size=16, device=DEV)
    cache.begin_step([cache.add_sequence()], [3])
    q, kv = torch.ones(3, 4, 128, dtype=torch.float16, device=DEV), torch.ones(3, 2, 128, dtype=torch.float16, device=DEV)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            cache.append_and_attend(0, q, kv, kv)
    assert not cache.pages.any()
    cache.append_and_attend(0, q, kv, kv)
    assert cache.pages.any()
    cache.check_status()


def _kernels(call):
    """Kernels in a graph of the call, by the runtime's own count."""
    import ctypes as C
    cudart = C.CDLL("libcudart.so.12")
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = call()
    n = C.c_size_t(0)
    assert cudart.cudaGraphGetNodes(C.c_void_p(graph.raw_cuda_graph()), None, C.byref(n)) == 0
    del held
    return n.value


@pytest.mark.parametrize("form,rows,t,expected", [(0, 1, 40, 1), (15, 1, 40, 1), (15, 1, 4000, 2), (8, 1, 4000, 1), (15, 3, 700, 2), (14, 3, 700, 3), (14, 300, 700, 3)])
def test_launches_are_counted_as_they_are_made(form, rows, t, expected, monkeypatch):
    from blockgtq_b200 import _lib, paged, paged_kv4_append, paged_kv4_decode_attention, paged_kv4_prefill_attention, paged_kv4_read
    monkeypatch.setattr(paged, "_FORM", form)
    gen = torch.Generator().manual_seed(form)
    pages, table, slots = _sequence(gen, t)
    lens = torch.tensor([t], **I32)
    q = torch.randn(rows, 4, 128, generator=gen).half().to(DEV)
    odd = torch.randn(rows, 4, 129, generator=gen).half().to(DEV)[:, :, 1:]           # rows that are copied first, in the binding's other path
    cu = torch.tensor([0, rows], **I32)
    def attend(q):
        return paged_kv4_decode_attention(q, pages, table, lens) if rows == 1 and form != 14 else paged_kv4_prefill_attention(q, pages, table, lens, cu)
    def counted(call):
        before = _lib.launches
        call()
        return _lib.launches - before
    assert counted(lambda: attend(q)) == counted(lambda: attend(odd)) == expected
    assert _kernels(lambda: attend(q)) == expected
    kv = torch.zeros(5, 2, 128, dtype=torch.float16, device=DEV)
    at = slots[:5].to(DEV)
    for n in (0, 5):
        for call in (lambda: paged_kv4_append(pages, at[:n], kv[:n], kv[:n]), lambda: paged_kv4_read(pages, at[:n]),
                     lambda: paged_kv4_append(pages, at[:n].repeat(2)[::2], kv[:n], kv[:n])):
            assert counted(call) == (1 if n else 0)
    assert counted(lambda: paged_kv4_prefill_attention(q[:0], pages, table, lens, cu)) == 0


def test_an_error_on_another_stream_is_told():
    from blockgtq_b200 import PagedKV4Cache
    cache = PagedKV4Cache(1, 4, 2, n_pages=4, max_seq_len=60, page_size=16, device=DEV)
    cache.begin_step([cache.add_sequence()], [3])
    q, kv = torch.ones(3, 4, 128, dtype=torch.float16, device=DEV), torch.ones(3, 2, 128, dtype=torch.float16, device=DEV)
    cos = torch.ones(2, 64, device=DEV)                         # the third token has no angle
    side = torch.cuda.Stream(DEV)
    cache.append_and_attend(0, q, kv, kv)
    cache.check_status()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        cache.append_and_attend(0, q, kv, kv, rope=(cos, cos))
    with pytest.raises(RuntimeError, match="position"):
        cache.check_status()
    cache.check_status()
