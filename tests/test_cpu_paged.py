"""CPU: what the paged 4-bit cache refuses, its page book-keeping, and that its values are numbers that fp16 holds exactly."""
import ctypes as C

import pytest
import torch

import paged_reference as R
from blockgtq_b200 import (PagedKV4Cache, _lib, page_bytes, paged_kv4_append, paged_kv4_decode_attention, paged_kv4_prefill_attention,
                           paged_kv4_read)


def _pages(n=3, h=2, page=32):
    return torch.zeros(n, h, page_bytes(page), dtype=torch.uint8)


def _rows(n=4, h=2, dtype=torch.float16):
    return torch.zeros(n, h, 128, dtype=dtype)


def test_page_bytes():
    assert page_bytes(16) == 2304 and page_bytes(128) == 8 * 2304
    for bad in (0, 8, 17, -16):
        with pytest.raises(ValueError):
            page_bytes(bad)


def test_valid_calls_want_the_gpu():
    slots = torch.arange(4)
    lens, table = torch.ones(4, dtype=torch.int32), torch.zeros(4, 1, dtype=torch.int32)
    for call in (lambda: paged_kv4_append(_pages(), slots, _rows(), _rows()), lambda: paged_kv4_read(_pages(), slots),
                 lambda: paged_kv4_decode_attention(_rows(h=4), _pages(), table, lens)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("change,error", [
    (dict(pages=torch.zeros(3, 2, 2305, dtype=torch.uint8)), ValueError),
    (dict(pages=torch.zeros(3, 2, 2304)), ValueError),
    (dict(pages=torch.zeros(3, 2304, dtype=torch.uint8)), ValueError),
    (dict(pages=torch.zeros(3, 2, 2 * 2304, dtype=torch.uint8)[..., 8:8 + 2304]), ValueError),
    (dict(slots=torch.arange(4, dtype=torch.int32)), ValueError),
    (dict(slots=torch.arange(5)), ValueError),
    (dict(k=torch.zeros(4, 3, 128, dtype=torch.float16)), ValueError),
    (dict(k=torch.zeros(4, 2, 64, dtype=torch.float16)), ValueError),
    (dict(k=torch.zeros(4, 2, 128)), TypeError),
    (dict(v=torch.zeros(4, 2, 128, dtype=torch.bfloat16)), TypeError),
    (dict(v=torch.zeros(3, 2, 128, dtype=torch.float16)), ValueError),
    (dict(q=torch.zeros(4, 4, 128, dtype=torch.float16)), ValueError),                 # without tables
    (dict(cos=torch.zeros(9, 64)), ValueError),
    (dict(cos=torch.zeros(9, 64), sin=torch.zeros(9, 64)), ValueError),
    (dict(cos=torch.zeros(9, 32), sin=torch.zeros(9, 32), positions=torch.arange(4)), ValueError),
    (dict(cos=torch.zeros(9, 64).half(), sin=torch.zeros(9, 64).half(), positions=torch.arange(4)), TypeError),
    (dict(cos=torch.zeros(9, 64), sin=torch.zeros(9, 64), positions=torch.arange(3)), ValueError),
    (dict(status=torch.zeros(1)), ValueError),
])
def test_append_refuses(change, error):
    args = dict(pages=_pages(), slots=torch.arange(4), k=_rows(), v=_rows()) | change
    with pytest.raises(error):
        paged_kv4_append(**args)


@pytest.mark.parametrize("change,error", [
    (dict(q=_rows(h=3)), ValueError),
    (dict(q=_rows(h=18)), ValueError),                                                # 9 heads per KV head
    (dict(q=_rows(h=4, dtype=torch.float32)), TypeError),
    (dict(q=_rows(n=3, h=4)), ValueError),
    (dict(block_table=torch.zeros(4, 1)), ValueError),
    (dict(block_table=torch.zeros(4, dtype=torch.int32)), ValueError),
    (dict(seq_lens=torch.ones(4, dtype=torch.int64)), ValueError),
    (dict(seq_lens=torch.ones(3, dtype=torch.int32)), ValueError),
    (dict(scale=float("nan")), ValueError),
    (dict(out=torch.zeros(4, 4, 128)), ValueError),
])
def test_decode_refuses(change, error):
    args = dict(q=_rows(h=4), pages=_pages(), block_table=torch.zeros(4, 1, dtype=torch.int32), seq_lens=torch.ones(4, dtype=torch.int32))
    with pytest.raises(error):
        paged_kv4_decode_attention(**(args | change))


def test_prefill_refuses():
    args = dict(q=_rows(h=4), pages=_pages(), block_table=torch.zeros(2, 1, dtype=torch.int32), seq_lens=torch.ones(2, dtype=torch.int32),
                cu_q=torch.tensor([0, 2, 4], dtype=torch.int32))
    for change in (dict(cu_q=torch.tensor([0, 4], dtype=torch.int32)), dict(cu_q=torch.tensor([0, 2, 4])), dict(max_seq_len=-1)):
        with pytest.raises(ValueError):
            paged_kv4_prefill_attention(**(args | change))
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_kv4_prefill_attention(**args)


def test_library_refuses_before_it_touches_the_device():
    lib, buf = _lib.lib(), C.create_string_buffer(4096)
    p = (C.addressof(buf) + 255) & ~255
    def append(**kw):
        a = dict(pages=p, ps=4608, hs=2304, n_pages=2, page=16, slots=p, k=p, kst=256, ksh=128, v=p, vst=256, vsh=128, q=0, qst=0, qsh=0, qo=0,
                 cos=0, sin=0, rst=0, pos=0, npos=0, n=1, nkv=2, nq=0, flags=0, status=0, stream=0) | kw
        return lib.bgtq_paged_append(*a.values())
    assert append(n=0) == _lib.OK
    for kw, code in ((dict(page=24), -1), (dict(page=0), -1), (dict(n_pages=0), -1), (dict(pages=0), -1), (dict(slots=0), -1), (dict(n=-1), -1),
                     (dict(pages=p + 8), -3), (dict(hs=2300), -3), (dict(k=p + 2), -3), (dict(kst=132), -3), (dict(cos=p), -1),
                     (dict(cos=p, sin=p, rst=64), -1), (dict(cos=p, sin=p, rst=66, pos=p, npos=1), -3), (dict(q=p, nq=1, qo=p), -1),
                     (dict(nq=1), -1), (dict(flags=2), -1), (dict(flags=64), -1)):
        assert append(**kw) == code, kw
    def attend(**kw):
        a = dict(q=p, qst=512, qsh=128, pages=p, ps=4608, hs=2304, n_pages=2, page=16, table=p, tst=1, cols=1, lens=p, cu=0, n_seq=1, n=1, nq=4, nkv=2,
                 max_q=1, most=16, scale=1.0, flags=0, ws=p, wsb=1 << 40, out=p, ost=512, osh=128, lse=0, status=0, stream=0) | kw
        return lib.bgtq_paged_attend(*a.values())
    assert attend(n_seq=0, n=0) == _lib.OK
    for kw, code in ((dict(nq=3), -1), (dict(nq=18), -2), (dict(n=2), -1), (dict(max_q=2), -1), (dict(max_q=0), -1), (dict(cols=1 << 28, most=1 << 40), -5), (dict(flags=14 << 8), -1), (dict(flags=13 << 8), -1),
                     (dict(q=p + 8), -3), (dict(qst=4), -3), (dict(out=p + 4), -3), (dict(ws=0, flags=15 << 8), -1), (dict(wsb=16, flags=15 << 8), -1), (dict(flags=3 << 8), -1), (dict(lens=0), -1),
                     (dict(table=0), -1), (dict(scale=float("nan")), -1), (dict(flags=2), -1), (dict(pages=p + 1), -3)):
        assert attend(**kw) == code, kw
    assert lib.bgtq_paged_workspace_bytes(1, 1, 18, 2, 1, 10, 0) == -2 and lib.bgtq_paged_workspace_bytes(1, 1, 3, 2, 1, 10, 0) == -1


def test_values_are_exact_in_half_precision():
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(400, 128, generator=gen) * torch.exp(6 * torch.randn(400, 1, generator=gen))
    codes, scale = R.quantised(x)
    value = codes.double() * scale.double().repeat_interleave(32, -1)
    assert torch.equal(value.half().double(), value)
    # half a step, the scale's rounding (2^-8 of a code of 7) and the smallest scale apart
    room = scale.double().repeat_interleave(32, -1) * (0.5 + 7 * 2.0 ** -8)
    inside = x.abs() <= 65000
    assert ((value - x.double()).abs() <= room)[inside].all()


def test_pages_are_handed_out_and_given_back():
    c = PagedKV4Cache(1, 4, 2, n_pages=6, max_seq_len=100, page_size=16, device="cpu")
    a, b = c.add_sequence(), c.add_sequence()
    c.begin_step([a, b], [17, 16])
    assert (c.seq_len(a), c.seq_len(b), c.free_pages) == (17, 16, 3)
    s = c._step
    assert s["ends"].tolist() == [0, 17, 33] and s["lens"].tolist() == [17, 16] and s["positions"].tolist() == [*range(17), *range(16)]
    table = s["table"]
    want = [int(table[0, t // 16]) * 16 + t % 16 for t in range(17)] + [int(table[1, 0]) * 16 + t for t in range(16)]
    assert s["slots"].tolist() == want and len(set(want)) == 33
    before = c._seqs[a][0], list(c._seqs[a][1]), c.free_pages
    with pytest.raises(RuntimeError, match="pages"):
        c.begin_step([a, b], [48, 17])                  # three and one more: one too many, and nothing is taken
    assert before == (c._seqs[a][0], c._seqs[a][1], c.free_pages)
    for bad in (([a, a], [1, 1]), ([a], [0]), ([], []), ([a], [1, 2]), ([a], [84])):
        with pytest.raises(ValueError):
            c.begin_step(*bad)
    with pytest.raises(KeyError):
        c.begin_step([99], [1])
    assert c.cache_memory_bytes() == 3 * 2 * 2304
    c.free_sequence(a)
    assert c.free_pages == 5
    with pytest.raises(KeyError):
        c.seq_len(a)
    c.begin_step([b], [1])
    assert c._step["slots"].tolist() == [int(c._step["table"][0, 1]) * 16]


def test_a_result_with_rows_of_its_own():
    q = _rows(h=4)
    args = (q, _pages(), torch.zeros(4, 1, dtype=torch.int32), torch.ones(4, dtype=torch.int32))
    for out in (q, torch.zeros(1, 4, 128, dtype=torch.float16).expand(4, 4, 128), torch.zeros(4, 1, 128, dtype=torch.float16).expand(4, 4, 128)):
        with pytest.raises(ValueError, match="of its own"):
            paged_kv4_decode_attention(*args, out=out)


def test_a_step_takes_its_tokens_and_ends_with_its_sequences():
    c = PagedKV4Cache(1, 4, 2, n_pages=6, max_seq_len=100, page_size=16, device="cpu")
    a, b, other = (c.add_sequence() for _ in range(3))
    c.begin_step([a, b], [3, 2])
    for n in (4, 6):                                    # rows of other numbers than the step's
        with pytest.raises(ValueError, match="step"):
            c.append_and_attend(0, _rows(n, 4), _rows(n), _rows(n))
    c.free_sequence(other)
    with pytest.raises(RuntimeError, match="CUDA"):
        c.append_and_attend(0, _rows(5, 4), _rows(5), _rows(5))
    c.free_sequence(b)                                  # its pages may be another's from here on
    with pytest.raises(RuntimeError, match="begin_step"):
        c.append_and_attend(0, _rows(5, 4), _rows(5), _rows(5))
