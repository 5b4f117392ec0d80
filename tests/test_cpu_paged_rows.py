"""CPU: where the result of the paged cache's attention may lie, in the binding and in the library."""
import ctypes as C

import pytest
import torch

from blockgtq_b200 import _lib, page_bytes, paged_kv4_decode_attention

N, H = 6, 4
ROW = 128


def _view(buffer, at, st, sh, n=N, h=H):
    return buffer.as_strided((n, h, ROW), (st, sh, 1), at)


# q (at, token stride, head stride), out, whether they may be used together; in elements of one buffer
PLACES = [
    ((0, 512, 128), (4096, 512, 128), True),
    ((0, 512, 128), (4096, 128, 768), True),                # heads outside
    ((0, 512, 128), (3584, 512, 128), True),
    ((0, 512, 128), (N * 512, 512, 128), True),             # right behind q
    ((N * 512, 512, 128), (0, 512, 128), True),
    ((0, 1536, 128), (512, 1536, 128), True),               # columns of one projection
    ((1024, 1536, 128), (0, 1536, 128), True),
    ((0, 128, 2 * N * 128), (N * 128, 128, 2 * N * 128), True),     # the same by heads
    ((0, 512, 128), (0, 512, 128), False),                  # q itself
    ((0, 512, 128), (512, 512, 128), False),                # one token on
    ((512, 512, 128), (0, 512, 128), False),
    ((0, 512, 128), (64, 512, 128), False),
    ((0, 512, 128), (N * 512 - 128, 512, 128), False),      # the last row
    ((0, 1536, 128), (384, 1536, 128), False),              # columns that share a head
    ((0, 1536, 128), (512, 1024, 128), False),
    ((0, 512, 128), (0, 128, 768), False),
    ((0, 512, 128), (4096, 128, 128), False),               # row (i, h + 1) is row (i + 1, h)
    ((0, 512, 128), (4096, 256, 128), False),
    ((0, 512, 128), (4096, 128, 256), False),
    ((0, 512, 128), (4096, 64, 768), False),
    ((0, 512, 128), (4096, 0, 128), False),
    ((0, 512, 128), (4096, 512, 0), False),
]


def _overlap(q, out):
    """By looking at every element."""
    at = [s * torch.arange(n)[:, None, None] + t * torch.arange(h)[:, None] + torch.arange(ROW) + a for a, s, t, n, h in (q, out)]
    a, b = (x.flatten().tolist() for x in at)
    return len(set(b)) < len(b) or bool(set(a) & set(b))


@pytest.mark.parametrize("q,out,fine", PLACES)
def test_a_result_lies_apart_from_the_queries_and_from_itself(q, out, fine):
    assert _overlap((*q, N, H), (*out, N, H)) is not fine
    buffer = torch.zeros(16384, dtype=torch.float16)
    args = (_view(buffer, *q), torch.zeros(3, 2, page_bytes(32), dtype=torch.uint8), torch.zeros(N, 1, dtype=torch.int32),
            torch.ones(N, dtype=torch.int32))
    with pytest.raises(RuntimeError if fine else ValueError, match="CUDA" if fine else "of its own"):
        paged_kv4_decode_attention(*args, out=_view(buffer, *out))


@pytest.mark.parametrize("q,out,fine", [x for x in PLACES if not x[2]])
def test_the_library_refuses_results_that_overlap(q, out, fine):
    raw = C.create_string_buffer(65536)
    p = (C.addressof(raw) + 255) & ~255
    rc = _lib.lib().bgtq_paged_attend(p + 2 * q[0], q[1], q[2], p, 2 * 4608, 4608, 3, 32, p, 1, 1, p, 0, N, N, H, 2, 1, 32, 1.0, 0, p, 1 << 30,
                                      p + 2 * out[0], out[1], out[2], 0, 0, 0)
    assert rc == -1


def test_one_token_or_one_head_has_no_stride():
    buffer = torch.zeros(4096, dtype=torch.float16)
    for n, h, st, sh in ((1, 4, 0, 128), (4, 2, 256, 128), (1, 2, 8, 128)):
        q, out = _view(buffer, 0, 256 * h, 128, n, h), _view(buffer, 2048, st, sh, n, h)
        with pytest.raises(RuntimeError, match="CUDA"):
            paged_kv4_decode_attention(q, torch.zeros(3, h, page_bytes(32), dtype=torch.uint8), torch.zeros(n, 1, dtype=torch.int32),
                                       torch.ones(n, dtype=torch.int32), out=out)


def test_pages_that_share_memory_are_not_written():
    """Read they may be: a head's pages for all heads, for instance."""
    from blockgtq_b200 import paged_kv4_append, paged_kv4_read
    k, slots = torch.zeros(4, 2, ROW, dtype=torch.float16), torch.arange(4)
    pool = torch.zeros(6, 2, page_bytes(32), dtype=torch.uint8)
    b = page_bytes(32)
    for pages in (pool, pool.transpose(0, 1).contiguous().transpose(0, 1), pool[::2], pool[:1], torch.zeros(2, 6, 2, b, dtype=torch.uint8)[1]):
        with pytest.raises(RuntimeError, match="CUDA"):
            paged_kv4_append(pages, slots, k, k)
    for pages in (pool[:, :1].expand(6, 2, b), pool[:1].expand(6, 2, b), pool.as_strided((3, 2, b), (b, b, 1)), pool.as_strided((3, 2, b), (2 * b, 2304, 1))):
        with pytest.raises(ValueError, match="of their own"):
            paged_kv4_append(pages, slots, k, k)
        with pytest.raises(RuntimeError, match="CUDA"):
            paged_kv4_read(pages, slots)
    raw = C.create_string_buffer(65536)
    p = (C.addressof(raw) + 255) & ~255
    for page_stride, head_stride in ((4608, 0), (0, 2304), (2304, 2304), (4608, 16)):
        rc = _lib.lib().bgtq_paged_append(p, page_stride, head_stride, 3, 16, p, p, 256, 128, p, 256, 128, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 2, 0, 0, 0, 0)
        assert rc == -1


@pytest.mark.parametrize("n,n_kv", [(1 << 28, 3), ((1 << 29) + 32, 1), (1 << 30, 1)])
def test_reading_counts_its_rows_in_32_bits(n, n_kv):
    """Four lanes to each of 2 n n_kv rows: beyond what 32 bits hold."""
    raw = C.create_string_buffer(4096)
    p = (C.addressof(raw) + 255) & ~255
    assert _lib.lib().bgtq_paged_read(p, 2304 * n_kv, 2304, 1, 16, p, n, n_kv, p, p, 0, 0, 0) == -5
