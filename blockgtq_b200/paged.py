"""A paged key/value cache in 4 bits, for batches whose sequences have lengths of their own.

The reference's caches are contiguous, of one length for the whole batch, and calibrated per head; this one needs
neither, and a sequence's tokens lie in whatever pages are free.  A token's K and V rows are quantised by themselves: four
groups of 32 dims, each with a bf16 scale and signed codes of 4 bits (4.5 bits per value).  ``include/bgtq.h`` has the layout
of a page.  The functions are the operators; :class:`PagedKV4Cache` keeps the pages of a model's layers and
hands them out to sequences.
"""
from __future__ import annotations

import ctypes as C
import math
import operator

import torch

from . import _lib

__all__ = ["PAGE_UNIT_BYTES", "page_bytes", "rope_axes", "paged_kv4_append", "paged_kv4_read", "paged_kv4_copy", "paged_kv4_decode_attention",
           "paged_kv4_prefill_attention", "PagedKV4Cache"]

HD = 128
UNIT = 16                       # tokens of a unit
PAGE_UNIT_BYTES = 2304          # bytes of a unit of one KV head
_FORM = 0                       # form of the attention's launch (bgtq.h, BGTQ_PAGED_FORM_SHIFT), 0: the library chooses
_KINDS = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_SCALE = 1.0 / math.sqrt(HD)
_TYPES = {torch.float16: 0, torch.bfloat16: _lib.PAGED_BF16}


def page_bytes(page_size: int) -> int:
    """Bytes of a page of ``page_size`` tokens of one KV head."""
    if page_size < UNIT or page_size % UNIT:
        raise ValueError(f"page_size must be a multiple of {UNIT}, got {page_size}")
    return page_size // UNIT * PAGE_UNIT_BYTES


def _pool(pages):
    """(page tokens) of a pool (n_pages, n_kv, page bytes) uint8, checked."""
    if pages.dtype != torch.uint8 or pages.dim() != 3:
        raise ValueError("pages must be uint8 (n_pages, n_kv, page bytes)")
    n, h, b = pages.shape
    if b < PAGE_UNIT_BYTES or b % PAGE_UNIT_BYTES or n < 1 or h < 1:
        raise ValueError(f"a page is a multiple of {PAGE_UNIT_BYTES} bytes per KV head, got pages of shape {tuple(pages.shape)}")
    if pages.stride(2) != 1 or pages.stride(0) % 16 or pages.stride(1) % 16 or pages.data_ptr() % 16:
        raise ValueError("pages must have contiguous rows whose addresses are multiples of 16 bytes")
    return b // PAGE_UNIT_BYTES * UNIT


def _rows(x, name, n, heads, dtype, device, align):
    """x (n, heads, 128) of the call's type on the call's device, with rows that the kernels can load."""
    if x.dim() != 3 or x.shape[2] != HD or (n is not None and x.shape[0] != n) or (heads is not None and x.shape[1] != heads):
        raise ValueError(f"{name} must be ({'tokens' if n is None else n}, {'heads' if heads is None else heads}, {HD}), got {tuple(x.shape)}")
    if x.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {x.dtype}")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, the pages on {device}")
    e = align // 2
    if x.stride(2) != 1 or x.stride(0) % e or x.stride(1) % e or x.data_ptr() % align:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _is(x, name, dtype, shape, device):
    if x.dtype != dtype or tuple(x.shape) != shape:
        raise ValueError(f"{name} must be {dtype} {shape}, got {x.dtype} {tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, the pages on {device}")


def _ints(x, name, dtype, shape, device):
    _is(x, name, dtype, shape, device)
    return x.contiguous()


def _spans(x):
    """(places, bytes from one to the next, bytes of all of them) along the two outer dimensions of x."""
    row = x.shape[2] * x.element_size()
    return [(n, x.element_size() * st, (max(n, 1) - 1) * x.element_size() * st + row) for n, st in zip(x.shape, x.stride()[:2])]


def _apart(x):
    """The places (i, j) of x do not overlap one another: those along the smaller stride fit into a step of the larger."""
    near, far = sorted(_spans(x), key=lambda d: (d[0] > 1, d[1]))
    row = x.shape[2] * x.element_size()
    return (near[0] <= 1 or near[1] >= row) and (far[0] <= 1 or far[1] >= near[2])


def _rows_clear(x, y):
    """The rows of y, of x's shape, are elsewhere, or between those of x with the same stride."""
    a, b, at = _spans(x), _spans(y), y.data_ptr() - x.data_ptr()
    if at >= a[0][2] + a[1][2] - 2 * HD or -at >= b[0][2] + b[1][2] - 2 * HD:
        return True
    return any(n > 1 and step > 0 and step == b[i][1] and a[1 - i][2] <= at % step <= step - b[1 - i][2] for i, (n, step, _) in enumerate(a))


def _status(status, device):
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1 or status.device != device):
        raise ValueError("status must be an int32 tensor on the pages' device")
    return _lib.ptr(status)


def _type_flag(dtype, name):
    if dtype not in _TYPES:
        raise TypeError(f"{name} must be float16 or bfloat16, got {dtype}")
    return _TYPES[dtype]


def rope_axes(sections, interleaved=False):
    """The ``axes`` of :func:`paged_kv4_append`: the axis of each of the 64 rotated pairs, as bytes.  ``sections``: how many pairs the axes have (1 to
    4 of them, 64 pairs in all), one axis behind the other, or ``interleaved``: the axes take turns, each while it has pairs left."""
    left = [operator.index(n) for n in sections]
    if not 1 <= len(left) <= 4 or min(left) < 0 or sum(left) != HD // 2:
        raise ValueError(f"sections must be 1 to 4 numbers of pairs, {HD // 2} in all, got {left}")
    if not interleaved:
        return bytes(a for a, n in enumerate(left) for _ in range(n))
    out = []
    while len(out) < HD // 2:
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return bytes(out)


def paged_kv4_append(pages, slots, k, v, q=None, cos=None, sin=None, positions=None, status=None, axes=None):
    """Quantise k and v (n, n_kv, 128) fp16 or bf16 into the slots of ``pages`` (n_pages, n_kv, page bytes) uint8.

    ``slots`` (n,) int64: page * page size + place in the page, distinct; a token with a negative one is not stored.
    ``cos`` / ``sin`` (n_positions, 64) fp32 with ``positions`` (n,) int64: k, and ``q`` (n, n_q, 128), go through the rotary
    embedding first (dims d and d + 64 are a pair; fp32, k quantised from the unrounded result).  Returns the rotated q (n, n_q, 128),
    or None without one.  ``status``: optional int32 tensor, set to 2 where a slot or position is out of range (the token is not stored).

    ``axes``: positions lie along several axes, ``positions`` is (axes, n), and the pair d is turned by the angle of its token's position along axis
    ``axes[d]``: 64 numbers of axes, as :func:`rope_axes` makes them."""
    host = _lib.host()
    if axes is None:
        r = host.paged_append(pages, slots, k, v, q, cos, sin, positions, status)
    else:
        r = host.paged_append(pages, slots, k, v, q, cos, sin, positions, status, axes)
        if type(r) is int and r < 0:        # (axes that positions do not have are named below)
            r = None
    if r is None:
        return _append(pages, slots, k, v, q, cos, sin, positions, status, axes)
    _lib.done(r, "bgtq_paged_append", host.paged_launched())
    return None if q is None else r


@torch.no_grad()
def _append(pages, slots, k, v, q, cos, sin, positions, status, axes=None):
    """:func:`paged_kv4_append` for what the extension module leaves: tensors that have to be copied, and errors."""
    page = _pool(pages)
    dev, n_kv = pages.device, pages.shape[1]
    if not _apart(pages):
        raise ValueError("tokens are stored in pages of their own, apart from one another")
    flags = _type_flag(k.dtype, "k")
    k = _rows(k, "k", None, n_kv, k.dtype, dev, 16)
    n = k.shape[0]
    v = _rows(v, "v", n, n_kv, k.dtype, dev, 16)
    slots = _ints(slots, "slots", torch.int64, (n,), dev)
    if (cos is None) != (sin is None) or (cos is None) != (positions is None):
        raise ValueError("cos, sin and positions belong together")
    n_q, q_out, qs, rope, entry = 0, None, (0, 0), (None, None, 0, None, 0), "bgtq_paged_append"
    if axes is not None and cos is None:
        raise ValueError("axes belong to cos, sin and positions")
    if cos is not None:
        if cos.dim() != 2 or cos.shape[1] != HD // 2 or cos.shape[0] < 1 or sin.shape != cos.shape:
            raise ValueError(f"cos and sin must be (positions, {HD // 2}), got {tuple(cos.shape)} and {tuple(sin.shape)}")
        if cos.dtype != torch.float32 or sin.dtype != torch.float32:
            raise TypeError("cos and sin must be float32")
        if cos.device != dev or sin.device != dev:
            raise ValueError(f"cos and sin must be on {dev}")
        if cos.stride(1) != 1 or cos.stride(0) % 4 or sin.stride() != cos.stride() or (cos.data_ptr() | sin.data_ptr()) % 16:
            cos, sin = (x.clone(memory_format=torch.contiguous_format) for x in (cos, sin))
        if axes is None:
            positions = _ints(positions, "positions", torch.int64, (n,), dev)
            rope = (cos.data_ptr(), sin.data_ptr(), cos.stride(0), positions.data_ptr(), cos.shape[0])
        else:
            n_axes = positions.shape[0] if positions.dim() == 2 else 0
            if not 1 <= n_axes <= 4:
                raise ValueError(f"positions must be (axes, {n}), 1 to 4 axes, got {tuple(positions.shape)}")
            positions = _ints(positions, "positions", torch.int64, (n_axes, n), dev)
            axes = bytes(axes)
            if len(axes) != HD // 2 or max(axes) >= n_axes:
                raise ValueError(f"axes must be {HD // 2} numbers below {n_axes}, the positions' axes")
            entry = "bgtq_paged_append_axes"
            rope = (cos.data_ptr(), sin.data_ptr(), cos.stride(0), positions.data_ptr(), n, axes, n_axes, cos.shape[0])
    if q is not None:
        if cos is None:
            raise ValueError("q is only taken to be rotated: pass cos, sin and positions")
        q = _rows(q, "q", n, None, k.dtype, dev, 16)
        n_q, qs = q.shape[1], q.stride()[:2]
        q_out = torch.empty(n, n_q, HD, dtype=q.dtype, device=dev)
        if n_q == 0:
            q = None
    status = _status(status, dev)
    _lib.require_cuda(pages, "pages")
    with torch.cuda.device(dev):
        _lib.check(getattr(_lib.lib(), entry)(
            pages.data_ptr(), pages.stride(0), pages.stride(1), pages.shape[0], page, slots.data_ptr(), k.data_ptr(), *k.stride()[:2],
            v.data_ptr(), *v.stride()[:2], _lib.ptr(q), *qs, _lib.ptr(q_out) if q is not None else 0, *rope, n, n_kv, n_q, flags,
            status, _lib.stream_ptr(dev)), entry)
    _lib.count_launch(_lib.lib().bgtq_paged_launches())
    return q_out


def paged_kv4_read(pages, slots, dtype=torch.float16, status=None):
    """The keys and values that the cache holds for ``slots`` (n,) int64: two tensors (n, n_kv, 128) of fp16 (exact), fp32
    (exact) or bf16.  A negative slot reads as zeros, and so does one out of range, with 2 in ``status``."""
    kind = _KINDS.get(dtype)
    host = _lib.host()
    r = None if kind is None else host.paged_read(pages, slots, kind, status)
    if r is None:
        return _read(pages, slots, dtype, status)
    return _lib.done(r, "bgtq_paged_read", host.paged_launched())


@torch.no_grad()
def _read(pages, slots, dtype, status):
    page = _pool(pages)
    dev, n_kv = pages.device, pages.shape[1]
    if dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError(f"dtype must be float16, bfloat16 or float32, got {dtype}")
    slots = _ints(slots, "slots", torch.int64, (slots.shape[0] if slots.dim() else 0,), dev)
    n, status = slots.shape[0], _status(status, dev)
    _lib.require_cuda(pages, "pages")
    k, v = (torch.empty(n, n_kv, HD, dtype=dtype, device=dev) for _ in range(2))
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().bgtq_paged_read(
            pages.data_ptr(), pages.stride(0), pages.stride(1), pages.shape[0], page, slots.data_ptr(), n, n_kv, k.data_ptr(), v.data_ptr(),
            _lib.PAGED_F32 if dtype == torch.float32 else _TYPES[dtype], status, _lib.stream_ptr(dev)), "bgtq_paged_read")
    _lib.count_launch(_lib.lib().bgtq_paged_launches())
    return k, v


def paged_kv4_copy(pages, src, dst, n_tokens=None, into=None):
    """Page ``dst[i]`` becomes page ``src[i]``, in every layer: ``pages`` (layers, n_pages, n_kv, page bytes) uint8, or one layer's
    (n_pages, n_kv, page bytes).

    ``src`` and ``dst`` are page numbers on the host (lists, or CPU tensors): no page is copied to twice, nor both copied to and from; one may be copied from
    many times.  ``n_tokens``, one number for each pair: only the units of 16 tokens that hold the page's first so many tokens are copied.  ``into``:
    another pool, of the same layers, heads and page size and apart from this one, that ``dst`` are pages of."""
    host = _lib.host()
    if pages.dim() == 3:
        r = host.paged_copy(pages.unsqueeze(0), src, dst, n_tokens, into if into is None or into.dim() == 4 else into.unsqueeze(0))
    else:
        r = host.paged_copy(pages, src, dst, n_tokens, into)
    if r is None:
        return _copy(pages, src, dst, n_tokens, into)
    _lib.done(r, "bgtq_paged_copy", host.paged_launched())


def _numbers(x, name):
    if isinstance(x, torch.Tensor):
        if x.is_cuda:
            raise ValueError(f"{name} must be numbers on the host: the call reads them before it returns")
        if x.dim() != 1 or x.is_floating_point() or x.is_complex() or x.dtype == torch.bool:
            raise ValueError(f"{name} must be whole numbers, one behind the other, got {x.dtype} {tuple(x.shape)}")
        return x.tolist()
    return [operator.index(i) for i in x]


def _copy(pages, src, dst, n_tokens, into):
    to, size = pages if into is None else into, None
    for x in (pages, to):
        if x.dtype != torch.uint8 or x.dim() not in (3, 4):
            raise ValueError("pages must be uint8 (layers, n_pages, n_kv, page bytes) or (n_pages, n_kv, page bytes)")
    if pages.dim() == 3:
        pages = pages.unsqueeze(0)
    to = pages if into is None else to.unsqueeze(0) if to.dim() == 3 else to
    for x in (pages, to):
        if x.shape[0] < 1:
            raise ValueError("pages of no layers")
        size = _pool(x[0])
        if x.stride(0) % 16:
            raise ValueError("pages must have rows whose addresses are multiples of 16 bytes")
    if to.device != pages.device or to.shape[0] != pages.shape[0] or to.shape[2:] != pages.shape[2:]:
        raise ValueError(f"into must have the layers, heads, page size and device of pages, got {tuple(to.shape)} on {to.device} for "
                         f"{tuple(pages.shape)} on {pages.device}")
    src, dst = _numbers(src, "src"), _numbers(dst, "dst")
    if len(src) != len(dst):
        raise ValueError(f"{len(src)} pages to copy from, {len(dst)} to copy to")
    for x, name, n in ((src, "src", pages.shape[1]), (dst, "dst", to.shape[1])):
        if x and not 0 <= min(x) <= max(x) < n:
            raise ValueError(f"{name} must be numbers of the pool's {n} pages")
    if len(set(dst)) != len(dst):
        raise ValueError("a page is copied to once")
    if into is None and not set(dst).isdisjoint(src):
        raise ValueError("a page is not both copied to and from")
    if n_tokens is not None:
        n_tokens = _numbers(n_tokens, "n_tokens")
        if len(n_tokens) != len(src) or (n_tokens and not 0 <= min(n_tokens) <= max(n_tokens) <= size):
            raise ValueError(f"n_tokens must be a number of 0 to {size} tokens for each pair")
    _lib.require_cuda(pages, "pages")
    if not src:
        return
    lib, n = _lib.lib(), len(src)
    with torch.cuda.device(pages.device):
        rc = lib.bgtq_paged_copy(
            pages.data_ptr(), *pages.stride()[:3], pages.shape[1], to.data_ptr(), *to.stride()[:3], to.shape[1], size, pages.shape[0], pages.shape[2],
            (C.c_int32 * n)(*src), (C.c_int32 * n)(*dst), None if n_tokens is None else (C.c_int32 * n)(*n_tokens), n,
            _lib.stream_ptr(pages.device))
    if rc == -1:                            # (all else has been looked at)
        raise ValueError("the pages that are copied to must lie apart from one another, and a pool from the one that it is copied into")
    _lib.check(rc, "bgtq_paged_copy")
    _lib.count_launch(lib.bgtq_paged_launches())


def _attend(q, pages, block_table, seq_lens, cu_q, max_q, max_tokens, causal, scale, return_lse, status, out, softcap, slopes, window, prefix_lens, max_prefix):
    scale = _SCALE if scale is None else float(scale)
    flags = (_lib.PAGED_CAUSAL if causal else 0) | _FORM << _lib.PAGED_FORM_SHIFT
    host = _lib.host()
    if softcap is None and slopes is None and window is None and prefix_lens is None:
        scored = False
        r = host.paged_attend(q, pages, block_table, seq_lens, cu_q, max_q, max_tokens, scale, flags, return_lse, status, out)
    else:
        scored = True
        r = host.paged_attend(q, pages, block_table, seq_lens, cu_q, max_q, max_tokens, scale, flags, return_lse, status, out, slopes, prefix_lens, softcap,
                              window, max_prefix)
    if r is None:
        scores = (slopes, prefix_lens, *_limits(softcap, window, causal), _most(max_prefix, "max_prefix_len")) if scored else None
        return _attend_any(q, pages, block_table, seq_lens, cu_q, max_q, max_tokens, flags, scale, return_lse, status, out, scores)
    return _lib.done(r, "bgtq_paged_attend", host.paged_launched())


def _limits(softcap, window, causal):
    """The cap and the window as numbers, 0 for none."""
    if softcap is None:
        softcap = 0.0
    else:
        softcap = float(softcap)
        if not 2.0 ** -64 <= softcap <= 2.0 ** 64:
            raise ValueError(f"softcap must be positive, 2^-64 to 2^64, got {softcap}")
    if window is None:
        return softcap, 0
    window = operator.index(window)
    if window < 1:
        raise ValueError(f"window must be at least one token, got {window}")
    if not causal:
        raise ValueError("a window is counted back from a row's own position: causal attention only")
    return softcap, min(window, 2 ** 31 - 1)


@torch.no_grad()
def _attend_any(q, pages, block_table, seq_lens, cu_q, max_q, max_tokens, flags, scale, return_lse, status, out, scores):
    """The attention for what the extension module leaves: tensors that have to be copied, empty ones, and errors."""
    page = _pool(pages)
    dev, n_kv = pages.device, pages.shape[1]
    flags |= _type_flag(q.dtype, "q")
    given, q = q, _rows(q, "q", None, None, q.dtype, dev, 16)
    n, n_q = q.shape[:2]
    if n_q < 1 or n_q % n_kv or n_q // n_kv > 8:
        raise ValueError(f"{n_q} query heads over {n_kv} KV heads: a KV head takes 1 to 8 of them")
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.device != dev:
        raise ValueError(f"block_table must be int32 (sequences, pages) on {dev}")
    n_seq = block_table.shape[0]
    if block_table.stride(1) != 1:
        block_table = block_table.contiguous()
    seq_lens = _ints(seq_lens, "seq_lens", torch.int32, (n_seq,), dev)
    if cu_q is None:
        if n != n_seq:
            raise ValueError(f"{n} queries for {n_seq} sequences")
    else:
        cu_q = _ints(cu_q, "cu_q", torch.int32, (n_seq + 1,), dev)
    if out is None:
        out = torch.empty(n, n_q, HD, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or out.stride(2) != 1 or out.stride(0) % 4 or out.stride(1) % 4 \
            or out.data_ptr() % 8:
        raise ValueError("out must be like q, with rows of 8-byte alignment")
    elif not _apart(out) or not _rows_clear(given, out):
        raise ValueError("out must have rows of its own, apart from one another and from q")
    lse = torch.empty(n, n_q, dtype=torch.float32, device=dev) if return_lse else None
    cap = block_table.shape[1] * page
    max_tokens = cap if max_tokens < 0 else min(max_tokens, cap)
    if math.isnan(scale):
        raise ValueError("scale is not a number")
    sc = None
    if scores is not None:
        slopes, prefix, softcap, window, longest = scores
        if slopes is not None:
            slopes = _ints(slopes, "slopes", torch.float32, (n_q,), dev)
        if prefix is not None:
            prefix = _ints(prefix, "prefix_lens", torch.int32, (n_seq,), dev)
        sc = _lib.PagedScores(_lib.ptr(slopes) or None, _lib.ptr(prefix) or None, softcap, window, max_tokens if longest < 0 else min(longest, max_tokens), 0)
    status, lib = _status(status, dev), _lib.lib()
    _lib.require_cuda(pages, "pages")
    if n and n_seq:
        with torch.cuda.device(dev):
            need = lib.bgtq_paged_scored_workspace_bytes(n_seq, n, n_q, n_kv, max_q, max_tokens, flags, sc)
            if need < 0:
                _lib.check(need, "bgtq_paged_workspace_bytes")
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            _lib.check(lib.bgtq_paged_attend_scored(
                q.data_ptr(), *q.stride()[:2], pages.data_ptr(), pages.stride(0), pages.stride(1), pages.shape[0], page,
                block_table.data_ptr(), block_table.stride(0), block_table.shape[1], seq_lens.data_ptr(), _lib.ptr(cu_q), n_seq, n, n_q, n_kv,
                max_q, max_tokens, scale, flags, sc, ws.data_ptr(), need, out.data_ptr(), *out.stride()[:2], _lib.ptr(lse), status,
                _lib.stream_ptr(dev)), "bgtq_paged_attend")
        _lib.count_launch(lib.bgtq_paged_launches())
    return (out, lse) if return_lse else out


def paged_kv4_decode_attention(q, pages, block_table, seq_lens, scale=None, return_lse=False, status=None, out=None, max_seq_len=None, *,
                               softcap=None, slopes=None, window=None, prefix_lens=None, max_prefix_len=None):
    """One query token of every sequence over its cached tokens: q (B, n_q, 128) fp16 or bf16 -> (B, n_q, 128) of the same type,
    with ``return_lse`` also (B, n_q) fp32, the natural logarithm of each row's sum of exponentials.

    ``block_table`` (B, pages per sequence) int32 and ``seq_lens`` (B,) int32: token t of sequence b lies in page ``block_table[b, t // page
    size]``; entries behind the sequence's end are not read.  A sequence without tokens gives zeros and -inf.  Query heads
    h * n_q / n_kv .. share KV head h, at most 8 of them.  ``max_seq_len``: sequences are held to it (default: what the table holds);
    a small one spares the launch what only long sequences need.  ``out``: where the result goes, like q, its rows apart from one
    another and from q's (other columns of one buffer will do).

    Layers that are no plain attention: ``softcap`` c: a logit x becomes c tanh(x / c).  ``slopes`` (n_q,) fp32, finite (negative ones times any
    distance, too): less slope times the distance between the query's position (the sequence's last) and the token's.  ``window``: of the tokens up to the
    query's own only the last so many are seen.
    ``prefix_lens`` (B,) int32: a sequence's first so many tokens are seen in any case (sinks in front of a window); ``max_prefix_len``: they are held
    to it (default: ``max_seq_len``), and with a window it chooses the launch: pass it with sinks, or the call is launched as if there were no window.  Pages that
    no query sees are not read."""
    return _attend(q, pages, block_table, seq_lens, None, 1, _most(max_seq_len), True, scale, return_lse, status, out, softcap, slopes, window, prefix_lens,
                   max_prefix_len)


def paged_kv4_prefill_attention(q, pages, block_table, seq_lens, cu_q, max_q_len=None, max_seq_len=None, causal=True, scale=None,
                                return_lse=False, status=None, out=None, *, softcap=None, slopes=None, window=None, prefix_lens=None,
                                max_prefix_len=None):
    """Several query tokens of every sequence over its cached tokens, their own among them: q (n, n_q, 128), rows ``cu_q[b]`` ..
    ``cu_q[b + 1] - 1`` (``cu_q`` (B + 1,) int32) are the last positions of sequence b, and when ``causal`` each sees the tokens up to itself.

    ``max_q_len``: no sequence has more query rows (default: all of them; it chooses the launch, 0 the one of 1, and one that has
    more is attended all the same).  ``max_seq_len``: sequences are held to it (default: what the table holds).  With many rows per sequence and KV head the
    tokens are unpacked into a workspace from torch's allocator, 512 bytes per token of ``max_seq_len`` and KV head for every sequence, at
    most 2 GiB at a time (with a ``window`` for every sequence ``max_prefix_len`` tokens and what the windows of all the call's rows together reach, where that
    is less).  Rows behind ``cu_q[B]`` are not written.  Otherwise as :func:`paged_kv4_decode_attention`: distances and the ``window`` (``causal`` only)
    count from the row's own position, and tokens of the prefix are seen by the rows in front of them too, at the distance between them."""
    if cu_q is None:
        raise ValueError("cu_q says which rows are whose")
    if max_q_len is not None and max_q_len < 0:
        raise ValueError("max_q_len must not be negative")
    rows = q.shape[0]
    max_q = max(1, rows if max_q_len is None else min(int(max_q_len), rows))
    return _attend(q, pages, block_table, seq_lens, cu_q, max_q, _most(max_seq_len), causal, scale, return_lse, status, out, softcap, slopes, window,
                   prefix_lens, max_prefix_len)


def _most(n, name="max_seq_len"):
    if n is None:
        return -1
    if n < 0:
        raise ValueError(f"{name} must not be negative")
    return int(n)


class PagedKV4Cache:
    """The pages of a model's layers, and which sequence holds which of them.

    A step is :meth:`begin_step` with the sequences that get new tokens and how many each, then
    :meth:`append_and_attend` once per layer with the tokens' rows one sequence behind the other.  What a step needs on the device
    (slots, positions, block table, lengths) is uploaded once and is the same for every layer.

    Sequences may share pages: :meth:`fork_sequence` makes one that begins with another's tokens and copies nothing.  A shared page is copied, in all
    layers, by the step that would write into it (on the stream of :meth:`begin_step`), and goes back to the pool with the last sequence that holds it.

    Copies wait for the layers of all streams, and steps and layers for the copies, whatever streams they are on.  Layers on several streams are the caller's to
    order otherwise, also where a page that one sequence gave back is another's next."""

    def __init__(self, n_layers, n_q_heads, n_kv_heads, head_dim=HD, *, n_pages, max_seq_len, page_size=64, device="cuda"):
        if head_dim != HD:
            raise ValueError(f"head_dim must be {HD}")
        if n_kv_heads < 1 or n_q_heads % n_kv_heads or not 1 <= n_q_heads // n_kv_heads <= 8:
            raise ValueError(f"{n_q_heads} query heads over {n_kv_heads} KV heads: a KV head takes 1 to 8 of them")
        self.n_layers, self.nq, self.nkv, self.hd, self.page_size = n_layers, n_q_heads, n_kv_heads, head_dim, page_size
        self.n_pages, self.max_seq_len, self.device = n_pages, max_seq_len, torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.pages = torch.zeros(n_layers, n_pages, n_kv_heads, page_bytes(page_size), dtype=torch.uint8, device=self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._free = list(range(n_pages - 1, -1, -1))
        self._held = [0] * n_pages          # sequences that hold a page
        self._seqs = {}                     # id -> [tokens, [pages, None: released]]
        self._gaps = set()                  # sequences that may have released pages (in all others none is looked for)
        self._next_id = 0
        self._step = None
        self._busy = set()                  # streams that layers have run on since pages were last copied
        self._copied = None                 # the event behind the last copies

    # ---- sequences -----------------------------------------------------------
    def add_sequence(self) -> int:
        """A new, empty sequence."""
        i = self._next_id
        self._next_id += 1
        self._seqs[i] = [0, []]
        return i

    def fork_sequence(self, seq: int, n_tokens=None) -> int:
        """A new sequence that begins with the first ``n_tokens`` (default: all) of another's tokens, in the same pages."""
        n, pages = self._first(seq, self._seqs[seq][0] if n_tokens is None else n_tokens)
        i = self.add_sequence()
        self._seqs[i] = [n, pages]
        if seq in self._gaps:
            self._gaps.add(i)
        for p in pages:
            if p is not None:
                self._held[p] += 1
        return i

    def truncate_sequence(self, seq: int, n_tokens: int):
        """Leaves the sequence its first ``n_tokens`` tokens, and gives the pages behind them back.  A step that it is part of ends with it."""
        n, pages = self._first(seq, n_tokens)
        behind = self._seqs[seq][1][len(pages):]
        self._seqs[seq] = [n, pages]
        self._let_go(behind)
        self._end_step(seq)

    def _first(self, seq, n_tokens):
        """A number of a sequence's first tokens, checked, and the pages that they are in."""
        t, pages = self._seqs[seq]
        n = operator.index(n_tokens)
        if not 0 <= n <= t:
            raise ValueError(f"sequence {seq} has {t} tokens, not {n}")
        pages = pages[:-(-n // self.page_size)]
        if n % self.page_size and pages[-1] is None:
            raise ValueError(f"the page that holds token {n - 1} of sequence {seq} has been released")
        return n, pages

    def release(self, seq: int, n_tokens: int, keep: int = 0):
        """Gives back the pages that lie as a whole behind the sequence's first ``keep`` tokens and in front of token ``n_tokens``: for models all of whose layers
        look through a window (with a prefix of up to ``keep`` tokens) that does not reach them any more.  An attention that sees one of their tokens is told
        of by :meth:`check_status`.  A step that the sequence is part of ends with it."""
        t, pages = self._seqs[seq]
        n, keep = operator.index(n_tokens), operator.index(keep)
        if not 0 <= n <= t or keep < 0:
            raise ValueError(f"sequence {seq} has {t} tokens: none of the first {n}, but for {keep}, can be released")
        gone = range(-(-keep // self.page_size), n // self.page_size)
        self._seqs[seq] = [t, [None if i in gone else p for i, p in enumerate(pages)]]
        self._gaps.add(seq)
        self._let_go([pages[i] for i in gone])
        self._end_step(seq)

    def free_sequence(self, seq: int):
        """Gives the sequence's pages back.  A step that it is part of ends with it."""
        self._let_go(self._seqs.pop(seq)[1])
        self._gaps.discard(seq)
        self._end_step(seq)

    def _let_go(self, pages):
        for p in reversed(pages):
            if p is None:
                continue
            self._held[p] -= 1
            if self._held[p] == 0:
                self._free.append(p)

    def _end_step(self, seq):
        if self._step is not None and seq in self._step["seqs"]:
            self._step = None

    def compact(self) -> int:
        """Moves the pages that sequences hold to the front of the pool, on the current stream, and returns how many they are.  The step ends."""
        self._not_captured()
        n = self.n_pages - len(self._free)
        places = sorted(p for p in self._free if p < n)
        moved = dict(zip((p for p in range(n, self.n_pages) if self._held[p]), places))
        if moved:
            self._copy(list(moved), list(moved.values()))
        self._renumber(moved, n, self.n_pages)
        return n

    def resize(self, n_pages: int):
        """Gives the pool another number of pages, no fewer than sequences hold; those come first, as after :meth:`compact`.  The step ends.  Waits for the
        device: nothing may be reading the old pool when it is given back."""
        self._not_captured()
        n, n_pages = self.n_pages - len(self._free), operator.index(n_pages)
        if n_pages < max(1, n):
            raise ValueError(f"{n} pages are held, more than {n_pages}" if n else "a pool has at least one page")
        held = [p for p in range(self.n_pages) if self._held[p]]
        pages = torch.zeros(self.n_layers, n_pages, *self.pages.shape[2:], dtype=torch.uint8, device=self.device)
        if held:
            self._copy(held, list(range(n)), into=pages)
        if self.device.type == "cuda":
            torch.cuda.synchronize(self.device)
        self.pages = pages
        self._renumber(dict(zip(held, range(n))), n, n_pages)

    def _renumber(self, moved, n, n_pages):
        for entry in self._seqs.values():
            entry[1] = [moved.get(p, p) for p in entry[1]]
        held = [0] * n_pages
        for p, h in enumerate(self._held):
            if h:
                held[moved.get(p, p)] = h
        self._held, self._free, self.n_pages, self._step = held, list(range(n_pages - 1, n - 1, -1)), n_pages, None

    def _copy(self, src, dst, **kw):
        """Copies pages on the current stream, behind the copies and the layers of every stream; steps and layers that follow on another one wait for it."""
        stream = self._stream()
        if self._copied is not None:        # (and so the last copies' event stands for all of them)
            stream.wait_event(self._copied)
        for other in self._busy:
            if other != stream:
                stream.wait_stream(other)
        paged_kv4_copy(self.pages, src, dst, **kw)
        if stream is not None:
            self._busy, self._copied = set(), stream.record_event()

    def _not_captured(self):
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a captured graph would go on moving the pages that are held now")

    def seq_len(self, seq: int) -> int:
        return self._seqs[seq][0]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def cache_memory_bytes(self) -> int:
        """Bytes of the pages that sequences hold, all layers."""
        return (self.n_pages - len(self._free)) * self.n_layers * self.nkv * page_bytes(self.page_size)

    # ---- a step --------------------------------------------------------------
    def begin_step(self, seqs, counts):
        """Makes room for ``counts[i]`` >= 1 new tokens of sequence ``seqs[i]`` (distinct); their rows follow one another in that order.
        Either every sequence gets its room or none does.  Pages that others hold too and that the step would write into are copied first."""
        seqs, counts = list(seqs), [int(c) for c in counts]
        if not seqs or len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or min(counts) < 1:
            raise ValueError("begin_step takes distinct sequences and a count of at least one token for each")
        need, parted, left = [], [], {}     # pages; sequences that get a copy of their last one; who holds that then
        for i, c in zip(seqs, counts):
            if i not in self._seqs:
                raise KeyError(f"no sequence {i}")
            t, held = self._seqs[i]
            if t + c > self.max_seq_len:
                raise ValueError(f"sequence {i} would have {t + c} tokens, more than {self.max_seq_len}")
            last = held[-1] if t % self.page_size else None
            parted.append(last is not None and left.get(last, self._held[last]) > 1)
            if parted[-1]:
                left[last] = left.get(last, self._held[last]) - 1
            need.append(-(-(t + c) // self.page_size) - len(held) + parted[-1])
        if sum(need) > len(self._free):
            raise RuntimeError(f"{sum(need)} pages needed, {len(self._free)} free")
        free = len(self._free)              # pages are taken from the end
        slots, positions, lens, ends, rows, copies = [], [], [], [0], [], []
        for i, c, n, part in zip(seqs, counts, need, parted):
            t, held = self._seqs[i]
            pages = (held[:-1] if part else held) + [self._free[free - 1 - k] for k in range(n)]
            if part:
                copies.append((held[-1], pages[len(held) - 1], t % self.page_size))
            free -= n
            at = range(t, t + c)
            positions.extend(at)
            slots.extend(pages[t // self.page_size] * self.page_size + t % self.page_size for t in at)
            lens.append(t + c)
            ends.append(ends[-1] + c)
            rows.append(pages)
        width = max(len(r) for r in rows)
        wide = torch.tensor([slots, positions], dtype=torch.int64).to(self.device)
        # (a step's time on the host goes with its table: 64 sequences of 4500 tokens in pages of 16 1.36 ms, 1.51 if each number were looked at)
        numbers = [[-1 if p is None else p for p in r] if i in self._gaps else r for i, r in zip(seqs, rows)]
        table = torch.tensor([r + [0] * (width - len(r)) for r in numbers], dtype=torch.int32).to(self.device)
        small = torch.tensor(lens + ends, dtype=torch.int32).to(self.device)
        if copies:
            self._not_captured()
            src, dst, n_tokens = (list(x) for x in zip(*copies))
            self._copy(src, dst, n_tokens=n_tokens)
        # (from here on nothing fails: a device without memory for the step leaves the sequences as they were)
        for i, t, pages in zip(seqs, lens, rows):
            self._seqs[i] = [t, pages]
        for p in self._free[free:]:
            self._held[p] = 1
        for src, _, _ in copies:
            self._held[src] -= 1
        del self._free[free:]
        if self._copied is not None:        # (pages may have been moved on another stream; other streams wait at their first layer)
            self._stream().wait_event(self._copied)
        self._step = {"slots": wide[0], "positions": wide[1], "table": table, "lens": small[:len(seqs)], "ends": small[len(seqs):],
                      "most_q": max(counts), "most": max(lens), "rows": len(slots), "seqs": frozenset(seqs),
                      "held": (wide, table, small), "streams": {self._stream()}}

    def _stream(self):
        return torch.cuda.current_stream(self.device) if self.device.type == "cuda" else None

    @torch.no_grad()
    def append_and_attend(self, layer_idx, q, k, v, rope=None, *, positions=None, axes=None, softcap=None, slopes=None, window=None,
                          prefix_lens=None, max_prefix_len=None):
        """The step's rows of one layer: k, v (n, n_kv, 128) are stored, q (n, n_q, 128) attends, causally, its own sequence ->
        (n, n_q, 128).  ``rope=(cos, sin)``, tables (positions, 64) fp32: q and k go through the rotary embedding first, at the tokens' places in
        their sequences, or at ``positions`` (n,) int64, or (axes, n) with ``axes`` as :func:`paged_kv4_append` takes them.  ``softcap``,
        ``slopes``, ``window``, ``prefix_lens`` (one for each of the step's sequences, in its order) and ``max_prefix_len`` are the attention's."""
        if self._step is None:
            raise RuntimeError("begin_step comes first")
        s, pages = self._step, self.pages[layer_idx]
        if q.shape != (s["rows"], self.nq, HD):
            raise ValueError(f"q must be ({s['rows']}, {self.nq}, {HD}), the step's tokens, got {tuple(q.shape)}")
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a captured graph would go on reading this step's slots and lengths, which end with the step: capture "
                               "paged_kv4_append and the attentions over tensors of your own")
        scores = dict(softcap=softcap, slopes=slopes, window=window, prefix_lens=prefix_lens, max_prefix_len=max_prefix_len)
        # (nothing is stored for an attention that is refused)
        _type_flag(q.dtype, "q")
        if q.device != self.device:
            raise ValueError(f"q is on {q.device}, the pages on {self.device}")
        if softcap is not None or slopes is not None or window is not None or prefix_lens is not None:
            _limits(softcap, window, True)
            if slopes is not None:
                _is(slopes, "slopes", torch.float32, (self.nq,), self.device)
            if prefix_lens is not None:     # (one for each of the step's sequences)
                _is(prefix_lens, "prefix_lens", torch.int32, tuple(s["lens"].shape), self.device)
            if max_prefix_len is not None:
                _most(operator.index(max_prefix_len), "max_prefix_len")
        stream = self._stream()
        if stream not in s["streams"]:      # (the next step's tensors must not take these tensors' memory before this stream is done with them)
            for t in s["held"]:
                t.record_stream(stream)
            s["streams"].add(stream)
            if self._copied is not None:
                stream.wait_event(self._copied)
        self._busy.add(stream)
        if rope is None:
            if positions is not None or axes is not None:
                raise ValueError("positions and axes belong to rope")
            paged_kv4_append(pages, s["slots"], k, v, status=self.status)
        else:
            if axes is not None and positions is None:
                raise ValueError("axes belong to positions")
            q = paged_kv4_append(pages, s["slots"], k, v, q=q, cos=rope[0], sin=rope[1], positions=s["positions"] if positions is None else positions,
                                 status=self.status, axes=axes)
        if s["most_q"] == 1:
            return paged_kv4_decode_attention(q, pages, s["table"], s["lens"], status=self.status, **scores)
        return paged_kv4_prefill_attention(q, pages, s["table"], s["lens"], s["ends"], max_q_len=s["most_q"], max_seq_len=s["most"],
                                           status=self.status, **scores)

    def check_status(self):
        """Raises when a launch since the last call, on whatever stream, reported an error (synchronises the device)."""
        if self.device.type == "cuda":
            torch.cuda.synchronize(self.device)
        code = int(self.status.item())
        self.status.zero_()
        if code:
            raise RuntimeError({1: "a kernel's wait ran out", 2: "a slot or position was out of range", 4: "a page number was out of range"}
                               .get(code, f"status {code}"))
