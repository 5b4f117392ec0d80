"""A paged key/value cache in 4 bits, for batches whose sequences have lengths of their own.

The reference's caches are contiguous, of one length for the whole batch, and calibrated per head; this one needs
neither, and a sequence's tokens lie in whatever pages are free.  A token's K and V rows are quantised by themselves: four
groups of 32 dims, each with a bf16 scale and signed codes of 4 bits (4.5 bits per value).  ``include/bgtq.h`` has the layout
of a page.  The functions are the operators; :class:`PagedKV4Cache` keeps the pages of a model's layers and
hands them out to sequences.
"""
from __future__ import annotations

import math

import torch

from . import _lib

__all__ = ["PAGE_UNIT_BYTES", "page_bytes", "paged_kv4_append", "paged_kv4_read", "paged_kv4_decode_attention",
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


def _ints(x, name, dtype, shape, device):
    if x.dtype != dtype or tuple(x.shape) != shape:
        raise ValueError(f"{name} must be {dtype} {shape}, got {x.dtype} {tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, the pages on {device}")
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


def paged_kv4_append(pages, slots, k, v, q=None, cos=None, sin=None, positions=None, status=None):
    """Quantise k and v (n, n_kv, 128) fp16 or bf16 into the slots of ``pages`` (n_pages, n_kv, page bytes) uint8.

    ``slots`` (n,) int64: page * page size + place in the page, distinct; a token with a negative one is not stored.
    ``cos`` / ``sin`` (n_positions, 64) fp32 with ``positions`` (n,) int64: k, and ``q`` (n, n_q, 128), go through the rotary
    embedding first (dims d and d + 64 are a pair; fp32, k quantised from the unrounded result).  Returns the rotated q (n, n_q, 128),
    or None without one.  ``status``: optional int32 tensor, set to 2 where a slot or position is out of range (the token is not stored)."""
    host = _lib.host()
    r = host.paged_append(pages, slots, k, v, q, cos, sin, positions, status)
    if r is None:
        return _append(pages, slots, k, v, q, cos, sin, positions, status)
    _lib.done(r, "bgtq_paged_append", host.paged_launched())
    return None if q is None else r


@torch.no_grad()
def _append(pages, slots, k, v, q, cos, sin, positions, status):
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
    n_q, q_out, qs, rope = 0, None, (0, 0), (None, None, 0, None, 0)
    if cos is not None:
        if cos.dim() != 2 or cos.shape[1] != HD // 2 or cos.shape[0] < 1 or sin.shape != cos.shape:
            raise ValueError(f"cos and sin must be (positions, {HD // 2}), got {tuple(cos.shape)} and {tuple(sin.shape)}")
        if cos.dtype != torch.float32 or sin.dtype != torch.float32:
            raise TypeError("cos and sin must be float32")
        if cos.device != dev or sin.device != dev:
            raise ValueError(f"cos and sin must be on {dev}")
        if cos.stride(1) != 1 or cos.stride(0) % 4 or sin.stride() != cos.stride() or (cos.data_ptr() | sin.data_ptr()) % 16:
            cos, sin = (x.clone(memory_format=torch.contiguous_format) for x in (cos, sin))
        positions = _ints(positions, "positions", torch.int64, (n,), dev)
        rope = (cos.data_ptr(), sin.data_ptr(), cos.stride(0), positions.data_ptr(), cos.shape[0])
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
        _lib.check(_lib.lib().bgtq_paged_append(
            pages.data_ptr(), pages.stride(0), pages.stride(1), pages.shape[0], page, slots.data_ptr(), k.data_ptr(), *k.stride()[:2],
            v.data_ptr(), *v.stride()[:2], _lib.ptr(q), *qs, _lib.ptr(q_out) if q is not None else 0, *rope, n, n_kv, n_q, flags,
            status, _lib.stream_ptr(dev)), "bgtq_paged_append")
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


def _attend(q, pages, block_table, seq_lens, cu_q, max_q, max_tokens, causal, scale, return_lse, status, out):
    scale = _SCALE if scale is None else float(scale)
    flags = (_lib.PAGED_CAUSAL if causal else 0) | _FORM << _lib.PAGED_FORM_SHIFT
    host = _lib.host()
    r = host.paged_attend(q, pages, block_table, seq_lens, cu_q, max_q, max_tokens, scale, flags, return_lse, status, out)
    if r is None:
        return _attend_any(q, pages, block_table, seq_lens, cu_q, max_q, max_tokens, flags, scale, return_lse, status, out)
    return _lib.done(r, "bgtq_paged_attend", host.paged_launched())


@torch.no_grad()
def _attend_any(q, pages, block_table, seq_lens, cu_q, max_q, max_tokens, flags, scale, return_lse, status, out):
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
    status, lib = _status(status, dev), _lib.lib()
    _lib.require_cuda(pages, "pages")
    if n and n_seq:
        with torch.cuda.device(dev):
            need = lib.bgtq_paged_workspace_bytes(n_seq, n, n_q, n_kv, max_q, max_tokens, flags)
            if need < 0:
                _lib.check(need, "bgtq_paged_workspace_bytes")
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            _lib.check(lib.bgtq_paged_attend(
                q.data_ptr(), *q.stride()[:2], pages.data_ptr(), pages.stride(0), pages.stride(1), pages.shape[0], page,
                block_table.data_ptr(), block_table.stride(0), block_table.shape[1], seq_lens.data_ptr(), _lib.ptr(cu_q), n_seq, n, n_q, n_kv,
                max_q, max_tokens, scale, flags, ws.data_ptr(), need, out.data_ptr(), *out.stride()[:2], _lib.ptr(lse), status,
                _lib.stream_ptr(dev)), "bgtq_paged_attend")
        _lib.count_launch(lib.bgtq_paged_launches())
    return (out, lse) if return_lse else out


def paged_kv4_decode_attention(q, pages, block_table, seq_lens, scale=None, return_lse=False, status=None, out=None, max_seq_len=None):
    """One query token of every sequence over its cached tokens: q (B, n_q, 128) fp16 or bf16 -> (B, n_q, 128) of the same type,
    with ``return_lse`` also (B, n_q) fp32, the natural logarithm of each row's sum of exponentials.

    ``block_table`` (B, pages per sequence) int32 and ``seq_lens`` (B,) int32: token t of sequence b lies in page ``block_table[b, t // page
    size]``; entries behind the sequence's end are not read.  A sequence without tokens gives zeros and -inf.  Query heads
    h * n_q / n_kv .. share KV head h, at most 8 of them.  ``max_seq_len``: sequences are held to it (default: what the table holds);
    a small one spares the launch what only long sequences need.  ``out``: where the result goes, like q, its rows apart from one
    another and from q's (other columns of one buffer will do)."""
    return _attend(q, pages, block_table, seq_lens, None, 1, _most(max_seq_len), True, scale, return_lse, status, out)


def paged_kv4_prefill_attention(q, pages, block_table, seq_lens, cu_q, max_q_len=None, max_seq_len=None, causal=True, scale=None,
                                return_lse=False, status=None, out=None):
    """Several query tokens of every sequence over its cached tokens, their own among them: q (n, n_q, 128), rows ``cu_q[b]`` ..
    ``cu_q[b + 1] - 1`` (``cu_q`` (B + 1,) int32) are the last positions of sequence b, and when ``causal`` each sees the tokens up to itself.

    ``max_q_len``: no sequence has more query rows (default: all of them; it chooses the launch, 0 the one of 1, and one that has
    more is attended all the same).  ``max_seq_len``: sequences are held to it (default: what the table holds).  With many rows per sequence and KV head the
    tokens are unpacked into a workspace from torch's allocator, 512 bytes per token of ``max_seq_len`` and KV head for every sequence, at
    most 2 GiB at a time.  Rows behind ``cu_q[B]`` are not written.  Otherwise as :func:`paged_kv4_decode_attention`."""
    if cu_q is None:
        raise ValueError("cu_q says which rows are whose")
    if max_q_len is not None and max_q_len < 0:
        raise ValueError("max_q_len must not be negative")
    rows = q.shape[0]
    max_q = max(1, rows if max_q_len is None else min(int(max_q_len), rows))
    return _attend(q, pages, block_table, seq_lens, cu_q, max_q, _most(max_seq_len), causal, scale, return_lse, status, out)


def _most(max_seq_len):
    if max_seq_len is None:
        return -1
    if max_seq_len < 0:
        raise ValueError("max_seq_len must not be negative")
    return int(max_seq_len)


class PagedKV4Cache:
    """The pages of a model's layers, and which sequence holds which of them.

    A step is :meth:`begin_step` with the sequences that get new tokens and how many each, then
    :meth:`append_and_attend` once per layer with the tokens' rows one sequence behind the other.  What a step needs on the device
    (slots, positions, block table, lengths) is uploaded once and is the same for every layer."""

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
        self._seqs = {}                     # id -> [tokens, [pages]]
        self._next_id = 0
        self._step = None

    # ---- sequences -----------------------------------------------------------
    def add_sequence(self) -> int:
        """A new, empty sequence."""
        i = self._next_id
        self._next_id += 1
        self._seqs[i] = [0, []]
        return i

    def free_sequence(self, seq: int):
        """Gives the sequence's pages back.  A step that it is part of ends with it."""
        self._free.extend(reversed(self._seqs.pop(seq)[1]))
        if self._step is not None and seq in self._step["seqs"]:
            self._step = None

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
        Either every sequence gets its room or none does."""
        seqs, counts = list(seqs), [int(c) for c in counts]
        if not seqs or len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or min(counts) < 1:
            raise ValueError("begin_step takes distinct sequences and a count of at least one token for each")
        need = []
        for i, c in zip(seqs, counts):
            if i not in self._seqs:
                raise KeyError(f"no sequence {i}")
            t, held = self._seqs[i]
            if t + c > self.max_seq_len:
                raise ValueError(f"sequence {i} would have {t + c} tokens, more than {self.max_seq_len}")
            need.append(-(-(t + c) // self.page_size) - len(held))
        if sum(need) > len(self._free):
            raise RuntimeError(f"{sum(need)} pages needed, {len(self._free)} free")
        free = len(self._free)              # pages are taken from the end
        slots, positions, lens, ends, rows = [], [], [], [0], []
        for i, c, n in zip(seqs, counts, need):
            t, held = self._seqs[i]
            pages = held + [self._free[free - 1 - k] for k in range(n)]
            free -= n
            at = range(t, t + c)
            positions.extend(at)
            slots.extend(pages[t // self.page_size] * self.page_size + t % self.page_size for t in at)
            lens.append(t + c)
            ends.append(ends[-1] + c)
            rows.append(pages)
        width = max(len(r) for r in rows)
        wide = torch.tensor([slots, positions], dtype=torch.int64).to(self.device)
        table = torch.tensor([r + [0] * (width - len(r)) for r in rows], dtype=torch.int32).to(self.device)
        small = torch.tensor(lens + ends, dtype=torch.int32).to(self.device)
        # (from here on nothing fails: a device without memory for the step leaves the sequences as they were)
        for i, t, pages in zip(seqs, lens, rows):
            self._seqs[i] = [t, pages]
        del self._free[free:]
        self._step = {"slots": wide[0], "positions": wide[1], "table": table, "lens": small[:len(seqs)], "ends": small[len(seqs):],
                      "most_q": max(counts), "most": max(lens), "rows": len(slots), "seqs": frozenset(seqs),
                      "held": (wide, table, small), "streams": {self._stream()}}

    def _stream(self):
        return torch.cuda.current_stream(self.device) if self.device.type == "cuda" else None

    @torch.no_grad()
    def append_and_attend(self, layer_idx, q, k, v, rope=None):
        """The step's rows of one layer: k, v (n, n_kv, 128) are stored, q (n, n_q, 128) attends, causally, its own sequence ->
        (n, n_q, 128).  ``rope=(cos, sin)``, tables (positions, 64) fp32: q and k go through the rotary embedding first."""
        if self._step is None:
            raise RuntimeError("begin_step comes first")
        s, pages = self._step, self.pages[layer_idx]
        if q.shape != (s["rows"], self.nq, HD):
            raise ValueError(f"q must be ({s['rows']}, {self.nq}, {HD}), the step's tokens, got {tuple(q.shape)}")
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a captured graph would go on reading this step's slots and lengths, which end with the step: capture "
                               "paged_kv4_append and the attentions over tensors of your own")
        stream = self._stream()
        if stream not in s["streams"]:      # (the next step's tensors must not take these tensors' memory before this stream is done with them)
            for t in s["held"]:
                t.record_stream(stream)
            s["streams"].add(stream)
        if rope is None:
            paged_kv4_append(pages, s["slots"], k, v, status=self.status)
        else:
            q = paged_kv4_append(pages, s["slots"], k, v, q=q, cos=rope[0], sin=rope[1], positions=s["positions"], status=self.status)
        if s["most_q"] == 1:
            return paged_kv4_decode_attention(q, pages, s["table"], s["lens"], status=self.status)
        return paged_kv4_prefill_attention(q, pages, s["table"], s["lens"], s["ends"], max_q_len=s["most_q"], max_seq_len=s["most"],
                                           status=self.status)

    def check_status(self):
        """Raises when a launch since the last call, on whatever stream, reported an error (synchronises the device)."""
        if self.device.type == "cuda":
            torch.cuda.synchronize(self.device)
        code = int(self.status.item())
        self.status.zero_()
        if code:
            raise RuntimeError({1: "a kernel's wait ran out", 2: "a slot or position was out of range", 4: "a page number was out of range"}
                               .get(code, f"status {code}"))
