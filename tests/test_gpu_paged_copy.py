"""GPU: copied pages byte for byte, and tokens appended with positions of several axes, bit for bit against plain operations."""
import random

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _pool(gen, *shape):
    return torch.randint(0, 256, shape, generator=gen, dtype=torch.uint8)


def _copied(pages, src, dst, n_tokens=None, into=None):
    """The bytes of `into` (or of pages) afterwards, (layers, pages, heads, bytes) on the CPU."""
    out = (pages if into is None else into).clone()
    for i, (a, b) in enumerate(zip(src, dst)):
        n = pages.shape[3] if n_tokens is None else -(-n_tokens[i] // 16) * R.UNIT_BYTES
        out[:, b, :, :n] = pages[:, a, :, :n]
    return out


@pytest.mark.parametrize("layers,heads,page,n_pages,pairs", [(1, 1, 16, 2, 1), (3, 2, 32, 9, 4), (2, 8, 64, 12, 5), (5, 3, 48, 30, 15), (1, 2, 16, 900, 450), (1, 1, 16, 6000, 2950)])
@pytest.mark.parametrize("whole", [True, False])
def test_pages_arrive_whole_and_nothing_else_changes(layers, heads, page, n_pages, pairs, whole):
    from blockgtq_b200 import page_bytes, paged_kv4_copy
    gen, rng = torch.Generator().manual_seed(pairs), random.Random(pairs)
    pages = _pool(gen, layers, n_pages, heads, page_bytes(page))
    order = rng.sample(range(n_pages), 2 * pairs)
    src, dst = order[:pairs], order[pairs:]
    if pairs > 1:
        src[1] = src[0]                                     # one page, copied twice
    tokens = None if whole else [rng.randint(0, page) for _ in src]
    if tokens and pairs > 2:
        tokens[:3] = 0, page, 1
    want = _copied(pages, src, dst, tokens)
    dev = pages.to(DEV)
    paged_kv4_copy(dev, src, dst, n_tokens=tokens)
    assert torch.equal(dev.cpu(), want)
    dev = pages.to(DEV)                                     # numbers in tensors, one layer's pages
    paged_kv4_copy(dev[0], torch.tensor(src), torch.tensor(dst, dtype=torch.int32), n_tokens=None if whole else torch.tensor(tokens))
    assert torch.equal(dev[0].cpu(), want[0]) and torch.equal(dev[1:].cpu(), pages[1:])


def test_pages_of_any_strides_and_of_another_pool():
    from blockgtq_b200 import page_bytes, paged_kv4_copy
    gen = torch.Generator().manual_seed(3)
    b = page_bytes(32)
    wide = _pool(gen, 3, 7, 6, b + 32)
    pages = wide[1:, :, 1:5, 16:16 + b]                     # some layers, some heads, rows with gaps
    into = _pool(gen, 2, 4, 4, b)
    src, dst, tokens = [6, 0, 3], [1, 3, 0], [32, 5, 17]
    for t in (None, tokens):
        dev, to = wide.to(DEV), into.to(DEV)
        paged_kv4_copy(dev[1:, :, 1:5, 16:16 + b], src, dst, n_tokens=t, into=to)
        assert torch.equal(to.cpu(), _copied(pages, src, dst, t, into)) and torch.equal(dev.cpu(), wide)
        paged_kv4_copy(dev[1:, :, 1:5, 16:16 + b], [1, 2], [4, 5], n_tokens=t and t[:2])
        want = wide.clone()
        want[1:, :, 1:5, 16:16 + b] = _copied(pages, [1, 2], [4, 5], t and t[:2])
        assert torch.equal(dev.cpu(), want)
        heads_first = torch.zeros(4, 2, 7, b, dtype=torch.uint8, device=DEV)              # (heads, layers, pages, bytes)
        paged_kv4_copy(dev[1:, :, 1:5, 16:16 + b], src, dst, n_tokens=t, into=heads_first.permute(1, 2, 0, 3))
        assert torch.equal(heads_first.permute(1, 2, 0, 3).cpu(), _copied(want[1:, :, 1:5, 16:16 + b], src, dst, t, torch.zeros(2, 7, 4, b, dtype=torch.uint8)))
    one, rows = dev[..., :b], dev.stride()
    for bad in (dict(pages=one[:2], into=one[1:]), dict(pages=one[:, :, :1].expand(-1, -1, 3, -1)), dict(pages=one.as_strided((3, 7, 6, b), (rows[0], 0, rows[2], 1)))):
        with pytest.raises(ValueError, match="apart"):      # layers of both; places that are one
            paged_kv4_copy(src=src, dst=dst if "into" in bad else [1, 2, 4], **bad)
    odd = torch.zeros(2 * 4 * b + 8, dtype=torch.uint8, device=DEV)[8:].view(1, 2, 4, b)
    with pytest.raises(ValueError, match="16 bytes"):
        paged_kv4_copy(odd, [0], [1])


def test_a_pool_of_more_than_four_gigabytes():
    from blockgtq_b200 import page_bytes, paged_kv4_copy
    b = page_bytes(128)
    pages = torch.empty(4, 9000, 8, b, dtype=torch.uint8, device=DEV)        # 5.3 GB
    gen = torch.Generator().manual_seed(9)
    for page in (0, 8999):
        pages[:, page] = _pool(gen, 4, 8, b).to(DEV)
    pages[:, 8998] = 0
    pages[:, 1] = 0
    paged_kv4_copy(pages, [0, 8999], [8998, 1], n_tokens=[128, 100])
    assert torch.equal(pages[:, 8998], pages[:, 0])
    assert torch.equal(pages[:, 1, :, :7 * 2304], pages[:, 8999, :, :7 * 2304]) and not pages[:, 1, :, 7 * 2304:].any()


def test_copies_on_another_stream_captured_and_counted():
    from blockgtq_b200 import _lib, page_bytes, paged_kv4_copy
    gen = torch.Generator().manual_seed(4)
    pages = _pool(gen, 2, 8, 2, page_bytes(16))
    dev, side = pages.to(DEV), torch.cuda.Stream(DEV)
    torch.cuda.synchronize()
    before = _lib.launches
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        paged_kv4_copy(dev, [0, 1], [4, 5])
        paged_kv4_copy(dev, [4], [6])                       # behind the first
        paged_kv4_copy(dev, [], [])
    assert _lib.launches - before == 2
    side.synchronize()
    want = _copied(_copied(pages, [0, 1], [4, 5]), [4], [6])
    assert torch.equal(dev.cpu(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_kv4_copy(dev, [2], [7], n_tokens=[3])
    assert torch.equal(dev.cpu(), want)
    dev[:, 2] = 77
    graph.replay()
    assert (dev[:, 7] == 77).all()


def _tables(n):
    angle = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    return angle.cos().float(), angle.sin().float()


def _rotated(x, cos, sin, positions, axes):
    """fp32, every product and sum rounded by itself."""
    pair = torch.arange(64)
    at = positions[torch.tensor(list(axes))].T
    c, s = cos[at, pair][:, None], sin[at, pair][:, None]
    a, b = x.float()[..., :64], x.float()[..., 64:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,n_kv,n_q,sections,interleaved", [
    (1, 1, 1, (16, 24, 24), False), (3, 2, 14, (24, 20, 20), True), (37, 8, 32, (16, 24, 24), False), (33, 3, 3, (1, 62, 1), False),
    (700, 8, 32, (16, 24, 24), False), (641, 8, 56, (16, 16, 16, 16), True), (5, 2, 4, (64,), False), (9, 2, 0, (31, 33), False), (700, 8, 8, (17, 0, 47), False)])
def test_several_axes_store_the_plain_quantisers_bytes(dtype, n, n_kv, n_q, sections, interleaved):
    from blockgtq_b200 import page_bytes, paged_kv4_append, rope_axes
    gen = torch.Generator().manual_seed(n)
    n_pages, page = -(-n // 32) + 2, 32
    slots = torch.randperm(n_pages * page, generator=gen)[:n]
    if n > 2:
        slots[1] = -1
    k, v, q = (torch.randn(n, h, 128, generator=gen).to(dtype) for h in (n_kv, n_kv, n_q))
    cos, sin = _tables(90)
    positions = torch.randint(0, 90, (len(sections), n), generator=gen)
    axes = rope_axes(sections, interleaved)
    pages = torch.randint(0, 256, (n_pages, n_kv, page_bytes(page)), generator=gen, dtype=torch.uint8)
    want, kr = pages.clone(), _rotated(k, cos, sin, positions, axes)
    for i in range(n):
        if slots[i] >= 0:
            R.write(want, int(slots[i]), kr[i], v[i].float())
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    wide = torch.cat([cos, sin], 1).to(DEV)
    spread = torch.zeros(len(sections), n + 3, dtype=torch.int64)
    spread[:, :n] = positions
    for turn, at, given in ((dict(cos=cos.to(DEV), sin=sin.to(DEV)), positions.to(DEV), axes),
                            (dict(cos=wide[:, :64], sin=wide[:, 64:]), spread.to(DEV)[:, :n], list(axes))):
        dev = pages.to(DEV)
        got = paged_kv4_append(dev, slots.to(DEV), k.to(DEV), v.to(DEV), q=q.to(DEV) if n_q else None, positions=at, axes=given, status=status, **turn)
        assert (dev.cpu() != want).sum() == 0 and status.item() == 0
        if n_q:
            assert torch.equal(got.cpu(), _rotated(q, cos, sin, positions, axes).to(dtype))
        else:
            assert got is None


@pytest.mark.parametrize("n", [1, 700])
@pytest.mark.parametrize("axis", [0, 1, 2])
def test_a_position_of_any_axis_outside_the_tables_leaves_its_token_out(n, axis):
    from blockgtq_b200 import page_bytes, paged_kv4_append, rope_axes
    cos, sin = (x.to(DEV) for x in _tables(4))
    rows = torch.ones(n, 8, 128, dtype=torch.float16, device=DEV)
    slots = torch.arange(n, device=DEV)
    for bad in (4, -1, 1 << 40):
        pages = torch.zeros(-(-n // 16), 8, page_bytes(16), dtype=torch.uint8, device=DEV)
        positions, status = torch.ones(3, n, dtype=torch.int64, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
        full = pages.clone()
        paged_kv4_append(full, slots, rows, rows, cos=cos, sin=sin, positions=positions, axes=rope_axes((16, 24, 24)), status=status)
        assert status.item() == 0
        positions[axis, n - 1] = bad
        paged_kv4_append(pages, slots, rows, rows, cos=cos, sin=sin, positions=positions, axes=rope_axes((16, 24, 24)), status=status)
        assert status.item() == 2
        # the token's V scales stay as they were, its neighbours' are there
        unit, t = pages[(n - 1) // 16].cpu(), (n - 1) % 16
        assert not unit[:, 64 * t:64 * t + 64].any() and not unit[:, 2176 + 8 * t:2184 + 8 * t].any()
        if n > 1:
            assert torch.equal(pages[:-1], full[:-1])
