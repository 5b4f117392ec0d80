"""CPU: what copying pages and positions of several axes refuse."""
import ctypes as C

import pytest
import torch

from blockgtq_b200 import _lib, page_bytes, paged_kv4_append, paged_kv4_copy, rope_axes


def _pool(layers=2, n=6, h=2, page=32):
    return torch.zeros(layers, n, h, page_bytes(page), dtype=torch.uint8)


def test_axes_of_sections():
    assert rope_axes((16, 24, 24)) == bytes([0] * 16 + [1] * 24 + [2] * 24)
    assert rope_axes([64]) == bytes(64)
    turns = rope_axes((24, 20, 20), interleaved=True)
    assert turns[:6] == bytes([0, 1, 2, 0, 1, 2]) and turns[60:] == bytes(4) and [turns.count(a) for a in range(3)] == [24, 20, 20]
    assert rope_axes((0, 64), interleaved=True) == bytes([1] * 64)
    for bad in ((16, 24), (16, 16, 16, 8, 8), (), (80, -16)):
        with pytest.raises(ValueError):
            rope_axes(bad)
    with pytest.raises(TypeError):
        rope_axes((32.0, 32.0))


@pytest.mark.parametrize("change,error", [
    (dict(axes=rope_axes((32, 32)), positions=torch.zeros(4, dtype=torch.int64)), ValueError),
    (dict(axes=rope_axes((16, 24, 24))), ValueError),                                       # two axes of positions
    (dict(axes=bytes(63)), ValueError),
    (dict(axes=[0, 1] * 31 + [2, 0]), ValueError),
    (dict(axes=[0, 1] * 31 + [256, 0]), ValueError),
    (dict(positions=torch.zeros(5, 4, dtype=torch.int64)), ValueError),
    (dict(positions=torch.zeros(2, 3, dtype=torch.int64)), ValueError),
    (dict(positions=torch.zeros(2, 4, dtype=torch.int32)), ValueError),
    (dict(axes=None), ValueError),                                                          # one axis, and positions of two
    (dict(cos=None, sin=None, positions=None), ValueError),
])
def test_append_refuses_axes_that_positions_do_not_have(change, error):
    rows = torch.zeros(4, 2, 128, dtype=torch.float16)
    args = dict(pages=_pool()[0], slots=torch.arange(4), k=rows, v=rows, cos=torch.zeros(9, 64), sin=torch.zeros(9, 64),
                positions=torch.zeros(2, 4, dtype=torch.int64), axes=rope_axes((32, 32)))
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_kv4_append(**args)
    with pytest.raises(error):
        paged_kv4_append(**(args | change))


@pytest.mark.parametrize("change,error", [
    (dict(pages=torch.zeros(2, 6, 2, 100, dtype=torch.uint8)), ValueError),
    (dict(pages=torch.zeros(2, 6, 2, 4608)), ValueError),
    (dict(pages=torch.zeros(6, 4608, dtype=torch.uint8)), ValueError),
    (dict(pages=_pool()[:0]), ValueError),
    (dict(src=[0]), ValueError),
    (dict(src=[0, 6]), ValueError),
    (dict(src=[-1, 0]), ValueError),
    (dict(dst=[3, 1 << 40]), ValueError),
    (dict(dst=[3, 3]), ValueError),
    (dict(dst=[0, 3]), ValueError),
    (dict(src=[0, 1.5]), TypeError),
    (dict(src=torch.tensor([0.0, 1.0])), ValueError),
    (dict(src=torch.tensor([[0, 1]])), ValueError),
    (dict(n_tokens=[1]), ValueError),
    (dict(n_tokens=[1, 33]), ValueError),
    (dict(n_tokens=[-1, 3]), ValueError),
    (dict(into=_pool(layers=3)), ValueError),
    (dict(into=_pool(h=4)), ValueError),
    (dict(into=_pool(page=16)), ValueError),
    (dict(into=_pool(n=3)), ValueError),                                                    # page 4 of three
])
def test_copy_refuses(change, error):
    args = dict(pages=_pool(), src=[0, 1], dst=[3, 4])
    for kw in ({}, dict(src=torch.tensor([0, 1])), dict(src=(0, 0)), dict(n_tokens=[0, 32]), dict(into=_pool(), dst=[0, 1]), dict(pages=_pool()[0])):
        with pytest.raises(RuntimeError, match="CUDA"):
            paged_kv4_copy(**(args | kw))
    with pytest.raises(error):
        paged_kv4_copy(**(args | change))


@pytest.mark.parametrize("n", [2, 100])
def test_library_refuses_before_it_touches_the_device(n):
    """Few pairs are compared with one another, many marked in a set: the same verdicts."""
    lib, buf = _lib.lib(), C.create_string_buffer(1 << 12)
    p = (C.addressof(buf) + 255) & ~255
    far = p + (1 << 40)
    pages, numbers = 2 * n, C.c_int32 * n
    own = dict(src=numbers(*range(n)), dst=numbers(*range(n, 2 * n)))
    def copy(**kw):
        a = dict(a=p, al=pages * 4608, ap=4608, ah=2304, na=pages, b=p, bl=pages * 4608, bp=4608, bh=2304, nb=pages, page=16, layers=2, h=2, **own, tokens=0, n=n,
                 stream=0) | kw
        return lib.bgtq_paged_copy(*a.values())
    assert copy(n=0) == _lib.OK
    twice, chain = numbers(*range(n, 2 * n - 1), n), numbers(*range(n - 1, 2 * n - 1))
    for kw, code in ((dict(dst=twice), -1), (dict(dst=chain), -1), (dict(src=numbers(*[-1] * n)), -1), (dict(src=numbers(*[pages] * n)), -1),
                     (dict(dst=numbers(*range(n + 1, 2 * n + 1))), -1), (dict(tokens=numbers(*[17] * n)), -1), (dict(tokens=numbers(*[-1] * n)), -1),
                     (dict(a=0), -1), (dict(b=0), -1), (dict(src=0), -1), (dict(dst=0), -1), (dict(n=-1), -1), (dict(page=8), -1), (dict(page=24), -1),
                     (dict(layers=0), -1), (dict(h=0), -1), (dict(na=0), -1), (dict(a=p + 8), -3), (dict(bh=2300), -3), (dict(ap=-4608, bp=-4608), -1),
                     (dict(b=p + 4608), -1), (dict(bl=pages * 4608 - 16), -1),            # pools that overlap one another
                     (dict(b=far, bl=16), -1), (dict(b=far, bp=2304), -1), (dict(b=far, bh=16), -1), (dict(b=far, bp=0), -1),      # or themselves
                     (dict(ah=0, bh=0), -1)):
        assert copy(**kw) == code, kw
    append = dict(pages=p, ps=4608, hs=2304, n_pages=2, page=16, slots=p, k=p, kst=256, ksh=128, v=p, vst=256, vsh=128, q=0, qst=0, qsh=0, qo=0, cos=p, sin=p,
                  rst=64, pos=p, pst=1, axes=rope_axes((32, 32)), n_axes=2, npos=1, n=1, nkv=2, nq=0, flags=0, status=0, stream=0)
    assert lib.bgtq_paged_append_axes(*(append | dict(n=0)).values()) == _lib.OK
    for kw in (dict(n_axes=1), dict(n_axes=0), dict(n_axes=5), dict(axes=None), dict(cos=0, sin=0), dict(pos=0), dict(axes=bytes([3] * 64))):
        assert lib.bgtq_paged_append_axes(*(append | kw).values()) == -1, kw
