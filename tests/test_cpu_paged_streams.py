"""CPU: what PagedKV4Cache's copies and layers are ordered behind, whatever streams they run on: streams that record it, and do nothing else."""
import random

import pytest
import torch

from blockgtq_b200 import PagedKV4Cache, paged


class Stream:
    """What lies behind its last work: numbers of copies and layers."""

    def __init__(self):
        self.behind = set()

    def wait_stream(self, other):
        self.behind |= other.behind

    def wait_event(self, event):
        self.behind |= event

    def record_event(self):
        return frozenset(self.behind)


class Cache(PagedKV4Cache):
    """The book-keeping on streams of its own: ``done`` holds (kind, what the work was ordered behind) of each copy and layer."""

    def __init__(self, n_pages=20):
        super().__init__(1, 4, 2, n_pages=n_pages, max_seq_len=100, page_size=16, device="cpu")
        self.done, self.now = [], Stream()

    def _stream(self):
        return self.now

    def run(self, kind):
        self.done.append((kind, set(self.now.behind)))
        self.now.behind.add(len(self.done) - 1)

    def begin_step(self, seqs, counts):
        super().begin_step(seqs, counts)
        self._step["held"] = ()                         # (no device, no memory that a stream holds on to)

    def layer(self):
        n = self._step["rows"]
        self.append_and_attend(0, torch.zeros(n, 4, 128).half(), *[torch.zeros(n, 2, 128).half()] * 2)

    def numbers(self, kind):
        return {i for i, (k, _) in enumerate(self.done) if k == kind}


@pytest.fixture
def cache(monkeypatch):
    c = Cache()
    monkeypatch.setattr(paged, "paged_kv4_copy", lambda *a, **kw: c.run("copy"))
    monkeypatch.setattr(paged, "paged_kv4_append", lambda *a, **kw: c.run("layer"))
    for name in ("paged_kv4_decode_attention", "paged_kv4_prefill_attention"):
        monkeypatch.setattr(paged, name, lambda *a, **kw: None)
    return c


def _two_sequences(c, first=40, second=20):
    a, b = c.add_sequence(), c.add_sequence()
    c.begin_step([a, b], [first, second])
    c.layer()
    return a, b


@pytest.mark.parametrize("same", [True, False])
def test_a_step_s_layers_wait_for_pages_that_another_stream_moved(cache, same):
    """same: the layers run on the stream of begin_step."""
    c, main, other, third = cache, cache.now, Stream(), Stream()
    a, b = _two_sequences(c)
    c.free_sequence(a)
    c.now = other
    assert c.compact() == 2
    c.now = main
    c.begin_step([b], [1])                              # (nothing to copy)
    c.now = main if same else third
    c.layer()
    assert len(c.numbers("copy")) == 1 and c.numbers("copy") <= c.done[-1][1]
    assert c.numbers("layer") - {len(c.done) - 1} <= c.done[1][1]              # and the copy for the layers before it


def test_a_step_waits_once_on_each_stream(cache):
    c, main, other = cache, cache.now, Stream()
    a, b = _two_sequences(c)
    c.free_sequence(a)
    c.now = other
    c.compact()
    c.now, waits = main, []
    main.wait_event = waits.append
    for i in range(3):
        c.begin_step([b], [1])
        c.layer()
        c.layer()
        assert len(waits) == i + 1


def _behind_all(c):
    """The last copy is ordered behind every copy and layer before it."""
    assert c.done[-1][0] == "copy" and c.done[-1][1] == set(range(len(c.done) - 1))


@pytest.mark.parametrize("second", ["compact", "resize", "step"])
def test_copies_wait_for_copies_on_another_stream(cache, second):
    """A step's copy of a shared page, or a compact, and before any layer runs a copy on another stream."""
    c = cache
    a, b = _two_sequences(c)
    d = c.fork_sequence(b)
    if second == "step":
        c.free_sequence(a)
        c.now = Stream()
        c.compact()
        c.now = Stream()
        c.begin_step([d], [1])
    else:
        c.now = Stream()
        c.begin_step([d], [1])
        c.free_sequence(a)
        c.now = Stream()
        c.compact() if second == "compact" else c.resize(9)
    assert len(c.numbers("copy")) == 2
    _behind_all(c)
    c.now = third = Stream()                            # the last copy's event stands for both
    c.begin_step([b], [1])
    assert c.numbers("copy") <= third.behind


@pytest.mark.parametrize("seed", range(10))
def test_any_order_of_streams(cache, seed):
    """Copies behind all copies and layers before them, layers behind all copies."""
    c, rng = cache, random.Random(seed)
    streams, seqs = [Stream() for _ in range(4)], []
    for _ in range(120):
        c.now = rng.choice(streams)
        kind = rng.choice(["add", "step", "step", "layer", "layer", "fork", "free", "compact", "resize"])
        some = rng.sample(seqs, min(len(seqs), rng.randint(1, 3)))
        before = len(c.done)
        if kind == "add" or not some:
            seqs.append(c.add_sequence())
        elif kind == "step":
            try:
                c.begin_step(some, [rng.randint(1, 20) for _ in some])
            except (RuntimeError, ValueError):
                continue
        elif kind == "layer" and c._step is not None:
            c.layer()
            assert c.numbers("copy") <= c.done[-1][1]
        elif kind == "fork":
            seqs.append(c.fork_sequence(some[0]))
        elif kind == "free":
            c.free_sequence(some[0])
            seqs.remove(some[0])
        elif kind == "compact":
            c.compact()
        elif kind == "resize":
            c.resize(max(1, c.n_pages - c.free_pages, rng.randint(10, 25)))
        if len(c.done) > before and c.done[-1][0] == "copy":
            _behind_all(c)
    assert len(c.numbers("copy")) > 3
