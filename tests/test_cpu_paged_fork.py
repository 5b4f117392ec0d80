"""CPU: which pages sequences of PagedKV4Cache share, and when they part."""
import random

import pytest
import torch

from blockgtq_b200 import PagedKV4Cache, paged


class Cache(PagedKV4Cache):
    """The book-keeping, with a pool of one byte per token in place of the pages: what a layer's append would store, stored."""

    def __init__(self, n_pages=12, page_size=16, max_seq_len=100):
        super().__init__(1, 4, 2, n_pages=n_pages, max_seq_len=max_seq_len, page_size=page_size, device="cpu")
        self.tokens = torch.full((n_pages, page_size), -1, dtype=torch.int64)
        self.copies = []

    def _copy(self, src, dst, n_tokens=None, into=None):
        assert len(set(dst)) == len(dst) and (into is not None or not set(dst) & set(src))
        if into is not None:
            new = torch.full((into.shape[1], self.page_size), -1, dtype=torch.int64)
            new[dst] = self.tokens[src]
            self.tokens = new
        else:
            for i, (a, b) in enumerate(zip(src, dst)):
                n = self.page_size if n_tokens is None else -(-n_tokens[i] // 16) * 16
                self.tokens[b, :n] = self.tokens[a, :n]
        self.copies.append(len(src))

    def resize(self, n_pages):
        super().resize(n_pages)
        if len(self.tokens) != n_pages:                 # (nothing was held, nothing copied)
            self.tokens = torch.full((n_pages, self.page_size), -1, dtype=torch.int64)

    def store(self, rows):
        slots = self._step["slots"]
        assert len(set(slots.tolist())) == len(slots)
        self.tokens.view(-1)[slots] = rows

    def read(self, seq):
        """The sequence's tokens, -1 where they have been released."""
        t, pages = self._seqs[seq]
        none = torch.full((1, self.page_size), -1, dtype=torch.int64)
        return torch.cat([none] * (not pages) + [none if p is None else self.tokens[p:p + 1] for p in pages]).reshape(-1)[:t]

    def check(self):
        held = [0] * self.n_pages
        for t, pages in self._seqs.values():
            there = [p for p in pages if p is not None]
            assert len(pages) == -(-t // self.page_size) and len(set(there)) == len(there)
            for p in pages:
                if p is not None:
                    held[p] += 1
        assert held == self._held and sorted(self._free) == [p for p in range(self.n_pages) if held[p] == 0]


def _step(c, seqs, counts, rows):
    c.begin_step(seqs, counts)
    c.store(torch.tensor(rows))
    c.check()


def test_a_fork_shares_pages_until_it_writes():
    c = Cache()
    a = c.add_sequence()
    _step(c, [a], [20], list(range(20)))
    b = c.fork_sequence(a)
    assert c.free_pages == 10 and c.seq_len(b) == 20 and c._seqs[a][1] == c._seqs[b][1] and c.copies == []
    _step(c, [a, b], [1, 1], [100, 200])                 # the first of the two takes a copy of the half-filled page, the other keeps it
    assert c.copies == [1] and c.free_pages == 9 and c._seqs[a][1][0] == c._seqs[b][1][0] and c._seqs[a][1][1] != c._seqs[b][1][1]
    assert c.read(a).tolist() == [*range(20), 100] and c.read(b).tolist() == [*range(20), 200]
    c.free_sequence(a)
    assert c.free_pages == 10
    _step(c, [b], [30], list(range(30)))
    assert c.copies == [1] and c.read(b).tolist() == [*range(20), 200, *range(30)]
    c.free_sequence(b)
    assert c.free_pages == 12


def test_forks_of_a_part_and_at_a_page_s_end():
    c = Cache()
    a = c.add_sequence()
    _step(c, [a], [40], list(range(40)))
    whole, part, none = c.fork_sequence(a, 32), c.fork_sequence(a, 5), c.fork_sequence(a, 0)
    assert [c.seq_len(i) for i in (whole, part, none)] == [32, 5, 0] and [len(c._seqs[i][1]) for i in (whole, part, none)] == [2, 1, 0]
    c.check()
    _step(c, [whole, none], [1, 1], [7, 8])              # nothing to copy: new pages
    assert c.copies == []
    _step(c, [part], [1], [9])
    assert c.copies == [1] and c.read(part).tolist() == [0, 1, 2, 3, 4, 9]
    for bad in (41, -1):
        with pytest.raises(ValueError):
            c.fork_sequence(a, bad)
    with pytest.raises(KeyError):
        c.fork_sequence(99)
    with pytest.raises(TypeError):
        c.fork_sequence(a, 1.5)
    c.check()


def test_truncating_gives_pages_back_and_parts_what_is_shared():
    c = Cache()
    a = c.add_sequence()
    _step(c, [a], [40], list(range(40)))
    b = c.fork_sequence(a)
    c.truncate_sequence(b, 18)
    assert c.free_pages == 9 and c.seq_len(b) == 18 and c._step is not None
    c.truncate_sequence(a, 36)
    assert c._step is None                              # its slots may be another's
    c.check()
    _step(c, [b, a], [2, 1], [50, 51, 60])
    assert c.copies == [1] and c.read(b).tolist() == [*range(18), 50, 51] and c.read(a).tolist() == [*range(36), 60]
    c.truncate_sequence(a, 0)
    assert c._seqs[a] == [0, []]
    for bad in (1, -1):
        with pytest.raises(ValueError):
            c.truncate_sequence(a, bad)
    c.check()


def test_a_step_that_lacks_pages_for_its_copies_takes_nothing():
    c = Cache(n_pages=3)
    a = c.add_sequence()
    _step(c, [a], [20], list(range(20)))
    forks = [c.fork_sequence(a) for _ in range(2)]
    before = {i: (t, list(p)) for i, (t, p) in c._seqs.items()}, list(c._free), list(c._held)
    with pytest.raises(RuntimeError, match="2 pages needed, 1 free"):
        c.begin_step([a, *forks], [1, 1, 1])
    assert before == ({i: (t, list(p)) for i, (t, p) in c._seqs.items()}, list(c._free), list(c._held)) and c.copies == []
    c.free_sequence(forks[0])
    _step(c, [a, forks[1]], [1, 1], [5, 6])
    assert c.free_pages == 0


@pytest.mark.parametrize("seed", range(20))
def test_any_order_of_calls_keeps_every_sequence_s_tokens(seed):
    rng = random.Random(seed)
    c = Cache(n_pages=40, page_size=rng.choice([16, 32]), max_seq_len=150)
    want, number = {}, 0
    for _ in range(150):
        kind = rng.choice(["add", "step", "step", "step", "fork", "fork", "truncate", "free", "release", "compact", "resize"])
        some = rng.sample(sorted(want), min(len(want), rng.randint(1, 5)))
        if kind == "add" or not some:
            want[c.add_sequence()] = []
        elif kind == "step":
            counts = [rng.randint(1, 30) for _ in some]
            rows = [list(range(number + 1000 * i, number + 1000 * i + n)) for i, n in enumerate(counts)]
            number += 10000
            try:
                c.begin_step(some, counts)
            except (RuntimeError, ValueError):
                c.check()
                continue
            c.store(torch.tensor([x for r in rows for x in r]))
            for i, r in zip(some, rows):
                want[i] = want[i] + r
        elif kind == "fork":
            n = rng.randint(0, len(want[some[0]]))
            if n and want[some[0]][n - 1] == -1 and n % c.page_size:
                with pytest.raises(ValueError, match="released"):
                    c.fork_sequence(some[0], n)
                continue
            want[c.fork_sequence(some[0], n)] = want[some[0]][:n]
        elif kind == "truncate":
            n = rng.randint(0, len(want[some[0]]))
            if n and want[some[0]][n - 1] == -1 and n % c.page_size:
                with pytest.raises(ValueError, match="released"):
                    c.truncate_sequence(some[0], n)
                continue
            c.truncate_sequence(some[0], n)
            want[some[0]] = want[some[0]][:n]
        elif kind == "release":
            n, keep, size = rng.randint(0, len(want[some[0]])), rng.choice([0, 1, 16, 40]), c.page_size
            c.release(some[0], n, keep)
            want[some[0]] = [-1 if -(-keep // size) <= i // size < n // size else x for i, x in enumerate(want[some[0]])]
        elif kind == "free":
            c.free_sequence(some[0])
            del want[some[0]]
        elif kind == "compact":
            n = c.compact()
            assert sorted({p for _, pages in c._seqs.values() for p in pages} - {None}) == list(range(n)) and c._step is None
        else:
            held = c.n_pages - c.free_pages
            c.resize(max(1, held, rng.randint(held, 40)))
            assert c.pages.shape[1] == c.n_pages == len(c._held)
        c.check()
        for i, rows in want.items():
            assert c.read(i).tolist() == rows


def test_released_pages_are_others_and_the_table_says_so():
    c = Cache()
    a = c.add_sequence()
    _step(c, [a], [70], list(range(70)))
    b = c.fork_sequence(a)
    c.release(a, 50, keep=4)                            # pages 1 and 2; b holds them still
    assert c._step is None and c.free_pages == 7
    c.release(b, 50)
    assert c.free_pages == 9 and [p is None for p in c._seqs[a][1]] == [False, True, True, False, False] and c._seqs[b][1][:3] == [None] * 3
    c.release(b, 50)
    c.release(b, 0)
    _step(c, [a, b], [1, 1], [100, 200])
    assert c._step["table"][:, :3].tolist() == [[c._seqs[a][1][0], -1, -1], [-1, -1, -1]] and c.copies == [1]
    assert c.read(a).tolist() == [*range(16), *[-1] * 32, *range(48, 70), 100] and c.read(b).tolist() == [*[-1] * 48, *range(48, 70), 200]
    for n in (17, 33, 47):
        for call in (c.truncate_sequence, c.fork_sequence):
            with pytest.raises(ValueError, match="released"):
                call(a, n)
    c.truncate_sequence(a, 32)
    _step(c, [a], [3], [7, 8, 9])
    assert c.read(a).tolist() == [*range(16), *[-1] * 16, 7, 8, 9]
    for bad in ((36, 0), (-1, 0), (0, -1)):
        with pytest.raises(ValueError):
            c.release(a, *bad)
    c.free_sequence(a)
    c.free_sequence(b)
    c.check()
    assert c.free_pages == 12


def test_a_pool_holds_what_is_held():
    c = Cache(n_pages=5)
    a = c.add_sequence()
    with pytest.raises(ValueError, match="at least one"):
        c.resize(0)
    _step(c, [a], [40], list(range(40)))
    with pytest.raises(ValueError, match="3 pages are held"):
        c.resize(2)
    c.resize(3)
    assert c.free_pages == 0 and c.cache_memory_bytes() == 3 * 2 * 2304 and c.read(a).tolist() == list(range(40))
    with pytest.raises(RuntimeError, match="begin_step"):
        c.append_and_attend(0, torch.zeros(40, 4, 128).half(), torch.zeros(40, 2, 128).half(), torch.zeros(40, 2, 128).half())


def test_positions_and_axes_belong_to_rope():
    c = PagedKV4Cache(1, 4, 2, n_pages=5, max_seq_len=100, page_size=16, device="cpu")
    c.begin_step([c.add_sequence()], [3])
    rows = torch.zeros(3, 4, 128).half(), torch.zeros(3, 2, 128).half(), torch.zeros(3, 2, 128).half()
    at = torch.zeros(3, dtype=torch.int64)
    for kw in (dict(positions=at), dict(axes=bytes(64)), dict(rope=(torch.zeros(9, 64),) * 2, axes=bytes(64))):
        with pytest.raises(ValueError):
            c.append_and_attend(0, *rows, **kw)
    with pytest.raises(TypeError):
        c.append_and_attend(0, *rows, causal=False)


@pytest.mark.parametrize("change", [dict(softcap=0.0), dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")), dict(softcap=1e-20), dict(softcap=1e20),
                                    dict(window=0), dict(window=-3), dict(max_prefix_len=-1, prefix_lens=torch.zeros(4, dtype=torch.int32)),
                                    dict(slopes=torch.zeros(3)), dict(slopes=torch.zeros(4).half()), dict(prefix_lens=torch.zeros(3, dtype=torch.int32)),
                                    dict(prefix_lens=torch.zeros(4, dtype=torch.int64))])
def test_scores_that_are_refused(change):
    args = dict(q=torch.zeros(4, 4, 128, dtype=torch.float16), pages=torch.zeros(3, 2, paged.page_bytes(32), dtype=torch.uint8),
                block_table=torch.zeros(4, 1, dtype=torch.int32), seq_lens=torch.ones(4, dtype=torch.int32))
    rows = args | dict(cu_q=torch.arange(5, dtype=torch.int32))
    good = dict(softcap=50.0, slopes=torch.zeros(4), window=1, prefix_lens=torch.zeros(4, dtype=torch.int32), max_prefix_len=0)
    for call in (lambda **kw: paged.paged_kv4_decode_attention(**args, **kw), lambda **kw: paged.paged_kv4_prefill_attention(**rows, **kw)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call(**good)
        with pytest.raises(ValueError):
            call(**change)
    with pytest.raises(ValueError, match="causal"):
        paged.paged_kv4_prefill_attention(**rows, causal=False, window=5)
    with pytest.raises(TypeError):
        paged.paged_kv4_decode_attention(**args, window=2.5)


def test_the_library_refuses_scores():
    import ctypes as C
    from blockgtq_b200 import _lib
    lib, buf = _lib.lib(), C.create_string_buffer(4096)
    p = (C.addressof(buf) + 255) & ~255
    def both(**kw):
        flags, sc = kw.pop("flags", 0), _lib.PagedScores(**(dict(softcap=0.0, window=0, max_prefix=0) | kw))
        attend = lib.bgtq_paged_attend_scored(p, 512, 128, p, 4608, 2304, 2, 16, p, 1, 0, p, p, 0, 0, 4, 2, 1, 16, 1.0, flags, sc, p, 0, p, 512, 128, 0, 0, 0)
        return attend, lib.bgtq_paged_scored_workspace_bytes(1, 1, 4, 2, 1, 16, flags, sc)
    assert both() == (_lib.OK, 0) and both(window=5, flags=4) == (_lib.OK, 0)
    for kw in (dict(window=-1), dict(max_prefix=-1), dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")), dict(softcap=5e-20), dict(softcap=2e19), dict(reserved=1)):
        assert both(**kw) == (-1, -1), kw
    assert both(window=5)[0] == -1                       # a window, and no causal queries
