"""GPU: pages moved on one stream, steps and layers on another: a cache whose copies come late answers as one that is asked on one stream alone."""
import pytest
import torch

import paged_scores as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _rows(gen, n):
    return [torch.randn(n, h, 128, generator=gen).half().to(DEV) for h in (4, 2, 2)]


def _cache():
    from blockgtq_b200 import PagedKV4Cache
    return PagedKV4Cache(2, 4, 2, n_pages=40, max_seq_len=200, page_size=16, device=DEV)


class Pair:
    """Two caches that are given the same calls: ``moved``'s layers and moves on streams of their own, ``plain``'s behind one another."""

    def __init__(self, seed):
        self.gen = torch.Generator().manual_seed(seed)
        self.moved, self.plain = _cache(), _cache()
        self.side = torch.cuda.Stream(DEV)

    def both(self, call):
        return [call(c) for c in (self.moved, self.plain)][0]

    def late(self, call):
        """On the side stream and behind a few ms of waiting there, for the cache whose pages move."""
        with torch.cuda.stream(self.side):
            torch.cuda._sleep(10_000_000)
            return call(self.moved)

    def step(self, seqs, counts):
        rows = [_rows(self.gen, sum(counts)) for _ in range(2)]
        outs = []
        for c in (self.moved, self.plain):
            c.begin_step(seqs, counts)
            outs.append([c.append_and_attend(i, *r) for i, r in enumerate(rows)])
        return outs

    def check(self, seqs, outs):
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(*outs))
        for s in seqs:
            slots = torch.arange(self.plain.seq_len(s), device=DEV)
            for layer in range(2):
                held = [S.read(c.pages[layer][c._seqs[s][1]], slots) for c in (self.moved, self.plain)]
                assert all(torch.equal(x, y) for x, y in zip(*held))
        for c in (self.moved, self.plain):
            c.check_status()


def _beginning(seed):
    """Three sequences, and the first one's pages free in front of the others'."""
    p = Pair(seed)
    seqs = [p.both(lambda c: c.add_sequence()) for _ in range(3)]
    p.step(seqs, [90, 37, 60])
    p.both(lambda c: c.free_sequence(seqs[0]))
    torch.cuda.synchronize()
    return p, seqs[1:]


def test_pages_moved_late_and_a_step_that_copies_nothing():
    p, seqs = _beginning(1)
    assert p.late(lambda c: c.compact()) == 7
    p.check(seqs, p.step(seqs, [1, 20]))


def test_pages_moved_late_and_a_step_that_parts_a_fork():
    p, seqs = _beginning(2)
    fork = p.both(lambda c: c.fork_sequence(seqs[1]))
    assert p.late(lambda c: c.compact()) == 7
    p.check([*seqs, fork], p.step([*seqs, fork], [1, 3, 1]))


@pytest.mark.parametrize("n_pages", [12, 60])
def test_pages_moved_late_and_a_pool_resized(n_pages):
    p, seqs = _beginning(3)
    assert p.late(lambda c: c.compact()) == 7
    p.moved.resize(n_pages)
    p.check(seqs, p.step(seqs, [1, 1]))


@pytest.mark.parametrize("move", ["compact", "resize"])
def test_a_fork_parted_late_and_its_copy_moved(move):
    """The step that copies the shared page is taken back before a layer runs; the copy moves on the main stream."""
    p, seqs = _beginning(4)
    fork = p.both(lambda c: c.fork_sequence(seqs[1]))
    p.late(lambda c: c.begin_step([fork], [2]))
    p.plain.begin_step([fork], [2])
    p.both(lambda c: c.truncate_sequence(fork, 60))
    p.moved.compact() if move == "compact" else p.moved.resize(9)
    p.check([*seqs, fork], p.step([fork, *seqs], [1, 1, 1]))
