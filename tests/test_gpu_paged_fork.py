"""GPU: forked, truncated and moved sequences answer as sequences of their own do; a model's step with all that a layer may do beside plain attention."""
import pytest
import torch

import paged_bounds as W
import paged_reference as R
import paged_scores as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I32 = dict(dtype=torch.int32, device=DEV)


def _rows(gen, n, n_q=4, n_kv=2):
    return [torch.randn(n, h, 128, generator=gen).half().to(DEV) for h in (n_q, n_kv, n_kv)]


def _cache(n_layers=2, n_pages=40, **kw):
    from blockgtq_b200 import PagedKV4Cache
    return PagedKV4Cache(n_layers, 4, 2, n_pages=n_pages, max_seq_len=200, page_size=16, device=DEV, **kw)


def _both(rows, n):
    """Rows of a step of n sequences, each the same ones."""
    return [x.repeat(n, 1, 1) for x in rows]


@pytest.mark.parametrize("late", [False, True])
@pytest.mark.parametrize("prompt", [1, 16, 37])
def test_beams_answer_as_sequences_of_their_own(prompt, late):
    """Three beams from one prompt, reordered after each step: the survivors' answers are those of sequences that were fed the same tokens one by one.
    late: layers on another stream, which nothing orders with the steps'."""
    gen = torch.Generator().manual_seed(prompt)
    shared, alone = _cache(), _cache(n_pages=300)
    side = torch.cuda.Stream(DEV)
    def layers(cache, rows):
        if not late:
            return [cache.append_and_attend(i, *r) for i, r in enumerate(rows)]
        with torch.cuda.stream(side):
            torch.cuda._sleep(2_000_000)
            return [cache.append_and_attend(i, *r) for i, r in enumerate(rows)]
    first = [_rows(gen, prompt) for _ in range(2)]
    torch.cuda.synchronize()
    root = shared.add_sequence()
    shared.begin_step([root], [prompt])
    layers(shared, first)
    history = {root: [first]}
    beams = [root, shared.fork_sequence(root), shared.fork_sequence(root)]
    history |= {b: [first] for b in beams[1:]}
    for parents in ((0, 0, 2), (1, 1, 1), (2, 0, 1), (0, 1, 2)):
        rows = [_rows(gen, 3) for _ in range(2)]
        shared.begin_step(beams, [1, 1, 1])
        got = layers(shared, rows)
        for j, b in enumerate(beams):
            history[b] = history[b] + [[[x[j:j + 1] for x in r] for r in rows]]
        side.synchronize()
        torch.cuda.synchronize()
        for j, b in enumerate(beams):                   # replayed from nothing
            s = alone.add_sequence()
            for part in history[b]:
                alone.begin_step([s], [part[0][0].shape[0]])
                want = [alone.append_and_attend(i, *r) for i, r in enumerate(part)]
            for g, w in zip(got, want):
                assert (g[j].float() - w[0].float()).abs().max() <= 2.0 ** -9 * w.float().abs().max()
            torch.cuda.synchronize()
            pages = [shared.pages[:, shared._seqs[b][1]], alone.pages[:, alone._seqs[s][1]]]
            slots = torch.arange(shared.seq_len(b), device=DEV)
            for layer in range(2):
                assert all(torch.equal(x, y) for x, y in zip(*[S.read(p[layer], slots) for p in pages]))
            alone.free_sequence(s)
        kept = [shared.fork_sequence(beams[p]) for p in parents]
        history |= {k: history[beams[p]] for k, p in zip(kept, parents)}
        for b in beams:
            shared.free_sequence(b)
        beams = kept
    for c in (shared, alone):
        c.check_status()
    for b in beams:
        shared.free_sequence(b)
    assert shared.free_pages == 40


def test_moved_pools_go_on_answering():
    gen = torch.Generator().manual_seed(8)
    a, b = _cache(n_pages=60), _cache(n_pages=60)
    def both(seqs, counts):
        rows = [_rows(gen, sum(counts)) for _ in range(2)]
        outs = []
        for c in (a, b):
            c.begin_step(seqs, counts)
            outs.append([c.append_and_attend(i, *r) for i, r in enumerate(rows)])
        assert all(torch.equal(x, y) for x, y in zip(*outs))
    seqs = [(a.add_sequence(), b.add_sequence())[0] for _ in range(5)]
    both(seqs, [40, 3, 70, 16, 33])
    for c in (a, b):
        c.free_sequence(seqs[0])
        c.truncate_sequence(seqs[2], 20)
        c.fork_sequence(seqs[4])
    assert a.compact() == 1 + 2 + 1 + 3 == a.n_pages - a.free_pages          # 3, 20, 16 and 33 tokens, the last ones twice
    both(seqs[1:] + [5], [1] * 5)
    a.resize(12)
    assert a.pages.shape[1] == 12
    both(seqs[1:] + [5], [1] * 5)
    a.resize(100)
    assert a.free_pages == 100 - (60 - b.free_pages)
    both(seqs[1:] + [5], [9, 1, 2, 30, 1])
    for c in (a, b):
        c.check_status()


@pytest.mark.parametrize("keep", [0, 4])
def test_a_windowed_model_in_a_pool_that_holds_its_window(keep):
    """200 tokens through a pool of 8 pages: released as the window leaves them behind, the answers are those of a cache that keeps everything."""
    gen = torch.Generator().manual_seed(keep)
    small, whole = _cache(n_pages=8), _cache()
    score = dict(window=60, prefix_lens=torch.full((1,), keep, **I32), max_prefix_len=keep)
    a, b = small.add_sequence(), whole.add_sequence()
    done = 0
    for n in (50, *[1] * 20, 30, *[4] * 25):
        rows = [_rows(gen, n) for _ in range(2)]
        outs = []
        for c, s in ((small, a), (whole, b)):
            c.begin_step([s], [n])
            outs.append([c.append_and_attend(i, *r, **score) for i, r in enumerate(rows)])
        assert all(torch.equal(x, y) for x, y in zip(*outs))
        done += n
        small.release(a, max(0, done + 1 - 60), keep)   # (the next row, at place done, sees from here on)
    assert done == 200 and small.free_pages == 8 - 5 - (keep > 0) and whole.free_pages == 40 - 13
    small.check_status()
    whole.check_status()
    small.truncate_sequence(a, 190)
    small.begin_step([a], [1])
    small.append_and_attend(0, *_rows(gen, 1))           # without the window: it looks for what is gone
    with pytest.raises(RuntimeError, match="page number"):
        small.check_status()


def test_moving_is_not_captured():
    cache = _cache()
    cache.begin_step([cache.add_sequence()], [20])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        for call in (cache.compact, lambda: cache.resize(50)):
            with pytest.raises(RuntimeError, match="captured"):
                call()


def test_a_step_with_axes_window_cap_and_prefix():
    """Layers of two kinds, as a model has them: append with positions of three axes, then capped logits behind a window that keeps sinks, or all tokens with
    a picture in front that both sides see and a bias by distance.  Against the operators' definition, layer by layer."""
    from blockgtq_b200 import rope_axes
    gen = torch.Generator().manual_seed(12)
    cache = _cache(n_pages=60)
    angle = torch.arange(60, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    cos, sin, axes = angle.cos().float(), angle.sin().float(), rope_axes((16, 24, 24))
    rope = cos.to(DEV), sin.to(DEV)
    slopes = 2.0 ** -torch.arange(1.0, 5.0)
    kinds = [dict(softcap=20.0, window=30, prefix=[2, 2]), dict(slopes=slopes, prefix=[25, 0])]
    seqs = [cache.add_sequence(), cache.add_sequence()]
    lens = [0, 0]
    for counts in ([90, 41], [1, 1], [1, 1], [4, 4]):
        cache.begin_step(seqs, counts)
        lens = [t + c for t, c in zip(lens, counts)]
        positions = torch.randint(0, 60, (3, sum(counts)), generator=gen)
        at = positions[torch.tensor(list(axes))].T
        for layer, kind in enumerate(kinds):
            q, k, v = _rows(gen, sum(counts))
            out = cache.append_and_attend(layer, q, k, v, rope=rope, positions=positions.to(DEV), axes=axes, softcap=kind.get("softcap"), window=kind.get("window"),
                                          slopes=slopes.to(DEV) if "slopes" in kind else None, prefix_lens=torch.tensor(kind["prefix"], **I32), max_prefix_len=25)
            a, b = q.float().cpu().chunk(2, -1)
            c, s = (x[at, torch.arange(64)][:, None] for x in (cos, sin))
            turned = torch.cat([a * c - b * s, b * c + a * s], -1).half()
            row = 0
            for i, n in enumerate(counts):
                slots = torch.arange(lens[i])
                slots = torch.tensor(cache._seqs[seqs[i]][1])[slots // 16] * 16 + slots % 16
                rows = sorted({0, n // 2, n - 1})
                given = {x: y for x, y in kind.items() if x != "prefix"}
                W.check(out, None, S.attention(turned[row:row + n], cache.pages[layer], slots, rows=rows, prefix=min(kind["prefix"][i], lens[i]), **given),
                        [row + r for r in rows])
                row += n
    cache.check_status()


def test_an_attention_that_is_refused_stores_nothing():
    cache = _cache()
    cache.begin_step([cache.add_sequence()], [3])
    rows = _rows(torch.Generator().manual_seed(1), 3)
    for kw in (dict(softcap=-1.0), dict(window=0), dict(prefix_lens=torch.zeros(2, **I32))):
        with pytest.raises(ValueError):
            cache.append_and_attend(0, *rows, **kw)
    assert not cache.pages.any()
