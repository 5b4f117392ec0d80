"""GPU: a layer whose attention is refused leaves the pages as they were, and can be asked again."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_pages_stay_as_they_were():
    from blockgtq_b200 import PagedKV4Cache
    gen = torch.Generator().manual_seed(1)
    cache = PagedKV4Cache(1, 4, 2, n_pages=9, max_seq_len=100, page_size=16, device=DEV)
    cache.begin_step([cache.add_sequence(), cache.add_sequence()], [3, 20])
    q, k, v = (torch.randn(23, h, 128, generator=gen).half().to(DEV) for h in (4, 2, 2))
    i32, good = dict(dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    for kw in (dict(slopes=torch.zeros(3, device=DEV)), dict(slopes=torch.zeros(4, device=DEV).half()), dict(slopes=torch.zeros(4)), dict(prefix_lens=good.long()),
               dict(prefix_lens=good.cpu()), dict(prefix_lens=torch.zeros(3, **i32)), dict(prefix_lens=good, max_prefix_len=-1), dict(window=9, max_prefix_len=1.5),
               dict(softcap=0.0), dict(window=0), dict(q=q.float()), dict(q=q.cpu())):
        with pytest.raises((ValueError, TypeError)):
            cache.append_and_attend(0, kw.pop("q", q), k, v, **kw)
        assert not cache.pages.any()
    slopes = torch.rand(4, generator=gen).to(DEV)
    want = cache.append_and_attend(0, q, k, v, slopes=slopes, prefix_lens=good)
    wide = slopes.repeat_interleave(2)[::2], good.repeat_interleave(3)[::3]
    assert torch.equal(cache.append_and_attend(0, q, k, v, slopes=wide[0], prefix_lens=wide[1]), want)
    cache.check_status()
