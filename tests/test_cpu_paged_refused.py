"""CPU: a layer whose attention is refused stores nothing, whatever it is refused for."""
import pytest
import torch

from blockgtq_b200 import PagedKV4Cache, paged

I32 = torch.int32


@pytest.fixture
def stored(monkeypatch):
    """What was appended."""
    calls = []
    monkeypatch.setattr(paged, "paged_kv4_append", lambda *a, **kw: calls.append(a) or kw.get("q"))
    return calls


def _layer(q=torch.float16, **kw):
    c = PagedKV4Cache(1, 4, 2, n_pages=5, max_seq_len=100, page_size=16, device="cpu")
    c.begin_step([c.add_sequence(), c.add_sequence()], [3, 1])
    c.append_and_attend(0, torch.zeros(4, 4, 128, dtype=q), *[torch.zeros(4, 2, 128).half()] * 2, **kw)


@pytest.mark.parametrize("change,error", [
    (dict(softcap=-1.0), ValueError), (dict(softcap="much"), ValueError), (dict(window=0), ValueError), (dict(window=1.5), TypeError),
    (dict(slopes=torch.zeros(3)), ValueError), (dict(slopes=torch.zeros(4, 1)), ValueError), (dict(slopes=torch.zeros(4).half()), ValueError),
    (dict(slopes=torch.zeros(4, device="meta")), ValueError),
    (dict(prefix_lens=torch.zeros(3, dtype=I32)), ValueError), (dict(prefix_lens=torch.zeros(2)), ValueError),
    (dict(prefix_lens=torch.zeros(2, dtype=torch.int64)), ValueError), (dict(prefix_lens=torch.zeros(2, dtype=I32, device="meta")), ValueError),
    (dict(prefix_lens=torch.zeros(2, dtype=I32), max_prefix_len=-1), ValueError), (dict(window=4, max_prefix_len=-1), ValueError),
    (dict(window=4, max_prefix_len=1.5), TypeError), (dict(q=torch.float32), TypeError),
])
def test_nothing_is_stored_for_an_attention_that_is_refused(stored, change, error):
    with pytest.raises(error):
        _layer(**change)
    assert stored == []


@pytest.mark.parametrize("change", [dict(), dict(slopes=torch.zeros(8)[::2]), dict(prefix_lens=torch.zeros(2, dtype=I32), max_prefix_len=0), dict(softcap=5, window=9),
                                    dict(max_prefix_len=-1)])      # (nothing that it is of)
def test_what_is_not_refused_is_stored(stored, change):
    with pytest.raises(RuntimeError, match="CUDA"):
        _layer(**change)
    assert len(stored) == 1
