"""CPU: what PagedKV4Cache keeps when a step cannot begin, and what it refuses."""
import pytest
import torch

from blockgtq_b200 import PagedKV4Cache, paged


def _cache():
    return PagedKV4Cache(1, 4, 2, n_pages=6, max_seq_len=100, page_size=16, device="cpu")


@pytest.mark.parametrize("fails", [0, 1, 2])
def test_a_step_that_the_device_has_no_memory_for_takes_nothing(monkeypatch, fails):
    c = _cache()
    a, b = c.add_sequence(), c.add_sequence()
    c.begin_step([a, b], [17, 3])
    def state():
        return {i: (t, list(p)) for i, (t, p) in c._seqs.items()}, list(c._free), c._step["slots"].tolist()
    before, make, made = state(), torch.tensor, []
    class Full:
        def to(self, device):
            raise torch.OutOfMemoryError("no memory")
    def tensor(*args, **kw):
        made.append(args)
        return Full() if len(made) == fails + 1 else make(*args, **kw)
    monkeypatch.setattr(paged.torch, "tensor", tensor)
    with pytest.raises(torch.OutOfMemoryError):
        c.begin_step([b, a], [40, 1])
    monkeypatch.undo()
    assert state() == before
    c.begin_step([b, a], [40, 1])
    assert (c.seq_len(a), c.seq_len(b), c.free_pages) == (18, 43, 1)
    held = [p for _, pages in c._seqs.values() for p in pages]
    assert sorted(held + c._free) == list(range(6))
    assert c._step["slots"].tolist() == [c._seqs[b][1][t // 16] * 16 + t % 16 for t in range(3, 43)] + [c._seqs[a][1][1] * 16 + 1]


def test_a_prefill_of_fewer_rows_than_none_is_refused():
    args = dict(q=torch.zeros(4, 4, 128, dtype=torch.float16), pages=torch.zeros(3, 2, paged.page_bytes(32), dtype=torch.uint8),
                block_table=torch.zeros(2, 1, dtype=torch.int32), seq_lens=torch.ones(2, dtype=torch.int32), cu_q=torch.tensor([0, 2, 4], dtype=torch.int32))
    with pytest.raises(ValueError, match="max_q_len"):
        paged.paged_kv4_prefill_attention(**args, max_q_len=-1)
    for n in (0, 1, 2, 100, None):
        with pytest.raises(RuntimeError, match="CUDA"):
            paged.paged_kv4_prefill_attention(**args, max_q_len=n)
