"""CPU: what a step of PagedKV4Cache costs on the host, counted in interpreted operations, and which sequences are looked through for released pages."""
import sys

import pytest

from blockgtq_b200 import PagedKV4Cache


def _cache(n_pages):
    return PagedKV4Cache(1, 1, 1, n_pages=n_pages, max_seq_len=100000, page_size=16, device="cpu")


def _operations(call):
    """How many of them ``call`` takes in the cache's own code."""
    count = [0]
    def trace(frame, event, arg):
        if not frame.f_code.co_filename.endswith("paged.py"):
            return None
        frame.f_trace_opcodes = True
        count[0] += event == "opcode"
        return trace
    before = sys.gettrace()
    sys.settrace(trace)
    try:
        call()
    finally:
        sys.settrace(before)
    return count[0]


def test_a_step_s_operations_do_not_go_with_its_pages():
    """(What does, the tables' lists, is made without looking at their numbers one by one.)"""
    counts = []
    for tokens in (100, 4004):             # (each with room in its last page: a new one is handed out operation by operation)
        c = _cache(2000)
        seqs = [c.add_sequence() for _ in range(3)]
        c.begin_step(seqs, [tokens] * 3)
        # (the first call that is traced tells the interpreter to, and is not counted)
        counts.append([_operations(lambda: c.begin_step(seqs, [1] * 3)) for _ in range(2)][1])
    assert counts[0] == counts[1] > 50


@pytest.mark.parametrize("fork", [False, True])
def test_tables_of_sequences_that_released_pages_and_of_others(fork):
    c = _cache(50)
    a, b = c.add_sequence(), c.add_sequence()
    c.begin_step([a, b], [70, 40])
    c.release(a, 50)
    if fork:
        first, a = a, c.fork_sequence(a)
        c.free_sequence(first)
    c.begin_step([b, a], [1, 1])
    table = c._step["table"].tolist()
    assert table[1][:3] == [-1] * 3 and table[1][3:] == c._seqs[a][1][3:] and table[0][:3] == c._seqs[b][1] and min(table[0]) >= 0
    c.free_sequence(a)
    assert c._gaps == set()
