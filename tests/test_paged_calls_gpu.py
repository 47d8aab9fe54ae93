"""Calls of the paged cache at its edges, against the definitions in 64 bits (oracle/paged_oracle.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_paged_gpu import BF16, FP16, LLAMA, MQA, QWEN, check_attend, filled, no_wait_ran_out, put, queries, trees  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout,rows,lengths", [(LLAMA, 1, [3000, 5]), (QWEN, 9, [700, 64]), (LLAMA, 70, [900, 0]), (MQA, 40, [2000])])
def test_results_in_the_queries_place(kt, layout, rows, lengths):
    cache = filled(layout, 32, BF16, lengths, rows)
    put(cache, rows)
    q = queries(cache, layout[0], rows)
    want = cache.attend(0, q, layout[0], rows)
    for _ in range(3):
        mine = q.clone()
        assert cache.attend(0, mine, layout[0], rows, out=mine) is mine
        assert torch.equal(mine, want)
    room = torch.zeros(q.numel() + 8, dtype=BF16, device="cuda")
    beside = room[8:].view(q.shape)
    beside.copy_(q)
    with pytest.raises(ValueError, match="overlap"):
        cache.attend(0, beside, layout[0], rows, out=room[:-8].view(q.shape))
    assert torch.equal(beside, q)
