"""8-bit paged serving and the per-head prologue at the edges of their calls:
memory that runs out, rows in front of the requests, refused row starts, status
words, values at the ends of their range."""

import pytest
import torch

from multics_b200.attention import hier_head_norm_rope
from multics_b200.paged8 import Paged8Cache, page_step, paged8_attention

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.fixture
def no_memory():
    """A limit on the process's memory: what it holds and 16 MB."""
    def limit():
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        total = torch.cuda.get_device_properties(0).total_memory
        torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (16 << 20)) / total)

    yield limit
    torch.cuda.set_per_process_memory_fraction(1.0)


def test_memory_run_out_is_an_error_of_the_call(no_memory):
    """Results that do not fit raise and leave nothing done; the same calls work
    when there is room."""
    T = 1 << 17
    q, k = torch.ones(T, 8 * 128, dtype=BF, device="cuda"), torch.ones(T, 128, dtype=BF, device="cuda")
    f, w = torch.ones(T, 64, 2, device="cuda"), torch.ones(128, device="cuda")
    c, table, lengths = Paged8Cache(2, 1), _i32([[0, 1]]), _i32([100])
    starts, add, free, count = _i32([0, T]), _i32([1]), _i32([]), _i32([0])
    calls = [lambda: hier_head_norm_rope(q, k, f, 8, 1, q_weight=w, k_weight=w),
             lambda: paged8_attention(q, c, table, lengths, starts, 8, block_frames=0),
             lambda: page_step(lengths, add, table, free, count, 1 << 24, in_place=True)]
    no_memory()
    for call in calls:
        with pytest.raises(torch.OutOfMemoryError):
            call()
    assert lengths.tolist() == [100]
    torch.cuda.set_per_process_memory_fraction(1.0)
    for call in calls:
        call()
    assert lengths.tolist() == [101]
    c.check()
