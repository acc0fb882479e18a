"""8-bit paged serving and the per-head prologue at the edges of their calls:
memory that runs out, rows in front of the requests, refused row starts, status
words, values at the ends of their range."""

import pytest
import torch

from multics_b200.attention import hier_head_norm_rope
from multics_b200.paged8 import Paged8Cache, page_step, paged8_append, paged8_attention

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


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("first", [1, 63, 64, 256, 2000])
@pytest.mark.parametrize("rows", [330, 5, 1])
def test_append_behind_rows_of_no_request(dtype, first, rows):
    """Only pages that new tokens are in are read or written: not those in front
    of them, whose entries may be gone (-1) or another request's by now."""
    heads, lengths = 3, [4000, 70]
    g = torch.Generator().manual_seed(first)
    c = Paged8Cache(12, heads, dtype=dtype)
    c.k.copy_(torch.randint(-100, 100, c.k.shape, generator=g).to(dtype))
    c.v.copy_(torch.randint(-100, 100, c.v.shape, generator=g).to(dtype))
    c.k_scale.fill_(2.0 ** -120), c.v_scale.fill_(2.0 ** -120)
    page0 = (4000 - rows) // 64
    table = torch.full((2, 63), -1, dtype=torch.int32)
    table[0, page0:] = torch.arange(63 - page0) + 2
    table[0, page0 - 1], table[0, page0 - 2] = 0, 1  # (the other request's pages)
    table[1, :2] = torch.tensor([0, 1])
    k, v = (torch.randn(first + rows + 40, heads * 128, generator=g).to(BF).cuda() for _ in range(2))
    starts = [first, first + rows, first + rows + 40]
    alone = Paged8Cache.from_tensors(c.k.clone(), c.v.clone(), c.k_scale.clone(), c.v_scale.clone())
    for b in range(2):
        part = slice(starts[b], starts[b + 1])
        paged8_append(alone, k[part], v[part], table[b:b + 1].cuda(), _i32(lengths[b:b + 1]),
                      _i32([0, starts[b + 1] - starts[b]]))
    paged8_append(c, k, v, table.cuda(), _i32(lengths), _i32(starts))
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(c, name).view(torch.int8), getattr(alone, name).view(torch.int8)), name
    c.check(), alone.check()
