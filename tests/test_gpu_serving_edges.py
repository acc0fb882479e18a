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


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("prompt", [100, 3000])
@pytest.mark.parametrize("at", [0, 31, 63])
def test_append_of_a_prompt_beside_single_tokens(dtype, prompt, at):
    """A step of continuous batching: every request's pages are those of an append
    of its own."""
    n, heads = 64, 2
    counts = [prompt if b == at else 1 for b in range(n)]
    held = [prompt if b == at else 1 + 7 * b % 90 for b in range(n)]
    pages = [-(-h // 64) for h in held]
    g = torch.Generator().manual_seed(at)
    order = torch.randperm(sum(pages), generator=g).to(torch.int32)
    table, used = torch.full((n, max(pages)), -1, dtype=torch.int32), 0
    for b, p in enumerate(pages):
        table[b, :p], used = order[used:used + p], used + p
    starts = torch.tensor([0] + counts).cumsum(0).tolist()
    k, v = (torch.randn(starts[-1], heads * 128, generator=g).to(BF).cuda() for _ in range(2))
    c, alone = (Paged8Cache(sum(pages), heads, dtype=dtype) for _ in range(2))
    paged8_append(c, k, v, table.cuda(), _i32(held), _i32(starts))
    for b in range(n):
        part = slice(starts[b], starts[b + 1])
        paged8_append(alone, k[part], v[part], table[b:b + 1].cuda(), _i32(held[b:b + 1]), _i32([0, counts[b]]))
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(c, name).view(torch.int8), getattr(alone, name).view(torch.int8)), name
    c.check(), alone.check()


def _pool(pages, heads, dtype=torch.int8, seed=0):
    g = torch.Generator().manual_seed(seed)
    c = Paged8Cache(pages, heads, dtype=dtype)
    for t in (c.k, c.v):
        t.copy_(torch.randint(-120, 120, t.shape, generator=g).to(dtype))
    c.k_scale.fill_(2.0 ** -7), c.v_scale.fill_(2.0 ** -6)
    return c, g


def _poisoned(call):
    """call() where the memory it gets for its results held other numbers."""
    out, lse = call()
    out.fill_(7.0), lse.fill_(7.0)
    del out, lse
    return call()


@pytest.mark.parametrize("first,rows,tail", [(0, 1, 3), (2, 40, 0), (64, 300, 5), (3, 3000, 7)])
@pytest.mark.parametrize("width", [4, 40])
@pytest.mark.parametrize("requests", [1, 2])
def test_log_sum_of_rows_of_no_request_beside_a_given_out(first, rows, tail, width, requests):
    """The log-sum-exp is always a new tensor: -inf where no request is."""
    heads, starts = 4, [first + b * rows for b in range(requests + 1)]
    T = starts[-1] + tail
    c, g = _pool(4, 2)
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    table[:, :4] = _i32([0, 1, 2, 3])
    q = torch.randn(T, heads * 128, generator=g).to(BF).cuda()
    args = (q, c, table, _i32([200] * requests), _i32(starts), heads)
    out, lse = _poisoned(lambda: paged8_attention(*args, block_frames=0, return_lse=True))
    given = torch.empty_like(q)

    def call():
        given.fill_(7.0)
        return paged8_attention(*args, block_frames=0, out=given, return_lse=True)[0].clone(), \
            paged8_attention(*args, block_frames=0, out=given, return_lse=True)[1]

    for i in range(2):
        kept, other = _poisoned(call)
        assert torch.equal(other, lse) and (lse[:first] == float("-inf")).all()
        assert (lse[starts[-1]:] == float("-inf")).all() and torch.isfinite(lse[first:starts[-1]]).all()
        assert torch.equal(kept[first:starts[-1]], out[first:starts[-1]])
        assert (kept[:first] == 7).all() and (kept[starts[-1]:] == 7).all()


@pytest.mark.parametrize("n,T", [(3, 40), (31, 700), (200, 9000), (1500, 5000)])
@pytest.mark.parametrize("width", [4, 40])
@pytest.mark.parametrize("seed", range(4))
def test_row_starts_that_are_anything(n, T, width, seed):
    """Whatever the row starts are, every row of a fresh result is some request's
    or zeros, and rows that no request can have are zeros."""
    heads, g = 2, torch.Generator().manual_seed(seed)
    c, _ = _pool(4, 1)
    qs = torch.randint(-20, T + 20, (n + 1,), generator=g)
    if seed % 2:  # ascending but for a few
        qs = qs.sort().values
        qs[torch.randint(0, n + 1, (2,), generator=g)] = torch.tensor([T + 7, -3])
    table = torch.full((n, width), -1, dtype=torch.int32)
    table[:, :2] = torch.randint(0, 4, (n, 2), generator=g)
    q = torch.randn(T, heads * 128, generator=g).to(BF).cuda()
    args = (q, c, table.cuda(), _i32([100] * n), qs.to(torch.int32).cuda(), heads)
    out, lse = _poisoned(lambda: paged8_attention(*args, block_frames=0, return_lse=True))
    with pytest.raises(ValueError, match="row starts"):
        c.check()
    first = min(max(int(qs[0]), 0), T)
    end = max(first, min(int(qs[-1]), T))
    had = torch.zeros(T, dtype=torch.bool)
    for a, e in zip(qs.tolist(), qs.tolist()[1:]):
        if first <= a < e <= end:
            had[a:e] = True
    o, s = out.view(T, heads, 128).cpu(), lse.cpu()
    assert (o[~had] == 0).all() and (s[~had] == float("-inf")).all()
    zero = (o == 0).all(2)
    assert torch.equal(zero, s == float("-inf"))
    assert torch.isfinite(s[~zero]).all() and not (o == 7).all(2).any()
    # values of up to 120 * 2^-6: nothing but averages of them
    assert (o.abs() <= 2).all() and (s[~zero] != 7).all()


def test_every_cache_has_its_status_word():
    """A fault in one layer's cache is that cache's: no other reports or clears it."""
    pools = [_pool(2, 1)[0] for _ in range(3)]
    layers = [Paged8Cache.from_tensors(c.k, c.v, c.k_scale, c.v_scale) for c in pools for _ in range(200)]
    assert len({c.status.data_ptr() for c in layers}) == len(layers)
    q, bad = torch.ones(1, 128, dtype=BF, device="cuda"), _i32([[-1]])
    for c in (layers[0], layers[450]):
        paged8_attention(q, c, bad, _i32([5]), _i32([0, 1]), 1)
    for i, c in enumerate(layers):
        if i in (0, 450):
            with pytest.raises(ValueError, match="page pool"):
                c.check()
        c.check()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c = Paged8Cache.from_tensors(pools[0].k, pools[0].v, pools[0].k_scale, pools[0].v_scale)
        c.check()


def test_faults_of_replays_are_kept_until_checked():
    """A cache made in a capture: no replay clears what an earlier one recorded,
    and nothing else gets its word when the cache object is gone."""
    c, _ = _pool(2, 1)
    q, table, lengths, starts = torch.ones(1, 128, dtype=BF, device="cuda"), _i32([[0]]), _i32([5]), _i32([0, 1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inner = [Paged8Cache.from_tensors(c.k, c.v, c.k_scale, c.v_scale) for _ in range(2)]
        paged8_attention(q, inner[0], table, lengths, starts, 1)
        paged8_attention(q, inner[1], table, lengths, starts, 1)
    graph.replay()
    inner[0].check(), inner[1].check()
    table.fill_(-1)
    graph.replay()
    table.fill_(0)
    graph.replay()
    for layer in inner:
        with pytest.raises(ValueError, match="page pool"):
            layer.check()
        layer.check()
    del layer, inner
    table.fill_(-1)
    others = [Paged8Cache.from_tensors(c.k, c.v, c.k_scale, c.v_scale) for _ in range(600)]
    graph.replay()
    for other in others:
        other.check()


def test_what_is_recorded_during_a_check_is_kept(monkeypatch):
    from test_paged8_status_cpu import late_record

    late_record(_pool(2, 1)[0], monkeypatch)


def _norm_leaves(T=64):
    g = torch.Generator().manual_seed(T)
    q, k = (torch.randn(T, n, generator=g).to(BF).cuda().requires_grad_() for n in (256, 128))
    return q, k, torch.randn(T, 64, 2, generator=g).cuda(), torch.ones(128, device="cuda", requires_grad=True)


def test_error_word_cleared_between_forward_and_backward():
    """The device's error word is no input of the gradients."""
    from multics_b200._lib import dev_err
    from multics_b200.train import head_norm_rope_grad

    q, k, f, w = _norm_leaves()
    want = torch.autograd.grad(sum(t.float().sum() for t in head_norm_rope_grad(
        q, k, f, 2, 1, q_weight=w, k_weight=w)), (q, k, w))
    out = head_norm_rope_grad(q, k, f, 2, 1, q_weight=w, k_weight=w)
    dev_err(q.device).zero_()
    got = torch.autograd.grad(sum(t.float().sum() for t in out), (q, k, w))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.fixture
def no_error_word():
    """As in a process that has called nothing yet."""
    from multics_b200 import _lib

    words = dict(_lib._DEV_ERR)
    _lib._DEV_ERR.clear()
    yield _lib
    _lib._DEV_ERR.clear()
    _lib._DEV_ERR.update(words)


def test_error_word_first_used_in_a_graph(no_error_word):
    """It is zero before the first replay, and no replay clears it."""
    from multics_b200.attention import device_error

    T, H = 9, 2
    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn(T, H * 128, generator=g).to(BF).cuda() for _ in range(2))
    f, w, pos = torch.randn(4, 64, 2, generator=g).cuda(), torch.ones(128, device="cuda"), _i32([1] * T)
    warm = [torch.randn(64, 64, device="cuda") for _ in range(8)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hier_head_norm_rope(q, k, f, H, H, q_weight=w, k_weight=w, positions=pos)
    del warm
    word = no_error_word.dev_err(q.device)
    assert device_error() == 0
    graph.replay()
    assert device_error() == 0 and (out[0] != 0).any()
    pos.fill_(4)
    graph.replay()
    assert device_error() == 2
    pos.fill_(1)
    graph.replay()
    assert device_error() == 2 and no_error_word.dev_err(q.device) is word
    word.zero_()
    graph.replay()
    assert device_error() == 0
    del graph
    torch.cuda.empty_cache()
    filled = [torch.full((1024,), 5, dtype=torch.int32, device="cuda") for _ in range(64)]
    assert device_error() == 0 and len(filled) == 64


def test_error_word_of_inference_mode_is_cleared_outside(no_error_word):
    with torch.inference_mode():
        word = no_error_word.dev_err(torch.device("cuda", 0))
    word.zero_()
    q, k, f, w = _norm_leaves()
    from multics_b200.train import head_norm_rope_grad

    out = head_norm_rope_grad(q, k, f, 2, 1, q_weight=w, k_weight=w)
    assert torch.isfinite(torch.autograd.grad(out[0].float().sum(), q)[0]).all()


@pytest.mark.parametrize("head_norm", [True, False])
def test_paged_forward_past_the_rotation_table(head_norm):
    """A request that outgrows the table: its new rows are NaN and the cache
    reports them, whichever norm the module has; the others are as ever."""
    from multics_b200._lib import dev_err
    from multics_b200.attention import SelfAttention

    torch.manual_seed(3)
    layer = SelfAttention(256, 2, head_norm=head_norm).to("cuda", BF)
    freqs = torch.randn(70, 64, 2, device="cuda")
    x = torch.randn(1, 70, 256, device="cuda").to(BF)

    def run(adds, rows):
        cache = Paged8Cache(6, 2)
        table, free, count = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), _i32(list(range(6))), _i32([6])
        lengths, outs = _i32([0, 0]), []
        for add in adds:
            st = page_step(lengths, _i32(add), table, free, count, rows)
            st.check()
            outs.append(layer.paged_forward(x[:, :rows], freqs, cache, table, st))
            lengths, count = st.lengths, st.free_count
        return outs, cache, st

    outs, cache, st = run([[66, 2], [3, 4]], 68)
    cache.check()  # 69 tokens
    assert torch.isfinite(outs[0]).all() and torch.isfinite(outs[1]).all()
    outs, cache, st = run([[66, 2], [3, 4], [4, 1]], 68)  # positions 69 to 72: three past the table
    with pytest.raises(ValueError, match="NaN"):
        cache.check()
    assert outs[2][0, 1:4].isnan().all()
    keep = [0, *range(4, 68)]
    assert torch.isfinite(outs[2][0, keep]).all()
    dev_err(x.device).zero_()


SCALES = [[-126] * 6, [-126, 0, -126, 0, -126, 0], [0, -126, 0, -126, 0, -126], [-100, 27, 27, 27, 27, 27],
          [27, -100, 27, -100, 60, 60], [-126, 126, -126, 126, -126, 126], [126, -126] * 3, [-126, -63, 0, 63, 119, 126],
          [126, 119, 63, 0, -63, -126], [126] * 6, [-90, 0, 90, -90, 0, 90]]


@pytest.mark.parametrize("scales", SCALES)
@pytest.mark.parametrize("rows", [1, 40, 1200])
@pytest.mark.parametrize("shape", ["short", "long", "split"])
@pytest.mark.parametrize("spread", [0.0, 0.3, 6.0])
def test_value_scales_at_the_ends_of_their_range(scales, rows, shape, spread):
    """The weights of a page count in the denominator whatever its values are:
    outputs and log-sum-exps of value scales from 2^-126 to 2^126, even scores
    (spread 0), near ones and ones that leave pages far behind."""
    import paged8_oracle as P

    pages, width = (3, 4) if shape == "short" else (6, 40) if shape == "long" else (66, 66)
    heads, kv, n = 2, 1, 1 if shape == "split" else 3
    c, g = _pool(pages * n, kv, seed=rows)
    order = torch.randperm(pages * n, generator=g).view(n, pages)
    table = torch.full((n, width), -1, dtype=torch.int32)
    table[:, :pages] = order
    e = torch.tensor([scales[p % 6] for p in range(pages)])
    vs, v = c.v_scale.cpu(), c.v.cpu()
    for b in range(n):
        vs[order[b]] = (2.0 ** e.double()).float()[:, None]
        big = order[b][e >= 119]
        v[big] = v[big].sign()  # values within bf16
        if -100 in scales:
            v[order[b][e == -100]] = 0
    c.v_scale.copy_(vs), c.v.copy_(v)
    held, starts = [pages * 64 - 5] * n, [b * rows for b in range(n + 1)]
    q = (torch.randn(n * rows, heads * 128, generator=g) * spread).to(BF)
    out, lse = paged8_attention(q.cuda(), c, table.cuda(), _i32(held), _i32(starts), heads, block_frames=0, return_lse=True)
    kk, vv = P.values(c)
    want, want_lse, mag = P.attention(q, kk, vv, table.tolist(), held, starts, heads, block=0)
    vmax = float(vv.abs().max())
    tol = P.attention_bound(want, mag, held[0], vmax) + 2.0 ** -126  # (and fp32's least normal number)
    err = (out.cpu().double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())
    # the bound of the other tests: sums off by 2^-11, and fp32's own step
    assert ((lse.cpu().double() - want_lse).abs() <= 2.0 ** -10 + want_lse.abs() * 2.0 ** -20).all()
    c.check()


@pytest.mark.parametrize("rows", [1, 40, 1500])
def test_scores_of_nothing_between_huge_numbers(rows):
    """Queries and keys so large that their factor passes fp32's range, and no
    dimension in common: the scores are 0, and every key weighs the same."""
    c, g = _pool(8, 1)
    c.k.view(8, 1, 2, 64, 64)[:, :, 1] = 0
    c.k_scale.fill_(2.0 ** 100)
    q = torch.zeros(rows, 256, dtype=BF)
    q[:, 64:128], q[:, 192:] = 2.0 ** 90, -2.0 ** 60
    table = torch.full((1, 40), -1, dtype=torch.int32, device="cuda")
    table[0, :8] = torch.arange(8)
    out, lse = paged8_attention(q.cuda(), c, table, _i32([500]), _i32([0, rows]), 2, block_frames=0, return_lse=True)
    v = (c.v.double() * c.v_scale.double()[..., None, None]).transpose(2, 3).reshape(512, 128)[:500]
    want = v.mean(0).repeat(2)
    # bf16's half step of the value, and fp16's of the weights (all 1) and of their fp32 sum
    assert ((out.double() - want).abs() <= want.abs() * 2.0 ** -8 + v.abs().mean() * 2.0 ** -10).all()
    assert ((lse.double() - torch.tensor(500.0, device="cuda").log2()).abs() <= 2.0 ** -10).all()


@pytest.mark.parametrize("first", [True, False])
def test_values_of_zeros_beside_large_ones_weigh(first):
    """By appends alone: a page of zero values and one of 1e10, all scores equal:
    half the weight is on the zeros."""
    c, table = Paged8Cache(2, 1), _i32([[0, 1]])
    k = torch.ones(128, 128, dtype=BF, device="cuda")
    v = torch.zeros(128, 128, dtype=BF, device="cuda")
    v[slice(64, 128) if first else slice(0, 64)] = 1e10
    paged8_append(c, k, v, table, _i32([128]), _i32([0, 128]))
    large = float(v.max())
    for rows in (1, 200):
        q = torch.zeros(rows, 128, dtype=BF, device="cuda")
        out, lse = paged8_attention(q, c, table, _i32([128]), _i32([0, rows]), 1, block_frames=0, return_lse=True)
        # codes within half a step of 2^-7 (large has 8 bits), weights of 2^-10
        assert ((out.double() / (large / 2) - 1).abs() <= 2.0 ** -6).all()
        assert ((lse - 7).abs() <= 2.0 ** -10).all()


# row starts in units of R rows, of 2 R; the rows (in R) that only refused requests or none have
REFUSED = [([0, 1, 3], [(1, 2)]), ([-1, 1, 2], [(0, 1)]), ([0, 5, 2], [(0, 2)]), ([1, 0, 2], [(0, 2)]),
           ([0, 3], [(0, 2)]), ([-1, 2], [(0, 2)]), ([3, 4], [(0, 2)]), ([1, 3], [(0, 2)]), ([2, 0], [(0, 2)]),
           ([1, 2, -3, 7, 2], [(0, 1)]), ([0, 0, 1, 5, 5], [(1, 2)]), ([0, 1, 7, 1, 2], []), ([0, 9, 0, 9, 2], [(0, 2)])]


@pytest.mark.parametrize("starts,none", REFUSED)
@pytest.mark.parametrize("rows", [1, 33, 300, 1500])
@pytest.mark.parametrize("width", [4, 40])
def test_rows_of_refused_requests_are_zeros(starts, none, rows, width):
    """As those of refused lengths: nothing of a result is left as allocated."""
    n, heads = len(starts) - 1, 4
    c, g = _pool(n * 4, 2)
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    table[:, :4] = _i32([[4 * b, 4 * b + 1, 4 * b + 2, 4 * b + 3] for b in range(n)])
    q = torch.randn(2 * rows, heads * 128, generator=g).to(BF).cuda()
    lengths = _i32([200] * n)
    qs = _i32([s * rows for s in starts])
    out, lse = _poisoned(lambda: paged8_attention(q, c, table, lengths, qs, heads, block_frames=0, return_lse=True))
    with pytest.raises(ValueError, match="row starts"):
        c.check()
    dead = torch.zeros(2 * rows, dtype=torch.bool, device="cuda")
    for a, b in none:
        dead[a * rows:b * rows] = True
    assert (out[dead] == 0).all() and (lse[dead] == float("-inf")).all()
    for b in range(n):
        a, e = starts[b], starts[b + 1]
        if 0 <= a < e <= 2 and not dead[a * rows:e * rows].any():
            want, want_lse = paged8_attention(q[a * rows:e * rows], c, table[b:b + 1], lengths[:1],
                                              _i32([0, (e - a) * rows]), heads, block_frames=0, return_lse=True)
            got = out[a * rows:e * rows].float()
            # (which kernel, and which parts are joined, may differ: a rounding of the output)
            descend = any(x > y for x, y in zip(starts, starts[1:]))
            if descend and (got == 0).all():  # (starts that descend may hide a long request)
                assert (lse[a * rows:e * rows] == float("-inf")).all()
                continue
            assert ((got - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 2.0 ** -9 * want.float().abs().max()).all()
            assert torch.allclose(lse[a * rows:e * rows], want_lse, rtol=0, atol=2.0 ** -9)
    assert torch.isfinite(out).all()
    given = torch.full_like(q, 7.0)
    paged8_attention(q, c, table, lengths, qs, heads, block_frames=0, out=given)
    assert (given[dead] == 7).all()
    assert ((given[~dead] == out[~dead]) | ((given[~dead] == 7) & (out[~dead] == 0))).all()
