"""8-bit paged cache on the GPU against 64-bit restatements: block tables and
slot maps, the append, the attention, and a run of them together."""

import random

import pytest
import torch

import paged8_oracle as P
from multics_b200 import paged8
from multics_b200.attention import device_error
from multics_b200.paged8 import Paged8Cache, page_step, paged8_append, paged8_attention

pytestmark = pytest.mark.gpu

FORMATS = [torch.int8, torch.float8_e4m3fn]
BF = torch.bfloat16


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------- block tables

def _random_steps(n, width, pages, seed, steps=6, most=200):
    """Lengths, additions (growth, drops, ends, idle requests) that fit."""
    r = random.Random(seed)
    lengths, free = [0] * n, pages
    for _ in range(steps):
        add = []
        for b in range(n):
            kind = r.random()
            a = -lengths[b] if kind < 0.1 else -r.randint(0, lengths[b]) if kind < 0.2 else \
                0 if kind < 0.3 else r.choice((1, 1, r.randint(1, most)))
            a = min(a, width * 64 - lengths[b])
            grow = -(-(lengths[b] + a) // 64) - -(-lengths[b] // 64)
            if grow > free:
                a, grow = 0, 0
            free -= max(grow, 0)  # pages given up this step are counted from the next
            add.append(a)
        yield lengths, add
        lengths = [x + a for x, a in zip(lengths, add)]
        free = pages - sum(-(-x // 64) for x in lengths)


@pytest.mark.parametrize("n,width,seed", [(1, 1, 0), (1, 40, 1), (5, 9, 2), (33, 4, 3), (1500, 3, 4)])
@pytest.mark.parametrize("in_place", [False, True])
def test_page_step(n, width, seed, in_place):
    pages = n * width * 3 // 4 + 2
    ids = torch.randperm(pages, generator=_gen(seed)).tolist()
    table, free, count = [[-1] * width for _ in range(n)], ids[:], pages
    wide = torch.full((n, width + 3), -1, dtype=torch.int32, device="cuda")
    d_table, d_free, d_count, d_len = wide[:, :width], _i32(free), _i32([count]), _i32([0] * n)
    for lengths, add in _random_steps(n, width, pages, seed):
        rows = sum(max(a, 0) for a in add) + 2
        d_add = _i32(add)
        st = page_step(d_len, d_add, d_table, d_free, d_count, rows, in_place=in_place)
        st.check()
        after, count, q_start, slots, positions = P.step(lengths, add, table, free, count)
        assert st.lengths.tolist() == after and st.free_count.tolist() == [count]
        assert st.q_start.tolist() == q_start
        assert st.slots.tolist() == slots + [-1, -1]
        assert st.positions.tolist() == positions + [-1, -1]
        assert d_table.tolist() == table
        assert d_free.tolist()[:count] == free[:count]
        assert (wide[:, width:] == -1).all()
        if in_place:
            assert st.lengths is d_len and st.free_count is d_count
        d_len, d_count = st.lengths, st.free_count


def test_page_step_maps_many_rows():
    """More rows than one block maps: one long request between short ones."""
    lengths, add, width = [70, 0, 63], [1, 20000, 2], 400
    table = [[-1] * width for _ in lengths]
    table[0][:2], table[2][:1] = [3, 1], [0]
    free = [2] + list(range(4, 400))
    d = [_i32(lengths), _i32(add), _i32(table), _i32(free), _i32([len(free)])]
    st = page_step(*d, 20100)
    st.check()
    after, count, q_start, slots, positions = P.step(lengths, add, table, free, len(free))
    assert st.q_start.tolist() == q_start and st.free_count.tolist() == [count]
    assert st.slots.tolist() == slots + [-1] * (20100 - len(slots))
    assert st.positions.tolist() == positions + [-1] * (20100 - len(slots))
    assert d[2].tolist() == table


@pytest.mark.parametrize("n", [1, 33, 1200, 5000])
@pytest.mark.parametrize("most", [1, 300])
def test_page_step_maps_rows_between_requests_without_any(n, most):
    """Rows of requests that lie far apart, few or hundreds each, mapped by the
    step itself or by a grid of their own."""
    r, width = random.Random(n + most), 8
    lengths = [r.randint(0, 90) for _ in range(n)]
    add = [0] * n
    for b in [0, n - 1] + [r.randrange(n) for _ in range(min(n, 60))]:
        add[b] = r.randint(1, most)
    if n > 1:
        add[n // 2] = -lengths[n // 2]
    table, at = [], 0
    for x in lengths:
        p = -(-x // 64)
        table.append(list(range(at, at + p)) + [-1] * (width - p))
        at += p
    free = list(range(at, at + 7 * n))
    rows = sum(max(x, 0) for x in add) + 70
    d = [_i32(lengths), _i32(add), _i32(table), _i32(free + [-1] * at), _i32([len(free)])]
    st = page_step(*d, rows)
    st.check()
    after, count, q_start, slots, positions = P.step(lengths, add, table, free + [-1] * at, len(free))
    assert st.lengths.tolist() == after and st.q_start.tolist() == q_start
    assert st.slots.tolist() == slots + [-1] * 70
    assert st.positions.tolist() == positions + [-1] * 70
    assert d[2].tolist() == table


@pytest.mark.parametrize("n", [1025, 2048, 5003])
def test_page_step_of_many_requests_is_taken_or_refused_whole(n):
    """More requests than a block has threads: pages change hands between the
    blocks' requests, and one request's fault refuses the step of all."""
    r, width = random.Random(n), 3
    lengths = [r.randint(0, 190) for _ in range(n)]
    add = [-r.randint(0, x) if r.random() < 0.6 else r.randint(0, 192 - x) for x in lengths]
    table, at = [], 0
    for x in lengths:
        p = -(-x // 64)
        table.append(list(range(at, at + p)) + [-1] * (width - p))
        at += p
    free = list(range(at, at + n // 4)) + [-1] * at
    rows = sum(max(x, 0) for x in add)
    for change in (None, 0, n // 2, n - 1):
        d = [_i32(lengths), _i32(add), _i32(table), _i32(free), _i32([n // 4])]
        if change is not None:
            d[1][change] = 193
        st = page_step(*d, rows)
        if change is None:
            st.check()
            t, f = [x[:] for x in table], free[:]
            after, count, q_start, slots, positions = P.step(lengths, add, t, f, n // 4)
            assert st.lengths.tolist() == after and st.free_count.tolist() == [count]
            assert st.q_start.tolist() == q_start and st.slots.tolist() == slots
            assert st.positions.tolist() == positions
            assert d[2].tolist() == t and d[3].tolist()[:count] == f[:count]
        else:
            with pytest.raises(ValueError, match="block table"):
                st.check()
            assert torch.equal(st.lengths, d[0]) and st.free_count.tolist() == [n // 4]
            assert not st.q_start.any() and (st.slots == -1).all() and (st.positions == -1).all()
            assert d[2].tolist() == table and d[3].tolist() == free


@pytest.mark.parametrize("change,match", [
    (dict(add=[60, 64]), "free pages"), (dict(rows=5), "rows"), (dict(add=[4, 300]), "block table"),
    (dict(add=[-11, 0]), "below -length"), (dict(most=3), "above the step"),
    (dict(lengths=[-1, 3]), "block table"), (dict(count=9), "free list"), (dict(count=-1), "free list")])
def test_page_step_refused_whole(change, match):
    """A step that cannot be taken leaves everything and maps no row."""
    c = dict(lengths=[10, 60], add=[2, 4], table=[[1, -1], [0, -1]], free=[7], count=1, rows=8, most=None)
    c.update(change)
    table, free = _i32(c["table"]), _i32(c["free"])
    st = page_step(_i32(c["lengths"]), _i32(c["add"]), table, free, _i32([c["count"]]), c["rows"],
                   most_new=c["most"])
    with pytest.raises(ValueError, match=match):
        st.check()
    assert st.lengths.tolist() == c["lengths"] and st.free_count.tolist() == [c["count"]]
    assert st.q_start.tolist() == [0, 0, 0]
    assert set(st.slots.tolist()) == set(st.positions.tolist()) == {-1}
    assert table.tolist() == c["table"] and free.tolist() == c["free"]


def test_page_step_without_requests_or_rows():
    st = page_step(_i32([]), _i32([]), torch.empty(0, 4, dtype=torch.int32, device="cuda"), _i32([3]),
                   _i32([1]), 2)
    st.check()
    assert st.q_start.tolist() == [0] and st.slots.tolist() == [-1, -1]
    st = page_step(_i32([5]), _i32([-5]), _i32([[2]]), _i32([0]), _i32([0]), 0)
    st.check()
    assert st.lengths.tolist() == [0] and st.free_count.tolist() == [1] and st.slots.numel() == 0


# ------------------------------------------------------------------- append

class _Session:
    """Requests on a cache, with the appended bf16 rows kept for the oracle."""

    def __init__(self, n, heads, dtype, width=12, pages=None, seed=0):
        pages = n * width if pages is None else pages
        self.cache = Paged8Cache(pages, heads, dtype=dtype)
        self.g = _gen(seed)
        order = torch.randperm(pages, generator=self.g).to(torch.int32)
        self.table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
        self.free, self.count = order.cuda(), _i32([pages])
        self.lengths = _i32([0] * n)
        self.heads, self.n = heads, n
        self.k = [torch.zeros(0, heads, 128, dtype=BF) for _ in range(n)]
        self.v = [torch.zeros(0, heads, 128, dtype=BF) for _ in range(n)]

    def append(self, add, scale=1.0, spare=0, k=None, v=None):
        total = sum(max(a, 0) for a in add)
        rows = total + spare
        st = page_step(self.lengths, _i32(add), self.table, self.free, self.count, rows)
        st.check()
        k = torch.randn(rows, self.heads * 128, generator=self.g).mul(scale).to(BF) if k is None else k
        v = torch.randn(rows, self.heads * 128, generator=self.g).mul(scale).to(BF) if v is None else v
        paged8_append(self.cache, k.cuda(), v.cuda(), self.table, st.lengths, st.q_start)
        at = 0
        for b, a in enumerate(add):
            if a < 0:
                self.k[b], self.v[b] = self.k[b][:a], self.v[b][:a]
            else:
                for mine, x in ((self.k, k), (self.v, v)):
                    mine[b] = torch.cat([mine[b], x[at:at + a].view(a, self.heads, 128)])
                at += a
        self.lengths, self.count, self.step = st.lengths, st.free_count, st
        return st

    def held(self):
        """Keys and values held by each request, float64 [held, heads, 128]."""
        k, v = P.values(self.cache)
        table, lengths = self.table.cpu().long(), self.lengths.tolist()
        out = []
        for b, n in enumerate(lengths):
            pg = table[b][:-(-n // 64)]
            out.append((k[pg].transpose(1, 2).flatten(0, 1)[:n], v[pg].transpose(1, 2).flatten(0, 1)[:n]))
        return out


def _near(held, rows, scale, dtype, growths):
    """Every held value within the roundings it went through: half a step of
    its block's scale (int8), or half a step of its own binade or of the
    subnormals (e4m3), once and once more per growth of the scale."""
    x = rows.double()
    if dtype == torch.int8:
        tol = scale / 2 * (1 + growths)
    else:
        tol = torch.maximum(x.abs() * 2.0 ** -4, scale * 2.0 ** -10) * (1 + growths)
    assert ((held - x).abs() <= tol * (1 + 1e-12)).all()


def _scales(s, b, which):
    n = int(s.lengths[b])
    pg = s.table[b].cpu().long()[:-(-n // 64)]
    sc = getattr(s.cache, which).cpu().double()[pg]  # [pages, heads]
    return sc.repeat_interleave(64, 0)[:n, :, None]


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("heads", [1, 5, 24])
def test_append_fresh_pages_are_the_nearest_codes(dtype, heads):
    """Pages written in one call: the scale and every code are exactly those of
    the definition."""
    s = _Session(4, heads, dtype, seed=heads)
    s.append([1, 64, 130, 0], spare=3)
    for b, (k, v) in enumerate(s.held()):
        for x, held, which in ((s.k[b], k, "k_scale"), (s.v[b], v, "v_scale")):
            sc = _scales(s, b, which)
            for p in range(0, x.shape[0], 64):
                for h in range(heads):
                    blk = x[p:p + 64, h].double()
                    want = P.scale_for(float(blk.abs().max()), dtype)
                    assert float(sc[p, h]) == want
                    assert torch.equal(held[p:p + 64, h], P.encode(blk / want, dtype) * want)
    s.cache.check()


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("sizes", [[1] * 70, [63, 2, 64, 7], [130, 1, 1, 200, 15]])
def test_append_into_partly_held_pages(dtype, sizes):
    """Appends of rising magnitude: scales only grow, held codes follow them,
    and untouched tokens keep their bytes."""
    s = _Session(2, 3, dtype, seed=len(sizes))
    for i, n in enumerate(sizes):
        before = [(k.clone(), v.clone()) for k, v in s.held()]
        s.append([n, n // 2], scale=2.0 ** (i % 7 - 3))
        for (k0, v0), (k1, v1) in zip(before, s.held()):
            whole = k0.shape[0] // 64 * 64
            assert torch.equal(k0[:whole], k1[:whole]) and torch.equal(v0[:whole], v1[:whole])
    for b, (k, v) in enumerate(s.held()):
        _near(k, s.k[b], _scales(s, b, "k_scale"), dtype, 6)
        _near(v, s.v[b], _scales(s, b, "v_scale"), dtype, 6)
    s.cache.check()


@pytest.mark.parametrize("dtype", FORMATS)
def test_append_growth_re_encodes_once(dtype):
    """A page held at a small scale and grown by one large token: the held codes
    are those of the old values under the new scale, rounded to nearest even."""
    s = _Session(1, 2, dtype)
    s.append([37])
    old_k, old_v = s.held()[0]
    s.append([1], scale=300.0)
    for x, old, (which, new) in ((s.k[0], old_k, ("k_scale", s.held()[0][0])),
                                 (s.v[0], old_v, ("v_scale", s.held()[0][1]))):
        sc = _scales(s, 0, which)
        for h in range(2):
            assert float(sc[0, h]) == P.scale_for(float(x[37, h].double().abs().max()), dtype)
        assert torch.equal(new[:37], P.encode(old / sc[:37], dtype) * sc[:37])


@pytest.mark.parametrize("dtype", FORMATS)
def test_append_zeros_huge_tiny_and_not_finite(dtype):
    s = _Session(1, 1, dtype)
    k = torch.zeros(6, 128, dtype=BF)
    k[1], k[2, 5], k[3, 7] = 3.0e38, float("inf"), float("nan")
    v = torch.full((6, 128), 1e-38, dtype=BF)
    v[4, 100] = float("-inf")
    s.append([6], k=k, v=v)
    with pytest.raises(ValueError, match="NaN"):
        s.cache.check()
    hk, hv = s.held()[0]
    top = P.TOP[dtype]
    sk, sv = P.scale_for(float(k[1, 0]), dtype), 2.0 ** -100
    assert torch.equal(hk[0], torch.zeros(1, 128, dtype=torch.float64))
    assert float(hk[2, 0, 5]) == top * sk and float(hk[3, 0, 7]) == 0.0
    assert torch.isfinite(hk).all() and torch.isfinite(hv).all()
    assert float(hv[4, 0, 100]) == -top * sv and float(hv[0, 0, 0]) == 0.0


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("heads", [2, 30])
@pytest.mark.parametrize("adds", [[3, 0, 0, 1, 0, 5, 0, 0, 0], [2, 3, 4, 1, 0, 0, 4, 3, 2],
                                  [7, 0, 1, 9, 2, 12, 0, 17, 1], [1] * 9, [4] * 9, [0] * 8 + [2]])
def test_append_a_few_tokens_at_a_time(dtype, heads, adds):
    """Every token has the code of its value whatever it comes with, at every
    place of a page; what is not finite too."""
    s = _Session(9, heads, dtype, width=3, seed=heads)
    top = P.TOP[dtype]
    for i in range(-1, 10):
        add = [1 + b for b in range(9)] if i < 0 else adds
        total = sum(add)
        k, v = (torch.randn(total, heads * 128, generator=s.g).clamp(-4, 4).to(BF) for _ in range(2))
        at = 0
        for b, n in enumerate(add):  # every page's first token has the largest value: scales stay
            held = s.k[b].shape[0]
            for t in range(n):
                if (held + t) % 64 == 0:
                    k[at + t], v[at + t] = 4.0, -4.0
            at += n
        if i == 3 and total > 1:
            k[1, 5], v[total - 1, 7], k[total - 1, 130], v[1, 131] = (float(x) for x in ("nan", "nan", "inf", "-inf"))
        s.append(add, k=k, v=v)
    for b, (k, v) in enumerate(s.held()):
        for got, x in ((k, s.k[b].double()), (v, s.v[b].double())):
            sc = P.scale_for(4.0, dtype)
            want = P.encode(torch.where(x.isfinite(), x, torch.zeros_like(x)) / sc, dtype) * sc
            want = torch.where(x.isinf(), x.sign() * top * sc, want)
            assert torch.equal(got, want)
    if sum(adds) > 1:
        with pytest.raises(ValueError, match="NaN"):
            s.cache.check()
    s.cache.check()


def test_append_rows_with_strides_and_another_stream():
    s, ref = _Session(2, 3, torch.int8, seed=5), _Session(2, 3, torch.int8, seed=5)
    k = torch.randn(90, 3 * 128, generator=_gen(1)).to(BF)
    v = torch.randn(90, 3 * 128, generator=_gen(2)).to(BF)
    ref.append([50, 40], k=k, v=v)
    st = page_step(s.lengths, _i32([50, 40]), s.table, s.free, s.count, 90)
    wide = torch.cat([k, v], 1).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged8_append(s.cache, wide[:, :384], wide[None, :, 384:], s.table, st.lengths, st.q_start)
    torch.cuda.current_stream().wait_stream(side)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(s.cache, name), getattr(ref.cache, name))


def test_append_skips_what_its_tables_get_wrong():
    """Bad pages, lengths and row starts are recorded and skipped; the pool's
    other bytes stay."""
    for table, lengths, q_start, match in (
            ([[5, 1]], [70], [0, 70], "page pool"), ([[-1, 1]], [70], [0, 70], "page pool"),
            ([[0, 1]], [200], [0, 70], "block table"), ([[0, 1]], [60], [0, 70], "block table"),
            ([[0, 1]], [70], [0, 90], "row starts"), ([[0, 1]], [70], [-3, 70], "row starts"),
            ([[0, 1]], [70], [9, 3], "row starts")):
        c = Paged8Cache(2, 2)
        x = torch.ones(80, 256, dtype=BF, device="cuda")
        paged8_append(c, x, x, _i32(table), _i32(lengths), _i32(q_start))
        with pytest.raises(ValueError, match=match):
            c.check()
        keep = 0 if "page pool" in match else slice(None)
        assert (c.k[keep] == 0).all() and (c.v[keep] == 0).all()


# ---------------------------------------------------------------- attention

def _filled(lengths, heads, dtype, seed=0, width=None, extra=0):
    """A cache holding `lengths` tokens per request in shuffled pages, all
    other bytes at their largest code."""
    g = _gen(seed)
    pages = [-(-n // 64) for n in lengths]
    width = max(pages + [1]) if width is None else width
    total = sum(pages) + 2 + extra
    c = Paged8Cache(total, heads, dtype=dtype)
    if dtype == torch.int8:
        c.k.copy_((torch.randn(c.k.shape, generator=g) * 40).round().clamp(-127, 127))
        c.v.copy_((torch.randn(c.v.shape, generator=g) * 40).round().clamp(-127, 127))
    else:
        c.k.copy_((torch.randn(c.k.shape, generator=g) * 100).clamp(-448, 448).to(dtype))
        c.v.copy_((torch.randn(c.v.shape, generator=g) * 100).clamp(-448, 448).to(dtype))
    e = torch.randint(-8, -4, (total, heads), generator=g)
    c.k_scale.copy_(2.0 ** e)
    c.v_scale.copy_(2.0 ** torch.randint(-9, -3, (total, heads), generator=g))
    order = torch.randperm(total, generator=g).tolist()
    table, at = [], 0
    for p in pages:
        table.append(order[at:at + p] + [-7] * (width - p))
        at += p
    return c, table, g


def _check(c, table, lengths, counts, heads, g, *, spare=0, q=None, **kw):
    q_start = [0]
    for n in counts:
        q_start.append(q_start[-1] + n)
    T = q_start[-1] + spare
    if q is None:
        q = (torch.randn(T, heads * 128, generator=g) * 1.5).to(BF)
    args = (q.cuda(), c, _i32(table).view(len(lengths), -1), _i32(lengths), _i32(q_start), heads)
    names = dict(tokens_per_frame=kw.pop("frame", 1), block_frames=kw.pop("block", 1),
                 window=kw.pop("window", -1))
    out, lse = paged8_attention(*args, return_lse=True, **names, **kw)
    again = paged8_attention(*args, **names, **kw)
    assert torch.equal(out, again)
    k, v = P.values(c)
    want, want_lse, mag = P.attention(q, k, v, table, lengths, q_start, heads,
                                      frame=names["tokens_per_frame"], block=names["block_frames"],
                                      window=names["window"], scale=kw.get("softmax_scale"))
    vmax = float(v[[p for row, n in zip(table, lengths) for p in row[:-(-n // 64)]]].abs().max()) \
        if any(lengths) else 0.0
    err = (out.cpu().double() - want).abs()
    tol = P.attention_bound(want, mag, max(lengths + [0]), vmax)
    assert (err <= tol).all(), float((err / tol).max())
    lse = lse.cpu().double()
    assert torch.equal(lse.isinf(), want_lse.isinf())
    fin = ~want_lse.isinf()
    # log2 of a sum whose terms are off by 2^-11 at most, and fp32's own step
    assert ((lse - want_lse)[fin].abs() <= 2.0 ** -10 + want_lse[fin].abs() * 2.0 ** -20).all()
    c.check()
    assert device_error() == 0
    return out


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (8, 1), (12, 4), (15, 3)])
def test_attention_single_rows(dtype, heads, kv):
    lengths = [1, 64, 65, 200, 1000, 63, 0, 129]
    c, table, g = _filled(lengths, kv, dtype, seed=heads)
    _check(c, table, lengths, [1, 1, 1, 1, 1, 1, 0, 1], heads, g, max_rows=1)


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("mask", [(1, 1, -1), (1, 0, -1), (7, 3, -1), (7, 1, 4), (1, 3, 21), (5, 0, 2),
                                  (220, 1, 1)])
@pytest.mark.parametrize("heads,kv", [(2, 2), (6, 2)])
def test_attention_rows_and_masks(dtype, mask, heads, kv):
    lengths, counts = [5, 700, 64, 130, 1, 333], [5, 300, 3, 130, 1, 17]
    c, table, g = _filled(lengths, kv, dtype, seed=mask[0])
    _check(c, table, lengths, counts, heads, g, spare=3, frame=mask[0], block=mask[1], window=mask[2])


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("lengths,counts", [([3000], [1]), ([3001, 20], [2, 1]), ([4097], [9]),
                                            ([2500, 1], [600, 1]), ([129], [129])])
def test_attention_long_keys_few_heads(dtype, lengths, counts):
    """Few tiles: the keys are split between blocks and joined."""
    c, table, g = _filled(lengths, 2, dtype, seed=7)
    _check(c, table, lengths, counts, 2, g)
    _check(c, table, lengths, counts, 4, g, max_rows=max(counts))


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("counts", [[17, 128, 127, 64, 65], [100, 129, 256, 64, 1], [257, 200, 120, 33, 40]])
@pytest.mark.parametrize("heads", [1, 4])
def test_attention_tiles_of_one_half(dtype, counts, heads):
    """Up to 128 pairs in a tile, one, two and many key tiles, whole and split."""
    lengths = [1500, 700, 400, 64, 130]
    c, table, g = _filled(lengths, 1, dtype, seed=heads)
    for mask in ((1, 1, -1), (3, 0, -1), (10, 2, 9)):
        _check(c, table, lengths, counts, heads, g, frame=mask[0], block=mask[1], window=mask[2])


@pytest.mark.parametrize("width", [None, 90])
def test_attention_max_rows_chooses_kernels_not_results(width):
    """Requests of more rows than the caller said, short and split keys."""
    lengths, counts = [300, 40, 2000 if width else 200], [30, 17, 9]
    c, table, g = _filled(lengths, 2, torch.int8, width=width)
    for most in (1, 8, 9, 20, None):
        _check(c, table, lengths, counts, 4, g, spare=5, max_rows=most)


def test_attention_rows_of_other_sequences_than_the_cache():
    """block_frames=0: the rows need not be tokens of the cache."""
    lengths, counts = [30, 0, 100], [70, 5, 3]
    c, table, g = _filled(lengths, 2, torch.int8)
    out = _check(c, table, lengths, counts, 2, g, block=0)
    assert (out[70:75] == 0).all()


def test_attention_rows_beyond_the_held_tokens_see_nothing():
    lengths, counts = [3, 66], [5, 70]
    c, table, g = _filled(lengths, 1, torch.int8)
    for frame, block, window in ((1, 1, -1), (2, 0, 3)):
        out = _check(c, table, lengths, counts, 1, g, frame=frame, block=block, window=window)
        assert (out[:2] == 0).all() and (out[5:9] == 0).all()


@pytest.mark.parametrize("dtype", FORMATS)
def test_attention_page_scales_far_apart(dtype):
    """Value scales from 2^-60 to 2^40 and queries of very different size: each
    row's output keeps its relative accuracy."""
    lengths = [64 * 6]
    c, table, g = _filled(lengths, 1, dtype)
    ks, vs = c.k_scale.clone(), c.v_scale.clone()
    for i, (a, b) in enumerate([(-5, -60), (-5, 0), (-5, 40), (-20, -30), (-5, 5), (-60, 10)]):
        ks[table[0][i]], vs[table[0][i]] = 2.0 ** a, 2.0 ** b
    c.k_scale.copy_(ks), c.v_scale.copy_(vs)
    q = (torch.randn(40, 128, generator=g) * 10.0 ** torch.linspace(-30, 1, 40)[:, None]).to(BF)
    _check(c, table, lengths, [40], 1, g, q=q, block=0)
    # rows whose weight is all on the page of tiny values
    k, _ = P.values(c)
    c.k_scale[table[0][0]] = 2.0 ** 3
    q = (k[table[0][0], 0, :40].sign() * 4).to(BF)
    _check(c, table, lengths, [40], 1, g, q=q, block=0)


@pytest.mark.parametrize("counts", [[1], [40], [300]])
def test_attention_query_not_finite_stays_in_its_row(counts):
    lengths = [400]
    c, table, g = _filled(lengths, 1, torch.int8)
    q = torch.randn(counts[0], 256, generator=g).to(BF)
    clean = paged8_attention(q.cuda(), c, _i32(table), _i32(lengths), _i32([0] + counts), 2)
    q[0, 3], q[-1, 130] = float("nan"), float("inf")
    out = paged8_attention(q.cuda(), c, _i32(table), _i32(lengths), _i32([0] + counts), 2)
    assert out[0, :128].isnan().all()
    assert not torch.isfinite(out[-1, 128:]).any()
    assert torch.equal(out[-1, :128], clean[-1, :128]) or counts[0] == 1
    assert torch.equal(out[1:-1], clean[1:-1])


@pytest.mark.parametrize("counts", [[1], [40], [300]])
def test_attention_query_not_finite_has_no_log_sum(counts):
    lengths = [400]
    c, table, g = _filled(lengths, 1, torch.int8)
    q = torch.randn(counts[0], 256, generator=g).to(BF)
    args = (c, _i32(table), _i32(lengths), _i32([0] + counts), 2)
    _, clean = paged8_attention(q.cuda(), *args, return_lse=True)
    q[0, 3] = float("nan")
    _, lse = paged8_attention(q.cuda(), *args, return_lse=True)
    assert lse[0, 0].isnan()
    assert torch.equal(lse.flatten()[1:], clean.flatten()[1:])


@pytest.mark.parametrize("counts", [[3, 2], [9, 300], [200, 5, 300], [300, 5], [1, 1, 1]])
@pytest.mark.parametrize("width", [9, 40])
def test_attention_rows_before_the_first_request(counts, width):
    """The last requests of a batch by themselves, in its rows: those of the
    others are zeros, or left."""
    lengths = [300, 520, 400][:len(counts)]
    c, table, g = _filled(lengths, 2, torch.int8, width=width)
    ends = [0]
    for n in counts:
        ends.append(ends[-1] + n)
    T, first = ends[-1] + 3, counts[0]
    q = torch.randn(T, 512, generator=g).to(BF).cuda()
    args = (c, _i32(table[1:]), _i32(lengths[1:]), _i32(ends[1:]), 4)
    out, lse = paged8_attention(q, *args, return_lse=True)
    want, want_lse = paged8_attention(q[first:].contiguous(), c, _i32(table[1:]), _i32(lengths[1:]),
                                      _i32([e - first for e in ends[1:]]), 4, return_lse=True)
    # (which parts are joined may differ: a rounding of the output)
    tol = 2.0 ** -7 * want.float().abs() + 2.0 ** -9 * want.float().abs().max()
    assert ((out[first:].float() - want.float()).abs() <= tol).all()
    assert torch.allclose(lse[first:-3], want_lse[:-3], rtol=0, atol=2.0 ** -9)
    for rows in (slice(0, first), slice(T - 3, T)):
        assert (out[rows] == 0).all() and (lse[rows] == float("-inf")).all()
    given = torch.full_like(q, 7.0)
    paged8_attention(q, *args, out=given)
    assert torch.equal(given[first:-3], out[first:-3])
    assert (given[:first] == 7).all() and (given[-3:] == 7).all()
    c.check()


@pytest.mark.parametrize("lengths,counts", [([100], [1]), ([3000], [1]), ([3000, 900], [5, 2]),
                                            ([2500] * 30, [1] * 30), ([300], [300]), ([900, 500], [100, 3])])
def test_attention_over_its_queries(lengths, counts):
    c, table, g = _filled(lengths, 2, torch.float8_e4m3fn)
    q = torch.randn(sum(counts) + 2, 512, generator=g).to(BF).cuda()
    starts = torch.cumsum(torch.tensor([0] + counts), 0)
    args = (c, _i32(table), _i32(lengths), _i32(starts.tolist()), 4)
    want, tail = paged8_attention(q, *args), q[-2:].clone()
    assert paged8_attention(q, *args, out=q) is q
    assert torch.equal(q[:-2], want[:-2]) and torch.equal(q[-2:], tail)


def test_attention_few_requests_with_rows_among_many():
    """Requests without rows, before, between and behind those with some."""
    lengths, counts = [0] * 3000, [0] * 3000
    for b, held, n in ((7, 2400, 1), (8, 2300, 3), (1500, 700, 40), (2990, 90, 2)):
        lengths[b], counts[b] = held, n
    lengths[1501] = 130
    for heads in (2, 16):
        c, table, g = _filled(lengths, 1, torch.int8)
        _check(c, table, lengths, counts, heads, g, spare=4)


def test_attention_strided_rows_given_out_and_tail():
    lengths, counts = [90, 200], [2, 100]
    c, table, g = _filled(lengths, 2, torch.int8)
    q = torch.randn(110, 512, generator=g).to(BF).cuda()
    args = (c, _i32(table), _i32(lengths), _i32([0, 2, 102]), 2)
    want = paged8_attention(q[:, 256:].contiguous(), *args)
    assert (want[102:] == 0).all()
    wide = torch.full((110, 300), 7.0, dtype=BF, device="cuda")
    got = paged8_attention(q[None, :, 256:], *args, out=wide[:, 8:264])
    assert got.data_ptr() == wide[:, 8:264].data_ptr()
    assert torch.equal(got[:102], want[:102])
    assert (wide[102:] == 7).all() and (wide[:, :8] == 7).all() and (wide[:, 264:] == 7).all()
    one = torch.full((2, 259), 7.0, dtype=BF, device="cuda")  # one row, of odd stride and place
    one[:1, 3:] = q[:1, :256]
    alone = (c, _i32(table[:1]), _i32(lengths[:1]), _i32([0, 1]), 2)
    assert torch.equal(paged8_attention(one[:1, 3:], *alone, out=one[1:, 3:]),
                       paged8_attention(q[:1, :256], *alone))
    assert (one[1, :3] == 7).all()
    assert paged8_attention(q[:0, :256], *args).shape == (0, 256)
    none = paged8_attention(q[:3, :256], c, _i32([]).view(0, 1), _i32([]), _i32([0]), 2)
    assert (none == 0).all()


@pytest.mark.parametrize("rows", [1, 150])
def test_attention_skips_what_its_tables_get_wrong(rows):
    """A page outside the pool drops its keys, a length outside the table or
    row starts outside the rows their request; all are recorded."""
    c, table, g = _filled([200, 200], 1, torch.int8)
    q = torch.randn(2 * rows, 128, generator=g).to(BF).cuda()
    starts = _i32([0, rows, 2 * rows])
    good = paged8_attention(q, c, _i32(table), _i32([200, 200]), starts, 1, block_frames=0)
    for bad in (c.num_pages, -1, 2 ** 31 - 1, -2 ** 31):
        t = [table[0][:], table[1]]
        t[0][1] = bad
        out = paged8_attention(q, c, _i32(t), _i32([200, 200]), starts, 1, block_frames=0)
        with pytest.raises(ValueError, match="page pool"):
            c.check()
        assert torch.equal(out[rows:], good[rows:]) and torch.isfinite(out).all()
        drop = [table[0][0], table[0][2], table[0][3]]
        want = paged8_attention(q[:rows], c, _i32([drop]), _i32([136]), _i32([0, rows]), 1,
                                block_frames=0)
        assert (out[:rows].float() - want.float()).abs().max() <= 2.0 ** -6 * want.float().abs().max()
    for lengths, match in (([300, 200], "block table"), ([-1, 200], "block table")):
        out = paged8_attention(q, c, _i32(table), _i32(lengths), starts, 1, block_frames=0)
        with pytest.raises(ValueError, match=match):
            c.check()
        assert (out[:rows] == 0).all() and torch.equal(out[rows:], good[rows:])
    for bad in ([0, rows, 3 * rows], [-5, rows, 2 * rows], [0, 5 * rows, 2 * rows]):
        paged8_attention(q, c, _i32(table), _i32([200, 200]), _i32(bad), 1)
        with pytest.raises(ValueError, match="row starts"):
            c.check()


def test_attention_offsets_beyond_32_bits():
    """A pool of more than 2^31 bytes of keys, read and written at its end."""
    heads, pages = 24, 11500
    c = Paged8Cache(pages, heads)
    assert c.k.numel() > 2 ** 31
    lengths, table = [100], [[pages - 1, pages - 2]]
    k = torch.randn(100, heads * 128, generator=_gen(0)).to(BF)
    v = torch.randn(100, heads * 128, generator=_gen(1)).to(BF)
    paged8_append(c, k.cuda(), v.cuda(), _i32(table), _i32(lengths), _i32([0, 100]))
    small = Paged8Cache(2, heads)
    paged8_append(small, k.cuda(), v.cuda(), _i32([[0, 1]]), _i32(lengths), _i32([0, 100]))
    assert torch.equal(c.k[-1], small.k[0]) and torch.equal(c.v[-2], small.v[1])
    for n in (1, 100):
        q = torch.randn(n, heads * 128, generator=_gen(n)).to(BF).cuda()
        got = paged8_attention(q, c, _i32(table), _i32(lengths), _i32([0, n]), heads)
        want = paged8_attention(q, small, _i32([[0, 1]]), _i32(lengths), _i32([0, n]), heads)
        assert torch.equal(got, want)


def test_attention_mixed_batch_is_each_request_alone():
    """Single rows and long chunks in one call, and pages shared by two
    requests: within a rounding of each request by itself."""
    lengths, counts = [700, 700, 65, 300, 64], [1, 513, 1, 2, 64]
    c, table, g = _filled(lengths, 3, torch.float8_e4m3fn)
    table[1][:5] = table[0][:5]
    _check(c, table, lengths, counts, 6, g)


@pytest.mark.parametrize("dtype", FORMATS)
def test_attention_of_new_data_is_that_of_old(dtype):
    """The first call on a cache just written gives the bits of the calls after
    it, when its pages are in the L2 cache: no load is used before it is there."""
    for seed in range(60):
        lengths, counts = [700, 64, 130, 333], [300, 3, 130, 17]
        c, table, g = _filled(lengths, 2, dtype, seed=seed)
        q = (torch.randn(450, 256, generator=g) * 1.5).to(BF)
        args = (q.cuda(), c, _i32(table), _i32(lengths), _i32([0, 300, 303, 433, 450]), 2)
        kw = dict(tokens_per_frame=1 + seed % 7, block_frames=seed % 3)
        first, second = (paged8_attention(*args, **kw) for _ in range(2))
        assert torch.equal(first, second), seed


@pytest.mark.parametrize("lengths", [[1500] * 20 + [2000, 2600], [100] * 200 + [240, 200, 130],
                                     [9000, 2000]])
def test_attention_of_short_and_long_requests_is_done_when_it_returns_to_the_stream(lengths):
    """Both kernels (and their merges) run beside one another: what follows on
    the stream changes the cache under neither."""
    counts = [1 if n in (100, 1500, 9000) else min(n, 500) for n in lengths]
    c, table, g = _filled(lengths, 2, torch.int8)
    q = torch.randn(sum(counts), 12 * 128, generator=g).to(BF).cuda()
    starts = torch.cumsum(torch.tensor([0] + counts), 0).tolist()
    args = (_i32(table), _i32(lengths), _i32(starts), 12)
    kept = c.k.clone(), c.v.clone()
    torch.cuda.synchronize()
    want = paged8_attention(q, c, *args)
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        outs.append(paged8_attention(q, c, *args))
        c.k.zero_(), c.v.zero_()
        c.k.copy_(kept[0]), c.v.copy_(kept[1])
    for out in outs:
        assert torch.equal(out, want)


def test_attention_on_two_streams_at_once():
    c, table, g = _filled([2000], 2, torch.int8)
    args = (c, _i32(table), _i32([2000]), None, 2)
    q = [torch.randn(n, 256, generator=g).to(BF).cuda() for n in (1, 1, 300, 300)]
    starts = [_i32([0, x.shape[0]]) for x in q]
    want = [paged8_attention(x, c, args[1], args[2], s, 2) for x, s in zip(q, starts)]
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    got = [[] for _ in q]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(paged8_attention(q[i], c, args[1], args[2], starts[i], 2))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


# ------------------------------------------------------------ used together

@pytest.mark.parametrize("dtype", FORMATS)
def test_steps_append_attention_together(dtype):
    """Sessions that start, grow, drop tokens and end, attention after each step."""
    s = _Session(4, 2, dtype, width=6, pages=16, seed=3)
    for add in ([100, 1, 0, 7], [1, 1, 130, 1], [1, -2, 1, 57], [-101, 64, 1, 1], [70, 1, -131, 1]):
        st = s.append(add, spare=2)
        counts = [max(a, 0) for a in add]
        T = sum(counts) + 2
        q = torch.randn(T, 4 * 128, generator=s.g).to(BF)
        out = paged8_attention(q.cuda(), s.cache, s.table, s.lengths, st.q_start, 4, tokens_per_frame=5,
                               block_frames=2, window=9)
        k, v = P.values(s.cache)
        want, _, mag = P.attention(q, k, v, s.table.tolist(), s.lengths.tolist(), st.q_start.tolist(), 4,
                                   frame=5, block=2, window=9)
        tol = P.attention_bound(want, mag, 400, float(v.abs().max()))
        assert ((out.cpu().double() - want).abs() <= tol).all()
    s.cache.check()


def test_captured_step_replays():
    """One decode step captured into a graph and replayed, against the same
    steps run one by one; a second graph on the same cache does not disturb it."""
    def build():
        s = _Session(3, 2, torch.int8, width=8, seed=11)
        s.append([70, 3, 130])
        return s

    add = _i32([1, 1, 1])
    xs = [torch.randn(3, 3, 256, generator=_gen(20 + i)).to(BF).cuda() for i in range(6)]

    def one(s, x):
        st = page_step(s.lengths, add, s.table, s.free, s.count, 3, in_place=True, most_new=1)
        paged8_append(s.cache, x[0], x[1], s.table, st.lengths, st.q_start)
        return paged8_attention(x[2], s.cache, s.table, st.lengths, st.q_start, 2, max_rows=1), st

    ref = build()
    want = [one(ref, x)[0] for x in xs]
    s = build()
    x = xs[0].clone()
    state = [t.clone() for t in (s.lengths, s.count, s.table, s.free, s.cache.k, s.cache.v,
                                 s.cache.k_scale, s.cache.v_scale)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(s, x)
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out, st = one(s, x)
    q2 = torch.randn(3, 256, device="cuda").to(BF)
    with torch.cuda.graph(g2):
        paged8_attention(q2, s.cache, s.table, s.lengths, st.q_start, 2, max_rows=1)
    for t, old in zip((s.lengths, s.count, s.table, s.free, s.cache.k, s.cache.v, s.cache.k_scale,
                       s.cache.v_scale), state):
        t.copy_(old)
    for xi, w in zip(xs, want):
        x.copy_(xi)
        g1.replay()
        g2.replay()
        assert torch.equal(out, w)
    st.check()
    assert s.lengths.tolist() == ref.lengths.tolist()
    assert torch.equal(s.cache.k, ref.cache.k) and torch.equal(s.cache.v, ref.cache.v)


def test_cache_made_while_a_graph_is_captured():
    """Its status word is the graph's own: later caches keep theirs."""
    lengths = [70]
    c, table, g = _filled(lengths, 1, torch.int8)
    q = torch.randn(1, 128, generator=g).to(BF).cuda()
    t, n, s = _i32(table), _i32(lengths), _i32([0, 1])
    want = paged8_attention(q, c, t, n, s, 1)
    made, words = [], dict(paged8._STATUS)
    paged8._STATUS.clear()
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            inner = Paged8Cache.from_tensors(c.k, c.v, c.k_scale, c.v_scale)
            made.append(paged8_attention(q, inner, t, n, s, 1))
        outer = Paged8Cache.from_tensors(c.k, c.v, c.k_scale, c.v_scale)
        assert outer.status.data_ptr() != inner.status.data_ptr()
        t[0, 0] = -1
        graph.replay()
        torch.cuda.synchronize()
        outer.check()
        with pytest.raises(ValueError, match="page pool"):
            inner.check()
        t.copy_(_i32(table))
        graph.replay()
        assert torch.equal(made[0], want)
        inner.check()
    finally:
        paged8._STATUS.update(words)


class _Apart:
    """The bind module without its whole calls: Python checks, allocates and
    calls the entry points."""

    def __init__(self, module):
        self.module = module

    def __getattr__(self, name):
        if name in ("append", "attention", "page_step", "head_norm", "layout"):
            return lambda *args: 0 if name == "layout" else None
        return getattr(self.module, name)


@pytest.mark.parametrize("dtype", FORMATS)
def test_whole_calls_are_those_of_the_checked_path(dtype, monkeypatch):
    """The same results and the same refusals either way."""
    from multics_b200 import _lib
    from multics_b200.attention import hier_head_norm_rope

    lengths, add, width = [70, 0, 500], [30, 1, 64], 9
    counts = [100, 1, 564]
    g = _gen(4)
    k, v = (torch.randn(95, 256, generator=g).to(BF).cuda() for _ in range(2))
    q = torch.randn(97, 512, generator=g).to(BF).cuda()
    f, w = torch.randn(97, 64, 2, generator=g).cuda(), torch.rand(128, generator=g).to(BF).cuda()

    def run():
        table = torch.full((3, width), -1, dtype=torch.int32)
        table[0, :2], table[2, :8] = _i32([4, 2]).cpu(), torch.arange(10, 18)
        table, free = table.cuda(), _i32([0, 1, 3, 5, 6, 7])
        st = page_step(_i32(lengths), _i32(add), table, free, _i32([6]), 97, most_new=64)
        st.check()
        c = Paged8Cache(18, 2, dtype=dtype)
        c = Paged8Cache.from_tensors(c.k, c.v, c.k_scale, c.v_scale, c.status)
        paged8_append(c, k, v, table, st.lengths, st.q_start)
        out, lse = paged8_attention(q, c, table, st.lengths, st.q_start, 4, tokens_per_frame=3, window=9,
                                    softmax_scale=0.1, max_rows=64, return_lse=True)
        given = paged8_attention(q, c, table, st.lengths, st.q_start, 4, out=torch.ones_like(q))
        qn, kn = hier_head_norm_rope(q, q[:, :256], f, 4, 2, q_weight=w, k_weight=w, eps=1e-5)
        again = page_step(st.lengths, _i32([-100, 0, 1]), table, free, st.free_count, 4, in_place=True)
        assert again.lengths is st.lengths and again.free_count is st.free_count
        assert st.lengths.tolist() == [0, 1, counts[2] + 1]
        return [*st, *again, table, free, c.k.view(torch.int8), c.v.view(torch.int8), c.k_scale, c.v_scale,
                out, lse, given, qn, kn]

    whole = run()
    module = _lib.calls()
    c, t, n, s = Paged8Cache(2, 2, dtype=dtype), _i32([[0, 1]]), _i32([3]), _i32([0, 3])

    def refuse():
        seen = []
        for fn, a in ((paged8_append, (c, k[:3], v[:2], t, n, s)), (paged8_append, (c, k[:3], v[:3], t, n, n)),
                      (paged8_append, (c, k[:3].float(), v[:3], t, n, s)),
                      (paged8_append, (c, k[:3].cpu(), v[:3], t, n, s)),
                      (paged8_attention, (q[:3], c, t, n, s, 3)), (paged8_attention, (q[:3], c, t, n.long(), s, 4)),
                      (paged8_attention, (q[:3], c, t, n, s, 2)), (page_step, (n, n, t, n, n, -1)),
                      (page_step, (n, s, t, n, n, 1))):
            with pytest.raises((ValueError, NotImplementedError)) as e:
                fn(*a)
            seen.append((e.type, str(e.value)))
        return seen

    refused = refuse()
    monkeypatch.setattr(_lib, "calls", lambda: _Apart(module))
    for a, b in zip(whole, run()):
        assert torch.equal(a, b)
    assert refused == refuse()
