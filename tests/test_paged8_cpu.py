"""8-bit paged cache and per-head prologue: refusals, sizes and the oracle's own
formulas (no GPU work)."""

import ctypes

import pytest
import torch

import paged8_oracle as P
from multics_b200 import _lib
from multics_b200.attention import hier_head_norm_rope
from multics_b200.paged8 import Paged8Cache, page_step, paged8_append, paged8_attention

BF = torch.bfloat16


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def _cache(pages=2, heads=2, dtype=torch.int8):
    return Paged8Cache(pages, heads, dtype=dtype, device="cpu")


def test_cache_refusals():
    with pytest.raises(NotImplementedError, match="head_dim 128"):
        Paged8Cache(1, 1, device="cpu", head_dim=64)
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        Paged8Cache(1, 1, device="cpu", dtype=BF)
    with pytest.raises(ValueError, match="num_pages=0"):
        Paged8Cache(0, 1, device="cpu")
    c = _cache()
    args = [c.k, c.v, c.k_scale, c.v_scale]
    for i, bad in ((0, c.k.flatten(3)), (0, c.k.float()), (1, c.v[:1]), (2, c.k_scale.double()),
                   (3, c.v_scale[:, :1]), (1, c.v.transpose(0, 1).contiguous().transpose(0, 1))):
        with pytest.raises(ValueError):
            Paged8Cache.from_tensors(*(bad if j == i else a for j, a in enumerate(args)))
    with pytest.raises(ValueError, match="status"):
        Paged8Cache.from_tensors(*args, status=torch.zeros(1))
    Paged8Cache.from_tensors(*args).check()


def test_cache_check_reports_and_clears():
    c = _cache()
    c.status.fill_(4 | 8)
    with pytest.raises(ValueError, match="page pool.*NaN"):
        c.check()
    c.check()


def test_page_step_refusals():
    good = dict(lengths=_i32(1), add=_i32(1), table=torch.zeros(1, 2, dtype=torch.int32),
                free_pages=_i32(1, 2), free_count=_i32(2), rows=4)
    for key, bad in (("lengths", _i32(1, 2)), ("add", torch.tensor([1])), ("table", _i32(0, 0)),
                     ("free_count", _i32()), ("rows", -1), ("rows", 1 << 31),
                     ("table", torch.zeros(2, 2, dtype=torch.int32).t()[:1].t()[:1].expand(1, 2).t())):
        with pytest.raises(ValueError):
            page_step(**{**good, key: bad})
    with pytest.raises(ValueError, match="most_new"):
        page_step(**good, most_new=-1)
    with pytest.raises(NotImplementedError, match="CUDA"):
        page_step(**good)


def test_append_and_attention_refusals():
    c = _cache()
    k = torch.zeros(3, 256, dtype=BF)
    t, n, s = torch.zeros(1, 2, dtype=torch.int32), _i32(3), _i32(0, 3)
    for args in ((k[:, :128], k, t, n, s), (k, k[:2], t, n, s), (k, k, t, n, _i32(0, 1, 3)),
                 (k, k, t, _i32(3, 3), s), (k, k, t.long(), n, s)):
        with pytest.raises(ValueError):
            paged8_append(c, *args)
    with pytest.raises(NotImplementedError, match="bf16"):
        paged8_append(c, k.float(), k, t, n, s)
    with pytest.raises(NotImplementedError, match="CUDA"):
        paged8_append(c, k, k, t, n, s)
    q = torch.zeros(3, 512, dtype=BF)
    for kw in (dict(num_heads=3), dict(num_heads=0), dict(window=0), dict(window=-2),
               dict(tokens_per_frame=0), dict(block_frames=-1), dict(window=(1 << 30) + 1),
               dict(max_rows=-1), dict(softmax_scale=0.0),
               dict(softmax_scale=-0.1), dict(softmax_scale=float("nan")), dict(out=torch.zeros(3, 512)), dict(out=torch.zeros(2, 512, dtype=BF))):
        with pytest.raises(ValueError):
            paged8_attention(q, c, t, n, s, **{"num_heads": 4, **kw})
    with pytest.raises(ValueError, match="q must be"):
        paged8_attention(q, c, t, n, s, 2)
    with pytest.raises(NotImplementedError, match="CUDA"):
        paged8_attention(q, c, t, n, s, 4)


def test_head_norm_refusals():
    q, k, w = torch.zeros(4, 256, dtype=BF), torch.zeros(4, 128, dtype=BF), torch.ones(128)
    f = torch.zeros(4, 64, 2)
    good = dict(q=q, k=k, freqs=f, num_heads=2, num_kv_heads=1, q_weight=w, k_weight=w)
    for kw in (dict(num_heads=3), dict(k=k[:3]), dict(k=q), dict(q_weight=w[:64]),
               dict(freqs=f[:, :32]), dict(freqs=f[:3]), dict(positions=torch.zeros(4)),
               dict(positions=_i32(0, 1))):
        with pytest.raises(ValueError):
            hier_head_norm_rope(**{**good, **kw})
    with pytest.raises(NotImplementedError, match="head_dim"):
        hier_head_norm_rope(**{**good, "num_heads": 8})
    with pytest.raises(NotImplementedError, match="bf16"):
        hier_head_norm_rope(**{**good, "q": q.float()})
    with pytest.raises(NotImplementedError, match="CUDA"):
        hier_head_norm_rope(**good)


def test_entry_points_refuse_before_any_device_work():
    L = _lib.lib()

    def attn(rows=1, heads=2, kv=2, D=128, fmt=0, stride=1, width=1, frame=1, block=1, window=-1,
             q=None):
        return L.hier_paged8_attn(q, 256, rows, heads, kv, D, fmt, None, None, None, None, 1, None,
                                  stride, width, None, None, 1, frame, block, window, 0.1, 0, None,
                                  256, None, 1, None, None, None, None)

    for kw, exc in ((dict(D=64), NotImplementedError), (dict(heads=3), ValueError),
                    (dict(fmt=2), ValueError), (dict(stride=0), ValueError),
                    (dict(window=0), ValueError), (dict(frame=0), ValueError),
                    (dict(rows=1 << 30, heads=8, kv=2), ValueError),
                    (dict(width=1 << 26, stride=1 << 26), ValueError), (dict(q=8), ValueError),
                    (dict(rows=-1), ValueError)):
        with pytest.raises(exc):
            _lib.check(attn(**kw))
    assert attn(rows=0) == 0
    floats = ctypes.c_int64(-1)
    _lib.check(L.hier_paged8_attn_workspace(0, 2, 2, 1, 1, 0, ctypes.byref(floats)))
    assert floats.value == 0
    with pytest.raises(ValueError):
        _lib.check(L.hier_paged8_append(4, 256, None, 256, 1, 2, 0, None, None, None, None, 1, None,
                                        1, 1, None, None, 1, None, None))
    with pytest.raises(ValueError):
        _lib.check(L.hier_page_step(None, None, 1, None, 1, 2, None, 0, None, 0, -1, None, None,
                                    None, None, None, None, None))
    n = ctypes.c_int32()
    with pytest.raises(NotImplementedError):
        _lib.check(L.hier_head_norm_rope_bwd_partials(1, 1, 1, 96, ctypes.byref(n)))


def test_a_pool_has_pages_and_heads():
    """An entry of no page is read as page 0's scales: there must be one."""
    for pages, heads in ((0, 2), (2, 0)):
        z = torch.zeros(pages, heads)
        with pytest.raises(ValueError, match="no pages or no heads"):
            Paged8Cache.from_tensors(torch.zeros(pages, heads, 2, 64, 64, dtype=torch.int8),
                                     torch.zeros(pages, heads, 128, 64, dtype=torch.int8), z, z)
    L = _lib.lib()
    with pytest.raises(ValueError):
        _lib.check(L.hier_paged8_attn(None, 256, 1, 2, 2, 128, 0, None, None, None, None, 0, None, 1, 1,
                                      None, None, 1, 1, 1, -1, 0.1, 0, None, 256, None, 1, None, None,
                                      None, None))
    with pytest.raises(ValueError):
        _lib.check(L.hier_paged8_append(None, 256, None, 256, 1, 2, 0, None, None, None, None, 0, None,
                                        1, 1, None, None, 1, None, None))


@pytest.mark.parametrize("requests", [1, 30, 3000, 200000])
def test_workspace_follows_the_rows_not_the_requests(requests):
    """At most 300 large tiles of 256 rows or 2^14 small ones of 8, of 130 floats."""
    for rows in (1, 10, 5000):
        for heads, kv in ((1, 1), (24, 4), (64, 8)):
            for width in (4, 150, 5000):
                floats = ctypes.c_int64(-1)
                _lib.check(_lib.lib().hier_paged8_attn_workspace(rows, heads, kv, requests, width, 0,
                                                                 ctypes.byref(floats)))
                assert 0 <= floats.value <= 130 * (300 * 256 + (1 << 14) * 8)


def test_calls_module_reads_the_declared_signatures():
    letters = {ctypes.c_void_p: "p", ctypes.c_int64: "q", ctypes.c_int32: "i", ctypes.c_float: "f"}
    C = _lib.calls()
    names = [n for n in dir(C) if n.startswith("hier_")]
    assert len(names) == 5
    for n in names:
        assert getattr(C, n).__doc__ == "".join(letters[t] for t in _lib._SIGS[n][1])
    args = [None, 256, None, 256, 0, 2, 0, None, None, None, None, 1, None, 1, 1, None, None, 1, None, None]
    assert C.hier_paged8_append(*args) == 0  # no rows
    with pytest.raises(ValueError):
        _lib.check(C.hier_paged8_append(*args[:6], 2, *args[7:]))
    with pytest.raises(TypeError, match="takes 20 arguments, got 19"):
        C.hier_paged8_append(*args[1:])
    with pytest.raises(ValueError, match="32 bits"):
        C.hier_paged8_append(*args[:4], 1 << 31, *args[5:])
    with pytest.raises(TypeError):
        C.hier_paged8_append(1.5, *args[1:])
    with pytest.raises(ValueError, match="no entry"):
        C.bind("hier_none", 0)


@pytest.mark.parametrize("dtype", list(P.TOP))
def test_scale_is_the_least_power_of_two(dtype):
    for amax in (1e-38, 2.0 ** -20, 0.1, 1.0, 126.9, 127.0, 127.5, 448.0, 449.0, 3e38):
        s = P.scale_for(amax, dtype)
        assert s * P.TOP[dtype] >= amax
        assert s == 2.0 ** -100 or s / 2 * P.TOP[dtype] < amax


def test_oracle_gradient_of_the_head_norm_against_differences():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 2 * 64, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(64, generator=g, dtype=torch.float64, requires_grad=True)
    a = torch.rand(5, 32, generator=g, dtype=torch.float64) * 6
    table = torch.stack([a.cos(), a.sin()], -1)
    pos = torch.tensor([4, -1, 0])
    assert torch.autograd.gradcheck(lambda x, w: P.head_norm(x, w, table, pos, 2), (x, w))


def test_oracle_mask_is_the_frame_mask():
    from multics_b200.action import cached_frame_mask

    for frame, block, window in ((1, 1, -1), (3, 2, 4), (7, 3, -1), (2, 1, 1)):
        pos = torch.arange(11, 23)
        want = cached_frame_mask(pos // frame, torch.arange(23) // frame, block, window)
        got = torch.stack([P.sees(int(p), 23, frame, block, window) for p in pos])
        assert torch.equal(got, want)
