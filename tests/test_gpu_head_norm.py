"""Per-head RMSNorm with the rotation in the same pass, forward and backward,
against the formulas in 64 bits."""

import pytest
import torch

import paged8_oracle as P
from multics_b200.attention import hier_head_norm_rope
from multics_b200.train import head_norm_rope_grad

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _inputs(T, H, Hk, D, F, seed, wdtype=BF):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand(F, D // 2, generator=g) * 6.3
    return dict(q=(torch.randn(T, H * D, generator=g) * 3).to(BF), k=torch.randn(T, Hk * D, generator=g).to(BF),
                wq=(1 + 0.3 * torch.randn(D, generator=g)).to(wdtype),
                wk=(1 + 0.3 * torch.randn(D, generator=g)).to(wdtype),
                table=torch.stack([a.cos(), a.sin()], -1),
                pos=torch.randint(0, F, (T,), generator=g, dtype=torch.int32),
                gq=torch.randn(T, H * D, generator=g).to(BF), gk=torch.randn(T, Hk * D, generator=g).to(BF))


def _run(x, H, Hk, pos, **kw):
    return hier_head_norm_rope(x["q"].cuda(), x["k"].cuda(), x["table"].cuda(), H, Hk,
                               q_weight=x["wq"].cuda(), k_weight=x["wk"].cuda(),
                               positions=None if pos is None else pos.cuda(), **kw)


def _near(got, want, slack):
    """One bf16 rounding (2^-8 of the value) and fp32 arithmetic on the terms."""
    err = (got.detach().cpu().double() - want).abs()
    tol = want.abs() * 2.0 ** -8 + slack * 2.0 ** -18 + 1e-37
    assert (err <= tol).all(), float((err / tol).max())


def _terms(x, w, heads):
    """|y| before the rotation, spread over the pair: the size of its terms."""
    T, D = x.shape[0], x.shape[1] // heads
    y = x.double().view(T, heads, D)
    y = (y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.double()).abs()
    return y.view(T, heads, D // 2, 2).sum(-1, keepdim=True).expand(T, heads, D // 2, 2).reshape(T, heads * D)


@pytest.mark.parametrize("T,H,Hk,D", [(1, 1, 1, 128), (7, 24, 24, 128), (301, 24, 8, 128), (33, 17, 3, 128),
                                      (50, 5, 1, 64), (9, 40, 33, 64), (20, 9, 2, 256)])
@pytest.mark.parametrize("wdtype", [BF, torch.float32])
def test_forward(T, H, Hk, D, wdtype):
    x = _inputs(T, H, Hk, D, 13, T + H, wdtype)
    q, k = _run(x, H, Hk, x["pos"])
    _near(q, P.head_norm(x["q"], x["wq"], x["table"], x["pos"], H), _terms(x["q"], x["wq"], H))
    _near(k, P.head_norm(x["k"], x["wk"], x["table"], x["pos"], Hk), _terms(x["k"], x["wk"], Hk))


def test_forward_without_positions_and_complex_table():
    x = _inputs(36, 3, 2, 128, 12, 0)
    every = torch.arange(36, dtype=torch.int32) % 12
    want = _run(x, 3, 2, every)
    assert all(torch.equal(a, b) for a, b in zip(_run(x, 3, 2, None), want))
    x["table"] = torch.view_as_complex(x["table"].double())[:, None]
    assert all(torch.equal(a, b) for a, b in zip(_run(x, 3, 2, None), want))


def test_forward_zero_huge_and_not_finite_rows():
    x = _inputs(6, 2, 2, 128, 4, 1)
    x["q"][0] = 0
    x["q"][1] = 1e-25
    x["q"][2, :128] = float("inf")
    x["q"][3, 5] = float("nan")
    q, _ = _run(x, 2, 2, x["pos"])
    want = P.head_norm(x["q"], x["wq"], x["table"], x["pos"], 2)
    for r, c in ((0, slice(None)), (1, slice(None)), (2, slice(128, None)), (3, slice(128, None)),
                 (4, slice(None))):
        _near(q[r, c], want[r, c], _terms(x["q"], x["wq"], 2)[r, c])
    assert q[2, :128].isnan().all() and q[3, :128].isnan().all()


def test_forward_strided_rows_given_out_row_maps_and_skipped_rows():
    x = _inputs(40, 3, 2, 128, 9, 2)
    x["pos"][4], x["pos"][17] = -1, -1
    want_q, want_k = _run(x, 3, 2, x["pos"])
    assert (want_q[4] == 0).all() and (want_k[17] == 0).all()
    wide = torch.cat([x["q"], x["k"]], 1).cuda()
    perm = torch.randperm(50, generator=torch.Generator().manual_seed(3))[:40].to(torch.int32)
    k_rows = perm.flip(0).clone()
    k_rows[8] = -1
    qo, ko = torch.full((50, 392), 5.0, dtype=BF, device="cuda"), torch.full((60, 256), 5.0, dtype=BF, device="cuda")
    hier_head_norm_rope(wide[:, :384], wide[:, 384:], x["table"].cuda(), 3, 2, q_weight=x["wq"].cuda(),
                        k_weight=x["wk"].cuda(), positions=x["pos"].cuda(), out=(qo[:, 8:], ko),
                        out_rows=perm.cuda(), k_out_rows=k_rows.cuda())
    live = x["pos"] >= 0
    assert torch.equal(qo[perm[live].long().cuda(), 8:], want_q[live.cuda()])
    assert (qo[:, :8] == 5).all()
    untouched = torch.ones(50, dtype=torch.bool)
    untouched[perm[live].long()] = False
    assert (qo[untouched.cuda(), 8:] == 5).all()
    live_k = live & (k_rows >= 0)
    assert torch.equal(ko[k_rows[live_k].long().cuda()], want_k[live_k.cuda()])
    untouched = torch.ones(60, dtype=torch.bool)
    untouched[k_rows[live_k].long()] = False
    assert (ko[untouched.cuda()] == 5).all()


def test_positions_and_rows_past_the_end_are_skipped_and_recorded():
    from multics_b200.attention import _dev_err, device_error

    x = _inputs(5, 1, 1, 128, 4, 4)
    assert device_error() == 0
    x["pos"][2] = 4
    q, _ = _run(x, 1, 1, x["pos"])
    assert (q[2] == 0).all() and device_error() == 2
    _dev_err(q.device).zero_()
    x["pos"][2] = 0
    out = (torch.zeros(5, 128, dtype=BF, device="cuda"), torch.zeros(3, 128, dtype=BF, device="cuda"))
    _run(x, 1, 1, x["pos"], out=out, k_out_rows=torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32).cuda())
    assert device_error() == 2
    _dev_err(q.device).zero_()


def test_no_rows():
    x = _inputs(0, 2, 1, 128, 4, 0)
    q, k = _run(x, 2, 1, x["pos"])
    assert q.shape == (0, 256) and k.shape == (0, 128)


@pytest.mark.parametrize("T,H,Hk,D", [(1, 1, 1, 128), (7, 24, 24, 128), (1501, 6, 2, 128), (33, 17, 3, 64),
                                      (20, 5, 2, 256)])
@pytest.mark.parametrize("wdtype", [BF, torch.float32])
def test_gradients(T, H, Hk, D, wdtype):
    x = _inputs(T, H, Hk, D, 11, T, wdtype)
    if T > 4:
        x["pos"][3] = -1
    leaves = [x[n].cuda().requires_grad_(True) for n in ("q", "k", "wq", "wk")]
    q, k = head_norm_rope_grad(leaves[0], leaves[1], x["table"].cuda(), H, Hk, q_weight=leaves[2],
                               k_weight=leaves[3], positions=x["pos"].cuda())
    got = torch.autograd.grad((q, k), leaves, (x["gq"].cuda(), x["gk"].cuda()))
    for xi, w, gi, heads, dx, dw in ((x["q"], x["wq"], x["gq"], H, got[0], got[2]),
                                     (x["k"], x["wk"], x["gk"], Hk, got[1], got[3])):
        a, b = xi.double().requires_grad_(True), w.double().requires_grad_(True)
        y = P.head_norm(a, b, x["table"], x["pos"], heads)
        wx, ww = torch.autograd.grad(y, (a, b), gi.double())
        xh = a.detach().view(T, heads, D)
        rstd = torch.rsqrt((xh * xh).mean(-1, keepdim=True) + 1e-6)
        size = (gi.double().view(T, heads, D).abs().amax(-1, keepdim=True) * 2 * w.double().abs().max()
                * rstd * (1 + (xh * rstd).abs())).reshape(T, heads * D)
        _near(dx, wx, size)
        # sums of up to a thousand fp32 additions per lane, rounded once to the weight's type
        total = (gi.double().view(T, heads, D).abs() * 2 * (xh * rstd).abs()).sum((0, 1))
        half = 2.0 ** -8 if wdtype == BF else 2.0 ** -24
        assert dw.dtype == wdtype
        assert ((dw.cpu().double() - ww).abs() <= ww.abs() * half + total * 2.0 ** -14).all()
        if T > 4:
            assert (dx[3] == 0).all()


def test_gradient_of_one_output_and_repeats():
    """Only q used: k's gradients are zero; the sums do not depend on timing."""
    x = _inputs(700, 4, 4, 128, 7, 9)
    leaves = [x[n].cuda().requires_grad_(True) for n in ("q", "k", "wq", "wk")]

    def grads():
        q, _ = head_norm_rope_grad(leaves[0], leaves[1], x["table"].cuda(), 4, 4, q_weight=leaves[2],
                                   k_weight=leaves[3], positions=x["pos"].cuda())
        return torch.autograd.grad(q, leaves, x["gq"].cuda().expand_as(q))

    a, b = grads(), grads()
    assert all(torch.equal(p, r) for p, r in zip(a, b))
    assert (a[1] == 0).all() and (a[3] == 0).all() and (a[0] != 0).any()


def test_gradient_broadcast_and_shared_weight():
    """A gradient expanded from one row, and one weight for q and k."""
    x = _inputs(30, 2, 2, 128, 5, 10)
    q0, k0 = x["q"].cuda().requires_grad_(True), x["k"].cuda().requires_grad_(True)
    w = x["wq"].cuda().requires_grad_(True)
    q, k = head_norm_rope_grad(q0, k0, x["table"].cuda(), 2, 2, q_weight=w, k_weight=w,
                               positions=x["pos"].cuda())
    g = x["gq"][:1].cuda().expand(30, 256)
    got = torch.autograd.grad((q, k), (w,), (g, g))[0]
    q, k = head_norm_rope_grad(q0, k0, x["table"].cuda(), 2, 2, q_weight=w, k_weight=w.detach().clone().requires_grad_(True),
                               positions=x["pos"].cuda())
    assert got.shape == w.shape and torch.isfinite(got.float()).all()
    a = w.detach().cpu().double().requires_grad_(True)
    y = (P.head_norm(x["q"], a, x["table"], x["pos"], 2) * g.cpu().double()).sum() + \
        (P.head_norm(x["k"], a, x["table"], x["pos"], 2) * g.cpu().double()).sum()
    want = torch.autograd.grad(y, a)[0]
    # two sums rounded to bf16, and the rounding of their sum
    assert ((got.cpu().double() - want).abs() <= want.abs().max() * 2.0 ** -6).all()


def test_backward_in_a_graph():
    x = _inputs(64, 2, 1, 128, 8, 12)
    leaves = [x[n].cuda().requires_grad_(True) for n in ("q", "k", "wq", "wk")]
    table, pos, gq, gk = (x[n].cuda() for n in ("table", "pos", "gq", "gk"))

    def step():
        q, k = head_norm_rope_grad(leaves[0], leaves[1], table, 2, 1, q_weight=leaves[2],
                                   k_weight=leaves[3], positions=pos)
        return torch.autograd.grad((q, k), leaves, (gq, gk))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------ SelfAttention

def _layer(H, seed, head_norm, cam=True):
    from multics_b200.attention import SelfAttention

    g = torch.Generator().manual_seed(seed)
    layer = SelfAttention(H * 128, H, head_norm=head_norm)
    if cam:
        layer.enable_camera_pose_qk(12, dropout_p=0.0)
    with torch.no_grad():
        for name, p in layer.named_parameters():
            p.copy_(torch.randn(p.shape, generator=g) * 0.05 + (1.0 if "norm" in name else 0.0))
    return layer.to("cuda", BF).eval()


def _module_math(layer, x, cam, table, mask):
    """The module in float64 on [B, L, dim], differentiable."""
    B, L, dim = x.shape
    H, D = layer.num_heads, layer.head_dim
    lin = lambda m, t: torch.nn.functional.linear(t, m.weight.double(),  # noqa: E731
                                                  None if m.bias is None else m.bias.double())
    pos = torch.arange(L).repeat(B).to(torch.int32)
    q = lin(layer.q, x) + (0 if cam is None else lin(layer.cam_q, cam))
    k = lin(layer.k, x) + (0 if cam is None else lin(layer.cam_k, cam))
    q = P.head_norm(q.reshape(B * L, dim), layer.norm_q.weight, table, pos, H, layer.norm_q.eps)
    k = P.head_norm(k.reshape(B * L, dim), layer.norm_k.weight, table, pos, H, layer.norm_k.eps)
    q, k, v = (t.reshape(B, L, H, D).transpose(1, 2) for t in (q, k, lin(layer.v, x)))
    s = (q @ k.transpose(2, 3)) / D ** 0.5
    s = s.masked_fill(~mask, float("-inf"))
    return lin(layer.o, (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B, L, dim))


@pytest.mark.parametrize("B,L", [(1, 200), (5, 21)])
@pytest.mark.parametrize("cam", [False, True])
def test_selfattention_with_head_norm(B, L, cam):
    """Forward and gradients of the module, one sequence and a batch, at the
    bars of the framework's other module tests."""
    layer = _layer(2, B, True, cam)
    assert layer.norm_q.weight.shape == (128,)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(B, L, 256, generator=g).to(BF)
    c = torch.randn(B, L, 12, generator=g).to(BF) if cam else None
    a = torch.rand(L, 64, generator=g) * 6.3
    table = torch.stack([a.cos(), a.sin()], -1)
    mask = torch.arange(L)[None] // 3 <= torch.arange(L)[:, None] // 3
    args = (table.cuda(), mask.cuda(), None if c is None else c.cuda())
    with torch.no_grad():
        out = layer(x.cuda(), *args)
    import copy
    ref = copy.deepcopy(layer).cpu().double()
    xr = x.double().requires_grad_(True)
    want = _module_math(ref, xr, None if c is None else c.double(), table, mask)
    assert (out.cpu().double() - want).abs().max() <= 2e-2 * max(1.0, float(want.detach().abs().max()))
    xg = x.cuda().requires_grad_(True)
    dy = torch.randn(want.shape, generator=g).to(BF)
    layer(xg, *args).backward(dy.cuda())
    want.backward(dy.double())
    got = {n: p.grad.cpu().double() for n, p in layer.named_parameters()} | {"x": xg.grad.cpu().double()}
    exp = {n: p.grad for n, p in ref.named_parameters()} | {"x": xr.grad}
    for n, e in exp.items():
        if n == "k.bias" and not cam:
            continue  # a residual of cancelling terms
        cos = torch.nn.functional.cosine_similarity(got[n].flatten(), e.flatten(), 0)
        assert (got[n] - e).abs().max() <= 6e-2 * e.abs().max() and cos >= 0.995, (n, float(cos))


@pytest.mark.parametrize("head_norm", [True, False])
@pytest.mark.parametrize("cam", [False, True])
def test_paged_forward_steps(head_norm, cam):
    """Three steps of two requests through the module: the output is the
    projection of the 64-bit attention over what the cache then holds."""
    from multics_b200.paged8 import Paged8Cache, page_step

    H = 2
    layer = _layer(H, 3, head_norm, cam)
    g = torch.Generator().manual_seed(5)
    a = torch.rand(300, 64, generator=g) * 6.3
    freqs = torch.stack([a.cos(), a.sin()], -1).cuda()
    cache = Paged8Cache(9, H)
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    free, count = torch.arange(9, dtype=torch.int32, device="cuda"), torch.tensor([9], dtype=torch.int32, device="cuda")
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    kept = []
    orig = layer.o.forward
    layer.o.forward = lambda t: (kept.append(t), orig(t))[1]
    for add in ((70, 33), (1, 1), (40, 0)):
        rows = sum(add) + 2
        st = page_step(lengths, torch.tensor(add, dtype=torch.int32, device="cuda"), table, free, count, rows)
        x = torch.randn(1, rows, H * 128, generator=g).to(BF).cuda()
        c = torch.randn(1, rows, 12, generator=g).to(BF).cuda() if cam else None
        y = layer.paged_forward(x, freqs, cache, table, st, tokens_per_frame=5, block_frames=2, window=9,
                                cam_tokens=c)
        assert y.shape == x.shape
        # the rotated queries by the module's own kernels, row by row of the table
        pos = st.positions
        rows_t = freqs[pos.clamp(min=0).long()]
        with torch.no_grad():
            q, k = layer._prologue(layer.q(x[0]), layer.k(x[0]), rows_t, None if c is None else c[0])
        kk, vv = P.values(cache)
        want, _, mag = P.attention(q, kk, vv, table.tolist(), st.lengths.tolist(), st.q_start.tolist(), H,
                                   frame=5, block=2, window=9)
        tol = P.attention_bound(want, mag, 200, float(vv.abs().max()))
        assert ((kept[-1].cpu().double() - want).abs() <= tol).all()
        # the cache holds this step's keys within half a step of its scales
        live = pos >= 0
        page, tok = (st.slots[live] // 64).long().cpu(), (st.slots[live] % 64).long().cpu()
        held = kk[page, :, tok].reshape(-1, H * 128)
        step_k = cache.k_scale.cpu().double()[page].repeat_interleave(128, 1)
        assert ((held - k[live].cpu().double()).abs() <= step_k / 2).all()
        lengths, count = st.lengths, st.free_count
    st.check(), cache.check()
    with pytest.raises(ValueError, match="rows"):
        layer.paged_forward(x[:, 1:], freqs, cache, table, st)
    del layer.o.forward


@pytest.mark.parametrize("H,Hk,D", [(5, 1, 64), (3, 1, 128)])
def test_gradients_without_eps(H, Hk, D):
    """Lanes that no head fills add nothing to the weights' gradients."""
    x = _inputs(9, H, Hk, D, 13, 3)
    ref, leaf = {}, {}
    for n in ("q", "k", "wq", "wk"):
        ref[n] = x[n].double().requires_grad_()
        leaf[n] = x[n].cuda().requires_grad_()
    q, k = head_norm_rope_grad(leaf["q"], leaf["k"], x["table"].cuda(), H, Hk, q_weight=leaf["wq"],
                               k_weight=leaf["wk"], positions=x["pos"].cuda(), eps=0.0)
    torch.autograd.backward((q, k), (x["gq"].cuda(), x["gk"].cuda()))
    torch.autograd.backward((P.head_norm(ref["q"], ref["wq"], x["table"], x["pos"], H, eps=0.0),
                             P.head_norm(ref["k"], ref["wk"], x["table"], x["pos"], Hk, eps=0.0)),
                            (x["gq"].double(), x["gk"].double()))
    for n in leaf:
        # one bf16 rounding, and fp32 sums of terms no larger than the largest gradient times their number
        top = ref[n].grad.abs().max()
        err = (leaf[n].grad.cpu().double() - ref[n].grad).abs()
        assert (err <= ref[n].grad.abs() * 2.0 ** -8 + top * 2.0 ** -14).all(), n


@pytest.mark.parametrize("wdtype", [BF, torch.float32])
@pytest.mark.parametrize("positions", [True, False])
def test_gradients_by_either_way_are_the_same(wdtype, positions, monkeypatch):
    """Through the bind module's function and through Python's; gradients that
    are broadcast, strided or missing too."""
    from multics_b200 import _lib

    x = _inputs(26, 6, 3, 128, 13, 1, wdtype)
    pos = x["pos"].cuda() if positions else None

    def run():
        leaf = {n: x[n].cuda().requires_grad_() for n in ("q", "k", "wq", "wk")}
        got = []
        wide = torch.cat([x["gk"], x["gk"]], 1).cuda()
        for grads in ((x["gq"].cuda(), x["gk"].cuda()), (x["gq"].cuda(), None), (None, wide[:, 384:]),
                      (torch.ones(1, 1, dtype=BF, device="cuda").expand(26, 768), wide[:, 1:385])):
            q, k = head_norm_rope_grad(leaf["q"], leaf["k"], x["table"].cuda(), 6, 3, q_weight=leaf["wq"],
                                       k_weight=leaf["wk"], positions=pos, eps=1e-5)
            pairs = [(o, g) for o, g in zip((q, k), grads) if g is not None]
            got += [q, k, *torch.autograd.grad([o for o, _ in pairs], list(leaf.values()),
                                               [g for _, g in pairs], create_graph=grads[1] is not None)]
        with pytest.raises(RuntimeError):  # (no gradient of a gradient)
            got[2].sum().backward()
        return [t.detach() for t in got]

    fast = run()
    module = _lib.calls()

    class Apart:
        def __getattr__(self, name):
            return (lambda *args: None) if name.startswith("head_norm") else getattr(module, name)

    monkeypatch.setattr(_lib, "calls", lambda: Apart())
    for a, b in zip(fast, run()):
        assert torch.equal(a, b)
