"""Cases of the 8-bit paged serving operators and of the per-head prologue.

Four operators, each in its plain form (elementary torch operations in 32
bits) and as the calls a user makes of ``multics_b200``:

* ``norm``    RMSNorm of every head of q and k with the position rotation in
  the same pass, forward and (``train``) with its gradients;
* ``pages``   block tables, slot maps and row positions from request lengths;
* ``append``  new keys and values written to the pages of a cache held in 8
  bits, one power-of-two scale per 64-token page and head;
* ``attend``  attention of the new rows over such a cache, from one row per
  request to whole sequences.

Token counts come from the repository's configurations: 220 tokens per latent
frame, blocks of 3 frames, a window of 21 frames, 42 frames per sequence, 24
heads of 128, 880 patch sequences of the per-frame attention.
"""

import random

import torch

own = False

D = 128      # head size
PAGE = 64    # tokens of a page
# the codes of both formats are returned as the numbers they are, beside their power-of-two scales
FMT = {"int8": (torch.int8, 127.0, 7), "e4m3": (torch.float8_e4m3fn, 448.0, 9)}
E_MIN = -100  # the smallest scale is 2 ** E_MIN


# ------------------------------------------------------------------- cases

def listed():
    return [
        # the hub rows of one frame: a call whose launch is most of its time
        dict(name="norm_hub_rows", op="norm", rows=38, heads=24, kv_heads=24, table=38, train=False),
        # all rows of the full-size layer, inference
        dict(name="norm_sequence", op="norm", rows=38556, heads=24, kv_heads=24, table=9240, train=False),
        # a training pass over one player's rows and one more, shared key heads
        dict(name="norm_train", op="norm", rows=9241, heads=24, kv_heads=8, table=9241, train=True),
        # four players' sessions, one token each
        dict(name="pages_tokens", op="pages", requests=4, held=9240, new=1, width=160, shrink=False),
        # the patch sequences of the per-frame attention: new frames for some,
        # dropped frames and ended sessions for others
        dict(name="pages_frames", op="pages", requests=3520, held=42, new=27, width=4, shrink=True),
        # one token for each of 67 requests
        dict(name="append_tokens", op="append", fmt="int8", requests=67, held=500, new=1, heads=24),
        # three new frames of each of four players, pages that start mid-way
        dict(name="append_frames", op="append", fmt="e4m3", requests=4, held=1100, new=660, heads=24),
        # one row over a player's whole history
        dict(name="attend_token", op="attend", fmt="int8", requests=1, new=1, held=9240, heads=24,
             kv_heads=24, frame=1, block=1, window=-1),
        # three new frames of 880 patch sequences over their window
        dict(name="attend_action", op="attend", fmt="int8", requests=880, new=3, held=24, heads=24,
             kv_heads=24, frame=1, block=3, window=21),
        # single rows of many requests of uneven length, eight query heads to a key head
        dict(name="attend_shared_heads", op="attend", fmt="e4m3", requests=37, new=1, held=19001,
             heads=32, kv_heads=4, frame=1, block=1, window=-1),
        # three new frames of four players, block-causal over the window
        dict(name="attend_players", op="attend", fmt="int8", requests=4, new=660, held=9240, heads=24,
             kv_heads=24, frame=220, block=3, window=21),
        # a whole sequence at once, causal by frame
        dict(name="attend_sequence", op="attend", fmt="e4m3", requests=1, new=9240, held=9240, heads=24,
             kv_heads=24, frame=220, block=1, window=-1),
    ]


def _log(rng, lo, hi):
    """A whole number, spread over the logarithm of the range."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("norm", "pages", "append", "attend", "attend"))
    fmt = rng.choice(("int8", "e4m3"))
    if op == "norm":
        heads = rng.randint(1, 32)
        rows = _log(rng, 1, 900000 // (heads * 2))
        return dict(op=op, rows=rows, heads=heads, kv_heads=rng.randint(1, heads),
                    table=rng.choice((rows, _log(rng, 1, 9240))), train=rng.random() < 0.5)
    if op == "pages":
        held = _log(rng, 1, 9240)
        return dict(op=op, requests=_log(rng, 1, 3520), held=held, new=_log(rng, 1, 27),
                    width=(held + 27 + PAGE - 1) // PAGE + rng.randint(0, 3),
                    shrink=rng.random() < 0.5)
    if op == "append":
        heads = rng.randint(1, 32)
        tokens = _log(rng, 1, 60000 // heads)
        requests = _log(rng, 1, min(tokens, 256))
        new = max(1, tokens // requests)
        return dict(op=op, fmt=fmt, requests=requests, held=new + _log(rng, 1, 800) - 1, new=new,
                    heads=heads)
    kv = rng.choice((1, 2, 3, 4, 8, 12, 24))
    group = rng.choice((1, 1, 2, 3, 4, 8)) if kv <= 8 else 1
    frame = rng.choice((1, 1, 7, 38, 220))
    requests = _log(rng, 1, 880)
    held = _log(rng, 1, max(8, min(19001, 1200000 // (requests * kv))))
    new = rng.choice((1, _log(rng, 1, held), _log(rng, 1, min(held, 64))))
    while requests * new * held * kv * group > 9240 * 9240 * 12 or requests * new * kv * group > 220000:
        new = max(1, new // 2)
    return dict(op=op, fmt=fmt, requests=requests, new=new, held=held, heads=kv * group, kv_heads=kv,
                frame=frame, block=rng.choice((0, 1, 1, 3)), window=rng.choice((-1, -1, rng.randint(1, 30))))


def _requests(case):
    """(held after the call, new) of each request: up to the case's numbers,
    uneven, the first request at the full size."""
    r = random.Random("%(requests)s %(held)s %(new)s" % case)
    got = []
    for b in range(case["requests"]):
        held = case["held"] if b == 0 else r.randint(max(1, case["held"] // 2), case["held"])
        new = case["new"] if b == 0 or r.random() < 0.7 else r.randint(1, case["new"])
        got.append((held, min(new, held)))
    return got


def _visible(case, held, new):
    """(first, end) of the keys that the rows of one request see between
    them, and the number of (row, key) pairs."""
    L, n, w = case["frame"], case["block"], case["window"]
    first, last, pairs = held, 0, 0
    p, end = held - new, held
    while p < end:
        f = p // L
        rows = min(end, (f + 1) * L) - p
        lo = max(0, (f - w + 1) * L) if w >= 0 else 0
        hi = held if n == 0 else min(held, (f // n + 1) * n * L)
        first, last = min(first, lo), max(last, hi)
        pairs += rows * max(0, hi - lo)
        p += rows
    return first, max(first, last), pairs


def work(case):
    op = case["op"]
    if op == "norm":
        values = case["rows"] * (case["heads"] + case["kv_heads"]) * D
        table = min(case["rows"], case["table"]) * D * 4 + case["rows"] * 4
        return {"bytes": values * (8 if case["train"] else 4) + table,
                "flops": values * (25 if case["train"] else 8)}
    if op == "pages":
        rows = sum(max(0, a) for _, a in _steps(case))
        pages = sum(max(0, -(-(h + a) // PAGE) - -(-h // PAGE)) for h, a in _steps(case))
        return {"bytes": case["requests"] * 16 + pages * 8 + rows * 8, "flops": 0}
    if op == "append":
        values = sum(n for _, n in _requests(case)) * case["heads"] * D
        pages = sum(-(-h // PAGE) - (h - n) // PAGE for h, n in _requests(case)) * case["heads"]
        return {"bytes": 2 * values * 3 + pages * 8, "flops": 4 * values}
    keys = pairs = rows = 0
    for held, new in _requests(case):
        first, end, p = _visible(case, held, new)
        keys, pairs, rows = keys + end - first, pairs + p, rows + new
    return {"bytes": rows * case["heads"] * D * 4 + keys * case["kv_heads"] * (2 * D + 8 / PAGE),
            "flops": 4 * D * pairs * case["heads"]}


def _steps(case):
    """(held before, added) of each request of a ``pages`` case; ``shrink``:
    some requests drop tokens and some end."""
    r = random.Random("%(requests)s %(held)s %(new)s %(shrink)s" % case)
    got = []
    for b in range(case["requests"]):
        held = case["held"] if b == 0 else r.randint(case["held"] // 2, case["held"])
        add = case["new"] if b == 0 else r.randint(0, case["new"])
        kind = r.random()
        if case["shrink"] and b and kind < 0.2:
            add = -held if kind < 0.1 else -r.randint(0, held)
        got.append((held, add))
    return got


# ------------------------------------------------------------------ inputs

def _rand(g, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _shuffled(g, n):
    return torch.randperm(n, generator=g, device="cuda").to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "norm":
        rows, hq, hk = case["rows"], case["heads"], case["kv_heads"]
        angle = torch.rand(case["table"], D // 2, generator=g, device="cuda") * 6.2831853
        s = {"case": case, "q": _rand(g, rows, hq * D, scale=2.0), "k": _rand(g, rows, hk * D, scale=2.0),
             "wq": 1 + _rand(g, D, scale=0.1), "wk": 1 + _rand(g, D, scale=0.1),
             "freqs": torch.stack([angle.cos(), angle.sin()], -1).contiguous(),
             "positions": torch.randint(0, case["table"], (rows,), generator=g, device="cuda",
                                        dtype=torch.int32)}
        if case["train"]:
            s["gq"], s["gk"] = _rand(g, rows, hq * D), _rand(g, rows, hk * D)
            for n in ("q", "k", "wq", "wk"):
                s[n].requires_grad_(True)
        return s
    order = random.Random(seed)
    if op == "pages":
        steps = _steps(case)
        order.shuffle(steps)
        owned = [-(-h // PAGE) for h, _ in steps]
        spare = sum(max(0, -(-(h + a) // PAGE) - o) for (h, a), o in zip(steps, owned)) + 5
        ids = _shuffled(g, sum(owned) + spare)
        table = torch.full((len(steps), case["width"]), -1, dtype=torch.int32, device="cuda")
        held = torch.arange(case["width"], device="cuda")[None] < _ints(owned)[:, None]
        table[held] = ids[:sum(owned)]
        free = torch.full((ids.numel(),), -1, dtype=torch.int32, device="cuda")
        free[:spare] = ids[sum(owned):]
        return {"case": case, "lengths": _ints([h for h, _ in steps]), "add": _ints([a for _, a in steps]),
                "table": table, "free": free, "free_count": _ints([spare]),
                "rows": sum(max(0, a) for _, a in steps) + 3}
    reqs = _requests(case)
    order.shuffle(reqs)
    pages = [-(-h // PAGE) for h, _ in reqs]
    heads = case["heads"] if op == "append" else case["kv_heads"]
    total, rows = sum(pages), sum(n for _, n in reqs)
    start = [0]
    for _, n in reqs:
        start.append(start[-1] + n)
    width = max(pages)
    table = torch.full((len(reqs), width), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda")[None] < _ints(pages)[:, None]] = _shuffled(g, total)
    dtype = FMT[case["fmt"]][0]

    def codes(*shape):
        if dtype == torch.int8:
            return (torch.randn(*shape, generator=g, device="cuda") * 35).round().clamp(-127, 127).to(dtype)
        return (torch.randn(*shape, generator=g, device="cuda") * 100).clamp(-448, 448).to(dtype)

    e0 = -5 if dtype == torch.int8 else -7

    def scales():
        e = torch.randint(e0 - 1, e0 + 2, (total, heads), generator=g, device="cuda")
        return _pow2(e)

    s = {"case": case, "table": table, "lengths": _ints([h for h, _ in reqs]), "q_start": _ints(start),
         # [pages, heads, dimension half, token, 64 dimensions] and [pages, heads, dimension, token]
         "k8": codes(total, heads, 2, PAGE, D // 2), "v8": codes(total, heads, D, PAGE),
         "k_scale": scales(), "v_scale": scales(), "new": max(n for _, n in reqs)}
    if op == "append":
        s["k"], s["v"] = _rand(g, rows, heads * D), _rand(g, rows, heads * D, scale=0.7)
    else:
        s["q"] = _rand(g, rows, case["heads"] * D, scale=1.5)
    return s


# ------------------------------------------------------------------- plain

def _pow2(e):
    """2 ** e in 32 bits, from the exponent's bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _plain_norm(s):
    c = s["case"]

    def one(x, w, heads):
        y = x.float().view(c["rows"], heads, D)
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.float()
        f = s["freqs"][s["positions"].long()][:, None]
        a, b, cs, sn = y[..., 0::2], y[..., 1::2], f[..., 0], f[..., 1]
        return torch.stack([a * cs - b * sn, a * sn + b * cs], -1).reshape(c["rows"], heads * D).bfloat16()

    q, k = one(s["q"], s["wq"], c["heads"]), one(s["k"], s["wk"], c["kv_heads"])
    if not c["train"]:
        return q, k
    grads = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
    return (q.detach(), k.detach()) + grads


def _plain_pages(s):
    before, add, rows = s["lengths"].long(), s["add"].long(), s["rows"]
    table, free, count = s["table"].clone(), s["free"].clone(), s["free_count"].long()
    after = before + add
    p0, p1 = (before + PAGE - 1) // PAGE, (after + PAGE - 1) // PAGE
    col = torch.arange(table.shape[1], device="cuda")[None]
    # pages given back go to the end of the list in request order, pages taken come off its end
    back = (col >= p1[:, None]) & (col < p0[:, None])
    given = table[back]
    free[count + torch.arange(given.numel(), device="cuda")] = given
    count = count + given.numel()
    take = (col >= p0[:, None]) & (col < p1[:, None])
    n = int(take.sum())
    table[take] = free[count - 1 - torch.arange(n, device="cuda")]
    count = count - n
    new = add.clamp(min=0)
    q_start = torch.cat([new.new_zeros(1), new.cumsum(0)])
    r = torch.arange(rows, device="cuda")
    b = torch.searchsorted(q_start[1:], r, right=True)
    live = b < new.numel()
    b = b.clamp(max=new.numel() - 1)
    pos = torch.where(live, before[b] + r - q_start[b], torch.full_like(r, -1))
    page = table[b, (pos.clamp(min=0) // PAGE)].long()
    slot = torch.where(live, page * PAGE + pos % PAGE, torch.full_like(r, -1))
    i = torch.int32
    return after.to(i), table, free, count.to(i), q_start.to(i), slot.to(i), pos.to(i)


def _fresh_exponent(amax, top, bits):
    """The least e with top * 2**e >= amax (top = m * 2**bits, 0.5 <= m < 1)."""
    m, x = torch.frexp(amax)
    e = x - bits + (m > top / 2.0 ** bits).to(x.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(min=E_MIN)


def _plain_append(s):
    c = s["case"]
    dtype, top, bits = FMT[c["fmt"]]
    H, rows = c["heads"], s["k"].shape[0]
    q_start, lengths = s["q_start"].long(), s["lengths"].long()
    r = torch.arange(rows, device="cuda")
    b = torch.searchsorted(q_start[1:], r, right=True)
    pos = lengths[b] - q_start[b + 1] + r
    page, off = s["table"][b, pos // PAGE].long(), pos % PAGE
    kept = torch.zeros(s["k_scale"].shape[0], dtype=torch.long, device="cuda")  # tokens held before
    first = (lengths - (q_start[1:] - q_start[:-1]))[b] - pos // PAGE * PAGE
    kept[page] = first.clamp(0, PAGE)
    touched = torch.zeros(kept.shape[0], dtype=torch.bool, device="cuda")
    touched[page] = True

    def one(x, codes, scale, tokens_last):
        x = x.float().view(rows, H, D)
        amax = torch.zeros(scale.shape, device="cuda")
        amax.index_reduce_(0, page, x.abs().amax(-1), "amax")
        need = _pow2(_fresh_exponent(amax, top, bits))
        new = torch.where((kept > 0)[:, None], torch.maximum(scale, need), need)
        new = torch.where(touched[:, None], new, scale)

        def encode(v):
            return (v.round() if dtype == torch.int8 else v).to(dtype)

        held = torch.arange(PAGE, device="cuda")[None] < kept[:, None]
        ratio = (scale / new)[:, :, None, None]
        if tokens_last:
            out = torch.where(held[:, None, None, :], codes.float() * ratio, codes.float())
        else:
            out = torch.where(held[:, None, None, :, None], codes.float() * ratio[..., None], codes.float())
        out = encode(out)
        y = encode(x / new[page][:, :, None])
        raw, yr = out.view(torch.int8), y.view(torch.int8)
        if tokens_last:
            raw[page, :, :, off] = yr
        else:
            raw[page, :, :, off] = yr.view(rows, H, 2, D // 2)
        return out, new

    k8, ks = one(s["k"], s["k8"], s["k_scale"], False)
    v8, vs = one(s["v"], s["v8"], s["v_scale"], True)
    return k8, v8, ks, vs


def _dense(s, dtype):
    """Keys and values of every request ``[B, H, width * 64, 128]``."""
    t = s["table"].clamp(min=0).long()
    B, W = t.shape
    H = s["k8"].shape[1]
    k = s["k8"][t].to(dtype) * s["k_scale"][t][..., None, None, None].to(dtype)  # [B, W, H, 2, 64, 64]
    v = s["v8"][t].to(dtype) * s["v_scale"][t][..., None, None].to(dtype)        # [B, W, H, 128, 64]
    return (k.permute(0, 2, 1, 4, 3, 5).reshape(B, H, W * PAGE, D),
            v.permute(0, 2, 1, 4, 3).reshape(B, H, W * PAGE, D))


def _edges(c, pos, lengths):
    """First key and end of the keys of rows at positions ``pos`` ``[B, n]``."""
    f = torch.div(pos, c["frame"], rounding_mode="floor")
    lo = (f - c["window"] + 1) * c["frame"] if c["window"] >= 0 else torch.zeros_like(pos)
    hi = lengths[:, None].expand_as(pos)
    if c["block"]:
        n = c["block"]
        hi = torch.minimum(hi, (torch.div(f, n, rounding_mode="floor") + 1) * n * c["frame"])
    return lo, hi


def _plain_attend(s):
    c = s["case"]
    H, Hk, B, n = c["heads"], c["kv_heads"], s["table"].shape[0], s["new"]
    G = H // Hk
    q_start, lengths = s["q_start"].long(), s["lengths"].long()
    count = q_start[1:] - q_start[:-1]
    i = torch.arange(n, device="cuda")[None]
    live = i < count[:, None]
    row = (q_start[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    pos = torch.where(live, (lengths - count)[:, None] + i, torch.full_like(row, -1))
    q = s["q"][row].float().view(B, n, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, n * G, D)
    k, v = _dense(s, torch.float32)
    lo, hi = _edges(c, pos, lengths)
    j = torch.arange(k.shape[2], device="cuda")
    sees = ((j >= lo[..., None]) & (j < hi[..., None]) & (pos >= 0)[..., None])[:, None, :, None]
    x = torch.matmul(q, k.transpose(2, 3)).view(B, Hk, n, G, -1).mul_(D ** -0.5)
    x.masked_fill_(~sees, float("-inf"))
    m = x.amax(-1, keepdim=True)
    x.sub_(torch.where(torch.isfinite(m), m, torch.zeros_like(m))).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, Hk, n * G, -1), v).view(B, Hk, n, G, D)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(0, 2, 1, 3, 4).reshape(B, n, H * D)[live].bfloat16()


# --------------------------------------------------------------------- run

def run(state):
    op, c = state["case"]["op"], state["case"]
    if not own:
        return {"norm": _plain_norm, "pages": _plain_pages, "append": _plain_append,
                "attend": _plain_attend}[op](state)
    s = state
    if op == "norm":
        if c["train"]:
            from multics_b200.train import head_norm_rope_grad

            q, k = head_norm_rope_grad(s["q"], s["k"], s["freqs"], c["heads"], c["kv_heads"],
                                       q_weight=s["wq"], k_weight=s["wk"], positions=s["positions"])
            grads = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
            return (q.detach(), k.detach()) + grads
        from multics_b200.attention import hier_head_norm_rope

        return hier_head_norm_rope(s["q"], s["k"], s["freqs"], c["heads"], c["kv_heads"],
                                   q_weight=s["wq"], k_weight=s["wk"], positions=s["positions"])
    from multics_b200.paged8 import Paged8Cache, page_step, paged8_append, paged8_attention

    if op == "pages":
        st = page_step(s["lengths"], s["add"], s["table"], s["free"], s["free_count"], s["rows"])
        return st.lengths, s["table"], s["free"], st.free_count, st.q_start, st.slots, st.positions
    cache = Paged8Cache.from_tensors(s["k8"], s["v8"], s["k_scale"], s["v_scale"])
    if op == "append":
        paged8_append(cache, s["k"], s["v"], s["table"], s["lengths"], s["q_start"])
        return cache.k, cache.v, cache.k_scale, cache.v_scale
    return paged8_attention(s["q"], cache, s["table"], s["lengths"], s["q_start"], c["heads"],
                            tokens_per_frame=c["frame"], block_frames=c["block"], window=c["window"],
                            max_rows=s["new"])


# ------------------------------------------------------------------- exact

def exact(case, seed):
    """What ``run`` returns, in 64 bits, one request and head at a time."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "pages":
        return None
    if op == "norm":
        return _exact_norm(s)
    if op == "append":
        return _exact_append(s)
    if sum(n * h for h, n in _requests(case)) * case["heads"] > 4e9:
        return None
    H, G = case["heads"], case["heads"] // case["kv_heads"]
    starts, lengths, table = s["q_start"].tolist(), s["lengths"].tolist(), s["table"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, held in enumerate(lengths):
        a, e = starts[b], starts[b + 1]
        pages = torch.tensor(table[b][:-(-held // PAGE)], device="cuda")
        kb = s["k8"][pages].double() * s["k_scale"][pages].double()[:, :, None, None, None]
        vb = s["v8"][pages].double() * s["v_scale"][pages].double()[:, :, None, None]
        kb = torch.cat([kb[:, :, 0], kb[:, :, 1]], -1).transpose(0, 1).flatten(1, 2)[:, :held]
        vb = vb.permute(1, 0, 3, 2).flatten(1, 2)[:, :held]
        p = torch.arange(held - (e - a), held, device="cuda")
        fq, fk = p[:, None] // case["frame"], torch.arange(held, device="cuda")[None] // case["frame"]
        ok = torch.ones(e - a, held, dtype=torch.bool, device="cuda")
        if case["block"]:
            ok &= fk // case["block"] <= fq // case["block"]
        if case["window"] >= 0:
            ok &= fq - fk < case["window"]
        qb = s["q"][a:e].double().view(e - a, H, D)
        for kv in range(case["kv_heads"]):
            qh = qb[:, kv * G:(kv + 1) * G].transpose(0, 1)
            x = (qh @ kb[kv].t()) / D ** 0.5
            x = torch.softmax(x.masked_fill(~ok, float("-inf")), -1).nan_to_num(0.0)
            out[a:e].view(e - a, H, D)[:, kv * G:(kv + 1) * G] = (x @ vb[kv]).transpose(0, 1)
    return out


def _exact_norm(s):
    c = s["case"]
    z = torch.complex(s["freqs"][..., 0].double(), s["freqs"][..., 1].double())[s["positions"].long()]

    def one(x, w, g, heads):
        x = x.detach().double().view(c["rows"], heads, D)
        w = w.detach().double()
        inv = (x.square().sum(-1, keepdim=True) / D + 1e-6) ** -0.5
        y = torch.view_as_complex((x * inv * w).view(c["rows"], heads, D // 2, 2)) * z[:, None]
        y = torch.view_as_real(y).reshape(c["rows"], heads * D)
        if g is None:
            return y, None, None
        # the rotation undone, then d(x inv w) = inv (w g - xh mean(w g xh))
        g = torch.view_as_complex(g.double().view(c["rows"], heads, D // 2, 2)) * z.conj()[:, None]
        g = torch.view_as_real(g).reshape(c["rows"], heads, D)
        xh = x * inv
        dx = inv * (w * g - xh * (w * g * xh).mean(-1, keepdim=True))
        return y, dx.reshape(c["rows"], heads * D), (g * xh).sum((0, 1))

    q, dq, dwq = one(s["q"], s["wq"], s.get("gq"), c["heads"])
    k, dk, dwk = one(s["k"], s["wk"], s.get("gk"), c["kv_heads"])
    return (q, k, dq, dk, dwq, dwk) if c["train"] else (q, k)


def _exact_append(s):
    """The scales alone: the codes are whole steps of the formats, equal or not."""
    c = s["case"]
    _, top, _ = FMT[c["fmt"]]
    starts, lengths, table = s["q_start"].tolist(), s["lengths"].tolist(), s["table"].tolist()
    out = []
    for x, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])):
        x = x.double().view(-1, c["heads"], D).abs().amax(-1)
        new = scale.double().clone()
        for b, held in enumerate(lengths):
            begin = held - (starts[b + 1] - starts[b])
            for pg in range(begin // PAGE, -(-held // PAGE)):
                r0 = starts[b] + max(0, pg * PAGE - begin)
                r1 = starts[b] + min(held, (pg + 1) * PAGE) - begin
                e = torch.ceil(torch.log2(x[r0:r1].amax(0) / top))
                e = torch.where(torch.exp2(e - 1) * top >= x[r0:r1].amax(0), e - 1, e)
                need = torch.exp2(e)
                at = table[b][pg]
                new[at] = torch.maximum(new[at], need) if begin > pg * PAGE else need
        out.append(new)
    return None, None, out[0], out[1]
