"""64-bit restatement of the 8-bit paged cache and the per-head prologue, one
request and head at a time, for the tests."""

import math

import torch

PAGE = 64
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def step(lengths, add, table, free, count):
    """One step on Python lists: (lengths, count, q_start, slots, positions),
    ``table`` and ``free`` updated in place."""
    after = [n + a for n, a in zip(lengths, add)]
    pages = [(-(-n // PAGE), -(-m // PAGE)) for n, m in zip(lengths, after)]
    for b, (p0, p1) in enumerate(pages):
        for p in range(p1, p0):
            free[count] = table[b][p]
            count += 1
    for b, (p0, p1) in enumerate(pages):
        for p in range(p0, p1):
            count -= 1
            table[b][p] = free[count]
    q_start, slots, positions = [0], [], []
    for b, a in enumerate(add):
        for t in range(lengths[b], max(lengths[b], after[b])):
            positions.append(t)
            slots.append(table[b][t // PAGE] * PAGE + t % PAGE)
        q_start.append(len(slots))
    return after, count, q_start, slots, positions


def scale_for(amax, dtype):
    """The least power of two whose top code reaches ``amax``, 2^-100 at least."""
    if amax == 0:
        return 2.0 ** -100
    e = math.floor(math.log2(amax / TOP[dtype])) - 1
    while TOP[dtype] * 2.0 ** e < amax:
        e += 1
    return 2.0 ** max(e, -100)


def encode(x, dtype):
    """Codes (as float64) of values already divided by their scale."""
    if dtype == torch.int8:
        return x.round().clamp(-127, 127)
    return x.float().to(torch.float8_e4m3fn).double()


def values(cache):
    """Keys and values of the pool, float64 ``[pages, heads, 64, 128]``."""
    k = cache.k.cpu().double() * cache.k_scale.cpu().double()[..., None, None, None]
    v = cache.v.cpu().double() * cache.v_scale.cpu().double()[..., None, None]
    return torch.cat([k[:, :, 0], k[:, :, 1]], -1), v.transpose(2, 3)


def sees(pos, held, frame, block, window):
    """Which of ``held`` tokens the row at ``pos`` sees, bool [held]."""
    j = torch.arange(held)
    if pos < 0 and not (block == 0 and window < 0):
        return torch.zeros(held, dtype=torch.bool)
    ok = torch.ones(held, dtype=torch.bool)
    f, fj = pos // frame, j // frame
    if block:
        ok &= fj // block <= f // block
    if window >= 0:
        ok &= f - fj < window
    return ok


def attention(q, k, v, table, lengths, q_start, heads, *, frame=1, block=1, window=-1, scale=None):
    """(out, log2-sum-exp, bound's terms) in float64; ``k``, ``v`` from
    :func:`values`.  The terms are sum p |v| / sum p and the largest |v|."""
    T, Hk = q.shape[0], k.shape[1]
    G = heads // Hk
    scale = 128 ** -0.5 if scale is None else scale
    out = torch.zeros(T, heads, 128, dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.full((T, heads), float("-inf"), dtype=torch.float64)
    qd = q.detach().cpu().double().view(T, heads, 128)
    for b, held in enumerate(lengths):
        a, e = q_start[b], q_start[b + 1]
        if e <= a or held == 0:
            continue
        pages = torch.tensor(table[b][:-(-held // PAGE)])
        kb, vb = k[pages].transpose(0, 1).flatten(1, 2)[:, :held], v[pages].transpose(0, 1).flatten(1, 2)[:, :held]
        ok = torch.stack([sees(held - (e - a) + i, held, frame, block, window) for i in range(e - a)])
        for h in range(heads):
            s = (qd[a:e, h] @ kb[h // G].t()) * scale
            s = s.masked_fill(~ok, float("-inf"))
            m = s.amax(1, keepdim=True)
            p = torch.where(ok, torch.exp(s - torch.where(m.isinf(), torch.zeros_like(m), m)),
                            torch.zeros_like(s))
            tot = p.sum(1, keepdim=True)
            w = p / torch.where(tot > 0, tot, torch.ones_like(tot))
            out[a:e, h], mag[a:e, h] = w @ vb[h // G], w @ vb[h // G].abs()
            lse[a:e, h] = torch.where(tot > 0, m + tot.log(), torch.full_like(m, float("-inf")))[:, 0] / math.log(2)
    return out.view(T, -1), lse, mag.view(T, -1)


def attention_bound(out, mag, n_keys, vmax):
    """How far a bf16 output may be from ``out``: its own rounding (2^-8 of the
    value); weights rounded to fp16 (2^-11 of sum p |v| / sum p, and half a step
    of 2^-24 per key for the weights below 2^-14); scores from 128 products
    added in fp32 and exponentials of two roundings (another 2^-11)."""
    return out.abs() * 2.0 ** -8 + mag * 2.0 ** -10 + n_keys * vmax * 2.0 ** -25 + 1e-30


def head_norm(x, w, table, positions, heads, eps=1e-6):
    """Per-head RMSNorm and rotation in float64 (differentiable); rows with a
    position outside the table are 0."""
    T, D = x.shape[0], x.shape[1] // heads
    y = x.double().view(T, heads, D)
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    live = (positions >= 0) & (positions < table.shape[0])
    f = table.double()[positions.long().clamp(0, table.shape[0] - 1)][:, None]
    a, b, c, s = y[..., 0::2], y[..., 1::2], f[..., 0], f[..., 1]
    y = torch.stack([a * c - b * s, a * s + b * c], -1).reshape(T, heads * D)
    return torch.where(live[:, None], y, torch.zeros_like(y))
