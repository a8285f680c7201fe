"""Plain restatements, in 64 bits, of the serving operators: causal attention over packed
prompts, the 8-bit paged key/value cache, attention over the cache.

Each attention returns, beside the output, ``A = sum_j softmax_j |v_j|``: a relative error u in
every probability moves the output by at most u * A, which is what the tests' bounds count."""
import math

import torch

E4M3_MAX, SCALE_EXP_MIN = 448.0, -117
# the largest value of 4 significant bits in a type: what is larger is stored as this, so that it can be read back
LARGEST = {torch.float16: 1.875 * 2.0 ** 15, torch.bfloat16: 1.875 * 2.0 ** 127, torch.float32: math.inf, torch.float64: math.inf}


def attend(q, k, v, seen, scale):
    """q [r, D], k, v [m, D]; row i sees the first seen[i] keys -> (o, lse, A).  Only visible keys enter."""
    q, k, v = q.double(), k.double(), v.double()
    o = torch.zeros_like(q)
    lse = torch.full((q.shape[0],), -math.inf, dtype=torch.float64, device=q.device)
    A = torch.zeros_like(q)
    hidden = torch.arange(k.shape[0], device=q.device)[None] >= seen[:, None]
    if k.shape[0] == 0 or q.shape[0] == 0:
        return o, lse, A
    s = (q @ k.T * scale).masked_fill(hidden, -math.inf)
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[:, None])
    bad = ~torch.isfinite(v).all(1)
    fine = torch.where(bad[:, None], 0.0, v)
    o, A = p @ fine, p @ fine.abs()
    for j in bad.nonzero().flatten().tolist():       # a value that is not finite: its own rows only
        rows = ~hidden[:, j]
        o[rows] = o[rows] + p[rows, j][:, None] * v[j]
    return o, lse, A


def prompt(q, k, v, cu_q, cu_k, scale, causal=True):
    """q [Tq, Hq, D], k, v [Tk, Hkv, D], offsets as lists -> (o, lse, A); rows of no sequence are NaN."""
    g = q.shape[1] // k.shape[1]
    o = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    lse, A = o[..., 0].clone(), o.clone()
    for a, b, c, d in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        n, m = b - a, d - c
        seen = torch.arange(n, device=q.device) + 1 + m - n if causal else torch.full((n,), m, device=q.device)
        for h in range(q.shape[1]):
            o[a:b, h], lse[a:b, h], A[a:b, h] = attend(q[a:b, h], k[c:d, h // g], v[c:d, h // g], seen, scale)
    return o, lse, A


def pow2(e):
    """2^e in 64 bits, exactly (exp2 and log2 may be an ulp off, which moves ties)."""
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64), e)


def round_e4m3(x):
    """To the nearest e4m3 value, ties to even; |x| <= 448; NaN and infinities give NaN."""
    x = x.double()
    fin = torch.isfinite(x)
    y = torch.where(fin, x, 0.0)
    step = pow2((torch.frexp(y)[1] - 1).clamp_min(-6) - 3)
    return torch.where(fin, torch.round(y / step) * step, math.nan)


def scale_exponent(amax):
    """The smallest e with amax <= 448 * 2^e, at least SCALE_EXP_MIN."""
    e = torch.frexp(amax.double().clamp_min(2.0 ** -140))[1] - 11
    for _ in range(3):
        e = torch.where(amax.double() > E4M3_MAX * pow2(e), e + 1, e)
    return e.clamp_min(SCALE_EXP_MIN)


def append(codes, scale, x, table, lengths, cu):
    """codes [P, H, page, D] (values of the codes, 64 bits), scale [P, H], both changed in place; x [T, H, D];
    the rest lists."""
    page = codes.shape[2]
    for b in range(len(lengths)):
        n = cu[b + 1] - cu[b]
        first = lengths[b] - n
        pos = first
        while pos < lengths[b]:
            pg, off = table[b][pos // page], pos % page
            cnt = min(page - off, lengths[b] - pos)
            new = x[cu[b] + pos - first: cu[b] + pos - first + cnt].double().transpose(0, 1)   # [H, cnt, D]
            new = torch.where(torch.isfinite(new), new.clamp(-LARGEST[x.dtype], LARGEST[x.dtype]), new)
            e = scale_exponent(torch.where(torch.isfinite(new), new.abs(), 0.0).amax((1, 2)))
            if off:
                e_old = torch.frexp(scale[pg].double())[1] - 1
                e = torch.maximum(e, e_old)
                codes[pg, :, :off] = round_e4m3(codes[pg, :, :off] * pow2(e_old - e)[:, None, None])
            codes[pg, :, off:off + cnt] = round_e4m3(new * pow2(-e)[:, None, None])
            scale[pg] = pow2(e).to(scale.dtype)
            pos += cnt


def gather(codes, scale, table, starts, counts):
    """-> [sum of counts, H, D] in 64 bits."""
    page, rows = codes.shape[2], []
    for b, n in enumerate(counts):
        for pos in range(starts[b], starts[b] + n):
            pg = table[b][pos // page]
            rows.append(codes[pg, :, pos % page].double() * scale[pg].double()[:, None])
    return torch.stack(rows) if rows else codes.new_zeros(0, codes.shape[1], codes.shape[3]).double()


def cached(q, k_codes, v_codes, k_scale, v_scale, table, lengths, scale):
    """q [B, Sq, Hq, D], codes as values -> (o, lse, A).  Tokens of pages outside the pool are left out."""
    B, Sq, Hq, D = q.shape
    P, H, page, _ = k_codes.shape
    g = Hq // H
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse, A = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=q.device), o.clone()
    for b in range(B):
        m = lengths[b]
        if m == 0:
            continue
        ids = torch.tensor(table[b][:-(-m // page)], device=q.device)
        there = ((ids >= 0) & (ids < P)).repeat_interleave(page)[:m]
        ids = ids.clamp(0, P - 1)
        before = torch.cat([there.new_zeros(1, dtype=torch.int64), there.cumsum(0)])
        for h in range(H):
            k, v = ((c[ids, h].double() * s[ids, h].double()[:, None, None]).reshape(-1, D)[:m][there]
                    for c, s in ((k_codes, k_scale), (v_codes, v_scale)))
            seen = before[(m - Sq + 1 + torch.arange(Sq, device=q.device)).clamp(0, m)].repeat_interleave(g)
            rows = attend(q[b, :, h * g:(h + 1) * g].reshape(Sq * g, D), k, v, seen, scale)
            o[b, :, h * g:(h + 1) * g] = rows[0].view(Sq, g, D)
            lse[b, :, h * g:(h + 1) * g] = rows[1].view(Sq, g)
            A[b, :, h * g:(h + 1) * g] = rows[2].view(Sq, g, D)
    return o, lse, A
