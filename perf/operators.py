"""Cases of the serving operators: causal attention over packed prompts (``attention_prompt``), the 8-bit
paged key/value cache (``kv_cache_append``, ``kv_cache_gather``) and attention over it (``attention_cached``).

Each case is one call (or the append and the gather that reads it back) as a program that serves the hybrid
chain makes it.  ``run`` computes it in plain torch, or with the framework's kernels where ``own`` is true."""
import math

import torch

own = False

E4M3_MAX = 448.0
SCALE_EXP_MIN = -117      # smallest scale exponent: 2^-9 * 2^-117 is still a normal bf16 number
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one short chat turn: a launch's latency counts
        dict(name="prompt_turn", kind="prompt", q="17", k="17", heads=8, kv=2, dim=64, type="f16", lse=False),
        # a server's batch of prompts, packed: lengths from one token to some thousands, odd ones
        dict(name="prompt_packed", kind="prompt", q="1+63+129+511+1000+2047+345+2600", k="1+63+129+511+1000+2047+345+2600",
             heads=24, kv=8, dim=128, type="bf16", lse=False),
        # pieces of two long prompts over the context that is already cached (queries at the end of the keys)
        dict(name="prompt_piece", kind="prompt", q="512+300", k="12345+8000", heads=32, kv=8, dim=128, type="bf16", lse=True),
        # one long prompt with as many key heads as query heads
        dict(name="prompt_long", kind="prompt", q="16380", k="16380", heads=24, kv=24, dim=128, type="bf16", lse=False),
        # a decode step's append: one token for each of 64 sequences, read back from its page's start
        dict(name="append_step", kind="append", new="1x64", old="1000", heads=8, dim=128, page=64, type="bf16"),
        # pieces of a few prompts, small pages, starting inside a page
        dict(name="append_pieces", kind="append", new="500+77+1+1030", old="333+0+15+4097", heads=4, dim=64, page=16, type="f16"),
        # a whole long prompt
        dict(name="append_prompt", kind="append", new="32760", old="0", heads=8, dim=128, page=64, type="bf16"),
        # one user's next token
        dict(name="decode_one", kind="decode", lens="1000", sq=1, heads=24, kv=8, dim=128, page=64, type="bf16", lse=False),
        # an ordinary batch, ragged, with an idle slot
        dict(name="decode_batch", kind="decode", lens="4096+0+1+2500+777+3333+64+65+1500+4000+2048+2049+128+900+3800+3100",
             sq=1, heads=24, kv=8, dim=128, page=64, type="bf16", lse=False),
        # two very long contexts
        dict(name="decode_long", kind="decode", lens="131072+100001", sq=1, heads=32, kv=8, dim=128, page=128, type="f16", lse=True),
        # four drafted tokens of each sequence at once, small heads and pages
        dict(name="decode_drafts", kind="decode", lens="6007x16", sq=4, heads=32, kv=4, dim=64, page=16,
             type="bf16", lse=False),
        # a full server: many sequences, as many key heads as query heads
        dict(name="decode_many", kind="decode", lens="2900x96", sq=1, heads=24, kv=24, dim=128, page=32,
             type="bf16", lse=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _text(values):
    return "+".join(str(v) for v in values)


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "append", "decode", "decode"])
    dim = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 3, 4, 8, 12])
    kind_of = rng.choice(["bf16", "bf16", "f16"])
    if kind == "prompt":
        n = rng.randint(1, 10)
        q = [_log(rng, 1, 6000 // n + 200) for _ in range(n)]
        k = [x + (0 if rng.random() < 0.5 else _log(rng, 1, 5000)) for x in q]
        return dict(kind="prompt", q=_text(q), k=_text(k), heads=kv * rng.choice([1, 1, 2, 3, 4, 5]), kv=kv, dim=dim,
                    type=kind_of, lse=rng.random() < 0.3)
    page = rng.choice([16, 32, 64, 128])
    if kind == "append":
        n = rng.randint(1, 24)
        most = rng.choice([1, 40, 24000 // n])
        return dict(kind="append", new=_text(_log(rng, 1, most) for _ in range(n)),
                    old=_text(0 if rng.random() < 0.2 else _log(rng, 1, 4000) for _ in range(n)), heads=kv, dim=dim, page=page,
                    type=kind_of)
    n = _log(rng, 1, 64)
    return dict(kind="decode", lens=_text(0 if rng.random() < 0.05 else _log(rng, 1, 200000 // n) for _ in range(n)),
                sq=rng.choice([1, 1, 1, 2, 3, 5, 8]), heads=kv * rng.choice([1, 2, 3, 4, 7, 8, 16]), kv=kv, dim=dim, page=page,
                type=kind_of, lse=rng.random() < 0.3)


def _lens(text):
    """"5+6" are two lengths, "5x3" three of five."""
    if "x" in text:
        n, times = text.split("x")
        return [int(n)] * int(times)
    return [int(n) for n in text.split("+")]


def _sums(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pairs(n, m):
    """Visible (query, key) pairs of n queries at the end of m keys."""
    first = m - n + 1
    if first >= 1:
        return n * (first + m) // 2
    return m * (m + 1) // 2


def _table(lens, page, gen):
    """Pages for sequences of these lengths, in shuffled order: (table on the host, number of pages in the pool)."""
    need = [-(-n // page) for n in lens]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=gen).tolist()
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (max(max(need), 1) - n))
        at += n
    return table, pool


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    t, dim = TYPES[case["type"]], case["dim"]
    s = dict(case)
    if case["kind"] == "prompt":
        # q, k, v are column views of one fused projection where the tokens agree, as a layer has them
        nq, nk, hq, hk = _lens(case["q"]), _lens(case["k"]), case["heads"], case["kv"]
        s["nq"], s["nk"] = nq, nk
        if nq == nk:
            x = torch.randn(sum(nq), hq + 2 * hk, dim, generator=gen, device="cuda").to(t)
            s["q"], s["k"], s["v"] = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
        else:
            s["q"] = torch.randn(sum(nq), hq, dim, generator=gen, device="cuda").to(t)
            s["k"] = torch.randn(sum(nk), hk, dim, generator=gen, device="cuda").to(t)
            s["v"] = torch.randn(sum(nk), hk, dim, generator=gen, device="cuda").to(t)
        s["cu_q"], s["cu_k"] = _int32(_sums(nq)), _int32(_sums(nk))
        return s
    page, hk = case["page"], case["heads"] if case["kind"] == "append" else case["kv"]
    if case["kind"] == "append":
        new, old = _lens(case["new"]), _lens(case["old"])
        old = old * len(new) if len(old) == 1 else old
        lens = [a + b for a, b in zip(new, old)]
    else:
        lens = _lens(case["lens"])
    table, pool = _table(lens, page, host)
    # keys and values of a model: normal, a few channels larger, every token of its own size
    big = 1 + 3 * (torch.rand(dim, generator=gen, device="cuda") < 0.05)
    exps, codes = [], []
    for _ in range(2):
        x = torch.randn(pool, hk, page, dim, generator=gen, device="cuda") * big
        x *= 0.5 + torch.rand(pool, hk, page, 1, generator=gen, device="cuda")
        e = _exponent(x.abs().amax((2, 3)))
        exps.append(_pow2(e))
        codes.append((x * _pow2(-e)[..., None, None]).to(torch.float8_e4m3fn))
        del x
    s["pool"] = pool
    s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"] = *codes, *exps
    s["page_table"], s["lengths"] = _int32(table), _int32(lens)
    s["lens"] = lens
    if case["kind"] == "append":
        s["k"], s["v"] = ((torch.randn(sum(new), hk, dim, generator=gen, device="cuda") * big * 1.3).to(t) for _ in range(2))
        s["cu_new"] = _int32(_sums(new))
        # what is read back: each sequence from the start of the first page that is written
        first = [o // page * page for o in old]
        s["starts"], s["cu_read"] = _int32(first), _int32(_sums([n - f for n, f in zip(lens, first)]))
        s["new"], s["read"] = sum(new), sum(lens) - sum(first)
    else:
        s["q"] = torch.randn(len(lens), case["sq"], case["heads"], dim, generator=gen, device="cuda").to(t)
    return s


def _exponent(amax):
    """The smallest e with amax <= 448 * 2^e, and at least SCALE_EXP_MIN."""
    m, x = torch.frexp(amax)              # amax = m * 2^x, m in [0.5, 1); 448 = 0.875 * 2^9
    return torch.where(amax > 0, x - 9 + (m > 0.875), SCALE_EXP_MIN).clamp_min(SCALE_EXP_MIN)


def _pow2(e):
    """2^e in 32 bits, exactly (its exponent field); 2^-126 below that."""
    return ((e.clamp_min(-126) + 127) << 23).view(torch.float32)


def _softmax_v(scores, v):
    """(softmax(scores) v, logsumexp); masked scores are -inf, a row without any gives 0 and -inf."""
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = scores.sub_(top).exp_()
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(l == 0, 1.0, l)
    return o, (top + l.log()).squeeze(-1)


def _plain_prompt(s):
    hk, dim = s["kv"], s["dim"]
    g = s["heads"] // hk
    outs, lses, q0, k0 = [], [], 0, 0
    for n, m in zip(s["nq"], s["nk"]):    # a packed sequence at a time
        q = s["q"][q0:q0 + n].float().reshape(n, hk, g, dim).permute(1, 2, 0, 3).reshape(hk, g * n, dim)
        k = s["k"][k0:k0 + m].float().permute(1, 2, 0)
        v = s["v"][k0:k0 + m].float().permute(1, 0, 2)
        scores = torch.matmul(q, k).mul_(dim ** -0.5).view(hk, g, n, m)
        i = torch.arange(n, device="cuda")[:, None]
        j = torch.arange(m, device="cuda")
        scores.masked_fill_(j > i + (m - n), -math.inf)
        o, lse = _softmax_v(scores.view(hk, g * n, m), v)
        outs.append(o.view(hk * g, n, dim).permute(1, 0, 2))
        lses.append(lse.view(hk * g, n).permute(1, 0))
        q0, k0 = q0 + n, k0 + m
    o = torch.cat(outs).to(s["q"].dtype)
    return (o, torch.cat(lses)) if s["lse"] else o


def _token_pages(s, cu, first, total):
    """For each packed token: its page and its slot in the page; token j of sequence b is at first[b] + j."""
    page = s["page"]
    at = torch.arange(total, device="cuda")
    b = torch.searchsorted(cu[1:].contiguous(), at, right=True)
    pos = at - cu[b] + first[b]
    return s["page_table"][b, pos // page].long(), pos % page


def _plain_append(s):
    pool, page = s["pool"], s["page"]
    cu = s["cu_new"]
    first = s["lengths"] - (cu[1:] - cu[:-1])                     # position of each sequence's first new token
    pg, slot = _token_pages(s, cu, first, s["new"])
    # which slots of the pages hold tokens from before: those under the sequence's old end
    last = s["page_table"].gather(1, (first // page)[:, None].long().clamp_max(s["page_table"].shape[1] - 1)).squeeze(1).long()
    part = (first % page > 0) & (cu[1:] > cu[:-1])
    kept = torch.zeros(pool + 1, dtype=torch.bool, device="cuda")
    kept[torch.where(part, last, pool)] = True
    kept = kept[:pool]
    last = torch.where(part, last, 0)
    read_pg, read_slot = _token_pages(s, s["cu_read"], s["starts"], s["read"])
    outs = []
    for name in ("k", "v"):
        x, codes, scale = s[name].float(), s[name + "_pages"], s[name + "_scale"]
        amax = x.abs().amax(-1)                                   # [tokens, heads]
        top = torch.zeros(pool, x.shape[1], device="cuda").index_reduce_(0, pg, amax, "amax")
        e_new = _exponent(top)
        e_old = torch.frexp(scale)[1] - 1
        touched = torch.zeros(pool, dtype=torch.bool, device="cuda")
        touched[pg] = True
        e = torch.where(kept[:, None], torch.maximum(e_old, e_new), e_new)
        e = torch.where(touched[:, None], e, e_old)
        grown = (e > e_old) & kept[:, None]
        old = codes[last].float() * _pow2(e_old - e)[last][..., None, None]
        codes[last] = torch.where(grown[last][..., None, None], old, codes[last].float()).to(codes.dtype)
        scale.copy_(_pow2(e))
        h = torch.arange(x.shape[1], device="cuda")
        codes[pg[:, None], h, slot[:, None]] = (x * _pow2(-e[pg])[..., None]).to(codes.dtype)
        outs.append((codes[read_pg[:, None], h, read_slot[:, None]].float() * scale[read_pg][..., None]).to(s[name].dtype))
    return outs[0], outs[1], s["k_scale"], s["v_scale"]


def _plain_decode(s):
    b, sq, hq, dim = s["q"].shape
    hk = s["kv"]
    g = hq // hk
    pt = s["page_table"].clamp_min(0).long()
    m = pt.shape[1] * s["page"]
    k, v = ((s[x + "_pages"][pt].float() * s[x + "_scale"][pt][..., None, None]).transpose(1, 2).reshape(b, hk, m, dim)
            for x in ("k", "v"))                                   # [b, kv heads, tokens, dim]
    q = s["q"].float().view(b, sq, hk, g, dim).permute(0, 2, 3, 1, 4).reshape(b, hk, g * sq, dim)
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(dim ** -0.5).view(b, hk, g, sq, m)
    j = torch.arange(m, device="cuda")
    seen = s["lengths"][:, None] - sq + 1 + torch.arange(sq, device="cuda")      # keys that query i sees
    scores.masked_fill_(j >= seen[:, None, None, :, None], -math.inf)
    o, lse = _softmax_v(scores.view(b, hk, g * sq, m), v)
    o = o.view(b, hk, g, sq, dim).permute(0, 3, 1, 2, 4).reshape(b, sq, hq, dim).to(s["q"].dtype)
    lse = lse.view(b, hk, g, sq).permute(0, 3, 1, 2).reshape(b, sq, hq)
    return (o, lse) if s["lse"] else o


def run(s):
    if not own:
        return {"prompt": _plain_prompt, "append": _plain_append, "decode": _plain_decode}[s["kind"]](s)
    from kairos_sensenova_b200 import KVCache, attention_cached, attention_prompt, kv_cache_append, kv_cache_gather
    if s["kind"] == "prompt":
        return attention_prompt(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], return_lse=s["lse"])
    cache = KVCache(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
    if s["kind"] == "append":
        kv_cache_append(cache, s["k"], s["v"], s["page_table"], s["lengths"], s["cu_new"])
        k, v = kv_cache_gather(cache, s["page_table"], s["starts"], s["cu_read"], total=s["read"], dtype=s["k"].dtype)
        return k, v, cache.k_scale, cache.v_scale
    return attention_cached(s["q"], cache, s["page_table"], s["lengths"], return_lse=s["lse"])


def work(case):
    dim = case["dim"]
    if case["kind"] == "prompt":
        nq, nk = _lens(case["q"]), _lens(case["k"])
        pairs = sum(_pairs(n, m) for n, m in zip(nq, nk))
        return {"bytes": 2 * dim * (2 * sum(nq) * case["heads"] + 2 * sum(nk) * case["kv"]) + 4 * sum(nq) * case["heads"] * case["lse"],
                "flops": 4 * dim * case["heads"] * pairs}
    if case["kind"] == "append":
        new, old, page = _lens(case["new"]), _lens(case["old"]), case["page"]
        old = old * len(new) if len(old) == 1 else old
        read = sum(a + b - b // page * page for a, b in zip(new, old))
        # new tokens read in 16 bits and written in 8; the tokens read back from 8 to 16 bits (k and v each)
        return {"bytes": 2 * case["heads"] * dim * (3 * sum(new) + 2 * read + (read - sum(new))), "flops": 2 * case["heads"] * dim * sum(new)}
    lens, page = _lens(case["lens"]), case["page"]
    pages = sum(-(-n // page) for n in lens)
    rows = len(lens) * case["sq"] * case["heads"]
    return {"bytes": 2 * case["kv"] * (dim * sum(lens) + 4 * pages) + 4 * dim * rows + 4 * rows * case["lse"] + 4 * pages,
            "flops": 4 * dim * case["heads"] * sum(_pairs(case["sq"], n) for n in lens)}


def _exact_attention(q, k, v, seen):
    """q [r, d], k, v [m, d] in 64 bits; row i sees the first seen[i] keys."""
    p = torch.einsum("rd,md->rm", q, k) / math.sqrt(q.shape[1])
    hidden = torch.arange(k.shape[0], device=q.device).unsqueeze(0) >= seen.unsqueeze(1)
    p[hidden] = -math.inf
    lse = torch.logsumexp(p, 1)
    w = torch.exp(p - lse.unsqueeze(1)).nan_to_num_(0.0)
    return torch.einsum("rm,md->rd", w, v), lse


def exact(case, seed):
    s = prepare(case, seed)
    dim = case["dim"]
    if case["kind"] == "append":
        return _exact_append(s)
    heads, kv = case["heads"], case["kv"]
    g = heads // kv
    if case["kind"] == "prompt":
        o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.zeros(o.shape[:2], dtype=torch.float64, device="cuda")
        cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
        for n in range(len(cq) - 1):
            rows, keys = slice(cq[n], cq[n + 1]), slice(ck[n], ck[n + 1])
            off = (ck[n + 1] - ck[n]) - (cq[n + 1] - cq[n])
            seen = torch.arange(cq[n + 1] - cq[n], device="cuda") + off + 1
            for h in range(heads):
                o[rows, h], lse[rows, h] = _exact_attention(s["q"][rows, h].double(), s["k"][keys, h // g].double(),
                                                            s["v"][keys, h // g].double(), seen)
    else:
        b, sq = s["q"].shape[:2]
        o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.full(o.shape[:3], -math.inf, dtype=torch.float64, device="cuda")
        for n in range(b):
            m = s["lens"][n]
            if m == 0:
                continue
            pages = s["page_table"][n, : -(-m // case["page"])].long()
            seen = (m - sq + 1 + torch.arange(sq, device="cuda")).repeat_interleave(g)
            for h in range(kv):
                k, v = ((s[x + "_pages"][pages, h].double() * s[x + "_scale"][pages, h].double()[:, None, None]).reshape(-1, dim)[:m]
                        for x in ("k", "v"))
                rows = s["q"][n, :, h * g:(h + 1) * g].double().reshape(sq * g, dim)
                a, c = _exact_attention(rows, k, v, seen)
                o[n, :, h * g:(h + 1) * g], lse[n, :, h * g:(h + 1) * g] = a.view(sq, g, dim), c.view(sq, g)
    return (o, lse) if case["lse"] else o


def _exact_codes(x):
    """x, finite and at most 448 in magnitude, to the nearest e4m3 value, ties to the even one: steps of 2^(x - 3), 2^-9 at least."""
    step = torch.exp2((torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -20))) - 3).clamp_min(-9))
    return torch.round(x / step) * step


def _exact_append(s):
    page, lens, table = s["page"], s["lens"], s["page_table"].tolist()
    cu, starts = s["cu_new"].tolist(), s["starts"].tolist()
    outs = []
    for name in ("k", "v"):
        scale = s[name + "_scale"].double()
        read = []
        for b, m in enumerate(lens):
            n = cu[b + 1] - cu[b]
            lo = starts[b]
            ids = torch.tensor(table[b][lo // page: -(-m // page)], device="cuda")
            kept = (m - n) - lo                                       # tokens of the first page that were there
            x = torch.zeros(len(ids) * page, s[name].shape[1], s["dim"], dtype=torch.float64, device="cuda")
            x[kept:m - lo] = s[name][cu[b]:cu[b + 1]].double()
            x = x.view(len(ids), page, -1, s["dim"]).transpose(1, 2)
            # 1e-9 below: log2 of a power of two may come out an ulp above it, and the next 16-bit value is 1e-3 away
            e = torch.ceil(torch.log2(x.abs().amax((2, 3)) / 448.0) - 1e-9).clamp_min(SCALE_EXP_MIN)
            new = torch.exp2(e)
            if kept:
                new[0] = torch.maximum(new[0], scale[ids[0]])
                x[0, :, :kept] = s[name + "_pages"][ids[0], :, :kept].double() * scale[ids[0]][:, None, None]
            x = _exact_codes(x / new[..., None, None]) * new[..., None, None]
            scale[ids] = new
            read.append(x.transpose(1, 2).reshape(len(ids) * page, -1, s["dim"])[:m - lo])
        outs.append((torch.cat(read), scale))
    return outs[0][0], outs[1][0], outs[0][1], outs[1][1]
