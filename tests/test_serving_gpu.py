"""attention_prompt, the 8-bit paged cache and attention_cached against ``oracle.serving`` (64 bits).

Bounds.  With u the half step of the output type (bf16 2^-8, fp16 2^-11) and u_p that of the
probabilities (attention_prompt rounds them to the input type, attention_cached to fp16),
|o - ref| <= u_p A + u |ref| + c A, A = sum_j softmax_j |v_j|.  c covers the fp32 chain: a score's error
is at most D 2^-24 sum_d |q_d k_d| scale <= 128 * 2^-24 * |q| |k| scale, and |q| |k| scale < 32 for the data
here, so 2 * 128 * 32 * 2^-24 = 2^-11 relative in a probability at the very most; the sums add n 2^-24."""
import ctypes
import math

import pytest
import torch

from kairos_sensenova_b200 import KVCache, _lib, attention_cached, attention_prompt, kv_cache_append, kv_cache_gather
from oracle import serving as ref

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
CHAIN = 2.0 ** -11


def close(o, want, A, dtype, u_p=None):
    u = HALF_STEP[dtype]
    bound = (HALF_STEP[dtype] if u_p is None else u_p) * A + u * want.abs() + CHAIN * A + 1e-7
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(o), nan), 'NaN in other places'
    inf = torch.isinf(want)
    assert torch.equal(o[inf].double(), want[inf])
    off = torch.where(nan | inf, 0.0, (o.double() - want).abs() - bound)
    assert (off <= 0).all(), f'{off.max().item():.3e} over the bound at {(off > 0).nonzero()[:4].tolist()}'


def close_lse(lse, want):
    fin = torch.isfinite(want)
    assert torch.equal(lse[~fin].double(), want[~fin])
    assert ((lse.double() - want)[fin].abs() <= 2.0 ** -11 + want[fin].abs() * 2.0 ** -22).all()


def cu(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device='cuda')


def gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device='cuda').to(dtype)


# ------------------------------------------------------------------ prompts
LENS = [
    ([1], [1]), ([0], [0]), ([5, 0, 3], [5, 0, 3]), ([128], [128]), ([129, 1, 127], [129, 1, 127]),
    ([255, 256, 257], [255, 256, 257]), ([640, 33], [640, 33]),
    ([1, 7, 64], [300, 129, 64]),            # queries at the end of more keys
    ([0, 4], [50, 0]),                       # no queries; no keys at all
    ([300, 20], [40, 20]),                   # more queries than keys: the first see nothing
    ([3] * 70, [5] * 70),
]


@pytest.mark.parametrize('nq,nk', LENS)
@pytest.mark.parametrize('heads,kv,dim,dtype', [(4, 4, 128, torch.bfloat16), (6, 2, 64, torch.float16),
                                                (7, 1, 128, torch.float16), (5, 5, 64, torch.bfloat16)])
def test_prompt(nq, nk, heads, kv, dim, dtype):
    g = gen(len(nq) * 1000 + sum(nq) + heads)
    q, k, v = randn(g, sum(nq), heads, dim, dtype=dtype), randn(g, sum(nk), kv, dim, dtype=dtype), \
        randn(g, sum(nk), kv, dim, dtype=dtype)
    for causal in (True, False):
        o, lse = attention_prompt(q, k, v, i32(cu(nq)), i32(cu(nk)), causal=causal, return_lse=True, check=True)
        want, wlse, A = ref.prompt(q, k, v, cu(nq), cu(nk), dim ** -0.5, causal)
        close(o, want, A, dtype)
        close_lse(lse, wlse)


@pytest.mark.parametrize('heads,kv,dim,dtype,n', [(24, 8, 128, torch.bfloat16, 3001), (32, 1, 64, torch.float16, 1500),
                                                  (2, 2, 128, torch.float16, 5000), (96, 1, 128, torch.bfloat16, 700),
                                                  (300, 1, 64, torch.bfloat16, 65)])
def test_prompt_long(heads, kv, dim, dtype, n):
    g = gen(n)
    x = randn(g, n, heads + 2 * kv, dim, dtype=dtype)         # views of a fused projection
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    o = attention_prompt(q, k, v, i32([0, n]))
    want, _, A = ref.prompt(q, k, v, [0, n], [0, n], dim ** -0.5)
    close(o, want, A, dtype)
    assert torch.equal(o, attention_prompt(q, k, v, i32([0, n])))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('value', [math.nan, math.inf])
def test_prompt_masked_values_do_not_leak(dtype, value):
    """K and V of one token not finite: rows that do not see it, in its sequence and in the neighbours, keep within
    the bound of the formula without it.  (Not the same bits: a tile that meets a NaN is summed in another order, so the
    two results differ by up to the bound each has of the formula.)"""
    g = gen(3)
    nq = [200, 150, 90]
    q, k, v = (randn(g, sum(nq), 3, 128, dtype=dtype) for _ in range(3))
    want, _, A = ref.prompt(q, k, v, cu(nq), cu(nq), 128 ** -0.5)
    at = 200 + 100                                            # token 100 of the second sequence
    kb, vb = k.clone(), v.clone()
    vb[at, 1, 5] = value
    kb[at, 2] = value
    o = attention_prompt(q, kb, vb, i32(cu(nq)))
    hit = torch.zeros_like(o, dtype=torch.bool)
    hit[at:350, 1, 5] = True
    hit[at:350, 2] = True
    close(o[~hit], want[~hit], A[~hit], dtype)
    assert not torch.isfinite(o[at:350, 1, 5]).any()
    assert torch.isnan(o[at:350, 2]).all() or value == math.inf
    # the first token of the next sequence: the sequence before ends in the same key tile
    vb = v.clone()
    vb[350] = value
    o = attention_prompt(q, k, vb, i32(cu(nq)))
    close(o[:350], want[:350], A[:350], dtype)


@pytest.mark.parametrize('keys', [400, 9000])
def test_prompt_nan_everywhere_and_no_keys(keys):
    """All of V, or of K, is NaN: so is the result, in no unusual time; no keys at all: 0.  (9000 keys of 400 queries are
    shared out over the SMs.)"""
    g = gen(17)
    q, k, v = randn(g, 400, 2, 128), randn(g, keys, 2, 128), randn(g, keys, 2, 128)
    nan = torch.full_like(v, math.nan)
    for a, b in ((k, nan), (nan, v)):
        assert torch.isnan(attention_prompt(q, a, b, i32([0, 400]), i32([0, keys]))).all()
    vb = v.clone()
    vb[keys - 30, 1, 9] = -math.inf                          # seen by the last 30 queries
    o, lse = attention_prompt(q, k, vb, i32([0, 400]), i32([0, keys]), return_lse=True)
    want, wlse, A = ref.prompt(q, k, vb, [0, 400], [0, keys], 128 ** -0.5)
    hit = torch.zeros_like(o, dtype=torch.bool)
    hit[370:, 1, 9] = True
    close(o[~hit], want[~hit], A[~hit], torch.bfloat16)
    assert (o[hit] == -math.inf).all()
    close_lse(lse, wlse)
    o, lse = attention_prompt(q, k[:0], v[:0], i32([0, 400]), i32([0, 0]), return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()


def milliseconds(f, n=5):
    """The median of n calls, after three."""
    times = []
    for i in range(n + 3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    return sorted(times[3:])[n // 2]


@pytest.mark.parametrize('nq,nk,heads,kv,dim,dtype', [
    ([3000], [3000], 24, 24, 128, torch.bfloat16),            # whole items of 256 tokens
    ([1000, 1, 333], [1500, 700, 300], 24, 8, 64, torch.float16),   # 84 tokens; more keys than queries, and fewer
    ([90] * 3, [90] * 3, 300, 1, 64, torch.bfloat16),         # the heads of a kv head in three parts
    ([200, 40], [9000, 2100], 6, 2, 128, torch.float16),      # key tiles in shares
])
def test_prompt_hidden_values_at_many_keys(nq, nk, heads, kv, dim, dtype):
    """V not finite at the newest keys, some channels of one kv head and all of another: infinities of both signs and NaN reach the
    rows that see them, no other, and do not slow the call down by more than the tiles at the diagonal."""
    g = gen(41)
    q, k, v = randn(g, sum(nq), heads, dim, dtype=dtype), randn(g, sum(nk), kv, dim, dtype=dtype), randn(g, sum(nk), kv, dim, dtype=dtype)
    bad = v.clone()
    for end, n in zip(cu(nk)[1:], nk):
        bad[end - 1, 0] = math.nan
        for back, ch, x in ((3, 5, math.inf), (3, 6, -math.inf), (40, 5, math.inf), (41, 6, math.inf), (70, 7, -math.inf)):
            if back < n:
                bad[end - back, kv - 1, ch] = x
    cq, ck = i32(cu(nq)), i32(cu(nk))
    o, lse = attention_prompt(q, k, bad, cq, ck, return_lse=True)
    want, wlse, A = ref.prompt(q, k, bad, cu(nq), cu(nk), dim ** -0.5)
    assert not torch.isfinite(want).all()
    close(o, want, A, dtype)
    close_lse(lse, wlse)
    clean = milliseconds(lambda: attention_prompt(q, k, v, cq, ck))
    assert milliseconds(lambda: attention_prompt(q, k, bad, cq, ck)) <= 2 * clean + 0.2


@pytest.mark.parametrize('clocks', [1, 2000, 10000, 50000])
@pytest.mark.parametrize('nq,nk,heads,kv,dim', [([300] * 20 + [40, 0, 1], [300] * 20 + [90, 5, 1], 12, 4, 128),   # whole items
                                                ([200, 30], [9000, 2100], 6, 2, 64)])                              # shares
def test_prompt_wait_gives_up(nq, nk, heads, kv, dim, clocks):
    """Waits of a few clocks run out: the status word says so, and a row is either finished or NaN, in o and in lse."""
    L = _lib.lib()
    g = gen(43)
    q, k, v = randn(g, sum(nq), heads, dim), randn(g, sum(nk), kv, dim), randn(g, sum(nk), kv, dim)
    cq, ck, status = i32(cu(nq)), i32(cu(nk)), i32([0])
    o, lse = torch.full_like(q, 5.0), torch.full((sum(nq), heads), 5.0, device='cuda')
    size = L.kb200_attn_prompt_workspace_size(sum(nq), sum(nk), len(nq), heads, kv, dim)
    assert (size > 0) == (len(nq) == 2)
    ws = torch.zeros(max(size, 16), device='cuda', dtype=torch.uint8)
    a = _lib.PromptArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), o=o.data_ptr(), lse=lse.data_ptr(), cu_q=cq.data_ptr(),
                        cu_k=ck.data_ptr(), Tq=sum(nq), Tk=sum(nk), N=len(nq), Hq=heads, Hkv=kv, D=dim, q_token_stride=heads * dim,
                        q_head_stride=dim, k_token_stride=kv * dim, k_head_stride=dim, v_token_stride=kv * dim, v_head_stride=dim,
                        o_token_stride=heads * dim, o_head_stride=dim, softmax_scale=dim ** -0.5, causal=1, dtype=0,
                        workspace=ws.data_ptr() if size else None, workspace_bytes=size, status=status.data_ptr(), wait_clocks=clocks)
    stream = torch.cuda.current_stream().cuda_stream
    assert L.kb200_attn_prompt_fwd(ctypes.byref(a), stream) == 0
    rc = L.kb200_read_error_word(status.data_ptr(), stream)
    gone = torch.isnan(lse)
    assert torch.equal(torch.isnan(o).any(-1), gone) and torch.equal(torch.isnan(o).all(-1), gone)
    assert rc in (0, _lib.ERRORS_BY_NAME['timeout']) and (rc or (clocks > 1 and not gone.any()))
    want, wlse, A = ref.prompt(q, k, v, cu(nq), cu(nk), dim ** -0.5)
    close(o[~gone], want[~gone], A[~gone], torch.bfloat16)
    close_lse(lse[~gone], wlse[~gone])
    o2, lse2 = attention_prompt(q, k, v, cq, ck, return_lse=True, check=True)     # the device is as it was
    close(o2, want, A, torch.bfloat16)
    close_lse(lse2, wlse)


@pytest.mark.parametrize('heads,kv,dim,dtype', [(32, 8, 128, torch.bfloat16), (10, 2, 64, torch.float16), (2, 1, 128, torch.float16)])
def test_prompt_shared_out(heads, kv, dim, dtype):
    """Few rows and many keys: the key tiles go to all SMs in shares, sequences of other lengths and empty ones among them."""
    g = gen(heads)
    nq, nk = [70, 0, 1, 300, 5], [6000, 10, 2100, 4097, 3]
    q, k, v = randn(g, sum(nq), heads, dim, dtype=dtype), randn(g, sum(nk), kv, dim, dtype=dtype), randn(g, sum(nk), kv, dim, dtype=dtype)
    for causal in (True, False):
        o, lse = attention_prompt(q, k, v, i32(cu(nq)), i32(cu(nk)), causal=causal, return_lse=True)
        want, wlse, A = ref.prompt(q, k, v, cu(nq), cu(nk), dim ** -0.5, causal)
        close(o, want, A, dtype)
        close_lse(lse, wlse)
        assert torch.equal(o, attention_prompt(q, k, v, i32(cu(nq)), i32(cu(nk)), causal=causal))


def test_prompt_many_sequences():
    """Thousands of sequences, runs of empty ones among them."""
    nq = [1, 0, 3, 130] * 40 + [0] * 500 + [2] * 3000 + [0, 300, 0]
    g = gen(31)
    q, k, v = randn(g, sum(nq), 3, 64), randn(g, sum(nq), 1, 64), randn(g, sum(nq), 1, 64)
    for causal in (True, False):
        o, lse = attention_prompt(q, k, v, i32(cu(nq)), causal=causal, return_lse=True)
        some = [i for i, n in enumerate(nq) if n][::7] + [len(nq) - 2]
        at = cu(nq)
        for i in some:
            a, b = at[i], at[i + 1]
            want, wlse, A = ref.prompt(q[a:b], k[a:b], v[a:b], [0, b - a], [0, b - a], 64 ** -0.5, causal)
            close(o[a:b], want, A, torch.bfloat16)
            close_lse(lse[a:b], wlse)


def test_cached_many_sequences():
    """More units than shares, and thousands of empty sequences."""
    lens = [0, 17, 0, 40, 1] * 300 + [0] * 1000 + [900, 0, 3]
    H, D, page = 2, 64, 16
    cache, table, _ = make_cache(lens, H, D, page, seed=12)
    q = randn(gen(12), len(lens), 1, 4, D)
    out = torch.full((len(lens), 1, 4, D), 3.0, device='cuda', dtype=torch.bfloat16)
    _, lse = attention_cached(q, cache, i32(table), i32(lens), out=out, return_lse=True)
    want, wlse, A = ref.cached(q, values(cache.k_pages), values(cache.v_pages), cache.k_scale, cache.v_scale, table, lens, D ** -0.5)
    close(out, want, A, torch.bfloat16, u_p=2.0 ** -11)
    close_lse(lse, wlse)


@pytest.mark.parametrize('heads,H,D,sq,dtype', [(24, 8, 128, 1, torch.bfloat16), (6, 3, 64, 4, torch.float16),
                                                (48, 12, 64, 8, torch.bfloat16), (12, 4, 128, 6, torch.float16)])
def test_cached_short_sequences(heads, H, D, sq, dtype):
    """Many units to a share: short ones, which a warp takes alone, with empty and long ones among them, an odd page
    count and a page that is not there."""
    lens = [1 + (i * 37) % 190 for i in range(260)] + [0, 5000, 0, 1] + [100] * 100 + [1111] + [16] * 60 + [0]
    page = 32
    cache, table, _ = make_cache(lens, H, D, page, seed=14)
    table = [list(r) for r in table]
    table[7][0] = -1
    q = randn(gen(15), len(lens), sq, heads, D, dtype=dtype)
    o, lse = attention_cached(q, cache, i32(table), i32(lens), return_lse=True)
    want, wlse, A = ref.cached(q, values(cache.k_pages), values(cache.v_pages), cache.k_scale, cache.v_scale, table, lens, D ** -0.5)
    close(o, want, A, dtype, u_p=2.0 ** -11)
    close_lse(lse, wlse)
    assert torch.equal(o, attention_cached(q, cache, i32(table), i32(lens)))


def test_first_call_captured():
    """A process whose first calls are made while a graph is captured."""
    import subprocess
    import sys
    code = """
import torch
from kairos_sensenova_b200 import *
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device='cuda')
x = torch.randn(40, 2, 64, device='cuda').bfloat16()
c = KVCache.empty(4, 2, 64, 16)
t, n, s, cu = i32([[0, 1, 2]]), i32([40]), i32([0]), i32([0, 40])
out = []
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    kv_cache_append(c, x, x, t, n, cu)
    k, v = kv_cache_gather(c, t, s, cu, 40)
    out = [k, v, attention_prompt(x, k, v, cu), attention_cached(x[None, -1:], c, t, n)]
g.replay()
torch.cuda.synchronize()
kv_cache_append(c, x, x, t, n, cu)
k, v = kv_cache_gather(c, t, s, cu, 40)
for a, b in zip(out, [k, v, attention_prompt(x, k, v, cu), attention_cached(x[None, -1:], c, t, n)]):
    assert torch.equal(a, b)
print('same')
"""
    r = subprocess.run([sys.executable, '-c', code], capture_output=True, text=True, timeout=200)
    assert r.returncode == 0 and 'same' in r.stdout, r.stderr[-2000:]


def test_derivatives_are_refused():
    """By autograd, in forward mode, and under torch.func: no operator drops a derivative without a word."""
    from torch.autograd import forward_ad
    x, cache = randn(gen(2), 8, 2, 64), KVCache.empty(2, 2, 64, 16)
    calls = (lambda t: attention_prompt(x, x, t, i32([0, 8])), lambda t: attention_prompt(t, x, x, i32([0, 8])),
             lambda t: kv_cache_append(cache, x, t, i32([[0]]), i32([8]), i32([0, 8])),
             lambda t: attention_cached(t[None], cache, i32([[0]]), i32([8])))
    for call in calls:
        with pytest.raises(NotImplementedError):
            call(x.clone().requires_grad_())
        with forward_ad.dual_level(), pytest.raises(NotImplementedError):
            call(forward_ad.make_dual(x, x))
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.jvp(call, (x,), (x,))
        with torch.no_grad():
            call(x.clone().requires_grad_())


def test_prompt_extremes():
    """Scores up to the largest finite ones, equal scores, and a row maximum that keeps rising along the keys."""
    n, dt = 700, torch.bfloat16
    g = gen(5)
    q, k, v = (randn(g, n, 2, 64, dtype=dt) for _ in range(3))
    k[:, 0] = (k[:, 0].float() * torch.linspace(0.1, 30, n, device='cuda')[:, None]).to(dt)
    k[:, 1] = 1.0
    o, lse = attention_prompt(q, k, v, i32([0, n]), return_lse=True)
    want, wlse, A = ref.prompt(q, k, v, [0, n], [0, n], 64 ** -0.5)
    # scores here reach 30 times the usual: so does the fp32 chain's bound
    close(o, want, A * 30 * CHAIN / (HALF_STEP[dt] + CHAIN) + A, dt)
    assert ((lse.double() - wlse).abs() <= 30 * 2.0 ** -11 + wlse.abs() * 2.0 ** -22).all()
    q[:] = 3e38
    k[:] = -1.0
    o = attention_prompt(q, k, v, i32([0, n]))               # every score is -inf: no key counts
    assert (o == 0).all()


@pytest.mark.parametrize('nq,nk', [([1, 200, 30], [1, 200, 300]), ([60, 2], [9000, 2100])])      # whole items; shares
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_prompt_largest_values(nq, nk, dtype):
    """V up to half of the type's largest value at 200 keys, in any channels and in one key that outweighs them, and values of 2^-90
    (fp16: its smallest) beside them: an output is an average, so none leaves the type."""
    g = gen(47)
    q, k, v = (randn(g, n, 2, 128, dtype=dtype) for n in (sum(nq), sum(nk), sum(nk)))
    top = torch.finfo(dtype).max / 2
    for end, n in zip(cu(nk)[1:], nk):
        rows = slice(max(end - 200, end - n), end)
        v[rows, 0] = (v[rows, 0] / 8).clamp(-1, 1) * top
        v[end - n:end, 1] *= 2.0 ** -90 if dtype == torch.bfloat16 else 2.0 ** -14
    o, lse = attention_prompt(q, k, v, i32(cu(nq)), i32(cu(nk)), return_lse=True)
    want, wlse, A = ref.prompt(q, k, v, cu(nq), cu(nk), 128 ** -0.5)
    unit = torch.tensor([top, 2.0 ** -90 if dtype == torch.bfloat16 else 1.0], device='cuda', dtype=torch.float64)[:, None]
    close(o.double() / unit, want / unit, A / unit, dtype)
    close_lse(lse, wlse)


def signs(g, *shape):
    return torch.randint(0, 2, shape, generator=g, device='cuda').double() * 2 - 1


def close_large_lse(lse, want):
    """Beside close_lse's terms, five fp32 roundings of the result."""
    assert ((lse.double() - want).abs() <= 2.0 ** -11 + want.abs() * 5 * 2.0 ** -24).all()


@pytest.mark.parametrize('nq,nk,dim', [([300], [300], 64), ([100, 40], [6000, 2500], 128)])    # whole items; shares
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('largest', [2.0 ** 12, 2.0 ** 17, 2.0 ** 22])
def test_prompt_large_scores(nq, nk, dim, dtype, largest):
    """Scores of up to 2^22, where fp32's steps are up to 1/2: of equal ones every key has its share.  (q and k are
    +-1 and the scale is large, so that every score's product is exact; those that differ, differ by two scales.)"""
    g = gen(53)
    q, k = (signs(g, n, 2, dim).to(dtype) for n in (sum(nq), sum(nk)))
    k[: sum(nk) // 2] = k[sum(nk) - sum(nk) // 2:]            # every key twice: ties in every row that sees both
    v = randn(g, sum(nk), 2, dim, dtype=dtype)
    for scale in (largest / dim, -largest / dim):
        o, lse = attention_prompt(q, k, v, i32(cu(nq)), i32(cu(nk)), softmax_scale=scale, return_lse=True)
        want, wlse, A = ref.prompt(q, k, v, cu(nq), cu(nk), scale)
        close(o, want, A, dtype)
        close_large_lse(lse, wlse)


@pytest.mark.parametrize('lens,sq,heads,H,D', [([300, 40], 1, 4, 2, 64), ([7000], 3, 12, 2, 128), ([90] * 600, 1, 8, 2, 128)])
@pytest.mark.parametrize('largest', [2.0 ** 12, 2.0 ** 17, 2.0 ** 22])
def test_cached_large_scores(lens, sq, heads, H, D, largest):
    cache, table, _ = make_cache(lens, H, D, 16, seed=22)
    g = gen(22)
    half = signs(g, cache.num_pages, H, 8, D).float()
    cache.k_pages.copy_(torch.cat([half, half], 2).to(torch.float8_e4m3fn))     # every key of a page twice
    cache.k_scale.fill_(2.0 ** 10)
    q = signs(g, len(lens), sq, heads, D).to(torch.bfloat16)
    for scale in (largest / D / 2 ** 10, -largest / D / 2 ** 10):
        o, lse = attention_cached(q, cache, i32(table), i32(lens), softmax_scale=scale, return_lse=True)
        want, wlse, A = ref.cached(q, values(cache.k_pages), values(cache.v_pages), cache.k_scale, cache.v_scale, table, lens, scale)
        close(o, want, A, torch.bfloat16, u_p=2.0 ** -11)
        close_large_lse(lse, wlse)


@pytest.mark.parametrize('scale', [-0.3, 0.0, 1e-3, 2.0])
def test_any_softmax_scale(scale):
    g = gen(13)
    q, k, v = (randn(g, 150, 2, 64) for _ in range(3))
    o, lse = attention_prompt(q, k, v, i32([0, 20, 150]), softmax_scale=scale, return_lse=True)
    want, wlse, A = ref.prompt(q, k, v, [0, 20, 150], [0, 20, 150], scale)
    close(o, want, A * (1 + abs(scale)), torch.bfloat16)      # |q| |k| scale < 32 (1 + |scale|) * 8 here
    assert ((lse.double() - wlse).abs() <= 2.0 ** -9 + wlse.abs() * 2.0 ** -22).all()
    cache, table, _ = make_cache([33, 100], 2, 64, 16, 3)
    q = randn(g, 2, 2, 2, 64)
    o = attention_cached(q, cache, i32(table), i32([33, 100]), softmax_scale=scale)
    want, _, A = ref.cached(q, values(cache.k_pages), values(cache.v_pages), cache.k_scale, cache.v_scale, table, [33, 100], scale)
    close(o, want, A * (1 + abs(scale)), torch.bfloat16, u_p=2.0 ** -11)


def test_prompt_rows_behind_the_last_sequence_and_out():
    g = gen(7)
    q, k, v = (randn(g, 300, 2, 128) for _ in range(3))
    out = torch.full((300, 4, 128), 7.0, device='cuda', dtype=torch.bfloat16)[:, 1:3]
    r = attention_prompt(q, k, v, i32([0, 100, 211]), out=out)
    assert r is out and (out[211:] == 7).all() and (out._base[:, 0] == 7).all() and (out._base[:, 3] == 7).all()
    want, _, A = ref.prompt(q, k, v, [0, 100, 211], [0, 100, 211], 128 ** -0.5)
    close(out[:211], want[:211], A[:211], torch.bfloat16)
    # offsets past the tokens are clamped to them
    out2 = attention_prompt(q, k, v, i32([0, 100, 5000]))
    want, _, A = ref.prompt(q, k, v, [0, 100, 300], [0, 100, 300], 128 ** -0.5)
    close(out2, want, A, torch.bfloat16)


def test_prompt_far_offsets():
    """Element offsets over 2^31 in k and v."""
    n, ld = 66000, 33000
    base = torch.empty(n, ld, device='cuda', dtype=torch.bfloat16)
    g = gen(9)
    k, v = base[:, 32872 - 128:32872].view(n, 1, 128), base[:, 32872:33000].view(n, 1, 128)
    k.copy_(randn(g, n, 1, 128))
    v.copy_(randn(g, n, 1, 128))
    q = randn(g, 40, 1, 128)
    o = attention_prompt(q, k, v, i32([0, 40]), i32([0, n]))
    want, _, A = ref.prompt(q, k, v, [0, 40], [0, n], 128 ** -0.5)
    close(o, want, A, torch.bfloat16)


# ------------------------------------------------------------------ the cache
def make_cache(lens, H, D, page, seed, extra=2):
    """A filled pool, shuffled pages, random codes (NaN codes on pages and slots that nobody owns)."""
    g = gen(seed)
    need = [-(-n // page) for n in lens]
    P = sum(need) + extra
    order = torch.randperm(P, generator=torch.Generator().manual_seed(seed)).tolist()
    table, at = [], 0
    width = max(max(need), 1)
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    used = torch.zeros(P, page, dtype=torch.bool, device='cuda')
    for b, n in enumerate(lens):
        for j, pg in enumerate(table[b][:need[b]]):
            used[pg, :min(page, n - j * page)] = True
    pools, scales = [], []
    for _ in range(2):
        x = (torch.randn(P, H, page, D, generator=g, device='cuda') * 60).clamp(-448, 448)
        c = x.to(torch.float8_e4m3fn)
        c.view(torch.uint8).masked_fill_(~used[:, None, :, None], 0x7f)
        pools.append(c)
        scales.append(torch.exp2(torch.randint(-8, -4, (P, H), generator=g, device='cuda').float()))
    return KVCache(*pools, *scales), table, used


def values(codes):
    return codes.float().double()


@pytest.mark.parametrize('new,old', [([1], [0]), ([1, 1, 1], [0, 15, 16]), ([16, 17, 1], [0, 0, 130]), ([200, 0, 3], [5, 40, 127]),
                                     ([1] * 40, list(range(40))), ([700], [0]), ([0], [9])])
@pytest.mark.parametrize('H,D,page,dtype', [(1, 128, 64, torch.bfloat16), (3, 64, 16, torch.float16),
                                            (2, 128, 128, torch.float16), (8, 64, 32, torch.bfloat16), (5, 128, 16, torch.bfloat16),
                                            (2, 64, 128, torch.bfloat16), (2, 64, 64, torch.float16), (3, 128, 32, torch.bfloat16)])
def test_append_and_gather(new, old, H, D, page, dtype):
    lens = [a + b for a, b in zip(new, old)]
    cache, table, used = make_cache(lens, H, D, page, seed=sum(lens) + H)
    g = gen(D + page)
    k, v = randn(g, sum(new), H, D, dtype=dtype) * 3, randn(g, sum(new), H, D, dtype=dtype)
    want = []
    for codes, scale, x in ((cache.k_pages, cache.k_scale, k), (cache.v_pages, cache.v_scale, v)):
        w, s = values(codes), scale.clone()
        ref.append(w, s, x, table, lens, cu(new))
        want.append((w, s))
    kv_cache_append(cache, k, v, i32(table), i32(lens), i32(cu(new)), check=True)
    for codes, scale, (w, s) in ((cache.k_pages, cache.k_scale, want[0]), (cache.v_pages, cache.v_scale, want[1])):
        assert torch.equal(scale, s)
        got = values(codes)
        assert torch.equal(torch.isnan(got), torch.isnan(w)) and torch.equal(got.nan_to_num(), w.nan_to_num())
    # all of it back, and a range from the middle
    for starts in ([0] * len(lens), [n // 2 for n in lens]):
        counts = [n - s for n, s in zip(lens, starts)]
        for dt in (torch.bfloat16, torch.float16):
            kg, vg = kv_cache_gather(cache, i32(table), i32(starts), i32(cu(counts)), sum(counts), dtype=dt, check=True)
            for got, (w, s) in ((kg, want[0]), (vg, want[1])):
                assert torch.equal(got, ref.gather(w, s, table, starts, counts).to(dt))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_append_extremes(dtype):
    """Zeros, subnormals, the borders of a scale, the largest values, NaN and infinities, token by token into one page."""
    H, D, page = 2, 64, 16
    cache = KVCache.empty(3, H, D, page)
    rows = torch.zeros(14, H, D, device='cuda', dtype=dtype)
    big = torch.finfo(dtype).max / 4
    for i, x in enumerate([0.0, 2.0 ** -20, 448.0, 449.0 if dtype == torch.float16 else 450.0, 0.4375, 3.0, math.nan, math.inf, -math.inf, 7.5,
                           big, -big, 1.0, 2.0 ** -24]):
        rows[i] = torch.linspace(-1, 1, D, device='cuda').to(dtype) * 0.01
        rows[i, 0, 3] = x
        rows[i, 1] = x
    w, s = values(cache.k_pages), cache.k_scale.clone()
    table = [[1]]
    for i in range(14):
        ref.append(w, s, rows[i:i + 1], table, [i + 1], [0, 1])
        kv_cache_append(cache, rows[i:i + 1], rows[i:i + 1], i32(table), i32([i + 1]), i32([0, 1]))
        assert torch.equal(cache.k_scale, s) and torch.equal(cache.v_scale, s), i
        got = values(cache.k_pages)
        assert torch.equal(torch.isnan(got), torch.isnan(w)) and torch.equal(got.nan_to_num(), w.nan_to_num()), i


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_append_largest(dtype):
    """Tokens up to the type's end come back finite and within e4m3's half step (2^-4), alone and under a scale that they raise."""
    H, D, page = 2, 64, 16
    end = torch.finfo(dtype).max
    x = torch.tensor([1.0, -0.25, 0.87, 0.9375, -0.953, 0.96875, 0.969, -0.999, 1.0], device='cuda', dtype=torch.float64)
    x = (x * end).to(dtype)[:, None, None].expand(9, H, D).contiguous()
    x[:, 1, ::3] /= 64
    cache, table = KVCache.empty(2, H, D, page), i32([[1]])
    w, s = values(cache.k_pages), cache.k_scale.clone()
    for i in range(9):
        ref.append(w, s, x[i:i + 1], [[1]], [i + 1], [0, 1])
        kv_cache_append(cache, x[i:i + 1], x[i:i + 1], table, i32([i + 1]), i32([0, 1]))
        assert torch.equal(cache.k_scale, s) and torch.equal(values(cache.k_pages), w), i
    for got in kv_cache_gather(cache, table, i32([0]), i32([0, 9]), 9, dtype=dtype):
        assert torch.isfinite(got).all() and ((got.double() - x.double()).abs() <= 2.0 ** -4 * x.double().abs()).all()
    o = attention_cached(torch.zeros(1, 1, H, D, device='cuda', dtype=dtype), cache, table, i32([9]))      # the mean
    mean = (w[1] * s[1].double()[:, None, None])[:, :9].mean(1)
    assert torch.isfinite(o).all() and ((o[0, 0].double() - mean).abs() <= 2.0 ** -7 * mean.abs().amax()).all()


def test_append_leaves_out_what_does_not_fit():
    """Pages outside the pool, lengths over the table row and new tokens over the length: nothing of them is written."""
    cache = KVCache.empty(4, 1, 64, 16)
    before = cache.k_pages.clone().view(torch.uint8)
    x = torch.ones(40, 1, 64, device='cuda', dtype=torch.bfloat16)
    table, lens, new = [[0, 9], [-1, -5], [1, 2], [3, 3]], [32, 16, 100, 2], [20, 10, 5, 5]
    kv_cache_append(cache, x, x, i32(table), i32(lens), i32(cu(new)))
    got = cache.k_pages.view(torch.uint8)
    assert torch.equal(got[1:], before[1:])                   # sequences 1, 2, 3 wrote nothing
    assert (got[0, 0, 12:] != 0).all() and (got[0, 0, :12] == 0).all()   # sequence 0: its page 9 is left out
    kg, _ = kv_cache_gather(cache, i32(table), i32([0, 0, 90, 0]), i32([0, 32, 48, 58, 60]), 64)
    assert (kg[12:16] == 1).all() and (kg[16:60] == 0).all()


def test_append_and_gather_many_sequences():
    """More sequences than a warp looks at together, runs of empty ones among them."""
    n = [1, 0, 3] * 30 + [0] * 70 + [5] * 40 + [0] * 33 + [70] + [1] * 900
    old = [i % 37 for i in range(len(n))]
    lens = [a + b for a, b in zip(n, old)]
    H, D, page = 1, 64, 16
    cache, table, _ = make_cache(lens, H, D, page, seed=8)
    g = gen(8)
    k, v = randn(g, sum(n), H, D), randn(g, sum(n), H, D)
    w, s = values(cache.k_pages), cache.k_scale.clone()
    ref.append(w, s, k, table, lens, cu(n))
    kv_cache_append(cache, k, v, i32(table), i32(lens), i32(cu(n)))
    assert torch.equal(cache.k_scale, s) and torch.equal(values(cache.k_pages).nan_to_num(), w.nan_to_num())
    kg, _ = kv_cache_gather(cache, i32(table), i32(old), i32(cu(n)), sum(n))
    assert torch.equal(kg, ref.gather(w, s, table, old, n).bfloat16())


@pytest.mark.parametrize('H,D,page,dtype,new,old', [
    (8, 128, 64, torch.bfloat16, [6000, 1, 300], [37, 63, 128]),
    (7, 64, 16, torch.float16, [9000, 5, 1, 2000], [9, 16, 15, 100]),
    (5, 128, 128, torch.bfloat16, [15000], [100]),
    (24, 128, 32, torch.float16, [2500, 0, 40], [31, 7, 0]),
    (32, 128, 16, torch.bfloat16, [600] * 3, [1, 2, 3]),
    (9, 64, 128, torch.float16, [20000, 17], [1, 127]),
])
def test_append_and_gather_at_size(H, D, page, dtype, new, old):
    """Enough pages that a block takes several (head, k or v) items one after the other, numbers of items that the blocks do not
    divide, scales that grow over the tokens of a page's first ones, and tokens of more than a block's threads."""
    lens = [a + b for a, b in zip(new, old)]
    cache, table, _ = make_cache(lens, H, D, page, seed=H + D)
    g = gen(H * page)
    grow = torch.exp2(torch.randint(-3, 7, (sum(new), H, 1), generator=g, device='cuda').float()).to(dtype)
    k, v = randn(g, sum(new), H, D, dtype=dtype) * grow, randn(g, sum(new), H, D, dtype=dtype) * grow.flip(1)
    want = []
    for codes, scale, x in ((cache.k_pages, cache.k_scale, k), (cache.v_pages, cache.v_scale, v)):
        w, s = values(codes), scale.clone()
        ref.append(w, s, x, table, lens, cu(new))
        want.append((w, s))
    kv_cache_append(cache, k, v, i32(table), i32(lens), i32(cu(new)), check=True)
    for codes, scale, (w, s) in ((cache.k_pages, cache.k_scale, want[0]), (cache.v_pages, cache.v_scale, want[1])):
        got = values(codes)
        assert torch.equal(scale, s) and torch.equal(torch.isnan(got), torch.isnan(w)) and torch.equal(got.nan_to_num(), w.nan_to_num())
    counts = [n - n // 3 for n in lens]
    kg, vg = kv_cache_gather(cache, i32(table), i32([n // 3 for n in lens]), i32(cu(counts)), sum(counts), dtype=dtype, check=True)
    for got, (w, s) in ((kg, want[0]), (vg, want[1])):
        flat = w * s.double()[:, :, None, None]              # [pages, H, page, D]
        for b, n in enumerate(lens):
            rows = flat[table[b][:-(-n // page)]].transpose(1, 2).reshape(-1, H, D)[n // 3:n] if n else flat.new_zeros(0, H, D)
            assert torch.equal(got[cu(counts)[b]:cu(counts)[b + 1]], rows.to(dtype))


def test_gather_leaves_other_rows():
    cache, table, _ = make_cache([30], 2, 128, 16, 1)
    out = [torch.full((50, 2, 128), 5.0, device='cuda', dtype=torch.bfloat16) for _ in range(2)]
    kv_cache_gather(cache, i32(table), i32([3]), i32([0, 27]), 50, out=out)
    assert all((t[27:] == 5).all() and (t[:27] != 5).any() for t in out)


# ------------------------------------------------------------------ attention over the cache
@pytest.mark.parametrize('lens,sq', [([1], 1), ([0, 5, 0], 1), ([127, 128, 129], 1), ([16, 17, 1000], 1), ([2, 300, 0], 4),
                                     ([64] * 33, 1), ([513], 9), ([3000, 1], 2)])
@pytest.mark.parametrize('heads,H,D,page,dtype', [(8, 2, 128, 64, torch.bfloat16), (3, 3, 64, 16, torch.float16),
                                                  (16, 1, 64, 32, torch.bfloat16), (14, 2, 128, 128, torch.float16),
                                                  (40, 1, 128, 16, torch.bfloat16), (5, 1, 64, 128, torch.bfloat16)])
def test_cached(lens, sq, heads, H, D, page, dtype):
    cache, table, _ = make_cache(lens, H, D, page, seed=len(lens) + sum(lens))
    q = randn(gen(heads), len(lens), sq, heads, D, dtype=dtype)
    o, lse = attention_cached(q, cache, i32(table), i32(lens), return_lse=True, check=True)
    want, wlse, A = ref.cached(q, values(cache.k_pages), values(cache.v_pages), cache.k_scale, cache.v_scale, table, lens,
                               D ** -0.5)
    close(o, want, A, dtype, u_p=2.0 ** -11)
    close_lse(lse, wlse)
    assert torch.equal(o, attention_cached(q, cache, i32(table), i32(lens)))


def test_cached_many_rows_and_long():
    for lens, sq, heads, H, D, page in (([700, 20], 40, 8, 2, 128, 64), ([40000, 3], 1, 4, 4, 64, 16), ([9000], 3, 200, 1, 128, 32)):
        cache, table, _ = make_cache(lens, H, D, page, seed=sq)
        q = randn(gen(sq), len(lens), sq, heads, D)
        o, lse = attention_cached(q, cache, i32(table), i32(lens), return_lse=True)
        want, wlse, A = ref.cached(q, values(cache.k_pages), values(cache.v_pages), cache.k_scale, cache.v_scale, table,
                                   lens, D ** -0.5)
        close(o, want, A, torch.bfloat16, u_p=2.0 ** -11)
        close_lse(lse, wlse)


def test_cached_scales_far_apart():
    """V scales 2^40 apart, the largest on a page whose keys get no weight; queries of any size; a strided q."""
    lens, H, D, page = [64], 1, 128, 16
    cache, table, _ = make_cache(lens, H, D, page, seed=2)
    cache.v_scale[table[0][1]] = 2.0 ** 30
    cache.v_scale[table[0][2]] = 2.0 ** -30
    k = values(cache.k_pages)
    cache.k_pages[table[0][1]] = torch.tensor(-448.0, device='cuda').to(torch.float8_e4m3fn)
    k = values(cache.k_pages)
    q = torch.full((1, 2, 6, D), 1.0, device='cuda', dtype=torch.bfloat16)
    q[:, :, 1] = 2.0 ** -100
    q[:, :, 2] = torch.randn(D, generator=gen(1), device='cuda').bfloat16() * 1e-3
    q = q[:, :, ::2]                                          # heads 0, 2, 4
    o = attention_cached(q, cache, i32(table), i32(lens), softmax_scale=0.02)
    want, _, A = ref.cached(q, k, values(cache.v_pages), cache.k_scale, cache.v_scale, table, lens, 0.02)
    close(o, want, A, torch.bfloat16, u_p=2.0 ** -11)


@pytest.mark.parametrize('lens,sq,heads,H,D,page', [([1, 300, 0, 20], 1, 4, 2, 128, 16), ([5000, 700], 2, 8, 1, 64, 32),
                                                    ([100] * 700, 1, 4, 2, 64, 64)])
@pytest.mark.parametrize('exponent', [118, -117])
def test_cached_largest_and_smallest_values(lens, sq, heads, H, D, page, exponent):
    """V of the first head up to 448 * 2^118 (the largest bf16 is 1.99 * 448 * 2^118), or under the smallest scale there is: an output
    is an average, so it is neither infinite nor lost.  (Whole units, joined ones, and short ones of a warp alone.)"""
    cache, table, _ = make_cache(lens, H, D, page, seed=19)
    cache.v_scale[:, 0] = 2.0 ** exponent
    q = randn(gen(20), len(lens), sq, heads, D)
    o, lse = attention_cached(q, cache, i32(table), i32(lens), return_lse=True)
    want, wlse, A = ref.cached(q, values(cache.k_pages), values(cache.v_pages), cache.k_scale, cache.v_scale, table, lens, D ** -0.5)
    unit = torch.ones(heads, 1, device='cuda', dtype=torch.float64)
    unit[:heads // H] = 2.0 ** exponent
    close(o.double() / unit, want / unit, A / unit, torch.bfloat16, u_p=2.0 ** -11)
    close_lse(lse, wlse)


@pytest.mark.parametrize('sq,heads,D,page,spread', [(1, 4, 128, 16, 30), (3, 4, 64, 32, 30), (6, 4, 128, 32, 40), (1, 4, 64, 16, 12)])
def test_cached_small_weights_of_large_values(sq, heads, D, page, spread):
    """Keys with weights of about 2^-28 (and 2^-10, in the second sequence) of the largest, on pages whose V scale is 2^30 (2^40, 2^12) larger than
    the others'.  Beside close's terms: a probability under 2^-22 of the row's largest P, which is 2^8 at least, is rounded in f16's
    subnormals, 2^-25 off at most, 2^-33 of the largest; that is 2^-33 of each |v| in the output."""
    lens = [1000, 700, 260]
    cache, table, _ = make_cache(lens, 1, D, page, seed=23)
    g = gen(23)
    cache.k_pages.copy_(torch.full(cache.k_pages.shape, 0.5, device='cuda').to(torch.float8_e4m3fn))
    cache.k_scale.fill_(2.0 ** -3)
    cache.v_scale.fill_(2.0 ** -6)
    q = (1 + 0.02 * torch.randn(3, sq, heads, D, generator=g, device='cuda')).to(torch.bfloat16)
    # a score is 1/16 a channel, times the scale: so far above those of keys of code -0.5
    bits = [28, 10, 28]
    for b, where in enumerate(([3, 17, 18], [0, 9], [2])):
        for i in where:
            pg = table[b][i]
            cache.k_pages[pg] = torch.tensor(-0.5 if bits[b] == 28 else 0.15625, device='cuda').to(torch.float8_e4m3fn)
            cache.v_scale[pg] = 2.0 ** (spread - 6)
    scale = 28 * math.log(2) / (D / 8)                       # between codes 0.5 and -0.5: 28 bits
    o, lse = attention_cached(q, cache, i32(table), i32(lens), softmax_scale=scale, return_lse=True)
    want, wlse, A = ref.cached(q, values(cache.k_pages), values(cache.v_pages), cache.k_scale, cache.v_scale, table, lens, scale)
    for b, n in enumerate(lens):
        total = sum((values(cache.v_pages[pg]) * cache.v_scale[pg].double()[:, None, None])[0, :n - i * page].abs().sum(0)
                    for i, pg in enumerate(table[b][:-(-n // page)]))
        close(o[b], want[b], A[b] + total * 2.0 ** -33 * 2.0 ** 11, torch.bfloat16, u_p=2.0 ** -11)
    close_lse(lse, wlse)


def test_cached_hidden_nan_and_missing_pages():
    """A NaN code of the newest token reaches only the queries that see it; a missing page is skipped."""
    lens, H, D, page = [100], 2, 128, 32
    cache, table, _ = make_cache(lens, H, D, page, seed=4)
    q = randn(gen(4), 1, 3, 4, D)
    clean = attention_cached(q, cache, i32(table), i32(lens))
    pg = table[0][99 // page]
    cache.v_pages.view(torch.uint8)[pg, 0, 99 % page, 7] = 0x7f     # the last token: query 2 alone sees it
    cache.k_pages.view(torch.uint8)[pg, 1, 98 % page] = 0xff        # the one before: queries 1 and 2
    o = attention_cached(q, cache, i32(table), i32(lens))
    hit = torch.zeros_like(o, dtype=torch.bool)
    hit[0, 2, :2, 7] = True
    hit[0, 1:, 2:] = True
    assert torch.equal(o[~hit], clean[~hit]) and torch.isnan(o[hit]).all()
    # all keys NaN: NaN, not 0
    cache.k_pages.view(torch.uint8)[:] = 0x7f
    assert torch.isnan(attention_cached(q, cache, i32(table), i32(lens))).all()
    # a table entry outside the pool: its tokens are not there
    cache, table, _ = make_cache([96], H, D, page, seed=5)
    holed = [[table[0][0], 10 ** 9, table[0][2]]]
    o, lse = attention_cached(q, cache, i32(holed), i32([96]), return_lse=True)
    short = [[table[0][0], table[0][2]]]
    w, wl = attention_cached(q, cache, i32(short), i32([64]), return_lse=True)
    assert (o.float() - w.float()).abs().max() <= 2.0 ** -7 * w.float().abs().max() and (lse - wl).abs().max() < 1e-3
    # lengths over the table row are cut to it
    assert torch.equal(attention_cached(q, cache, i32(table), i32([5000])), attention_cached(q, cache, i32(table), i32([96])))


def test_cached_far_pages():
    """Code offsets over 2^31 bytes."""
    H, D, page, P = 4, 128, 128, 40000                       # 2.6 GB each for k and v
    k = torch.zeros(P, H, page, D, device='cuda', dtype=torch.uint8).view(torch.float8_e4m3fn)
    v = torch.zeros_like(k)
    cache = KVCache(k, v, torch.ones(P, H, device='cuda'), torch.ones(P, H, device='cuda'))
    table, lens = [[39999, 39998, 7]], [300]
    g = gen(11)
    x, y = randn(g, 300, H, D), randn(g, 300, H, D)
    kv_cache_append(cache, x, y, i32(table), i32(lens), i32([0, 300]))
    xg, yg = kv_cache_gather(cache, i32(table), i32([0]), i32([0, 300]), 300)
    assert ((xg.float() - x.float()).abs() <= 2.0 ** -4 * x.float().abs() + 2.0 ** -10 * 4).all()
    q = randn(g, 1, 1, 8, D)
    o = attention_cached(q, cache, i32(table), i32(lens))
    want, _, A = ref.prompt(q[0], xg, yg, [0, 1], [0, 300], D ** -0.5)
    close(o[0], want, A, torch.bfloat16, u_p=2.0 ** -11)


# ------------------------------------------------------------------ together, as they are used
def test_serving_run_in_pieces_streams_and_graph():
    """Prompts, their next pieces over the gathered context, then decode steps replayed as a graph, on a side stream;
    every step against attention over the tokens that the cache holds."""
    H, heads, D, page, B = 2, 6, 128, 16, 3
    g = gen(21)
    lens = [37, 5, 130]
    cache = KVCache.empty(64, H, D, page)
    perm = torch.randperm(64, generator=torch.Generator().manual_seed(1)).tolist()
    table_l = [perm[i * 20:(i + 1) * 20] for i in range(B)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        table = i32(table_l)
        done = [0] * B
        for piece in (lens, [16, 0, 3]):
            q, k, v = randn(g, sum(piece), heads, D), randn(g, sum(piece), H, D), randn(g, sum(piece), H, D)
            done = [a + b for a, b in zip(done, piece)]
            kv_cache_append(cache, k, v, table, i32(done), i32(cu(piece)))
            kc, vc = kv_cache_gather(cache, table, i32([0] * B), i32(cu(done)), sum(done))
            o = attention_prompt(q, kc, vc, i32(cu(piece)), i32(cu(done)))
            want, _, A = ref.prompt(q, kc, vc, cu(piece), cu(done), D ** -0.5)
            close(o, want, A, torch.bfloat16)
        # a decode step as a graph: lengths grow inside it
        length = i32(done)
        q, k, v = randn(g, B, 1, heads, D), randn(g, B, H, D), randn(g, B, H, D)
        steps = i32(list(range(B + 1)))

        def step():
            length.add_(1)
            kv_cache_append(cache, k, v, table, length, steps)
            return attention_cached(q, cache, table, length)
        step()
        done = [n + 1 for n in done]
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o = step()
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other, stream=side):
        o2 = attention_cached(q, cache, table, length)
    for i in range(20):
        q.copy_(randn(g, B, 1, heads, D))
        k.copy_(randn(g, B, H, D))
        v.copy_(randn(g, B, H, D))
        graph.replay()
        other.replay()
        done = [n + 1 for n in done]
        assert length.tolist() == done and torch.equal(o, o2)
        want, _, A = ref.cached(q, values(cache.k_pages), values(cache.v_pages), cache.k_scale, cache.v_scale, table_l, done,
                                D ** -0.5)
        close(o, want, A, torch.bfloat16, u_p=2.0 ** -11)
