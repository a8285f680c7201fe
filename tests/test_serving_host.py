"""Refusals of the serving operators (no GPU: the checks run before anything is launched) and the oracle itself."""
import ctypes

import pytest
import torch

from kairos_sensenova_b200 import KVCache, _lib, attention_cached, attention_prompt, kv_cache_append, kv_cache_gather
from kairos_sensenova_b200.kv_cache import _int32, _refuse_grad, _rows, check_tables
from oracle import serving as ref

i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731


def test_cache_refuses_other_layouts():
    k, s = torch.zeros(4, 2, 16, 64, dtype=torch.uint8), torch.ones(4, 2)
    c = KVCache(k, k.clone(), s, s.clone())
    assert (c.num_pages, c.num_heads, c.page_size, c.head_dim) == (4, 2, 16, 64)
    assert KVCache.empty(3, 2, 128, 32, device='cpu').k_pages.dtype == torch.float8_e4m3fn
    for bad in ((k[0], k[0], s, s), (k, k[:3], s, s), (k, k, s[:3], s), (k, k, s.double(), s), (k.float(), k, s, s),
                (k[:, :, :8], k[:, :, :8], s, s), (k[..., :32], k[..., :32], s, s), (k.transpose(0, 1), k.transpose(0, 1), s.T, s.T),
                (k[:0], k[:0], s[:0], s[:0]), (torch.zeros(4, 2, 64, 16, dtype=torch.uint8).transpose(2, 3),) * 2 + (s, s)):
        with pytest.raises(ValueError, match='KVCache'):
            KVCache(*bad)


def test_operators_refuse_cpu_tensors():
    c = KVCache.empty(3, 2, 64, 16, device='cpu')
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match='CUDA'):
        attention_prompt(x, x, x, i32([0, 4]))
    with pytest.raises(RuntimeError, match='CUDA'):
        kv_cache_append(c, x, x, i32([[0]]), i32([4]), i32([0, 4]))
    with pytest.raises(RuntimeError, match='CUDA'):
        kv_cache_gather(c, i32([[0]]), i32([0]), i32([0, 4]), 4)
    with pytest.raises(RuntimeError, match='CUDA'):
        attention_cached(x[None], c, i32([[0]]), i32([4]))


def test_index_and_rows():
    assert _int32(torch.tensor([1, 2]), (2,), 'x', 'y', -1).dtype == torch.int32
    for bad in (torch.zeros(3), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int16)):
        with pytest.raises(ValueError, match='x: y'):
            _int32(bad, (3,), 'x', 'y', -1)
    with pytest.raises(ValueError, match='device 0'):
        _int32(i32([1, 2]), (2,), 'x', 'y', 0)
    x = torch.zeros(10, 6, 64, dtype=torch.bfloat16)
    rows = lambda t: _rows(t)[0]  # noqa: E731
    assert rows(x[:, 2:4]).data_ptr() == x[:, 2:4].data_ptr()
    assert rows(x[..., 1:]).is_contiguous() and rows(x.transpose(1, 2)).is_contiguous()
    assert rows(x[:, :1].expand(10, 3, 64)).is_contiguous()
    odd = torch.zeros(10 * 64 + 1, dtype=torch.bfloat16)[1:].view(10, 1, 64)    # contiguous, 2 bytes off
    assert rows(odd).data_ptr() % 16 == 0 and rows(odd[None]).data_ptr() % 16 == 0
    t, ptr, strides = _rows(x[:, 1:, ::2])
    assert t.is_contiguous() and strides == t.stride() and ptr == t.data_ptr()


def test_check_tables():
    c = KVCache.empty(4, 1, 64, 16, device='cpu')
    check_tables(c, i32([[0, 1], [2, -1]]), i32([32, 16]))
    check_tables(c, i32([[0, -1]]), i32([0]))
    check_tables(c, i32([[-1, 1]]), i32([20]), first=i32([16]))
    for table, last, first in (([[0, 1]], [33], None), ([[0, 4]], [17], None), ([[0, -1]], [17], None), ([[0, 1]], [-1], None),
                               ([[0, 1]], [3], i32([-1]))):
        with pytest.raises(ValueError):
            check_tables(c, i32(table), i32(last), first=first)
    with pytest.raises(ValueError, match='twice'):
        check_tables(c, i32([[0, 1], [1, 0]]), i32([17, 17]), first=i32([16, 16]) - 1, unique=True)


def test_c_entries_refuse():
    L = _lib.lib()
    cache = lambda **kw: _lib.KvCacheArgs(**{**dict(k_pages=16, v_pages=16, k_scale=16, v_scale=16, num_pages=4, H=2, page=16,  # noqa: E731
                                                   D=64), **kw})
    tables = dict(page_table=16, lengths=16, max_pages=4, B=1)

    def app(c=None, **kw):
        a = dict(cache=c or cache(), k=16, v=16, cu_new=16, k_token_stride=64, v_token_stride=64, T=1, **tables)
        return L.kb200_kv_append(ctypes.byref(_lib.KvAppendArgs(**{**a, **kw})), None)
    assert app(T=0) == 0 and app(B=0) == 0
    for bad in (dict(D=96), dict(page=8), dict(page=48), dict(H=0), dict(num_pages=0), dict(k_pages=0), dict(num_pages=1 << 40)):
        assert app(cache(**bad)) == 1, bad
    assert app(cache(k_pages=8)) == 2 and app(k=24) == 2 and app(k_token_stride=65) == 2
    assert app(dtype=2) == 1 and app(T=-1) == 1 and app(k=None) == 1 and app(lengths=None) == 1
    assert L.kb200_kv_append(None, None) == 1 and L.kb200_kv_gather(None, None) == 1 and L.kb200_attn_cached_fwd(None, None) == 1

    def gather(**kw):
        a = dict(cache=cache(), k=16, v=16, page_table=16, starts=16, cu=16, max_pages=4, B=1, T=5)
        return L.kb200_kv_gather(ctypes.byref(_lib.KvGatherArgs(**{**a, **kw})), None)
    assert gather(T=0, k=None) == 0 and gather(k=None) == 1 and gather(k=24) == 2 and gather(dtype=3) == 1

    size = lambda *a: L.kb200_attn_cached_workspace_size(*a)  # noqa: E731
    assert size(1, 1, 8, 2, 64, 16, 4) > 0 and size(1, 1, 7, 2, 64, 16, 4) == 0 and size(-1, 1, 8, 2, 64, 16, 4) == 0

    def att(**kw):
        a = dict(cache=cache(), q=16, o=16, q_batch_stride=64, q_token_stride=64, q_head_stride=64, Sq=1, Hq=4, softmax_scale=1.0,
                 **tables)
        return L.kb200_attn_cached_fwd(ctypes.byref(_lib.AttnCachedArgs(**{**a, **kw})), None)
    assert att(B=0) == 0 and att(Hq=3) == 1 and att(dtype=5) == 1 and att(q=None) == 1 and att(q=8) == 2
    assert att(q_head_stride=4) == 2
    assert att() == 3 and b'workspace' in L.kb200_last_error()
    assert att(workspace=16, workspace_bytes=64) == 3
    base = dict(q=16, k=16, v=16, o=16, cu_q=16, cu_k=16, Tq=4, Tk=4, N=1, Hq=4, Hkv=2, D=64, q_token_stride=64, softmax_scale=1.0)
    pr = lambda **kw: L.kb200_attn_prompt_fwd(ctypes.byref(_lib.PromptArgs(**{**base, **kw})), None)  # noqa: E731
    assert pr(N=0) == 0 and pr(Tq=0) == 0
    for bad in (dict(D=96), dict(Hq=3), dict(Hkv=0), dict(Tq=-1), dict(dtype=2), dict(q=None), dict(k=None), dict(cu_k=None)):
        assert pr(**bad) == 1, bad
    assert pr(v=8) == 2 and pr(o_head_stride=4) == 2
    for scale in (float('nan'), float('inf'), -float('inf')):
        assert pr(softmax_scale=scale) == 1 and att(softmax_scale=scale) == 1, scale
    assert pr(N=1 << 20, Hq=32, Hkv=32) == 1 and pr(N=(1 << 20) + 1) == 1


def test_oracle_rounds_as_torch_does():
    x = torch.cat([torch.linspace(-448, 448, 20001), torch.linspace(-0.05, 0.05, 4001), 2.0 ** torch.linspace(-12, 8, 999)])
    assert torch.equal(ref.round_e4m3(x).float(), x.to(torch.float8_e4m3fn).float())
    a = torch.tensor([0.0, 448.0, 448.5, 3.5, 3.51, 1e-30, 1.0])
    assert torch.equal(ref.scale_exponent(a), torch.tensor([-117, 0, 1, -7, -6, -108, -8], dtype=torch.int32))


def test_oracle_attention_is_the_formula():
    torch.manual_seed(0)
    q, k, v = torch.randn(3, 8), torch.randn(5, 8), torch.randn(5, 8)
    o, lse, A = ref.attend(q, k, v, torch.tensor([0, 2, 5]), 0.5)
    assert (o[0] == 0).all() and lse[0] == -float('inf')
    for i, n in ((1, 2), (2, 5)):
        w = torch.softmax(q[i].double() @ k[:n].double().T * 0.5, 0)
        assert torch.allclose(o[i], w @ v[:n].double()) and torch.allclose(A[i], w @ v[:n].double().abs())
    v[4] = float('nan')
    o2 = ref.attend(q, k, v, torch.tensor([0, 2, 5]), 0.5)[0]
    assert torch.equal(o2[:2], o[:2]) and torch.isnan(o2[2]).all()


def test_prompt_wait_bound():
    """The bound of a device-side wait: 0 (the default) to 4e9 clocks."""
    L = _lib.lib()
    base = dict(q=16, k=16, v=16, o=16, cu_q=16, cu_k=16, Tq=4, Tk=4, N=1, Hq=4, Hkv=2, D=64, q_token_stride=64, softmax_scale=1.0)
    for bad in (-1, 4_000_000_001):
        assert L.kb200_attn_prompt_fwd(ctypes.byref(_lib.PromptArgs(**base, wait_clocks=bad)), None) == 1
        assert b'wait_clocks' in L.kb200_last_error()


def test_cache_follows_its_tensors():
    """Addresses are those of the tensors at the call: a storage that is freed is refused, a moved one is followed, one of another
    layout is checked again."""
    k, s = torch.zeros(4, 2, 16, 64, dtype=torch.uint8), torch.ones(4, 2)
    tensors = [k, k.clone(), s, s.clone()]
    c = KVCache(*tensors)
    at = lambda: _lib.KV_CACHE_ARGS.unpack(c._args)  # noqa: E731
    assert at() == (*(t.data_ptr() for t in tensors), 4, 2, 16, 64)
    tensors[1].set_(torch.zeros(4, 2, 16, 64, dtype=torch.uint8))
    tensors[2].data = torch.ones(4, 2)
    c._look()
    assert at() == (*(t.data_ptr() for t in tensors), 4, 2, 16, 64)
    size = tensors[0].untyped_storage().nbytes()
    tensors[0].untyped_storage().resize_(0)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: kv_cache_append(c, x, x, i32([[0]]), i32([4]), i32([0, 4])), lambda: attention_cached(x[None], c, i32([[0]]), i32([4])),
                 lambda: kv_cache_gather(c, i32([[0]]), i32([0]), i32([0, 4]), 4)):
        with pytest.raises(ValueError, match='freed'):
            call()
    tensors[0].untyped_storage().resize_(size)
    c._look()
    assert at()[0] == tensors[0].data_ptr() != 0
    tensors[3].data = torch.ones(3, 2)
    with pytest.raises(ValueError, match='scales must be'):
        c._look()


def test_imports_without_cuda():
    """The package imports, and its host parts work, on a torch built without CUDA."""
    import subprocess
    import sys
    code = """
import torch
import torch._dynamo            # (torch's own modules of a build with CUDA take these names too)
for name in ('_cuda_getDevice', '_cuda_getCurrentRawStream'):
    delattr(torch._C, name)
from kairos_sensenova_b200 import KVCache, attention_cached
c = KVCache.empty(3, 2, 64, 16, device='cpu')
try:
    attention_cached(torch.zeros(1, 1, 2, 64).bfloat16(), c, torch.zeros(1, 1).int(), torch.zeros(1).int())
except RuntimeError as e:
    assert 'CUDA' in str(e)
    print('refused')
"""
    r = subprocess.run([sys.executable, '-c', code], capture_output=True, text=True, timeout=200)
    assert r.returncode == 0 and 'refused' in r.stdout, r.stderr[-2000:]


def test_derivatives_are_refused():
    """Autograd's leaves and forward-mode duals; nothing is refused where no derivative is asked for."""
    from torch.autograd import forward_ad
    x = torch.zeros(3)
    leaf = torch.zeros(3, requires_grad=True)
    _refuse_grad('op', x, x)
    with torch.no_grad():
        _refuse_grad('op', x, leaf)
    with pytest.raises(NotImplementedError, match='op is forward-only'):
        _refuse_grad('op', x, leaf)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        _refuse_grad('op', x)
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match='op is forward-only'):
                _refuse_grad('op', x, dual)


def test_copies_of_a_cache():
    """A deep copy and an unpickled cache have tensors and addresses of their own; a shallow copy has the same ones."""
    import copy
    import pickle
    pages, scale = torch.zeros(3, 2, 16, 64, dtype=torch.uint8), torch.ones(3, 2)    # (this torch pickles no float8 tensors)
    c = KVCache(pages, pages.clone(), scale, scale.clone())
    c.k_scale.fill_(4.0)
    for d, same in ((copy.deepcopy(c), False), (pickle.loads(pickle.dumps(c)), False), (copy.copy(c), True)):
        assert d.k_pages.shape == c.k_pages.shape and (d.k_scale == 4.0).all()
        at = _lib.KV_CACHE_ARGS.unpack(d._args)[:4]
        assert at == tuple(t.data_ptr() for t in (d.k_pages, d.v_pages, d.k_scale, d.v_scale))
        assert all((t.data_ptr() == u.data_ptr()) == same for t, u in zip(d._tensors, c._tensors))
        d._look()
        assert _lib.KV_CACHE_ARGS.unpack(d._args)[:4] == at
