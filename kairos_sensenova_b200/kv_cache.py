"""The 8-bit paged key/value cache and the attention that reads it.

``layers.Cache`` carries the GatedDeltaNet layers' state from piece to piece; this is its
counterpart for softmax attention.  A :class:`KVCache` is a pool of pages of 16 to 128
tokens, e4m3 codes with one fp32 scale per (page, head) that is always a power of two;
the caller keeps the page table ``[B, max_pages]`` and the lengths ``[B]`` (int32, on the
device), so none of the calls waits for the host:

* :func:`kv_cache_append` quantises new tokens (whole prompts, pieces, single tokens,
  packed) into the pages;
* :func:`kv_cache_gather` gives a token range of each sequence back as packed K and V
  (the context of a prompt's next piece, for ``attention.attention_prompt``);
* :func:`attention_cached` attends the last token, or the last few, of each sequence to
  the cache.

A page table entry outside the pool is a page that is not there: nothing is written to
it, attention skips its tokens and a gather reads 0.  ``check=True`` looks at the lengths
and the table on the host first (it synchronises) and raises ``ValueError``.
"""
from __future__ import annotations

import functools

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_I32 = torch.int32
# (short ways to the current device and stream; a torch built without CUDA has neither, and needs none)
_get_device = getattr(torch._C, '_cuda_getDevice', None)
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)
PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)


class KVCache:
    """Pages of one attention layer: ``k_pages``, ``v_pages`` ``[num_pages, heads, page, D]``
    (``torch.float8_e4m3fn`` or ``uint8`` codes), ``k_scale``, ``v_scale`` ``[num_pages, heads]``
    fp32 powers of two, all contiguous.  A value is ``code * scale``."""

    __slots__ = ('_tensors', '_pointers', '_at', '_args', '_shape', '_row', '_device', '_index')

    def __init__(self, k_pages, v_pages, k_scale, v_scale):
        self._tensors, self._at = (k_pages, v_pages, k_scale, v_scale), None
        self._pointers = k_pages.data_ptr, v_pages.data_ptr, k_scale.data_ptr, v_scale.data_ptr
        self._look()

    def _look(self):
        """Takes the addresses, and all that is checked, from the tensors if they have moved since the last call
        (``set_``, ``.data =``, a storage that was freed and allocated again); returns the device's index."""
        k, v, ks, vs = self._pointers
        at = (k(), v(), ks(), vs())
        if at == self._at:
            return self._index
        k_pages, v_pages, k_scale, v_scale = self._tensors
        if k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
            raise ValueError(f'KVCache: k_pages and v_pages must share shape [pages, heads, page, D], got '
                             f'{tuple(k_pages.shape)}, {tuple(v_pages.shape)}')
        P, H, page, D = k_pages.shape
        if page not in PAGE_SIZES or D not in HEAD_DIMS:
            raise ValueError(f'KVCache: pages of {page} tokens and head dim {D}; supported are {PAGE_SIZES} and {HEAD_DIMS}')
        if P < 1 or H < 1:
            raise ValueError(f'KVCache: {P} pages of {H} heads')
        if k_scale.shape != (P, H) or v_scale.shape != (P, H):
            raise ValueError(f'KVCache: scales must be [{P}, {H}], got {tuple(k_scale.shape)}, {tuple(v_scale.shape)}')
        for t in (k_pages, v_pages):
            if t.dtype not in (torch.float8_e4m3fn, torch.uint8):
                raise ValueError(f'KVCache: pages must be float8_e4m3fn or uint8, got {t.dtype}')
        for t in (k_scale, v_scale):
            if t.dtype != torch.float32:
                raise ValueError(f'KVCache: scales must be float32, got {t.dtype}')
        for t in (k_pages, v_pages, k_scale, v_scale):
            if t.device != k_pages.device:
                raise ValueError('KVCache: pages and scales must be on one device')
            if not t.is_contiguous():
                raise ValueError('KVCache: pages and scales must be contiguous')
            # (3 us for the four: when they have moved, not for a new cache)
            if self._at and t.untyped_storage().nbytes() < (t.storage_offset() + t.numel()) * t.element_size():
                raise ValueError('KVCache: the storage of the pages or scales has been freed')
        self._shape, self._row, self._device = (P, H, page, D), (H, D), k_pages.device
        self._index = k_pages.get_device()              # -1 on the CPU
        self._args = _lib.KV_CACHE_ARGS.pack(*at, P, H, page, D)
        self._at = at
        return self._index

    def __reduce__(self):                               # (a copy, or an unpickled one, is of its own tensors)
        return KVCache, self._tensors

    @classmethod
    def empty(cls, num_pages: int, num_heads: int, head_dim: int, page_size: int = 64, device='cuda'):
        """A pool without tokens (codes 0, scales 1)."""
        codes = [torch.zeros(num_pages, num_heads, page_size, head_dim, device=device, dtype=torch.uint8)
                 .view(torch.float8_e4m3fn) for _ in range(2)]
        return cls(*codes, *(torch.ones(num_pages, num_heads, device=device) for _ in range(2)))

    k_pages = property(lambda self: self._tensors[0])
    v_pages = property(lambda self: self._tensors[1])
    k_scale = property(lambda self: self._tensors[2])
    v_scale = property(lambda self: self._tensors[3])
    num_pages = property(lambda self: self._shape[0])
    num_heads = property(lambda self: self._shape[1])
    page_size = property(lambda self: self._shape[2])
    head_dim = property(lambda self: self._shape[3])
    device = property(lambda self: self._device)


def _int32(t, shape, what, name, index):
    """`t` as a contiguous int32 tensor of that shape on device `index` (None: any extent)."""
    if t.dtype is _I32 and t.get_device() == index and t.shape == shape and t.is_contiguous():
        return t
    got = t.shape
    if got != shape and (len(got) != len(shape) or any([n != m and n is not None for n, m in zip(shape, got)])):
        raise ValueError(f'{what}: {name} must be {list(shape)}, got {tuple(got)}')
    if t.get_device() != index:
        raise ValueError(f'{what}: {name} must be on device {index}, got {t.device}')
    if t.dtype is not _I32:
        if t.dtype is not torch.int64:
            raise ValueError(f'{what}: {name} must be int32, got {t.dtype}')
        t = t.to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def _rows(t):
    """(tensor, address, strides) of `t` if its rows can be read in 16-byte steps in place, else of a contiguous copy."""
    strides, ptr = t.stride(), t.data_ptr()
    bits = ptr >> 1                                 # 16-byte aligned, strides positive multiples of 8, channels contiguous
    if len(strides) == 3:
        a, b, c = strides
        if not (bits | a | b) & 7 and c == 1 and a > 0 and b > 0:
            return t, ptr, strides
    else:
        a, b, c, d = strides
        if not (bits | a | b | c) & 7 and d == 1 and a > 0 and b > 0 and c > 0:
            return t, ptr, strides
    t = t.clone(memory_format=torch.contiguous_format)   # (contiguous() would keep an unaligned start)
    return t, t.data_ptr(), t.stride()


def _refuse_grad(what, *tensors):
    """Raises if a derivative with respect to one of `tensors` would be lost: by autograd, or a forward-mode tangent."""
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled() or \
                _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f'kairos_sensenova_b200.{what} is forward-only')


def _refuse_cpu(what):
    raise RuntimeError(f'{what}: the cache must be on a CUDA device (no CPU path)')


def _launch(index, what, fn, args):
    """``fn(args, stream)`` on device `index`'s current stream, with that the current device."""
    if index == _get_device():
        rc = fn(args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(args, _raw_stream(index))
    if rc:
        _lib.check(rc, what)


def _table(t, rows, what, index):
    """``(table, rows, max_pages)``: `t` as an int32 table ``[rows, max_pages]`` (rows None: any)."""
    if t.dtype is not _I32 or t.get_device() != index or not t.is_contiguous():
        t = _int32(t, (rows, None), what, 'page_table', index)
    shape = t.shape
    if len(shape) != 2 or (rows is not None and shape[0] != rows):
        raise ValueError(f'{what}: page_table must be {[rows, None]}, got {tuple(shape)}')
    return t, shape[0], shape[1]


def check_tables(cache: KVCache, page_table, last, what='kv_cache', first=None, unique=False):
    """Raises ``ValueError`` if tokens ``first[b] .. last[b]`` (default from 0) of a sequence lie
    outside its table row or on a page outside the pool; with ``unique`` also if two of
    those pages are the same.  Reads the tensors on the host."""
    table, last = page_table.tolist(), last.tolist()
    first = [0] * len(last) if first is None else first.tolist()
    seen = set()
    for b, (lo, hi) in enumerate(zip(first, last)):
        if lo < 0 or hi < lo or hi > len(table[b]) * cache.page_size:
            raise ValueError(f'{what}: sequence {b} has tokens {lo} .. {hi}, its table row holds '
                             f'{len(table[b]) * cache.page_size}')
        for pg in table[b][lo // cache.page_size:-(-hi // cache.page_size)] if hi > lo else ():
            if not 0 <= pg < cache.num_pages:
                raise ValueError(f'{what}: sequence {b} names page {pg} of a pool of {cache.num_pages}')
            if unique and pg in seen:
                raise ValueError(f'{what}: page {pg} would be written twice')
            seen.add(pg)


def kv_cache_append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, cu_seqlens: torch.Tensor, check: bool = False) -> None:
    """Quantise new tokens into their pages, in place.

    ``k``, ``v``: ``[T, heads, D]`` bf16 or fp16, the new tokens of all sequences packed
    (views of a fused projection are read in place); those of sequence b are rows
    ``cu_seqlens[b] .. cu_seqlens[b+1]`` and are the LAST tokens of its ``lengths[b]``
    (the lengths count them already).  A sequence whose tokens do not fit its table row
    is left out.  The scale of a page and head is the smallest power of two that holds the
    largest finite magnitude within e4m3's 448; when a later token needs a larger one, the
    codes already there are re-encoded (exact but for subnormals).  NaN and infinities
    are stored as NaN and set no scale; magnitudes over 1.875 * 2^15 (fp16) or 1.875 * 2^127 (bf16) are stored as that, so
    that they stay inside the type.  The pages a call writes must each belong to one
    sequence (``check=True`` raises otherwise)."""
    what = 'kv_cache_append'
    index = cache._look()
    if index < 0:
        _refuse_cpu(what)
    shape, kd = k.shape, k.dtype
    if len(shape) != 3 or shape[1:] != cache._row or v.shape != shape:
        raise ValueError(f'{what}: k and v must be {["T", *cache._row]}, got {tuple(k.shape)}, {tuple(v.shape)}')
    dtype = _DTYPES.get(kd)
    if dtype is None or v.dtype is not kd:
        raise ValueError(f'{what}: k and v must both be bfloat16 or float16, got {k.dtype}, {v.dtype}')
    if k.get_device() != index or v.get_device() != index:
        raise ValueError(f'{what}: k and v must be on {cache.device}')
    if k.requires_grad or v.requires_grad or _forward_ad._current_level >= 0:   # (-1: not in a dual_level)
        _refuse_grad(what, k, v)
    page_table, B, max_pages = _table(page_table, None, what, index)
    lengths = _int32(lengths, (B,), what, 'lengths', index)
    cu = _int32(cu_seqlens, (B + 1,), what, 'cu_seqlens', index)
    if check:
        check_tables(cache, page_table, lengths, what, lengths - (cu[1:] - cu[:-1]), unique=True)
        if int(cu[0]) != 0 or int(cu[-1]) > shape[0]:
            raise ValueError(f'{what}: cu_seqlens runs from {int(cu[0])} to {int(cu[-1])}, there are {shape[0]} tokens')
    k, kp, ks = _rows(k)
    v, vp, vs = _rows(v)
    _launch(index, what, _lib.lib().kb200_kv_append, cache._args + _lib.KV_APPEND_ARGS.pack(
        kp, vp, page_table.data_ptr(), lengths.data_ptr(), cu.data_ptr(), ks[0], ks[1], vs[0], vs[1], max_pages, B,
        shape[0], dtype))


def kv_cache_gather(cache: KVCache, page_table: torch.Tensor, starts: torch.Tensor, cu_seqlens: torch.Tensor, total: int,
                    dtype: torch.dtype = torch.bfloat16, out=None, check: bool = False):
    """Tokens ``starts[b] ..`` of each sequence, ``cu_seqlens[b+1] - cu_seqlens[b]`` of them, as
    packed ``(k, v)`` ``[total, heads, D]`` in ``dtype`` (bf16: exact; fp16: rounded under 2^-14, infinities past 65504,
    which tokens appended in fp16 do not reach).  ``total`` is known to
    the host (``cu_seqlens[-1]``, or more: rows behind it are left as they were).  ``out``:
    ``(k, v)`` to write into, contiguous."""
    what = 'kv_cache_gather'
    index = cache._look()
    if index < 0:
        _refuse_cpu(what)
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f'{what}: dtype must be bfloat16 or float16, got {dtype}')
    page_table, B, max_pages = _table(page_table, None, what, index)
    starts = _int32(starts, (B,), what, 'starts', index)
    cu = _int32(cu_seqlens, (B + 1,), what, 'cu_seqlens', index)
    shape = (int(total), *cache._row)
    if shape[0] < 0:
        raise ValueError(f'{what}: total {total}')
    if check:
        check_tables(cache, page_table, starts + cu[1:] - cu[:-1], what, starts)
        if int(cu[0]) != 0 or int(cu[-1]) > shape[0]:
            raise ValueError(f'{what}: cu_seqlens runs from {int(cu[0])} to {int(cu[-1])}, total is {shape[0]}')
    if out is None:
        k = torch.empty(shape, device=cache._device, dtype=dtype)
        v = torch.empty_like(k)
    else:
        k, v = out
        for t in (k, v):
            if t.shape != shape or t.dtype != dtype or t.get_device() != index or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f'{what}: out must be contiguous 16-byte aligned {dtype} {list(shape)} on {cache.device}')
    _launch(index, what, _lib.lib().kb200_kv_gather, cache._args + _lib.KV_GATHER_ARGS.pack(
        k.data_ptr(), v.data_ptr(), page_table.data_ptr(), starts.data_ptr(), cu.data_ptr(), max_pages, B, shape[0], code))
    return k, v


@functools.lru_cache(maxsize=256)
def _cached_workspace(device_index, *sizes):
    """Workspace bytes for these sizes (they depend on the device's number of SMs)."""
    with torch.cuda.device(device_index):
        n = _lib.lib().kb200_attn_cached_workspace_size(*sizes)
    if n == 0:
        _lib.check(1, 'attention_cached')
    return -(-n // 16) * 16


def attention_cached(q: torch.Tensor, cache: KVCache, page_table: torch.Tensor, lengths: torch.Tensor,
                     softmax_scale: float | None = None, out: torch.Tensor | None = None, return_lse: bool = False,
                     check: bool = False):
    """Attention of the last Sq tokens of each sequence over its cached tokens.

    ``q``: ``[B, Sq, Hq, D]`` bf16 or fp16 (Hq a multiple of the cache's heads; query head h
    reads kv head ``h // (Hq / heads)``); ``lengths[b]`` counts the cached tokens, the Sq
    themselves included, and query i sees the first ``lengths[b] - Sq + 1 + i`` of them.  A
    query that sees none (an idle slot of length 0) gets 0.  Returns ``[B, Sq, Hq, D]`` in
    q's type (``out``: contiguous, to write into, apart from the inputs); with ``return_lse`` also the fp32 log of
    the softmax sum ``[B, Sq, Hq]`` (-inf where nothing is seen).  Scores (scale q . k) may reach 2^22 in magnitude; past that
    fp32's steps exceed what a probability bears, and results are not defined.  Probabilities are rounded to fp16: 2^-11 of
    themselves, or 2^-33 of the row's largest where they are under 2^-22 of it."""
    what = 'attention_cached'
    index = cache._look()
    if index < 0:
        _refuse_cpu(what)
    _, H, page, D = cache._shape
    shape = q.shape
    if len(shape) != 4 or shape[3] != D or shape[2] < 1 or shape[2] % H:
        raise ValueError(f'{what}: q must be [B, Sq, Hq, {D}] with Hq a multiple of {H}, got {tuple(shape)}')
    dtype = _DTYPES.get(q.dtype)
    if dtype is None:
        raise ValueError(f'{what}: q must be bfloat16 or float16, got {q.dtype}')
    if q.get_device() != index:
        raise ValueError(f'{what}: q must be on {cache.device}, got {q.device}')
    if q.requires_grad or _forward_ad._current_level >= 0:
        _refuse_grad(what, q)
    B, Sq, Hq, _ = shape
    page_table, _, max_pages = _table(page_table, B, what, index)
    lengths = _int32(lengths, (B,), what, 'lengths', index)
    if check:
        check_tables(cache, page_table, lengths, what)
    q, qp, qs = _rows(q)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    elif out.shape != shape or out.dtype != q.dtype or out.get_device() != index or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f'{what}: out must be contiguous 16-byte aligned {q.dtype} {list(shape)} on {cache.device}')
    lse = torch.empty(shape[:3], device=cache._device, dtype=torch.float32) if return_lse else None
    nbytes = _cached_workspace(index, B, Sq, Hq, H, D, page, max_pages)
    ws = lengths.new_empty(nbytes >> 2)
    _launch(index, what, _lib.lib().kb200_attn_cached_fwd, cache._args + _lib.ATTN_CACHED_ARGS.pack(
        qp, out.data_ptr(), lse.data_ptr() if return_lse else 0, page_table.data_ptr(), lengths.data_ptr(), ws.data_ptr(),
        nbytes, qs[0], qs[1], qs[2], max_pages, B, Sq, Hq, D ** -0.5 if softmax_scale is None else softmax_scale, dtype))
    return (out, lse) if return_lse else out
