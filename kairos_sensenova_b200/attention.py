"""FP8 attention module with the reference's ``AttentionModule`` interface.

``AttentionModule(num_heads).forward(q, k, v, attn_mask=None, window_size=(-1, -1))``
with q, k, v ``[B, S, N*D]`` bf16 returns ``[B, S, N*D]`` bf16
(``kairos/modules/dits/kairos_dit.py:362-373``).  The core is computed by the
sm_100a kernels behind ``kb200_attn_fp8_fwd``: per-(batch, head) amax scaling
of q/k to e4m3, non-causal softmax(q k^T / sqrt(D)) v with fp32 softmax and
accumulation; the P.V half runs on bf16 probabilities and the bf16 V (with P
and V in e4m3 too, the cosine similarity to the bf16 reference would sit near
0.9986 on N(0,1) data, below the 0.999 contract; this way it is ~0.9992).  Like the reference's
quantised backends (``SageAttention3Module``, ``kairos_dit.py:398-420``) it
raises ``NotImplementedError`` for an ``attn_mask``.  A sliding ``window_size``
(left, right) restricts query i to keys i - left .. i + right, as the reference's
flash-attention call does for ``SelfAttention`` (``kairos_dit.py:423-507``; its
dilation is a rearrangement before this call); key tiles outside every window of a
256-query block are skipped.
"""
from __future__ import annotations

import functools

import torch
import torch.nn as nn

from . import _lib
from .kv_cache import _DTYPES, _forward_ad, _int32, _launch, _refuse_grad, _rows


def attention_fp8(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, num_heads: int,
                  softmax_scale: float | None = None,
                  events=None, check: bool = False, window_size=(-1, -1)) -> torch.Tensor:
    """q, k, v: [B, S, H*D] (bf16; other float dtypes are converted) -> [B, S, H*D] bf16.

    ``events``: optional (start, end) CUDA events recorded on the launch stream
    around the attention kernel alone (after quantisation).  ``window_size``:
    (left, right) sliding window as in flash-attention (query i sees keys
    i - left .. i + right; -1 = unbounded)."""
    if q.device.type != 'cuda':
        raise RuntimeError('attention_fp8: inputs must be CUDA tensors (no CPU path)')
    if q.dim() != 3 or k.shape != q.shape or v.shape != q.shape:
        raise ValueError(f'attention_fp8: q/k/v must share shape [B,S,H*D], got {tuple(q.shape)}, '
                         f'{tuple(k.shape)}, {tuple(v.shape)}')
    B, S, HD = q.shape
    if HD % num_heads:
        raise ValueError(f'attention_fp8: hidden {HD} not divisible by num_heads {num_heads}')
    D = HD // num_heads
    if softmax_scale is None:
        softmax_scale = D ** -0.5
    dev = q.device
    with torch.cuda.device(dev):
        qc, kc, vc = (x.to(torch.bfloat16) for x in (q, k, v))
        ld = qc.stride(1)
        # strided row views (e.g. column slices of one projection) are read in place
        if not all(t.stride(2) == 1 and t.stride(1) == ld and (B == 1 or t.stride(0) == S * ld)
                   and t.data_ptr() % 16 == 0 for t in (qc, kc, vc)) or ld % 8:
            qc, kc, vc = (t.contiguous() for t in (qc, kc, vc))
            ld = HD
        o = torch.empty(B, S, HD, device=dev, dtype=torch.bfloat16)
        L = _lib.lib()
        nbytes = L.kb200_attn_fp8_workspace_size(B, S, num_heads, D)
        if nbytes == 0:
            raise ValueError(f'attention_fp8: unsupported shape B={B} S={S} H={num_heads} D={D} (D must be 128)')
        ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
        stream = torch.cuda.current_stream(dev).cuda_stream
        args = (qc.data_ptr(), kc.data_ptr(), vc.data_ptr(), o.data_ptr(), B, S, num_heads, D, ld,
                float(softmax_scale), ws.data_ptr(), nbytes, stream)
        wl, wr = (int(x) for x in window_size)
        windowed = wl >= 0 or wr >= 0
        if events is None:
            if windowed:
                _lib.check(L.kb200_attn_fp8_fwd_window(*args, wl, wr), 'attention_fp8')
            else:
                _lib.check(L.kb200_attn_fp8_fwd(*args), 'attention_fp8')
        else:
            _lib.check(L.kb200_attn_fp8_quantize(*args), 'attention_fp8 quantize')
            events[0].record()
            if windowed:
                _lib.check(L.kb200_attn_fp8_attend_window(*args, wl, wr), 'attention_fp8 attend')
            else:
                _lib.check(L.kb200_attn_fp8_attend(*args), 'attention_fp8 attend')
            events[1].record()
        if check:   # synchronises; raises if a bounded device wait gave up
            _lib.check(L.kb200_attn_fp8_status(ws.data_ptr(), B, S, num_heads, stream),
                       'attention_fp8')
    return o


class AttentionModule(nn.Module):
    """Drop-in for ``AttentionModule`` / ``SageAttention3Module`` (``kairos_dit.py:362-420``)."""

    def __init__(self, num_heads):
        super().__init__()
        self.num_heads = num_heads

    def forward(self, q, k, v, attn_mask=None, window_size=(-1, -1)):
        if attn_mask is not None:
            raise NotImplementedError('FP8 attention path does not support arbitrary attn_mask')
        return attention_fp8(q, k, v, self.num_heads, window_size=window_size)


FP8AttentionModule = AttentionModule


@functools.lru_cache(maxsize=256)
def _prompt_workspace(device_index, *sizes):
    """Workspace bytes for these sizes (they depend on the device's number of SMs)."""
    with torch.cuda.device(device_index):
        return _lib.lib().kb200_attn_prompt_workspace_size(*sizes)


def attention_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                     cu_seqlens_k: torch.Tensor | None = None, softmax_scale: float | None = None,
                     causal: bool = True, out: torch.Tensor | None = None, return_lse: bool = False, check: bool = False):
    """Causal attention over packed prompts with grouped heads, bf16 or fp16, forward.

    ``q``: ``[Tq, Hq, D]``, ``k``, ``v``: ``[Tk, Hkv, D]`` of one type, D 64 or 128, Hq a multiple
    of Hkv (query head h reads kv head ``h // (Hq / Hkv)``); views of a fused projection are
    read in place.  Sequence s has query rows ``cu_seqlens_q[s] .. [s+1]`` and key rows
    ``cu_seqlens_k[s] .. [s+1]`` (int32 on the device; default: the same).  With n queries and m
    keys the queries are the last n of the m tokens: query i sees the first ``i + 1 + m - n``
    keys (``causal=False``: all m).  A query that sees none gets 0; the values of keys that a
    query does not see never reach it, NaN and infinities included; V may be as large as the type allows (up to 256
    such bf16 keys; O is summed in fp32), and scores (scale q . k) up to 2^22 in magnitude (past that fp32's steps exceed what a
    probability bears, and results are not defined).  Returns ``[Tq, Hq, D]``
    (``out``: to write into, apart from the inputs; rows behind the last sequence are left as they
    were); with ``return_lse`` also the fp32 log of the softmax sum ``[Tq, Hq]``.  ``check=True``
    looks at the offsets on the host first (it synchronises) and raises ``ValueError``, and ``RuntimeError`` if a device-side
    wait gave up (without it such rows are NaN)."""
    what = 'attention_prompt'
    index = q.get_device()
    if index < 0:
        raise RuntimeError(f'{what}: inputs must be CUDA tensors (no CPU path)')
    shape, kshape, qd = q.shape, k.shape, q.dtype
    if len(shape) != 3 or len(kshape) != 3 or v.shape != kshape or kshape[2] != shape[2] or kshape[1] < 1 \
            or shape[1] < 1 or shape[1] % kshape[1]:
        raise ValueError(f'{what}: q must be [Tq, Hq, D] and k, v [Tk, Hkv, D] with Hq a multiple of Hkv, got '
                         f'{tuple(shape)}, {tuple(kshape)}, {tuple(v.shape)}')
    dtype = _DTYPES.get(qd)
    if dtype is None or k.dtype is not qd or v.dtype is not qd:
        raise ValueError(f'{what}: q, k and v must all be bfloat16 or all float16, got {q.dtype}, {k.dtype}, {v.dtype}')
    if k.get_device() != index or v.get_device() != index:
        raise ValueError(f'{what}: q, k and v must be on one device')
    if q.requires_grad or k.requires_grad or v.requires_grad or _forward_ad._current_level >= 0:   # (-1: not in a dual_level)
        _refuse_grad(what, q, k, v)
    cu_q = _int32(cu_seqlens_q, (None,), what, 'cu_seqlens_q', index)
    N = cu_q.shape[0] - 1
    if N < 0:
        raise ValueError(f'{what}: cu_seqlens_q must be [N + 1], got [0]')
    cu_k = cu_q if cu_seqlens_k is None else _int32(cu_seqlens_k, (N + 1,), what, 'cu_seqlens_k', index)
    Tq, Hq, D = shape
    Tk, Hkv, _ = kshape
    if check:
        for name, cu, T in (('cu_seqlens_q', cu_q, Tq), ('cu_seqlens_k', cu_k, Tk)):
            at = cu.tolist()
            if at[0] != 0 or at[-1] > T or any(b < a for a, b in zip(at, at[1:])):
                raise ValueError(f'{what}: {name} must rise from 0 to at most {T}')
    q, qp, qs = _rows(q)
    k, kp, ks = _rows(k)
    v, vp, vs = _rows(v)
    if out is None:
        out = q.new_empty(shape)
        op, os = out.data_ptr(), (Hq * D, D)
    else:
        same, op, os = _rows(out)
        if out.shape != shape or out.dtype != qd or out.get_device() != index or same is not out:
            raise ValueError(f'{what}: out must be {q.dtype} {list(shape)} on {q.device}, its rows 16-byte aligned')
    lse = torch.empty((Tq, Hq), device=q.device, dtype=torch.float32) if return_lse else None
    nbytes = _prompt_workspace(index, Tq, Tk, N, Hq, Hkv, D)
    ws = cu_q.new_empty(nbytes >> 2) if nbytes else None
    status = cu_q.new_zeros(1) if check else None
    args = _lib.PROMPT_ARGS.pack(
        qp, kp, vp, op, lse.data_ptr() if return_lse else 0, cu_q.data_ptr(), cu_k.data_ptr(), Tq, Tk, N, Hq, Hkv, D,
        qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0], os[1], D ** -0.5 if softmax_scale is None else softmax_scale,
        1 if causal else 0, dtype, ws.data_ptr() if nbytes else 0, nbytes, status.data_ptr() if check else 0, 0)
    _launch(index, what, _lib.lib().kb200_attn_prompt_fwd, args)
    if check:
        _launch(index, what, _lib.lib().kb200_read_error_word, status.data_ptr())
    return (out, lse) if return_lse else out
