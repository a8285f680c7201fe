// attn_prompt.cu -- causal softmax attention over packed prompts with grouped heads.
//
//   o_i = sum_{j <= i + m - n} softmax_j(scale q_i . k_j) v_j     (n queries at the end of m keys)
//
// One warp per (query token, head): the keys one after the other, the running maximum
// and sum of the softmax in fp32, D / 32 channels per lane.
#include "kb200_internal.h"
#include "kv_cache.cuh"

namespace kb {
namespace prompt {

struct Params {
  const void *q, *k, *v;
  void* o;
  float* lse;
  const int32_t *cu_q, *cu_k;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;
  int64_t Tq, Tk;
  int N, Hq, H, G;
  float scale_log2;
  int causal;
};

KB_DEVI float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// [start, end) of sequence s in the packed tokens, inside [0, T].
KB_DEVI int2 seq_range(const int32_t* cu, int s, int64_t T) {
  const int64_t a = min(max((int64_t)cu[s], (int64_t)0), T), b = min(max((int64_t)cu[s + 1], a), T);
  return make_int2((int)a, (int)b);
}

template <bool F16>
KB_DEVI float load16(const void* base, int64_t i) {
  if constexpr (F16) return __half2float(reinterpret_cast<const __half*>(base)[i]);
  else return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[i]);
}
template <bool F16>
KB_DEVI void store16(void* base, int64_t i, float x) {
  if constexpr (F16) reinterpret_cast<__half*>(base)[i] = __float2half_rn(x);
  else reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(x);
}

// Query token `tq` of head `h`, which sees the keys [k0, k0 + seen), by one warp.
template <int D, bool F16>
KB_DEVI void attend_row(const Params& p, int64_t tq, int h, int64_t k0, int64_t seen, int lane) {
  constexpr int C = D / 32;
  const int hk = h / p.G;
  float q[C], acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    q[c] = load16<F16>(p.q, tq * p.q_ts + h * p.q_hs + c * 32 + lane) * p.scale_log2;
    acc[c] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j = 0; j < seen; ++j) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) s = fmaf(q[c], load16<F16>(p.k, (k0 + j) * p.k_ts + hk * p.k_hs + c * 32 + lane), s);
    s = warp_sum(s);
    const float mn = fmaxf(m, s);
    if (mn > m) {
      const float a = ex2(m - mn);
      l *= a;
#pragma unroll
      for (int c = 0; c < C; ++c) acc[c] *= a;
      m = mn;
    }
    const float e = s == -INFINITY ? 0.f : ex2(s - m);
    l += e;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = fmaf(e, load16<F16>(p.v, (k0 + j) * p.v_ts + hk * p.v_hs + c * 32 + lane), acc[c]);
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) store16<F16>(p.o, tq * p.o_ts + h * p.o_hs + c * 32 + lane, acc[c] * inv);
  if (lane == 0 && p.lse) p.lse[tq * p.Hq + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

template <int D, bool F16>
__global__ void __launch_bounds__(256) attn_prompt_rows_kernel(Params p) {
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t tq = w / p.Hq;
  if (tq >= p.Tq || tq < p.cu_q[0] || tq >= p.cu_q[p.N]) return;
  const int s = kv::find_sequence(p.cu_q, p.N, tq);
  const int2 rq = seq_range(p.cu_q, s, p.Tq), rk = seq_range(p.cu_k, s, p.Tk);
  const int64_t m = rk.y - rk.x, i = tq - rq.x;
  const int64_t seen = p.causal ? min(m, max((int64_t)0, i + 1 + m - (rq.y - rq.x))) : m;
  attend_row<D, F16>(p, tq, (int)(w % p.Hq), rk.x, seen, lane);
}

}  // namespace prompt
}  // namespace kb

extern "C" int kb200_attn_prompt_fwd(const KB200PromptArgs* a, void* stream) {
  using namespace kb;
  if (!a) return set_error(KB200_ERR_INVALID, "attn_prompt: null arguments");
  if (a->N < 0 || a->Tq < 0 || a->Tk < 0 || a->N > (1 << 20) || a->Tq > 0x7fffff00LL || a->Tk > 0x7fffff00LL || a->Hq < 1 ||
      a->Hkv < 1 || a->Hq % a->Hkv || a->Hq > (1 << 16) || (a->dtype != 0 && a->dtype != 1))
    return set_error(KB200_ERR_INVALID, "attn_prompt: N=%lld Tq=%lld Tk=%lld Hq=%lld Hkv=%lld dtype=%d", (long long)a->N,
                     (long long)a->Tq, (long long)a->Tk, (long long)a->Hq, (long long)a->Hkv, a->dtype);
  if (a->D != 64 && a->D != 128) return set_error(KB200_ERR_INVALID, "attn_prompt: head dim %lld (64 or 128)", (long long)a->D);
  if (a->N == 0 || a->Tq == 0) return KB200_OK;
  if (!a->q || !a->o || !a->cu_q || !a->cu_k || (a->Tk > 0 && (!a->k || !a->v)))
    return set_error(KB200_ERR_INVALID, "attn_prompt: null pointer");
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->o) ||
      ((a->q_token_stride | a->q_head_stride | a->k_token_stride | a->k_head_stride | a->v_token_stride | a->v_head_stride |
        a->o_token_stride | a->o_head_stride) & 7))
    return set_error(KB200_ERR_ALIGN, "attn_prompt: q, k, v and o rows must be 16-byte aligned");
  prompt::Params p{a->q, a->k, a->v, a->o, a->lse, a->cu_q, a->cu_k, a->q_token_stride, a->q_head_stride,
                   a->k_token_stride, a->k_head_stride, a->v_token_stride, a->v_head_stride, a->o_token_stride,
                   a->o_head_stride, a->Tq, a->Tk, (int)a->N, (int)a->Hq, (int)a->Hkv, (int)(a->Hq / a->Hkv),
                   a->softmax_scale * 1.4426950408889634f, a->causal};
  cudaStream_t st = (cudaStream_t)stream;
  const unsigned grid = (unsigned)((a->Tq * a->Hq + 7) / 8);
  if (a->D == 64) {
    if (a->dtype) prompt::attn_prompt_rows_kernel<64, true><<<grid, 256, 0, st>>>(p);
    else prompt::attn_prompt_rows_kernel<64, false><<<grid, 256, 0, st>>>(p);
  } else {
    if (a->dtype) prompt::attn_prompt_rows_kernel<128, true><<<grid, 256, 0, st>>>(p);
    else prompt::attn_prompt_rows_kernel<128, false><<<grid, 256, 0, st>>>(p);
  }
  return check_launch("attn_prompt_rows_kernel");
}
