// kv_cache.cu -- filling and reading the 8-bit paged key/value cache (layout: kv_cache.cuh).
#include "kv_cache.cuh"

namespace kb {
namespace kv {

struct AppendParams {
  uint8_t *k_pages, *v_pages;
  float *k_scale, *v_scale;
  const void *k, *v;
  int64_t k_ts, k_hs, v_ts, v_hs;   // token and head strides, elements
  const int32_t *table, *lengths, *cu;
  int num_pages, H, max_pages, B;
  int64_t T;
};

// New tokens into their pages.  A unit is one page that a sequence writes; the new
// tokens of sequence b are the last cu[b+1] - cu[b] of its lengths[b] tokens.
// Sequence b owns the units [cu[b] / page + 2 b, ...): it touches at most
// n / page + 2 pages, so the ranges do not overlap and a unit finds its sequence by
// binary search, without a table and without the host knowing the lengths.
//
// Per (unit, head, k or v) one group of page * D / 32 threads holds the page's new
// values in registers (32 each), so that they are read once: amax over the group,
// exponent, codes.  Tokens that were in the page before keep their codes unless the
// exponent grows; then they are re-encoded under the new one.
// Bound: HBM.  2 B read and 1 B written per value.
template <int D, int PAGE, bool F16>
__global__ void __launch_bounds__(PAGE * D / 32 > 256 ? 512 : 256) kv_append_kernel(AppendParams p) {
  constexpr int GROUP = PAGE * D / 32;                 // threads of one (unit, head, k|v)
  constexpr int THREADS = GROUP > 256 ? GROUP : 256;
  constexpr int PER_BLOCK = THREADS / GROUP;
  constexpr int CPT = D / 8;                           // 8-value chunks of a token
  __shared__ float wmax[THREADS / 32];
  const int grp = threadIdx.x / GROUP, t = threadIdx.x % GROUP;
  const int item = blockIdx.y * PER_BLOCK + grp;       // (head, k|v)
  const bool is_v = item & 1;
  const int h = item >> 1;
  const int64_t unit = blockIdx.x;

  // the unit's sequence: largest b with cu[b] / PAGE + 2 b <= unit
  int lo = 0, hi = p.B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int64_t)max(0, p.cu[mid]) / PAGE + 2 * mid <= unit) lo = mid; else hi = mid - 1;
  }
  const int b = lo;
  const int64_t c0 = min((int64_t)max(0, p.cu[b]), p.T), c1 = min((int64_t)p.cu[b + 1], p.T);
  const int64_t n = c1 - c0, len = p.lengths[b], first = len - n;
  const int64_t pi = unit - (c0 / PAGE + 2 * b);       // index among the pages that b writes
  bool live = n > 0 && first >= 0 && pi >= 0 && len <= (int64_t)p.max_pages * PAGE && h < p.H;
  const int64_t slot = first / PAGE + pi;              // index into b's table row
  live = live && slot * PAGE < len;
  int pg = 0;
  if (live) {
    pg = p.table[(int64_t)b * p.max_pages + slot];
    live = pg >= 0 && pg < p.num_pages;
  }
  const int64_t pos0 = slot * PAGE;                    // position of the page's first token
  const int keep = (int)max((int64_t)0, min((int64_t)PAGE, first - pos0));   // tokens that were there
  const int end = (int)min((int64_t)PAGE, len - pos0);

  const char* src = reinterpret_cast<const char*>(is_v ? p.v : p.k);
  const int64_t ts = is_v ? p.v_ts : p.k_ts, hs = is_v ? p.v_hs : p.k_hs;
  uint4 x[4];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = t + i * GROUP, tok = c / CPT, d0 = (c % CPT) * 8;
    x[i] = make_uint4(0, 0, 0, 0);
    if (live && tok >= keep && tok < end)
      x[i] = __ldg(reinterpret_cast<const uint4*>(src + 2 * ((c0 + pos0 + tok - first) * ts + h * hs + d0)));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack16<F16>(w[e]);
      const float a = fabsf(f.x), c = fabsf(f.y);
      if (a < INFINITY) amax = fmaxf(amax, a);         // NaN and infinities do not set the scale
      if (c < INFINITY) amax = fmaxf(amax, c);
    }
  }
  amax = warp_max(amax);
  if constexpr (GROUP > 32) {
    if ((threadIdx.x & 31) == 0) wmax[threadIdx.x >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < GROUP / 32; ++w) amax = fmaxf(amax, wmax[grp * (GROUP / 32) + w]);
  }
  if (!live) return;

  float* scale = (is_v ? p.v_scale : p.k_scale) + (int64_t)pg * p.H + h;
  uint8_t* page = (is_v ? p.v_pages : p.k_pages) + ((int64_t)pg * p.H + h) * (PAGE * D);
  int e = scale_exponent(amax), e_old = 0;
  bool grown = false;
  if (keep > 0) {
    e_old = exponent_of(*scale);
    grown = e > e_old;
    e = max(e, e_old);
  }
  // x 2^-e in one product: e is at most 120, so 2^-e is normal
  const float inv = pow2(-e), up = grown ? pow2(e_old - e) : 1.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = t + i * GROUP, tok = c / CPT;
    uint2* dst = reinterpret_cast<uint2*>(page) + c;
    if (tok < keep) {
      if (grown) {
        const uint2 o = *dst;
        uint2 r;
        float2 f0 = half2_to_float2(decode2(o.x & 0xffff)), f1 = half2_to_float2(decode2(o.x >> 16));
        r.x = encode2(f0.x * up, f0.y * up) | encode2(f1.x * up, f1.y * up) << 16;
        f0 = half2_to_float2(decode2(o.y & 0xffff)), f1 = half2_to_float2(decode2(o.y >> 16));
        r.y = encode2(f0.x * up, f0.y * up) | encode2(f1.x * up, f1.y * up) << 16;
        *dst = r;
      }
    } else if (tok < end) {
      const float2 f0 = unpack16<F16>(x[i].x), f1 = unpack16<F16>(x[i].y), f2 = unpack16<F16>(x[i].z),
                   f3 = unpack16<F16>(x[i].w);
      uint2 r;
      r.x = encode2(f0.x * inv, f0.y * inv) | encode2(f1.x * inv, f1.y * inv) << 16;
      r.y = encode2(f2.x * inv, f2.y * inv) | encode2(f3.x * inv, f3.y * inv) << 16;
      *dst = r;
    }
  }
  // every thread of the group has read the old scale before it changes
  if constexpr (GROUP > 32) {
    // (whole blocks only: the groups of a block can differ in `live`)
    asm volatile("bar.sync %0, %1;\n" ::"r"(1 + grp), "r"(GROUP) : "memory");
  } else {
    __syncwarp();
  }
  if (t == 0) *scale = pow2(e);
}

struct GatherParams {
  const uint8_t *k_pages, *v_pages;
  const float *k_scale, *v_scale;
  const int32_t *table, *starts, *cu;
  void *k, *v;
  int num_pages, H, max_pages, B, page;
  int64_t T;
};

// Packed token i of sequence b is its cached token starts[b] + i - cu[b]; out [T, H, D].
// A block takes 32 packed tokens: a warp finds their pages, then every thread
// dequantises 16 codes at a time (one 16-byte load, two 16-byte stores), heads of a
// token next to each other so that the stores are contiguous.  Bound: HBM.  1 B read
// and 2 B written per value.  Tokens of a missing page read as 0; rows at and behind
// cu[B] are left as they were.
template <int D, bool F16>
__global__ void __launch_bounds__(256) kv_gather_kernel(GatherParams p) {
  constexpr int TOK = 32, CPR = D / 16;
  __shared__ int64_t row[TOK];     // code row of head 0 (a row has D codes), -1: no such token, -2: missing page
  __shared__ int pgs[TOK];
  const int64_t t0 = (int64_t)blockIdx.x * TOK;
  if (threadIdx.x < TOK) {
    const int64_t i = t0 + threadIdx.x;
    int64_t r = -1;
    int pg = 0;
    if (i < p.T && i < p.cu[p.B] && i >= p.cu[0]) {
      const int b = find_sequence(p.cu, p.B, i);
      const int64_t pos = p.starts[b] + i - p.cu[b];
      r = -2;
      if (pos >= 0 && pos < (int64_t)p.max_pages * p.page) {
        pg = p.table[(int64_t)b * p.max_pages + pos / p.page];
        if (pg >= 0 && pg < p.num_pages) r = (int64_t)pg * p.H * p.page + pos % p.page;
      }
    }
    row[threadIdx.x] = r;
    pgs[threadIdx.x] = pg;
  }
  __syncthreads();
  const int per_tok = p.H * CPR;
  for (int it = threadIdx.x; it < TOK * per_tok; it += 256) {
    const int tok = it / per_tok, rest = it % per_tok, h = rest / CPR, c = rest % CPR;
    const int64_t r = row[tok];
    if (r == -1) continue;
    const int64_t dst = ((t0 + tok) * p.H + h) * D + c * 16;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      uint4 codes = make_uint4(0, 0, 0, 0);
      float s = 0.f;
      if (r >= 0) {
        codes = __ldg(reinterpret_cast<const uint4*>((kv ? p.v_pages : p.k_pages) + (r + (int64_t)h * p.page) * D + c * 16));
        s = __ldg((kv ? p.v_scale : p.k_scale) + (int64_t)pgs[tok] * p.H + h);
      }
      const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
      uint32_t o[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f0 = half2_to_float2(decode2(w[e] & 0xffff)), f1 = half2_to_float2(decode2(w[e] >> 16));
        o[2 * e] = pack16<F16>(f0.x * s, f0.y * s);
        o[2 * e + 1] = pack16<F16>(f1.x * s, f1.y * s);
      }
      uint4* d = reinterpret_cast<uint4*>(reinterpret_cast<char*>(kv ? p.v : p.k) + 2 * dst);
      d[0] = make_uint4(o[0], o[1], o[2], o[3]);
      d[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
  }
}

int check_cache(const KB200KvCache* c, const char* what) {
  if (!c || !c->k_pages || !c->v_pages || !c->k_scale || !c->v_scale)
    return set_error(KB200_ERR_INVALID, "%s: null cache pointer", what);
  if (!aligned16(c->k_pages) || !aligned16(c->v_pages))
    return set_error(KB200_ERR_ALIGN, "%s: cache pages must be 16-byte aligned", what);
  if (c->D != 64 && c->D != 128) return set_error(KB200_ERR_INVALID, "%s: head dim %lld (64 or 128)", what, (long long)c->D);
  if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128)
    return set_error(KB200_ERR_INVALID, "%s: page of %lld tokens (16, 32, 64 or 128)", what, (long long)c->page);
  if (c->H < 1 || c->H > 4096 || c->num_pages < 1 || c->num_pages * c->H * c->page > 0x7fffffffLL)
    return set_error(KB200_ERR_INVALID, "%s: %lld pages of %lld heads (pages * heads * page tokens up to 2^31 - 1)", what,
                     (long long)c->num_pages, (long long)c->H);
  return KB200_OK;
}

template <int D, int PAGE, bool F16>
static void launch_append(const AppendParams& p, cudaStream_t st) {
  constexpr int GROUP = PAGE * D / 32, THREADS = GROUP > 256 ? GROUP : 256, PER = THREADS / GROUP;
  const int64_t units = p.T / PAGE + 2 * (int64_t)p.B;
  kv_append_kernel<D, PAGE, F16><<<dim3((unsigned)units, (unsigned)((2 * p.H + PER - 1) / PER)), THREADS, 0, st>>>(p);
}

template <int D, bool F16>
static void launch_append_page(const AppendParams& p, int page, cudaStream_t st) {
  if (page == 16) launch_append<D, 16, F16>(p, st);
  else if (page == 32) launch_append<D, 32, F16>(p, st);
  else if (page == 64) launch_append<D, 64, F16>(p, st);
  else launch_append<D, 128, F16>(p, st);
}

}  // namespace kv
}  // namespace kb

extern "C" int kb200_kv_append(const KB200KvCache* c, const void* k, const void* v, int64_t k_token_stride,
                               int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                               const int32_t* page_table, int64_t max_pages, const int32_t* lengths,
                               const int32_t* cu_new, int64_t B, int64_t T, int dtype, void* stream) {
  using namespace kb;
  if (int e = kv::check_cache(c, "kv_append")) return e;
  if (B < 0 || T < 0 || max_pages < 0 || B > (1 << 24) || T > 0x7fffffffLL || (dtype != 0 && dtype != 1))
    return set_error(KB200_ERR_INVALID, "kv_append: B=%lld T=%lld max_pages=%lld dtype=%d", (long long)B, (long long)T,
                     (long long)max_pages, dtype);
  if (B == 0 || T == 0) return KB200_OK;
  if (!k || !v || !page_table || !lengths || !cu_new) return set_error(KB200_ERR_INVALID, "kv_append: null pointer");
  if (!aligned16(k) || !aligned16(v) || ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7))
    return set_error(KB200_ERR_ALIGN, "kv_append: k and v rows must be 16-byte aligned");
  kv::AppendParams p{(uint8_t*)c->k_pages, (uint8_t*)c->v_pages, c->k_scale, c->v_scale, k, v, k_token_stride,
                     k_head_stride, v_token_stride, v_head_stride, page_table, lengths, cu_new, (int)c->num_pages,
                     (int)c->H, (int)max_pages, (int)B, T};
  cudaStream_t st = (cudaStream_t)stream;
  const int page = (int)c->page;
  if (c->D == 64) {
    if (dtype) kv::launch_append_page<64, true>(p, page, st); else kv::launch_append_page<64, false>(p, page, st);
  } else {
    if (dtype) kv::launch_append_page<128, true>(p, page, st); else kv::launch_append_page<128, false>(p, page, st);
  }
  return check_launch("kv_append_kernel");
}

extern "C" int kb200_kv_gather(const KB200KvCache* c, const int32_t* page_table, int64_t max_pages, const int32_t* starts,
                               const int32_t* cu, int64_t B, int64_t T, void* k, void* v, int dtype, void* stream) {
  using namespace kb;
  if (int e = kv::check_cache(c, "kv_gather")) return e;
  if (B < 0 || T < 0 || max_pages < 0 || B > (1 << 24) || T > 0x7fffffffLL || (dtype != 0 && dtype != 1))
    return set_error(KB200_ERR_INVALID, "kv_gather: B=%lld T=%lld max_pages=%lld dtype=%d", (long long)B, (long long)T,
                     (long long)max_pages, dtype);
  if (B == 0 || T == 0) return KB200_OK;
  if (!k || !v || !page_table || !starts || !cu) return set_error(KB200_ERR_INVALID, "kv_gather: null pointer");
  if (!aligned16(k) || !aligned16(v)) return set_error(KB200_ERR_ALIGN, "kv_gather: outputs must be 16-byte aligned");
  kv::GatherParams p{(const uint8_t*)c->k_pages, (const uint8_t*)c->v_pages, c->k_scale, c->v_scale, page_table, starts,
                     cu, k, v, (int)c->num_pages, (int)c->H, (int)max_pages, (int)B, (int)c->page, T};
  cudaStream_t st = (cudaStream_t)stream;
  const unsigned grid = (unsigned)((T + 31) / 32);
  if (c->D == 64) {
    if (dtype) kv::kv_gather_kernel<64, true><<<grid, 256, 0, st>>>(p); else kv::kv_gather_kernel<64, false><<<grid, 256, 0, st>>>(p);
  } else {
    if (dtype) kv::kv_gather_kernel<128, true><<<grid, 256, 0, st>>>(p); else kv::kv_gather_kernel<128, false><<<grid, 256, 0, st>>>(p);
  }
  return check_launch("kv_gather_kernel");
}
