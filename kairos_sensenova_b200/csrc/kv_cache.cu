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
// Bound: HBM.  2 B read and 1 B written per value (8 sequences of 16384 tokens, 8 heads of 128: 129 us,
// 6.0 TB/s).  A block takes several of a unit's
// (head, k|v) items, the next one's loads under way while one is encoded: the three
// dependent reads that find the page are paid once.
template <int D, int PAGE, bool F16>
__global__ void __launch_bounds__(PAGE * D / 32 > 256 ? 512 : 256) kv_append_kernel(AppendParams p) {
  constexpr int GROUP = PAGE * D / 32;                 // threads of one item
  constexpr int THREADS = GROUP > 256 ? GROUP : 256;
  constexpr int PER_BLOCK = THREADS / GROUP;
  constexpr int CPT = D / 8;                           // 8-value chunks of a token
  __shared__ float wmax[2][THREADS / 32];
  const int grp = threadIdx.x / GROUP, t = threadIdx.x % GROUP;
  const int64_t unit = blockIdx.x;
  const int part = blockIdx.y;

  // the unit's sequence: largest b with cu[b] / PAGE + 2 b <= unit
  const int b = warp_last(p.B, threadIdx.x & 31, [&](int i) { return (int64_t)max(0, p.cu[i]) / PAGE + 2 * i <= unit; });
  const int64_t c0 = min((int64_t)max(0, p.cu[b]), p.T), c1 = min((int64_t)p.cu[b + 1], p.T);
  const int64_t n = c1 - c0, len = p.lengths[b], first = len - n;
  const int64_t pi = unit - (c0 / PAGE + 2 * b);       // index among the pages that b writes
  if (n <= 0 || first < 0 || pi < 0 || len > (int64_t)p.max_pages * PAGE) return;
  const int64_t slot = first / PAGE + pi;              // index into b's table row
  if (slot * PAGE >= len) return;
  const int pg = p.table[(int64_t)b * p.max_pages + slot];
  if (pg < 0 || pg >= p.num_pages) return;
  const int64_t pos0 = slot * PAGE;                    // position of the page's first token
  const int keep = (int)max((int64_t)0, min((int64_t)PAGE, first - pos0));   // tokens that were there
  const int end = (int)min((int64_t)PAGE, len - pos0);
  const int64_t row0 = c0 + pos0 - first;              // packed row of the page's first token

  auto fetch = [&](int item, uint4* x) {
    const bool is_v = item & 1;
    const char* src = reinterpret_cast<const char*>(is_v ? p.v : p.k);
    const int64_t ts = is_v ? p.v_ts : p.k_ts, hs = is_v ? p.v_hs : p.k_hs;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = t + i * GROUP, tok = c / CPT, d0 = (c % CPT) * 8;
      x[i] = make_uint4(0, 0, 0, 0);
      if (item < 2 * p.H && tok >= keep && tok < end)
        x[i] = __ldg(reinterpret_cast<const uint4*>(src + 2 * ((row0 + tok) * ts + (item >> 1) * hs + d0)));
    }
  };
  const int stride = gridDim.y * PER_BLOCK;
  uint4 x[4], nx[4];
  fetch(part * PER_BLOCK + grp, x);
  int turn = 0;
  for (int base = part * PER_BLOCK; base < 2 * p.H; base += stride, turn ^= 1) {   // (items: head, k|v)
    const int item = base + grp;
    fetch(item + stride, nx);
    // the largest magnitude, as 16-bit integers in pairs (the order of the magnitudes; NaN and
    // infinities come out on top, and only if there are some is it done again without them).  TOP is
    // the type's largest magnitude of 4 significant bits, 1.875 * 2^15 or 2^127: what is larger would be
    // rounded to a code whose value the type does not have, and becomes TOP (2^-4 of the value off at
    // most, the half step of e4m3).
    constexpr uint32_t INF = F16 ? 0x7c00u : 0x7f80u, TOP = F16 ? 0x7b80u : 0x7f70u;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      top = __vmaxu2(__vmaxu2(__vmaxu2(top, x[i].x & 0x7fff7fffu), __vmaxu2(x[i].y & 0x7fff7fffu, x[i].z & 0x7fff7fffu)),
                     x[i].w & 0x7fff7fffu);
    uint32_t mag = max(top & 0xffffu, top >> 16);
    const bool odd = mag > TOP;                          // this thread has a value that is not finite, or behind TOP
    if (odd) {
      mag = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t lo = w[e] & 0x7fffu, hi = (w[e] >> 16) & 0x7fffu;
          if (lo > TOP && lo < INF) lo = TOP;
          if (hi > TOP && hi < INF) hi = TOP;
          w[e] = (w[e] & 0x80008000u) | hi << 16 | lo;
          if (lo < INF) mag = max(mag, lo);
          if (hi < INF) mag = max(mag, hi);
        }
        x[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    const float2 mag2 = unpack16<F16>(mag);
    float amax = mag2.x;
    const bool is_v = item & 1, live = item < 2 * p.H;
    const int h = item >> 1;
    float* scale = (is_v ? p.v_scale : p.k_scale) + (int64_t)pg * p.H + h;
    int e_old = 0;
    if (keep > 0 && live) e_old = exponent_of(*scale);   // (every thread reads it before the barrier, one writes it after)
    amax = warp_max(amax);
    if constexpr (GROUP > 32) {
      if ((threadIdx.x & 31) == 0) wmax[turn][threadIdx.x >> 5] = amax;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < GROUP / 32; ++w) amax = fmaxf(amax, wmax[turn][grp * (GROUP / 32) + w]);
    }
    if (live) {
      uint8_t* page = (is_v ? p.v_pages : p.k_pages) + ((int64_t)pg * p.H + h) * (PAGE * D);
      int e = scale_exponent(amax);
      const bool grown = keep > 0 && e > e_old;
      if (keep > 0) e = max(e, e_old);
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
          const float2 s2 = make_float2(inv, inv);
          const float2 f0 = fmul2(unpack16<F16>(x[i].x), s2), f1 = fmul2(unpack16<F16>(x[i].y), s2),
                       f2 = fmul2(unpack16<F16>(x[i].z), s2), f3 = fmul2(unpack16<F16>(x[i].w), s2);
          uint2 r;
          if (odd) {
            r.x = encode2(f0.x, f0.y) | encode2(f1.x, f1.y) << 16;
            r.y = encode2(f2.x, f2.y) | encode2(f3.x, f3.y) << 16;
          } else {
            r.x = encode2_finite(f0) | encode2_finite(f1) << 16;
            r.y = encode2_finite(f2) | encode2_finite(f3) << 16;
          }
          *dst = r;
        }
      }
      if constexpr (GROUP <= 32) __syncwarp();
      if (t == 0) *scale = pow2(e);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = nx[i];
  }
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
// dequantises 8 codes at a time (an 8-byte load, a 16-byte store), heads of a
// token next to each other so that the stores are contiguous.  Bound: HBM.  1 B read
// and 2 B written per value (the same sequences: 142 us, 5.3 TB/s; a kernel that only writes 3.6-3.9).  Tokens of a missing page read as 0; rows at and behind
// cu[B] are left as they were.
template <int D, bool F16>
__global__ void __launch_bounds__(256) kv_gather_kernel(GatherParams p) {
  constexpr int TOK = 32, CPR = D / 8, UNROLL = 8;
  __shared__ int64_t row[TOK];     // code row of head 0 (a row has D codes), -1: no such token, -2: missing page
  __shared__ int pgs[TOK];
  const int64_t t0 = (int64_t)blockIdx.x * TOK;
  if (threadIdx.x < TOK) {
    const int lane = threadIdx.x;
    const int64_t i = t0 + lane;
    // the first token's sequence, and of the 32 that begin after it those that begin at or before each token
    const int b0 = find_sequence(p.cu, p.B, t0, lane);
    const int next = b0 + 1 + lane < p.B ? p.cu[b0 + 1 + lane] : 0x7fffffff;
    int b = b0;
#pragma unroll
    for (int j = 0; j < 32; ++j) b += __shfl_sync(0xffffffffu, next, j) <= i ? 1 : 0;
    if (b - b0 >= 32)                // (more of them: empty ones)
      for (int end = p.B; end - b > 1;) {
        const int mid = b + (end - b) / 2;
        if (p.cu[mid] <= i) b = mid; else end = mid;
      }
    int64_t r = -1;
    int pg = 0;
    if (i < p.T && i < p.cu[p.B] && i >= p.cu[0]) {
      const int64_t pos = p.starts[b] + i - p.cu[b];
      r = -2;
      if (pos >= 0 && pos < (int64_t)p.max_pages * p.page) {
        pg = p.table[(int64_t)b * p.max_pages + pos / p.page];
        if (pg >= 0 && pg < p.num_pages) r = (int64_t)pg * p.H * p.page + pos % p.page;
      }
    }
    row[threadIdx.x] = r;
    pgs[threadIdx.x] = r >= 0 ? pg : 0;
  }
  __syncthreads();
  // a thread keeps its (head, chunk) and goes through the tokens, `lanes` of which are taken at once
  const int per_tok = p.H * CPR, lanes = per_tok >= 256 ? 1 : 256 / per_tok;
  const int tok0 = per_tok >= 256 ? 0 : threadIdx.x / per_tok;
  if (tok0 >= lanes) return;
  for (int rest = per_tok >= 256 ? threadIdx.x : threadIdx.x % per_tok; rest < per_tok; rest += 256) {
    const int h = rest / CPR, c = rest % CPR;
    const int64_t hoff = (int64_t)h * p.page;
    for (int tok = tok0; tok < TOK; tok += lanes * UNROLL) {
      uint2 codes[UNROLL][2];
      float s[UNROLL][2];
#pragma unroll
      for (int z = 0; z < UNROLL; ++z) {
        const int tt = tok + z * lanes;
        const int64_t r = tt < TOK ? row[tt] : -1;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          codes[z][kv] = make_uint2(0, 0);
          s[z][kv] = 0.f;
          if (r >= 0) {
            codes[z][kv] = __ldg(reinterpret_cast<const uint2*>((kv ? p.v_pages : p.k_pages) + (r + hoff) * D + c * 8));
            s[z][kv] = __ldg((kv ? p.v_scale : p.k_scale) + (int64_t)pgs[tt] * p.H + h);
          }
        }
      }
#pragma unroll
      for (int z = 0; z < UNROLL; ++z) {
        const int tt = tok + z * lanes;
        if (tt >= TOK || row[tt] == -1) continue;
        const int64_t dst = ((t0 + tt) * p.H + h) * D + c * 8;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const uint32_t w[2] = {codes[z][kv].x, codes[z][kv].y};
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t lo, hi;
            decode4(w[e], lo, hi);
            const float2 f0 = half2_to_float2(lo), f1 = half2_to_float2(hi);
            o[2 * e] = pack16<F16>(f0.x * s[z][kv], f0.y * s[z][kv]);
            o[2 * e + 1] = pack16<F16>(f1.x * s[z][kv], f1.y * s[z][kv]);
          }
          *reinterpret_cast<uint4*>(reinterpret_cast<char*>(kv ? p.v : p.k) + 2 * dst) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
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
static int launch_append(const AppendParams& p, cudaStream_t st) {
  constexpr int GROUP = PAGE * D / 32, THREADS = GROUP > 256 ? GROUP : 256, PER = THREADS / GROUP;
  // few units: a block for every item group of a unit; many: four of them one after the other
  // (32760 tokens of 8 heads: 46.8 us with four, 49 with two, 47.5 with eight; a unit's blocks next to
  // each other in a one-dimensional grid: 53.8)
  const int64_t units = p.T / PAGE + 2 * (int64_t)p.B, groups = (2 * p.H + PER - 1) / PER;
  const int64_t items = units * groups <= sm_count() * 8 ? 1 : 4;
  kv_append_kernel<D, PAGE, F16><<<dim3((unsigned)units, (unsigned)((groups + items - 1) / items)), THREADS, 0, st>>>(p);
  return check_launch("kv_append_kernel");
}

template <int D, bool F16>
static int launch_append_page(const AppendParams& p, int page, cudaStream_t st) {
  if (page == 16) return launch_append<D, 16, F16>(p, st);
  if (page == 32) return launch_append<D, 32, F16>(p, st);
  if (page == 64) return launch_append<D, 64, F16>(p, st);
  return launch_append<D, 128, F16>(p, st);
}

}  // namespace kv
}  // namespace kb

extern "C" int kb200_kv_append(const KB200KvAppendArgs* a, void* stream) {
  using namespace kb;
  if (!a) return set_error(KB200_ERR_INVALID, "kv_append: null arguments");
  const KB200KvCache* c = &a->cache;
  if (int e = kv::check_cache(c, "kv_append")) return e;
  if (a->B < 0 || a->T < 0 || a->max_pages < 0 || a->B > (1 << 24) || a->max_pages > (1 << 26) || a->T > 0x7fffffffLL ||
      (a->dtype != 0 && a->dtype != 1))
    return set_error(KB200_ERR_INVALID, "kv_append: B=%lld T=%lld max_pages=%lld dtype=%lld", (long long)a->B,
                     (long long)a->T, (long long)a->max_pages, (long long)a->dtype);
  if (a->B == 0 || a->T == 0) return KB200_OK;
  if (!a->k || !a->v || (a->max_pages > 0 && !a->page_table) || !a->lengths || !a->cu_new)
    return set_error(KB200_ERR_INVALID, "kv_append: null pointer");
  if (!aligned16(a->k) || !aligned16(a->v) ||
      ((a->k_token_stride | a->k_head_stride | a->v_token_stride | a->v_head_stride) & 7))
    return set_error(KB200_ERR_ALIGN, "kv_append: k and v rows must be 16-byte aligned");
  kv::AppendParams p{(uint8_t*)c->k_pages, (uint8_t*)c->v_pages, c->k_scale, c->v_scale, a->k, a->v, a->k_token_stride,
                     a->k_head_stride, a->v_token_stride, a->v_head_stride, a->page_table, a->lengths, a->cu_new,
                     (int)c->num_pages, (int)c->H, (int)a->max_pages, (int)a->B, a->T};
  cudaStream_t st = (cudaStream_t)stream;
  const int page = (int)c->page;
  if (c->D == 64) return a->dtype ? kv::launch_append_page<64, true>(p, page, st) : kv::launch_append_page<64, false>(p, page, st);
  return a->dtype ? kv::launch_append_page<128, true>(p, page, st) : kv::launch_append_page<128, false>(p, page, st);
}

extern "C" int kb200_kv_gather(const KB200KvGatherArgs* a, void* stream) {
  using namespace kb;
  if (!a) return set_error(KB200_ERR_INVALID, "kv_gather: null arguments");
  const KB200KvCache* c = &a->cache;
  if (int e = kv::check_cache(c, "kv_gather")) return e;
  if (a->B < 0 || a->T < 0 || a->max_pages < 0 || a->B > (1 << 24) || a->max_pages > (1 << 26) || a->T > 0x7fffffffLL ||
      (a->dtype != 0 && a->dtype != 1))
    return set_error(KB200_ERR_INVALID, "kv_gather: B=%lld T=%lld max_pages=%lld dtype=%lld", (long long)a->B,
                     (long long)a->T, (long long)a->max_pages, (long long)a->dtype);
  if (a->B == 0 || a->T == 0) return KB200_OK;
  if (!a->k || !a->v || (a->max_pages > 0 && !a->page_table) || !a->starts || !a->cu)
    return set_error(KB200_ERR_INVALID, "kv_gather: null pointer");
  if (!aligned16(a->k) || !aligned16(a->v)) return set_error(KB200_ERR_ALIGN, "kv_gather: outputs must be 16-byte aligned");
  kv::GatherParams p{(const uint8_t*)c->k_pages, (const uint8_t*)c->v_pages, c->k_scale, c->v_scale, a->page_table, a->starts,
                     a->cu, a->k, a->v, (int)c->num_pages, (int)c->H, (int)a->max_pages, (int)a->B, (int)c->page, a->T};
  cudaStream_t st = (cudaStream_t)stream;
  const unsigned grid = (unsigned)((a->T + 31) / 32);
  if (c->D == 64) {
    if (a->dtype) kv::kv_gather_kernel<64, true><<<grid, 256, 0, st>>>(p); else kv::kv_gather_kernel<64, false><<<grid, 256, 0, st>>>(p);
  } else {
    if (a->dtype) kv::kv_gather_kernel<128, true><<<grid, 256, 0, st>>>(p); else kv::kv_gather_kernel<128, false><<<grid, 256, 0, st>>>(p);
  }
  return check_launch("kv_gather_kernel");
}
