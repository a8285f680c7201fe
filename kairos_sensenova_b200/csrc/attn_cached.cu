// attn_cached.cu -- attention of a few query tokens per sequence over the 8-bit paged
// cache (kv_cache.cuh): the decode step of one token, or Sq drafted tokens at once.
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j,  j < length - Sq + 1 + i
//
// Bound: HBM, 2 D bytes per cached token and kv head.  Rows are the R = Sq * (Hq / Hkv)
// queries that share a kv head, so the cache is read once for all of them.
//
// Split of the work: the tiles of 128 cached tokens of all (sequence, kv head, row
// block) units are laid end to end and every CTA takes an equal, contiguous share; the
// shares are computed on the device from the lengths, so ragged batches balance without
// the host knowing them.  A unit inside one share is finished there; one that crosses
// shares leaves a partial (m, l, O) per CTA, joined in share order (no atomics: the
// result does not depend on timing) by a second kernel.
//
// A CTA: one producer warp streams K and V pages by TMA (128-byte swizzle) into a ring
// of 128-token stages; 8 consumer warps = key groups x row groups.  Per 16 tokens:
//   S^T = K Q^T  mma.m16n8k16 f16 (16 tokens x 8 rows), codes widened to f16 in
//                registers (exact); the contraction index is permuted so that a lane's
//                operands are 16 consecutive bytes of the page
//   P   = 2^(s - m), running max per row (per warp; the warps join at the end)
//   O^T += V^T P^T, P transposed between the two by movmatrix.  The products of 16
//                tokens are formed from zero and added times their page's V scale in
//                fp32, so scales of any spread keep full precision.
// bf16 queries are multiplied by a power of two per row into f16's range first (exact
// but for elements 2^-29 below the row's largest).  P is rounded to f16 (2^-12).
#include "kv_cache.cuh"
#include "tc_common.cuh"

namespace kb {
namespace cached {

constexpr int TK = 128;            // tokens per stage
constexpr int NW = 8;              // consumer warps
constexpr int THREADS = (NW + 1) * 32;
constexpr float SHIFT = 8.f;       // P = 2^(s - m + SHIFT), s <= m + TAU: below 2^12, inside f16
constexpr float TAU = 4.f;         // O and l are rescaled when the maximum grows by more than this (log2 units)

struct Params {
  const void* q;
  void* o;
  float* lse;
  const int32_t *table, *lengths;
  const float *k_scale, *v_scale;
  float* part;                     // [2 G][rows][D] partial O, then [2 G][rows][2] (m, l)
  int64_t q_bs, q_ts, q_hs;        // batch, token, head strides of q, elements
  int B, Sq, Hq, H, G, R;          // G = Hq / H query heads per kv head, R = Sq * G
  int rblocks, rows;               // row blocks per (sequence, kv head), rows of a block
  int num_pages, max_pages, page;
  float scale_log2;
};

struct Maps {
  CUtensorMap k, v;
};

KB_DEVI float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
KB_DEVI void mma_f16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
KB_DEVI uint32_t transpose8(uint32_t x) {   // 8x8 matrix of 16-bit values over the warp
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
  return r;
}

// Length of sequence b, inside its table row.
KB_DEVI int seq_len(const Params& p, int b) {
  const int64_t cap = (int64_t)p.max_pages * p.page;
  return (int)min(max((int64_t)p.lengths[b], (int64_t)0), min(cap, (int64_t)0x7fffff00));
}
KB_DEVI int seq_tiles(const Params& p, int b) { return (seq_len(p, b) + TK - 1) / TK; }

// Sum of the tiles of all sequences, by one warp.
KB_DEVI int64_t warp_total_tiles(const Params& p, int lane) {
  int64_t s = 0;
  for (int b = lane; b < p.B; b += 32) s += seq_tiles(p, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
// Sequence that holds the flat tile position `at` (tiles of one sequence: units * seq_tiles),
// and the position where it begins; by one warp.  at < total.
KB_DEVI void warp_find(const Params& p, int64_t units, int64_t at, int lane, int& b_out, int64_t& begin_out) {
  int64_t base = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int64_t mine = b0 + lane < p.B ? units * seq_tiles(p, b0 + lane) : 0;
    int64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, base + inc > at);
    if (hit) {
      const int l = __ffs(hit) - 1;
      b_out = b0 + l;
      begin_out = __shfl_sync(0xffffffffu, base + inc - mine, l);
      return;
    }
    base += __shfl_sync(0xffffffffu, inc, 31);
  }
  b_out = p.B;
  begin_out = base;
}

// What a CTA works on: shares of `per` flat tiles, CTA c has [c * per, (c + 1) * per).
struct Share {
  int64_t total, per;
};
KB_DEVI Share share_of(const Params& p, int64_t units, int64_t sum_tiles, int ctas) {
  Share s;
  s.total = sum_tiles * units;
  s.per = (s.total + ctas - 1) / ctas;
  return s;
}

template <int D, int NT, int WR, int STAGES>
struct Smem {
  static constexpr int ROWS = NT * 8 * WR;
  uint8_t k[STAGES][TK * D];       // swizzled page rows
  uint8_t v[STAGES][TK * D];
  float o[NW / WR][ROWS][D];       // the warps' O, joined at the end of a unit
  float ml[NW / WR][ROWS][2];
  float sk[STAGES][TK / 16], sv[STAGES][TK / 16];   // page scales of 16-token groups; sk < 0: no such page
  uint64_t full[STAGES], empty[STAGES];
  int64_t total, begin;
  int first_b;
  int abort_flag;
};

// 16-byte chunk `c` of page row `r` in a swizzled stage.
template <int D>
KB_DEVI uint32_t swz(int r, int c) {
  if constexpr (D == 128) return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
  else return (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

template <int D, bool F16, int NT, int WR, int STAGES, int OCC>
__global__ void __launch_bounds__(THREADS, OCC) attn_cached_kernel(const __grid_constant__ Maps maps, Params p) {
  using SM = Smem<D, NT, WR, STAGES>;
  constexpr int WK = NW / WR, ROWS = SM::ROWS;
  constexpr int MT = D / 16;               // 16-wide tiles of D
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  SM& sm = *reinterpret_cast<SM*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t units = (int64_t)p.H * p.rblocks;

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      tc::mbar_init(&sm.full[s], 32);
      tc::mbar_init(&sm.empty[s], NW);
    }
    sm.abort_flag = 0;
    tc::fence_barrier_init();
  }
  if (warp == 0) {
    const int64_t sum = warp_total_tiles(p, lane);
    const Share sh = share_of(p, units, sum, gridDim.x);
    int b = 0;
    int64_t begin = 0;
    if ((int64_t)blockIdx.x * sh.per < sh.total) warp_find(p, units, blockIdx.x * sh.per, lane, b, begin);
    if (lane == 0) {
      sm.total = sum;
      sm.first_b = b;
      sm.begin = begin;
    }
  }
  __syncthreads();
  const Share sh = share_of(p, units, sm.total, gridDim.x);
  const int64_t at0 = (int64_t)blockIdx.x * sh.per, at1 = min(at0 + sh.per, sh.total);
  if (at0 >= at1) return;
  auto aborted = [&]() { return *((volatile int*)&sm.abort_flag) != 0; };

  // Every warp walks the CTA's segments (unit, tile range) in the same order.
  int b = sm.first_b;
  int64_t begin = sm.begin, at = at0;
  int st = 0;                              // stage counter
  int seg = 0;
  if (warp == NW) {
    // ---------------------------------------------------------------- producer
    if (lane == 0) {
      tc::prefetch_tmap(&maps.k);
      tc::prefetch_tmap(&maps.v);
    }
    bool ok = true;
    const int per_stage = TK / p.page, gpp = p.page / 16;
    while (at < at1 && ok) {
      int nt = seq_tiles(p, b);
      while (nt == 0 || at >= begin + units * nt) {
        begin += units * nt;
        nt = seq_tiles(p, ++b);
      }
      const int len = seq_len(p, b), npages = (len + p.page - 1) / p.page;
      const int u = (int)((at - begin) / nt), t0 = (int)((at - begin) % nt);
      const int t1 = (int)min((int64_t)nt, t0 + (at1 - at));
      const int h = u / p.rblocks;
      const int32_t* row = p.table + (int64_t)b * p.max_pages;
      // lane i < per_stage holds page i of the stage
      const int pi0 = t0 * per_stage + lane;
      int next = lane < per_stage && pi0 < npages ? __ldg(row + pi0) : -1;
      for (int t = t0; t < t1; ++t, ++st) {
        const int pg = next;
        const int pn = (t + 1) * per_stage + lane;
        next = t + 1 < t1 && lane < per_stage && pn < npages ? __ldg(row + pn) : -1;
        const bool have = pg >= 0 && pg < p.num_pages;
        float ks = -1.f, vs = 0.f;
        if (have) {
          ks = __ldg(p.k_scale + (int64_t)pg * p.H + h);
          vs = __ldg(p.v_scale + (int64_t)pg * p.H + h);
        }
        const int s = st % STAGES;
        if (st >= STAGES && !tc::mbar_wait(&sm.empty[s], (st / STAGES - 1) & 1)) { sm.abort_flag = 1; ok = false; }
        ok = __all_sync(0xffffffffu, ok) && !aborted();
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane < per_stage)
          for (int g = 0; g < gpp; ++g) {
            sm.sk[s][lane * gpp + g] = ks;
            sm.sv[s][lane * gpp + g] = vs;
          }
        const int loads = __popc(__ballot_sync(0xffffffffu, have));
        if (lane == 0) tc::mbar_expect_tx(&sm.full[s], (uint32_t)(loads * 2 * p.page * D));
        __syncwarp();
        if (have) {
          const int y = (pg * p.H + h) * p.page;
          tc::tma_load_2d(sm.k[s] + lane * p.page * D, &maps.k, &sm.full[s], 0, y);
          tc::tma_load_2d(sm.v[s] + lane * p.page * D, &maps.v, &sm.full[s], 0, y);
        }
        if (lane != 0) tc::mbar_arrive(&sm.full[s]);
      }
      at += t1 - t0;
    }
    // every load lands before the CTA may exit
    for (int i = st > STAGES ? st - STAGES : 0; i < st; ++i) tc::mbar_wait(&sm.full[i % STAGES], (i / STAGES) & 1);
    return;
  }

  // ------------------------------------------------------------------ consumers
  const int wk = warp / WR, wr = warp % WR;
  const int g = lane >> 2, t4 = lane & 3;
  for (; at < at1; ++seg) {
    int nt = seq_tiles(p, b);
    while (nt == 0 || at >= begin + units * nt) {
      begin += units * nt;
      nt = seq_tiles(p, ++b);
    }
    const int len = seq_len(p, b);
    const int u = (int)((at - begin) / nt), t0 = (int)((at - begin) % nt);
    const int t1 = (int)min((int64_t)nt, t0 + (at1 - at));
    const int h = u / p.rblocks, rb = u % p.rblocks;

    // Q^T operands of this warp's rows: row n = g of each 8-row tile, this lane's D / 4
    // channels (t4 * 32 + ... for D = 128), as f16 under a power of two per row.
    constexpr int CH = D / 64;             // 16-byte code chunks per lane and row
    uint32_t qf[NT][CH * 8];
    float qs[NT][2];                       // log2-domain score factors of the rows 2 t4, 2 t4 + 1
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = rb * p.rows + (wr * NT + n) * 8 + g;
      float amax = 0.f;
      uint32_t raw[CH * 8];
      const bool in = r < p.R;
      const char* src = reinterpret_cast<const char*>(p.q);
      if (in) src += 2 * ((int64_t)b * p.q_bs + (int64_t)(r / p.G) * p.q_ts + (int64_t)(h * p.G + r % p.G) * p.q_hs +
                          t4 * (CH * 16));
#pragma unroll
      for (int c = 0; c < CH * 2; ++c) {
        const uint4 x = in ? __ldg(reinterpret_cast<const uint4*>(src) + c) : make_uint4(0, 0, 0, 0);
        raw[4 * c] = x.x; raw[4 * c + 1] = x.y; raw[4 * c + 2] = x.z; raw[4 * c + 3] = x.w;
      }
      float f = 1.f;
      if constexpr (F16) {
#pragma unroll
        for (int c = 0; c < CH * 8; ++c) qf[n][c] = raw[c];
      } else {
#pragma unroll
        for (int c = 0; c < CH * 8; ++c) {
          const float2 x = unpack_bf16(raw[c]);
          if (fabsf(x.x) < INFINITY) amax = fmaxf(amax, fabsf(x.x));
          if (fabsf(x.y) < INFINITY) amax = fmaxf(amax, fabsf(x.y));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int e = min(max(kv::exponent_of(amax) - 14, -112), 112);   // amax 2^-e in [2^14, 2^15)
        const float down = kv::pow2(-e);
        f = kv::pow2(e);
#pragma unroll
        for (int c = 0; c < CH * 8; ++c) {
          const float2 x = unpack_bf16(raw[c]);
          qf[n][c] = kv::pack16<true>(x.x * down, x.y * down);
        }
      }
      f *= p.scale_log2;
      // row 2 t4 (+1) of the tile is lane (2 t4 (+1)) * 4's row
      qs[n][0] = __shfl_sync(0xffffffffu, f, t4 * 8);
      qs[n][1] = __shfl_sync(0xffffffffu, f, t4 * 8 + 4);
    }

    float o[NT][MT][4], m[NT][2], l[NT][2];
    int seen[NT][2];                       // keys that the rows 2 t4, 2 t4 + 1 see
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[n][c] = -INFINITY;
        l[n][c] = 0.f;
        const int r = rb * p.rows + (wr * NT + n) * 8 + 2 * t4 + c;
        seen[n][c] = r < p.R ? len - p.Sq + 1 + r / p.G : len;
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
    }
    const int all_seen = len - p.Sq + 1;   // keys below are seen by every row

    for (int t = t0; t < t1; ++t, ++st) {
      const int s = st % STAGES;
      const bool ok = tc::mbar_wait(&sm.full[s], (st / STAGES) & 1);
      if (!ok) sm.abort_flag = 1;
      if (__any_sync(0xffffffffu, !ok)) break;
#pragma unroll 1
      for (int kg = wk; kg < TK / 16; kg += WK) {
        const int tok0 = t * TK + kg * 16;
        const float sk = sm.sk[s][kg], sv = sm.sv[s][kg];
        if (tok0 >= len || sk < 0.f) continue;
        // ---- S^T = K Q^T
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        const uint8_t* kb = sm.k[s];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const int r0 = kg * 16 + g;
          const uint4 x0 = *reinterpret_cast<const uint4*>(kb + swz<D>(r0, t4 * CH + c));
          const uint4 x1 = *reinterpret_cast<const uint4*>(kb + swz<D>(r0 + 8, t4 * CH + c));
          const uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t a[4] = {kv::decode2(w0[e] & 0xffff), kv::decode2(w1[e] & 0xffff), kv::decode2(w0[e] >> 16),
                                   kv::decode2(w1[e] >> 16)};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(acc[n], a, qf[n][c * 8 + 2 * e], qf[n][c * 8 + 2 * e + 1]);
          }
        }
        // ---- softmax; lane: tokens g, g + 8 of rows 2 t4, 2 t4 + 1
        const bool edge = tok0 + 16 > all_seen;
        uint32_t pf[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = acc[n][e] * (sk * qs[n][e & 1]);
          if (edge) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (tok0 + g + (e >> 1) * 8 >= seen[n][e & 1]) x[e] = -INFINITY;
          }
          float t0m = fmaxf(x[0], x[2]), t1m = fmaxf(x[1], x[3]);
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) {
            t0m = fmaxf(t0m, __shfl_xor_sync(0xffffffffu, t0m, w));
            t1m = fmaxf(t1m, __shfl_xor_sync(0xffffffffu, t1m, w));
          }
          const bool grow = t0m > m[n][0] + TAU || t1m > m[n][1] + TAU;
          if (__any_sync(0xffffffffu, grow)) {
            const float n0 = fmaxf(m[n][0], t0m), n1 = fmaxf(m[n][1], t1m);
            const float a0 = n0 == -INFINITY ? 1.f : ex2(m[n][0] - n0), a1 = n1 == -INFINITY ? 1.f : ex2(m[n][1] - n1);
            m[n][0] = n0; m[n][1] = n1;
            l[n][0] *= a0; l[n][1] *= a1;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              o[n][i][0] *= a0; o[n][i][1] *= a1; o[n][i][2] *= a0; o[n][i][3] *= a1;
            }
          }
          const float b0 = m[n][0] == -INFINITY ? 0.f : SHIFT - m[n][0], b1 = m[n][1] == -INFINITY ? 0.f : SHIFT - m[n][1];
          const float p0 = ex2(x[0] + b0), p1 = ex2(x[1] + b1), p2 = ex2(x[2] + b0), p3 = ex2(x[3] + b1);
          l[n][0] += p0 + p2;
          l[n][1] += p1 + p3;
          pf[n][0] = transpose8(kv::pack16<true>(p0, p1));
          pf[n][1] = transpose8(kv::pack16<true>(p2, p3));
        }
        // ---- O^T += sv V^T P^T; lane: tokens 2 t4, +1, +8, +9, channels g * D/8 ...
        const uint8_t* vb = sm.v[s];
        constexpr int VW = D / 32;         // 32-bit words of channels per lane
        uint32_t vr[4][VW];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = kg * 16 + 2 * t4 + (j & 1) + (j >> 1) * 8;
          if constexpr (D == 128) {
            const uint4 x = *reinterpret_cast<const uint4*>(vb + swz<D>(r, g));
            vr[j][0] = x.x; vr[j][1] = x.y; vr[j][2] = x.z; vr[j][3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(vb + swz<D>(r, g >> 1) + (g & 1) * 8);
            vr[j][0] = x.x; vr[j][1] = x.y;
          }
        }
        bool poison = false;               // a NaN code that some rows must not see
        if (edge) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int tok = tok0 + 2 * t4 + (j & 1) + (j >> 1) * 8;
#pragma unroll
            for (int w = 0; w < VW; ++w) {
              if (tok >= len) vr[j][w] = 0;      // behind the sequence: never looked at
              const uint32_t mag = vr[j][w] & 0x7f7f7f7fu;
              poison |= ((mag + 0x01010101u) & 0x80808080u) != 0;
            }
          }
          poison = __any_sync(0xffffffffu, poison);
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          const uint32_t lo01 = __byte_perm(vr[0][w], vr[1][w], 0x5140), hi01 = __byte_perm(vr[0][w], vr[1][w], 0x7362);
          const uint32_t lo89 = __byte_perm(vr[2][w], vr[3][w], 0x5140), hi89 = __byte_perm(vr[2][w], vr[3][w], 0x7362);
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const uint32_t u01 = z ? hi01 : lo01, u89 = z ? hi89 : lo89;
            uint32_t a[4] = {kv::decode2(u01 & 0xffff), kv::decode2(u01 >> 16), kv::decode2(u89 & 0xffff), kv::decode2(u89 >> 16)};
            if (poison) {
              // a NaN value reaches only the rows that see its token: it is taken out of the
              // product, and a second product counts the NaNs each row sees
              uint32_t bad[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t lo = (a[e] & 0x7fffu) > 0x7c00u, hi = (a[e] & 0x7fff0000u) > 0x7c000000u;
                bad[e] = (lo ? 0x3c00u : 0u) | (hi ? 0x3c000000u : 0u);
                a[e] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
              }
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                float cnt[4] = {0.f, 0.f, 0.f, 0.f};
                float vis[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) vis[e] = tok0 + g + (e >> 1) * 8 < seen[n][e & 1] ? 1.f : 0.f;
                mma_f16(cnt, bad, transpose8(kv::pack16<true>(vis[0], vis[1])), transpose8(kv::pack16<true>(vis[2], vis[3])));
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (cnt[e] > 0.f) o[n][2 * w + z][e] = __uint_as_float(0x7fffffffu);
              }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float d[4] = {0.f, 0.f, 0.f, 0.f};
              mma_f16(d, a, pf[n][0], pf[n][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e) o[n][2 * w + z][e] = fmaf(d[e], sv, o[n][2 * w + z][e]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sm.empty[s]);
    }
    at += t1 - t0;

    // ---- the warps' partial results join: O of key group wk at sm.o[wk]
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = l[n][c];
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
        const int r = (wr * NT + n) * 8 + 2 * t4 + c;
        if (g == 0) {
          sm.ml[wk][r][0] = m[n][c];
          sm.ml[wk][r][1] = x;
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          // channels g * D/8 + 2 i, + 1
          *reinterpret_cast<float2*>(&sm.o[wk][r][g * (D / 8) + 2 * i]) = make_float2(o[n][i][c], o[n][i][2 + c]);
        }
      }
    }
    tc::bar_sync_named(1, NW * 32);
    const bool whole = t0 == 0 && t1 == nt;
    const bool bad = aborted();
    const int slot = 2 * blockIdx.x + (t0 > 0 ? 0 : 1);   // a share's first segment may end a unit, its last may begin one
    for (int i = tid; i < ROWS * (D / 4); i += NW * 32) {
      const int r = i / (D / 4), c = i % (D / 4);
      float mx = -INFINITY;
#pragma unroll
      for (int k = 0; k < WK; ++k) mx = fmaxf(mx, sm.ml[k][r][0]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float ls = 0.f;
#pragma unroll
      for (int k = 0; k < WK; ++k) {
        // (m = -inf: no visible key, O and l are 0, or all of its scores are NaN, and so are they)
        const float f = sm.ml[k][r][0] == -INFINITY ? 1.f : ex2(sm.ml[k][r][0] - mx);
        const float4 x = *reinterpret_cast<const float4*>(&sm.o[k][r][c * 4]);
        acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
        ls += f * sm.ml[k][r][1];
      }
      if (bad) acc = make_float4(NAN, NAN, NAN, NAN);
      if (!whole) {
        float* dst = p.part + ((int64_t)slot * ROWS + r) * D + c * 4;
        *reinterpret_cast<float4*>(dst) = acc;
        if (c == 0) {
          float* ml = p.part + (int64_t)2 * gridDim.x * ROWS * D + ((int64_t)slot * ROWS + r) * 2;
          ml[0] = mx;
          ml[1] = ls;
        }
      } else {
        const int rr = rb * p.rows + r;
        if (rr < p.R) {
          const float inv = ls > 0.f || ls != ls ? 1.f / ls : 0.f;
          const int64_t orow = ((int64_t)b * p.Sq + rr / p.G) * p.Hq + h * p.G + rr % p.G;
          uint2 w;
          w.x = kv::pack16<F16>(acc.x * inv, acc.y * inv);
          w.y = kv::pack16<F16>(acc.z * inv, acc.w * inv);
          *reinterpret_cast<uint2*>(reinterpret_cast<char*>(p.o) + 2 * (orow * D + c * 4)) = w;
          if (c == 0 && p.lse) p.lse[orow] = ls == 0.f ? -INFINITY : (mx - SHIFT + log2f(ls)) * 0.6931471805599453f;
        }
      }
    }
    tc::bar_sync_named(1, NW * 32);
  }
}

// Joins the partials of the units that cross shares, and writes the empty sequences.
// One block per (sequence, kv head, row block).
template <int D, bool F16, int ROWS>
__global__ void __launch_bounds__(128) attn_cached_join_kernel(Params p, int ctas) {
  const int lane = threadIdx.x & 31;
  const int64_t units = (int64_t)p.H * p.rblocks;
  const int b = (int)(blockIdx.x / units), u = (int)(blockIdx.x % units);
  const int h = u / p.rblocks, rb = u % p.rblocks;
  const int nt = seq_tiles(p, b);
  // tiles of the sequences before b, and of all (every warp for itself)
  int64_t before = 0, sum = 0;
  for (int i = lane; i < p.B; i += 32) {
    const int x = seq_tiles(p, i);
    sum += x;
    if (i < b) before += x;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  const Share sh = share_of(p, units, sum, ctas);
  int c0 = 0, c1 = -1;                     // CTAs whose shares hold a part of this unit
  int64_t begin = 0;
  if (nt > 0) {
    begin = before * units + (int64_t)u * nt;
    c0 = (int)(begin / sh.per);
    c1 = (int)((begin + nt - 1) / sh.per);
    if (c0 == c1) return;                  // finished there
  }
  const float* mlp = p.part + (int64_t)2 * ctas * ROWS * D;
  for (int i = threadIdx.x; i < ROWS * (D / 4); i += 128) {
    const int r = i / (D / 4), c = i % (D / 4), rr = rb * p.rows + r;
    if (rr >= p.R) break;
    float mx = -INFINITY, ls = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    // the part that begins the unit is its CTA's last segment (slot 1), the later ones
    // continue it (slot 0)
    for (int k = c0; k <= c1; ++k) {
      const int64_t slot = 2 * (int64_t)k + (k == c0 ? 1 : 0);
      const float m = mlp[(slot * ROWS + r) * 2], l = mlp[(slot * ROWS + r) * 2 + 1];
      const float mn = fmaxf(mx, m), f0 = mx == -INFINITY ? 1.f : ex2(mx - mn), f1 = m == -INFINITY ? 1.f : ex2(m - mn);
      const float4 x = *reinterpret_cast<const float4*>(p.part + (slot * ROWS + r) * D + c * 4);
      acc.x = acc.x * f0 + x.x * f1; acc.y = acc.y * f0 + x.y * f1;
      acc.z = acc.z * f0 + x.z * f1; acc.w = acc.w * f0 + x.w * f1;
      ls = ls * f0 + l * f1;
      mx = mn;
    }
    const float inv = ls > 0.f || ls != ls ? 1.f / ls : 0.f;
    const int64_t orow = ((int64_t)b * p.Sq + rr / p.G) * p.Hq + h * p.G + rr % p.G;
    uint2 w;
    w.x = kv::pack16<F16>(acc.x * inv, acc.y * inv);
    w.y = kv::pack16<F16>(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(reinterpret_cast<char*>(p.o) + 2 * (orow * D + c * 4)) = w;
    if (c == 0 && p.lse) p.lse[orow] = ls == 0.f ? -INFINITY : (mx - SHIFT + log2f(ls)) * 0.6931471805599453f;
  }
}

// Rows that a CTA takes: 8, 16, 32 or 64 of the R = Sq * Hq / Hkv.
static int block_rows(int64_t R) { return R <= 8 ? 8 : R <= 16 ? 16 : R <= 32 ? 32 : 64; }

static int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  else cudaGetLastError();
  return n;
}

// CTAs of the main kernel: as many as fit on the GPU at once, no more than there can be tiles.
static int grid_of(int64_t B, int64_t H, int64_t R, int64_t max_tokens) {
  const int rows = block_rows(R);
  const int64_t most = B * H * ((R + rows - 1) / rows) * ((max_tokens + TK - 1) / TK);
  const int64_t fit = (int64_t)sm_count() * (rows == 8 ? 2 : 1);
  return (int)(most < 1 ? 1 : most < fit ? most : fit);
}

template <int D, bool F16, int NT, int WR, int STAGES, int OCC>
static int launch(const Maps& maps, const Params& p, int grid, cudaStream_t st) {
  using SM = Smem<D, NT, WR, STAGES>;
  const size_t smem = sizeof(SM) + 1024;
  auto* kern = attn_cached_kernel<D, F16, NT, WR, STAGES, OCC>;
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  kern<<<grid, THREADS, smem, st>>>(maps, p);
  if (int e = check_launch("attn_cached_kernel")) return e;
  attn_cached_join_kernel<D, F16, SM::ROWS><<<(unsigned)((int64_t)p.B * p.H * p.rblocks), 128, 0, st>>>(p, grid);
  return check_launch("attn_cached_join_kernel");
}

template <int D, bool F16>
static int launch_rows(const Maps& maps, const Params& p, int grid, cudaStream_t st) {
  constexpr int S8 = D == 128 ? 2 : 4, S16 = D == 128 ? 4 : 6;
  if (p.rows == 8) return launch<D, F16, 1, 1, S8, 2>(maps, p, grid, st);
  if (p.rows == 16) return launch<D, F16, 2, 1, S16, 1>(maps, p, grid, st);
  if (p.rows == 32) return launch<D, F16, 2, 2, S16, 1>(maps, p, grid, st);
  return launch<D, F16, 2, 4, S16, 1>(maps, p, grid, st);
}

static int make_map(CUtensorMap* m, const void* base, uint64_t rows, int D, int page) {
  tc::EncodeTiledFn fn = tc::encode_tiled_fn();
  if (!fn) return set_error(KB200_ERR_LAUNCH, "attn_cached: cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {(cuuint64_t)D, rows};
  cuuint64_t strides[1] = {(cuuint64_t)D};
  cuuint32_t box[2] = {(cuuint32_t)D, (cuuint32_t)page};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(KB200_ERR_LAUNCH, "attn_cached: tensor map encode failed (%d)", (int)r);
  return KB200_OK;
}

static int check_shape(int64_t B, int64_t Sq, int64_t Hq, int64_t H, int64_t max_pages) {
  if (B < 0 || Sq < 0 || B > (1 << 20) || Sq > 4096 || Hq < 1 || H < 1 || Hq % H || Hq > (1 << 16) || max_pages < 0 ||
      max_pages > (1 << 26) || B * Sq * Hq > 0x7fffffffLL)
    return set_error(KB200_ERR_INVALID, "attn_cached: B=%lld Sq=%lld Hq=%lld Hkv=%lld max_pages=%lld", (long long)B,
                     (long long)Sq, (long long)Hq, (long long)H, (long long)max_pages);
  return KB200_OK;
}

}  // namespace cached
}  // namespace kb

extern "C" size_t kb200_attn_cached_workspace_size(int64_t B, int64_t Sq, int64_t Hq, int64_t Hkv, int64_t D,
                                                   int64_t page, int64_t max_pages) {
  using namespace kb::cached;
  if (check_shape(B, Sq, Hq, Hkv, max_pages) || page < 1 || page > 128) return 0;
  if (B == 0 || Sq == 0) return 256;
  const int64_t R = Sq * (Hq / Hkv);
  const int grid = grid_of(B, Hkv, R, max_pages * page);
  return (size_t)2 * grid * block_rows(R) * (D + 2) * sizeof(float);
}

extern "C" int kb200_attn_cached_fwd(const void* q, int64_t q_batch_stride, int64_t q_token_stride, int64_t q_head_stride,
                                     const KB200KvCache* c, const int32_t* page_table, int64_t max_pages,
                                     const int32_t* lengths, void* o, float* lse, int64_t B, int64_t Sq, int64_t Hq,
                                     float softmax_scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace kb;
  if (int e = kv::check_cache(c, "attn_cached")) return e;
  if (int e = cached::check_shape(B, Sq, Hq, c->H, max_pages)) return e;
  if (dtype != 0 && dtype != 1) return set_error(KB200_ERR_INVALID, "attn_cached: dtype=%d", dtype);
  if (B == 0 || Sq == 0) return KB200_OK;
  if (!q || !o || !lengths || (max_pages > 0 && !page_table)) return set_error(KB200_ERR_INVALID, "attn_cached: null pointer");
  if (!aligned16(q) || !aligned16(o) || ((q_batch_stride | q_token_stride | q_head_stride) & 7))
    return set_error(KB200_ERR_ALIGN, "attn_cached: q and o rows must be 16-byte aligned");
  const size_t need = kb200_attn_cached_workspace_size(B, Sq, Hq, c->H, c->D, c->page, max_pages);
  if (!workspace || workspace_bytes < need || !aligned16(workspace))
    return set_error(KB200_ERR_WORKSPACE, "attn_cached: workspace of %zu bytes needed, got %zu", need, workspace_bytes);
  const int64_t G = Hq / c->H, R = Sq * G;
  const int rows = cached::block_rows(R);
  const int64_t rblocks = (R + rows - 1) / rows;
  if (B * c->H * rblocks > 0x7fffffffLL) return set_error(KB200_ERR_INVALID, "attn_cached: too many rows");
  cached::Params p{};
  p.q = q; p.o = o; p.lse = lse; p.table = page_table; p.lengths = lengths;
  p.k_scale = c->k_scale; p.v_scale = c->v_scale; p.part = (float*)workspace;
  p.q_bs = q_batch_stride; p.q_ts = q_token_stride; p.q_hs = q_head_stride;
  p.B = (int)B; p.Sq = (int)Sq; p.Hq = (int)Hq; p.H = (int)c->H; p.G = (int)G; p.R = (int)R;
  p.rblocks = (int)rblocks; p.rows = rows;
  p.num_pages = (int)c->num_pages; p.max_pages = (int)max_pages; p.page = (int)c->page;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  cached::Maps maps;
  const uint64_t mrows = (uint64_t)c->num_pages * c->H * c->page;
  if (int e = cached::make_map(&maps.k, c->k_pages, mrows, (int)c->D, (int)c->page)) return e;
  if (int e = cached::make_map(&maps.v, c->v_pages, mrows, (int)c->D, (int)c->page)) return e;
  const int grid = cached::grid_of(B, c->H, R, max_pages * c->page);
  cudaStream_t st = (cudaStream_t)stream;
  if (c->D == 64)
    return dtype ? cached::launch_rows<64, true>(maps, p, grid, st) : cached::launch_rows<64, false>(maps, p, grid, st);
  return dtype ? cached::launch_rows<128, true>(maps, p, grid, st) : cached::launch_rows<128, false>(maps, p, grid, st);
}
