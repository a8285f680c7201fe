// attn_prompt.cu -- causal softmax attention over packed prompts with grouped heads, on
// 5th-generation tensor cores (tcgen05 + TMEM + TMA).
//
//   o_i = sum_{j <= i + m - n} softmax_j(scale q_i . k_j) v_j     (n queries at the end of m keys)
//
// Bound: the tensor pipe and the exponentials together.  A tile of 256 rows x 128 keys is
// 4 * 256 * 128 * D flops (2048 cycles at D = 128) and 32768 exponentials (2048 cycles of MUFU).
//
// Rows.  The G = Hq / Hkv heads that share a kv head are rows of one matrix, row
// r = token * G + head in group, so a CTA of 256 rows reads each key tile once for all of
// them, and short prompts still fill the tile.  Any G works: Q is fetched with plain
// loads, K and V by TMA (boxes of 64 channels x 128 tokens of one head, any token stride).
//
// Order.  CTA c takes tile c / Hkv of all sequences' tiles sorted by their number of
// keys, most first (each CTA finds its own by a search over the levels: no host
// knowledge of the lengths, no extra launch); the short ones fill the end of the run.
//
// One CTA, 12 warps (one idles: registers are dealt by warpgroups of four):
//   warps 0-7  softmax: query tile t = w / 4, one row per thread (its 128 scores in registers)
//   warp 8     TMA producer: K and V tiles into their rings
//   warp 9     issues S = Q_t K_j^T, in the order QK_0(j) QK_1(j): the two query tiles share one
//              TMEM score buffer, which a tile gives back as soon as its scores are in registers
//   warp 10    issues O_t += P_t V_j (P_t from TMEM, V read MN-major from its TMA tile)
// What a period of 256 rows x 128 keys takes is the chain QK_0 - load - QK_1 - load: each link
// is 512 cycles of product, the two hand-offs and the load.  So the loads read whole lanes
// (32x32b; the 16-lane shapes run at half the rate) and the two kinds of products have
// an issuer each, so that no QK waits behind a PV's operands.
// The row maximum is kept lazily: O and l are rescaled only when it grows by more than
// TAU (log2 units), so P <= 2^(SHIFT + TAU) (inside f16) and most tiles rescale nothing.
// P is rounded to the input type (half a step, as the output is); l sums the unrounded P.
//
// Keys that a row does not see score -inf, so their P is 0.  V rows behind the sequence are
// zeroed in shared memory before the product.  A NaN or an infinity in V at a key that a
// row must not see still reaches it as 0 * NaN: so a row whose O is not finite is computed again,
// by its warp, over its visible keys alone (and if one of those is the cause, the result is
// what it should be).
//
// Every wait is bounded.  A warp whose wait gives up stops, so that the others' waits give up
// too; what is in flight is drained, and the CTA writes NaN.
#include <math.h>
#include <string.h>
#include "kb200_internal.h"
#include "kv_cache.cuh"
#include "tc_common.cuh"

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
  float scale_log2;        // |softmax scale| log2 e; its sign goes into q (flip)
  uint32_t flip;
  uint64_t g_magic;        // ceil(2^32 / G): x / G = x g_magic >> 32 for x G < 2^32
  int causal;
};

KB_DEVI float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^x for a pair on the FMA pipe: x = j + f, f in [-1/2, 1/2], by adding and taking away 1.5 * 2^23;
// 2^f by a polynomial of degree 4 (least squares on the relative error, reweighted towards the
// largest: 2.9e-6), times 2^j by its exponent field, which is 0 at j = -127: x below -126 gives 0.
// A NaN stays one.
KB_DEVI float2 exp2_poly(float2 x) {
  constexpr float C = 12582912.f;
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.x));      // -127
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.y));
  const float2 t = fadd2(x, make_float2(C, C));
  const float2 j = fadd2(t, make_float2(-C, -C));
  const float2 f = ffma2(j, make_float2(-1.f, -1.f), x);
  float2 q = ffma2(make_float2(0.00958285323f, 0.00958285323f), f, make_float2(0.055906426f, 0.055906426f));
  q = ffma2(q, f, make_float2(0.240240986f, 0.240240986f));
  q = ffma2(q, f, make_float2(0.693124193f, 0.693124193f));
  q = ffma2(q, f, make_float2(1.f, 1.f));
  return fmul2(q, make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000),
                              __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000)));
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
    q[c] = load16<F16>(p.q, tq * p.q_ts + h * p.q_hs + c * 32 + lane) * (p.flip ? -p.scale_log2 : p.scale_log2);
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

constexpr int BM = 128, BN = 128, QT = 2, ROWS = QT * BM;
constexpr float SHIFT = 6.f, TAU = 8.f;      // P = 2^(s - m + SHIFT) <= 2^14
constexpr int THREADS = 12 * 32;
// Registers: the launch gives each thread 168 (its 384 threads share the SM's 65536); the softmax
// warpgroups take 208 and the third leaves itself 88, 2 * 208 + 88 = 3 * 168.
constexpr int REGS_SOFTMAX = 208, REGS_OTHERS = 88;
constexpr int SORTED = 64;                   // up to this many sequences the tiles are sorted by their keys
constexpr uint32_t TM_O = 0, TM_S = 256, TM_P = 384;   // TMEM columns: O_t at 128 t, S, P_t at 64 t

struct Maps {
  CUtensorMap k, v;
};

template <int D>
struct Smem {
  static constexpr int KS = D == 128 ? 3 : 4, VS = D == 128 ? 2 : 4;
  static constexpr int ATOMS = D / 64;       // 64 channels: 128 swizzled bytes
  uint8_t q[QT][ATOMS][BM * 128];
  uint8_t k[KS][ATOMS][BN * 128];
  uint8_t v[VS][ATOMS][BN * 128];
  uint64_t q_full;
  uint64_t k_full[KS], k_empty[KS], v_full[VS], v_empty[VS];
  uint64_t s_full[QT], s_free[QT], p_full[QT], pv_done[QT], o_done, drain[2];
  uint32_t tmem_base;
  int seq, tile;                             // this CTA's sequence (-1: none) and row tile in it
  int4 range;                                // its queries and keys
  int abort_flag, keep_tmem;
};

// Tile `r` of the order above: sequence and tile in it, by one warp (seq = -1: there is none).
KB_DEVI void find_tile(const Params& p, int64_t r, int lane, int& seq, int& tile) {
  auto tiles_of = [&](int s, int& level) {   // row tiles of sequence s; level of its first one
    const int2 q = seq_range(p.cu_q, s, p.Tq), k = seq_range(p.cu_k, s, p.Tk);
    const int n = q.y - q.x;
    level = p.causal ? (int)(max(k.y - k.x - n, 0) * (int64_t)p.G / ROWS) : 0;
    return (int)(((int64_t)n * p.G + ROWS - 1) / ROWS);
  };
  seq = -1;
  tile = 0;
  if (p.causal && p.N <= SORTED) {
    int nt[SORTED / 32], lv[SORTED / 32], top = 0;
#pragma unroll
    for (int i = 0; i < SORTED / 32; ++i) {
      const int s = lane + 32 * i;
      nt[i] = lv[i] = 0;
      if (s < p.N) nt[i] = tiles_of(s, lv[i]);
      if (nt[i]) top = max(top, lv[i] + nt[i]);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    auto above = [&](int L) {                // tiles with level >= L
      int c = 0;
#pragma unroll
      for (int i = 0; i < SORTED / 32; ++i) c += min(max(lv[i] + nt[i] - L, 0), nt[i]);
      return (int)__reduce_add_sync(0xffffffffu, (unsigned)c);
    };
    if (r >= above(0)) return;
    int lo = 0, hi = top;                    // above(lo) > r >= above(hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (above(mid) > r) lo = mid; else hi = mid;
    }
    int k = (int)(r - above(lo + 1));        // k-th of the tiles of level lo
#pragma unroll
    for (int i = 0; i < SORTED / 32; ++i) {
      const bool mine = lo >= lv[i] && lo < lv[i] + nt[i];
      const uint32_t m = __ballot_sync(0xffffffffu, mine);
      if (seq < 0 && k < __popc(m)) {
        const int l = __fns(m, 0, k + 1);
        seq = l + 32 * i;
        tile = lo - __shfl_sync(0xffffffffu, lv[i], l);
      }
      if (seq < 0) k -= __popc(m);
    }
    return;
  }
  int64_t base = 0;
  for (int s0 = 0; s0 < p.N; s0 += 32) {
    int lv;
    const int mine = s0 + lane < p.N ? tiles_of(s0 + lane, lv) : 0;
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, base + inc > r);
    if (hit) {
      const int l = __ffs(hit) - 1;
      seq = s0 + l;
      tile = (int)(r - (base + __shfl_sync(0xffffffffu, inc - mine, l)));
      return;
    }
    base += __shfl_sync(0xffffffffu, inc, 31);
  }
}

// One arrival per warp, after its TMEM reads or writes.
KB_DEVI void warp_arrive(uint64_t* bar, int lane) {
  tc::tc_fence_before();
  __syncwarp();
  if (lane == 0) tc::mbar_arrive(bar);
}

// Which of every 8 pairs of exponentials go to the FMA pipe.
#ifndef KB_POLY
#define KB_POLY (D == 128 ? 0x88 : 0x88)
#endif

template <int D, bool F16>
__global__ void __launch_bounds__(THREADS, 1) attn_prompt_kernel(const __grid_constant__ Maps maps, Params p) {
  using SM = Smem<D>;
  constexpr int POLY = KB_POLY;
  constexpr int KS = SM::KS, VS = SM::VS, ATOMS = SM::ATOMS;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  SM& sm = *reinterpret_cast<SM*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hk = blockIdx.x % p.H;

  if (warp == 0) {
    int s, t;
    find_tile(p, blockIdx.x / p.H, lane, s, t);
    if (lane == 0) {
      sm.seq = s;
      sm.tile = t;
      if (s >= 0) {
        const int2 q = seq_range(p.cu_q, s, p.Tq), k = seq_range(p.cu_k, s, p.Tk);
        sm.range = make_int4(q.x, q.y, k.x, k.y);
      }
    }
  } else if (warp == 8) {
    if (lane == 0) {
      tc::mbar_init(&sm.q_full, 8);
      for (int s = 0; s < KS; ++s) {
        tc::mbar_init(&sm.k_full[s], 1);
        tc::mbar_init(&sm.k_empty[s], 1);
      }
      for (int s = 0; s < VS; ++s) {
        tc::mbar_init(&sm.v_full[s], 1);
        tc::mbar_init(&sm.v_empty[s], 1);
      }
      for (int i = 0; i < QT; ++i) {
        tc::mbar_init(&sm.s_full[i], 1);
        tc::mbar_init(&sm.s_free[i], 4);
        tc::mbar_init(&sm.p_full[i], 4);
        tc::mbar_init(&sm.pv_done[i], 1);
      }
      tc::mbar_init(&sm.o_done, 1);
      tc::mbar_init(&sm.drain[0], 1);
      tc::mbar_init(&sm.drain[1], 1);
      sm.abort_flag = 0;
      sm.keep_tmem = 0;
      tc::fence_barrier_init();
      tc::prefetch_tmap(&maps.k);
      tc::prefetch_tmap(&maps.v);
    }
  } else if (warp == 9) {
    tc::tmem_alloc(&sm.tmem_base, 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  const int seq = sm.seq;
  if (seq < 0) {
    if (warp == 9) tc::tmem_dealloc(tmem, 512);
    return;
  }
  const int2 rq = make_int2(sm.range.x, sm.range.y), rk = make_int2(sm.range.z, sm.range.w);
  const int n = rq.y - rq.x, m = rk.y - rk.x;
  const int64_t row0 = (int64_t)sm.tile * ROWS;              // first row (token * G + head)
  const int64_t nrows = min((int64_t)ROWS, (int64_t)n * p.G - row0);
  // keys that token t of the sequence sees
  auto seen_by = [&](int64_t t) { return p.causal ? (int)min((int64_t)m, max((int64_t)0, t + 1 + m - n)) : m; };
  const int ntiles = (seen_by((row0 + nrows - 1) / p.G) + BN - 1) / BN;
  const int full = seen_by(row0 / p.G) / BN;                 // key tiles below are seen fully by every row
  auto aborted = [&]() { return *((volatile int*)&sm.abort_flag) != 0; };

  if (warp >= 8) {
    tc::setmaxnreg_dec<REGS_OTHERS>();
  if (warp == 8) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0 && ntiles > 0) {
      int kiss = 0, viss = 0;
      for (int j = 0; j < ntiles; ++j) {
        const int sk = j % KS, sv = j % VS, tok = rk.x + j * BN;
        if (j >= KS && !tc::mbar_wait(&sm.k_empty[sk], (j / KS - 1) & 1)) { sm.abort_flag = 1; break; }
        tc::mbar_expect_tx(&sm.k_full[sk], ATOMS * BN * 128);
        for (int a = 0; a < ATOMS; ++a) tc::tma_load_3d(sm.k[sk][a], &maps.k, &sm.k_full[sk], a * 64, hk, tok);
        ++kiss;
        if (j >= VS && !tc::mbar_wait(&sm.v_empty[sv], (j / VS - 1) & 1)) { sm.abort_flag = 1; break; }
        tc::mbar_expect_tx(&sm.v_full[sv], ATOMS * BN * 128);
        for (int a = 0; a < ATOMS; ++a) tc::tma_load_3d(sm.v[sv][a], &maps.v, &sm.v_full[sv], a * 64, hk, tok);
        ++viss;
      }
      // before the CTA may exit, every load it issued must have landed
      bool drained = true;
      for (int j = kiss > KS ? kiss - KS : 0; j < kiss; ++j) drained &= tc::mbar_wait(&sm.k_full[j % KS], (j / KS) & 1);
      for (int j = viss > VS ? viss - VS : 0; j < viss; ++j) drained &= tc::mbar_wait(&sm.v_full[j % VS], (j / VS) & 1);
      if (!drained) { sm.abort_flag = 1; sm.keep_tmem = 1; }
    }
  } else if (warp == 9 || warp == 10) {
    // ------------------------------------------------------------ MMA issuers
    // The whole warp runs the schedule, so every operand is warp-uniform; one elected lane issues.
    if (ntiles > 0) {
      const bool leader = tc::elect_one();
      constexpr uint64_t ATOM = BN * 128 / 16;               // descriptor units between 64-channel atoms
      const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        const bool w = __all_sync(0xffffffffu, tc::mbar_wait(bar, parity));
        tc::tc_fence_after();
        return w;
      };
      bool ok = true;
      if (warp == 9) {
        constexpr uint32_t IDESC_QK = tc::idesc_f32acc(F16 ? 0 : 1, BM, BN, 0, 0);
        const uint64_t dq0 = tc::sdesc_sw128_kmajor(sm.q[0][0]);
        const uint64_t dk0 = tc::sdesc_sw128_kmajor(sm.k[0][0]);
        auto qk = [&](int t, int j) {   // S = Q_t K_j^T
          const uint64_t dq = dq0 + (uint64_t)(t * ATOMS) * ATOM, dk = dk0 + (uint64_t)((j % KS) * ATOMS) * ATOM;
          if (leader) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
              tc::mma_bf16(tmem_u + TM_S, dq + (ks >> 2) * ATOM + 2 * (ks & 3), dk + (ks >> 2) * ATOM + 2 * (ks & 3), IDESC_QK,
                           ks > 0 ? 1u : 0u);
            tc::tc_commit(&sm.s_full[t]);
            if (t == 1) tc::tc_commit(&sm.k_empty[j % KS]);
          }
          __syncwarp();
        };
        ok = wait(&sm.q_full, 0) && wait(&sm.k_full[0], 0);
        if (ok) qk(0, 0);
        for (int j = 0; ok && j < ntiles; ++j) {
          ok = wait(&sm.s_free[0], j & 1);
          if (!ok) break;
          qk(1, j);
          if (j + 1 < ntiles) {
            ok = wait(&sm.k_full[(j + 1) % KS], ((j + 1) / KS) & 1) && wait(&sm.s_free[1], j & 1);
            if (ok) qk(0, j + 1);
          }
        }
      } else {
        constexpr uint32_t IDESC_PV = tc::idesc_f32acc(F16 ? 0 : 1, BM, D, 0, 1);
        const uint64_t dv0 = tc::sdesc_sw128_mnmajor(sm.v[0][0], BN * 128);
        for (int j = 0; ok && j < ntiles; ++j) {
          ok = wait(&sm.v_full[j % VS], (j / VS) & 1);
          if (ok && (j + 1) * BN > m) {                      // the sequence ends in this tile
            uint4* v = reinterpret_cast<uint4*>(sm.v[j % VS][0]);
            for (int a = 0; a < ATOMS; ++a)
              for (int i = (m - j * BN) * 8 + lane; i < BN * 8; i += 32) v[a * BN * 8 + i] = make_uint4(0, 0, 0, 0);
            tc::fence_proxy_async_smem();
            __syncwarp();
          }
          const uint64_t dv = dv0 + (uint64_t)((j % VS) * ATOMS) * ATOM;
          for (int t = 0; ok && t < QT; ++t) {               // O_t += P_t V_j, 16 keys per instruction
            ok = wait(&sm.p_full[t], j & 1);
            if (ok && leader) {
#pragma unroll
              for (int ks = 0; ks < BN / 16; ++ks)
                tc::mma_bf16_ts(tmem_u + TM_O + t * 128, tmem_u + TM_P + t * 64 + ks * 8, dv + ks * (16 * 128 / 16), IDESC_PV,
                                (j > 0 || ks > 0) ? 1u : 0u);
              tc::tc_commit(&sm.pv_done[t]);
              if (t == 1) tc::tc_commit(&sm.v_empty[j % VS]);
            }
            __syncwarp();
          }
        }
        if (ok && leader) tc::tc_commit(&sm.o_done);
        __syncwarp();
      }
      if (!ok) sm.abort_flag = 1;
      // every MMA this warp issued must complete before TMEM is freed
      if (leader) tc::tc_commit(&sm.drain[warp - 9]);
      __syncwarp();
      if (!__all_sync(0xffffffffu, tc::mbar_wait(&sm.drain[warp - 9], 0))) {
        sm.abort_flag = 1;
        sm.keep_tmem = 1;
      }
    }
  }
  } else {
    // ------------------------------------------------------------ softmax
    tc::setmaxnreg_inc<REGS_SOFTMAX>();
    // Q into shared memory: 256 rows of D channels, 16 bytes at a time
    const uint32_t flip = p.flip;                            // 0x80008000: a negative scale, moved into q
    constexpr int CPR = D / 8, BATCH = 8;                    // 16-byte chunks of a row; loads in flight per thread
    const int64_t tok0 = row0 / p.G;
    const uint32_t rem0 = (uint32_t)(row0 - tok0 * p.G);
    // token of row r of the tile (from tok0) and head in the group
    auto split = [&](int r, int& dt, int& hg) {
      const uint32_t x = rem0 + r;
      dt = (int)((x * p.g_magic) >> 32);
      hg = (int)(x - dt * p.G);
    };
    const char* qbase = reinterpret_cast<const char*>(p.q) + 2 * ((rq.x + tok0) * p.q_ts + (int64_t)hk * p.G * p.q_hs);
    if (ntiles > 0) {
#pragma unroll 1
      for (int i0 = tid; i0 < ROWS * CPR; i0 += 256 * BATCH) {
        uint4 x[BATCH];
#pragma unroll
        for (int z = 0; z < BATCH; ++z) {
          const int i = i0 + z * 256, r = i / CPR, c = i % CPR;
          x[z] = make_uint4(0, 0, 0, 0);
          if (r < nrows) {
            int dt, hg;
            split(r, dt, hg);
            x[z] = __ldg(reinterpret_cast<const uint4*>(qbase + 2 * (dt * p.q_ts + hg * p.q_hs + c * 8)));
          }
        }
#pragma unroll
        for (int z = 0; z < BATCH; ++z) {
          const int i = i0 + z * 256, r = i / CPR, c = i % CPR, rr = r % BM;
          x[z].x ^= flip; x[z].y ^= flip; x[z].z ^= flip; x[z].w ^= flip;
          *reinterpret_cast<uint4*>(&sm.q[r / BM][c / 8][rr * 128 + (((c % 8) ^ (rr & 7)) << 4)]) = x[z];
        }
      }
    }
    tc::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&sm.q_full);

    const int qt = warp >> 2, w4 = warp & 3;
    const int r = qt * BM + w4 * 32 + lane;                  // this thread's row; its TMEM lane is r % 128
    const uint32_t lane_off = (uint32_t)(w4 * 32) << 16;
    const uint32_t tS = tmem + TM_S + lane_off, tO = tmem + TM_O + qt * 128 + lane_off, tP = tmem + TM_P + qt * 64 + lane_off;
    const float sl2 = p.scale_log2;
    const bool live = r < nrows;
    int my_dt, my_hg;
    split(r, my_dt, my_hg);
    const int lim = live ? seen_by(tok0 + my_dt) : 0x7fffffff;   // keys that the row sees
    float mref = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < ntiles; ++j) {
      if (!tc::mbar_wait(&sm.s_full[qt], j & 1)) { sm.abort_flag = 1; ok = false; }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc::tc_fence_after();
      uint32_t s[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tc::tmem_ld32(tS + c * 32, s + c * 32);
      tc::tmem_wait_ld();
      warp_arrive(&sm.s_free[qt], lane);
      if (j >= full) {
        const int end = lim - j * BN;
#pragma unroll
        for (int c0 = 0; c0 < BN; c0 += 32)
          if (__any_sync(0xffffffffu, end < c0 + 32)) {
#pragma unroll
            for (int c = c0; c < c0 + 32; ++c)
              if (c >= end) s[c] = __float_as_uint(-INFINITY);
          }
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < BN; c += 8)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mx[i] = fmaxf(mx[i], fmaxf(__uint_as_float(s[c + 2 * i]), __uint_as_float(s[c + 2 * i + 1])));
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2;
      const bool grow = __any_sync(0xffffffffu, top > mref + TAU);
      float alpha = 1.f;
      if (grow) {
        const float mn = fmaxf(mref, top);
        if (mn != -INFINITY) alpha = ex2(mref - mn);
        mref = mn;
        l *= alpha;
      }
      // (no key of the row seen yet: every score here is -inf, and so is x)
      const float b0 = mref == -INFINITY ? 0.f : SHIFT - mref;
      const float2 sc = make_float2(sl2, sl2), bias = make_float2(b0, b0);
      float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const int i = h * 64 + 2 * c;
          const float2 x = ffma2(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), sc, bias);
          const float2 e = ((POLY >> (c & 7)) & 1) ? exp2_poly(x) : make_float2(ex2(x.x), ex2(x.y));
          ls[c & 1] = fadd2(ls[c & 1], e);
          pk[c] = kv::pack16<F16>(e.x, e.y);
        }
        if (h == 0) {
          // P_t(j) overwrites P_t(j-1) and O_t may be rescaled: PV_t(j-1) must have completed
          if (j >= 1 && !tc::mbar_wait(&sm.pv_done[qt], (j - 1) & 1)) { sm.abort_flag = 1; ok = false; }
          ok = __all_sync(0xffffffffu, ok);
          tc::tc_fence_after();
        }
        if (ok) tc::tmem_st32(tP + h * 32, pk);
      }
      if (!ok) break;
      l += (ls[0].x + ls[0].y) + (ls[1].x + ls[1].y);
      if (grow && j >= 1) {
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tc::tmem_ld32(tO + c * 32, o);
          tc::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tc::tmem_st32(tO + c * 32, o);
        }
      }
      tc::tmem_wait_st();
      warp_arrive(&sm.p_full[qt], lane);
    }
    // ---- epilogue
    if (ok && ntiles > 0) ok = __all_sync(0xffffffffu, tc::mbar_wait(&sm.o_done, 0));
    if (!ok) sm.abort_flag = 1;
    tc::tc_fence_after();
    const float f = !ok || aborted() ? NAN : l == 0.f ? 0.f : 1.f / l;
    // through this warp's part of the Q tile (every product has read Q), so that rows are stored whole
    uint8_t* stage = sm.q[qt][0] + w4 * 32 * (D * 2);
    bool finite = true;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      uint32_t o[32];
      if (ntiles > 0 && ok) {
        tc::tmem_ld32(tO + c * 32, o);
        tc::tmem_wait_ld();
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0;
      }
      float worst = 0.f;                                     // NaN if some value is not finite: inf - inf
#pragma unroll
      for (int e = 0; e < 32; ++e) worst = fmaf(__uint_as_float(o[e]), 0.f, worst);
      finite &= worst == 0.f;
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        uint4 x;
        x.x = kv::pack16<F16>(__uint_as_float(o[8 * z + 0]) * f, __uint_as_float(o[8 * z + 1]) * f);
        x.y = kv::pack16<F16>(__uint_as_float(o[8 * z + 2]) * f, __uint_as_float(o[8 * z + 3]) * f);
        x.z = kv::pack16<F16>(__uint_as_float(o[8 * z + 4]) * f, __uint_as_float(o[8 * z + 5]) * f);
        x.w = kv::pack16<F16>(__uint_as_float(o[8 * z + 6]) * f, __uint_as_float(o[8 * z + 7]) * f);
        *reinterpret_cast<uint4*>(stage + lane * (D * 2) + (((c * 4 + z) ^ (lane & 7)) << 4)) = x;
      }
    }
    __syncwarp();
    char* obase = reinterpret_cast<char*>(p.o) + 2 * ((rq.x + tok0) * p.o_ts + (int64_t)hk * p.G * p.o_hs);
#pragma unroll 8
    for (int z = 0; z < CPR; ++z) {                          // 32 / CPR rows at a time
      const int i = z * 32 + lane, rr = i / CPR, ch = i % CPR, ri = qt * BM + w4 * 32 + rr;
      const uint4 x = *reinterpret_cast<const uint4*>(stage + rr * (D * 2) + ((ch ^ (rr & 7)) << 4));
      if (ri < nrows) {
        int dt, hg;
        split(ri, dt, hg);
        *reinterpret_cast<uint4*>(obase + 2 * (dt * p.o_ts + hg * p.o_hs + ch * 8)) = x;
      }
    }
    if (p.lse && live)
      p.lse[(rq.x + tok0 + my_dt) * p.Hq + hk * p.G + my_hg] =
          l == 0.f ? -INFINITY : (mref - SHIFT + log2f(l)) * 0.6931471805599453f;
    uint32_t again = __ballot_sync(0xffffffffu, live && ok && !finite);
    __syncwarp();
    while (again) {
      const int i = __ffs(again) - 1;
      again &= again - 1;
      int dt, hg;
      split(qt * BM + w4 * 32 + i, dt, hg);
      attend_row<D, F16>(p, rq.x + tok0 + dt, hk * p.G + hg, rk.x, seen_by(tok0 + dt), lane);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 9 && !sm.keep_tmem) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// [T, H, D] 16-bit with the given strides (elements): boxes of 64 channels x 1 head x 128 tokens.
static int make_map(CUtensorMap* m, const void* base, const Params& p, int D, int64_t ts, int64_t hs, int f16) {
  tc::EncodeTiledFn fn = tc::encode_tiled_fn();
  if (!fn) return set_error(KB200_ERR_LAUNCH, "attn_prompt: cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)p.H, (cuuint64_t)p.Tk};
  cuuint64_t strides[2] = {(cuuint64_t)hs * 2, (cuuint64_t)ts * 2};
  cuuint32_t box[3] = {64, 1, BN};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base),
                        dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(KB200_ERR_INVALID, "attn_prompt: k or v cannot be read by TMA (%d)", (int)r);
  return KB200_OK;
}

template <int D, bool F16>
static int launch(const Maps& maps, const Params& p, cudaStream_t st) {
  const size_t smem = sizeof(Smem<D>) + 1024;
  static std::atomic<uint64_t> done{0};
  if (int e = allow_smem((const void*)attn_prompt_kernel<D, F16>, smem, done)) return e;
  const int64_t tiles = p.Tq * p.G / ROWS + p.N;             // no fewer than the sequences have
  attn_prompt_kernel<D, F16><<<(unsigned)(tiles * p.H), THREADS, smem, st>>>(maps, p);
  return check_launch("attn_prompt_kernel");
}

}  // namespace prompt
}  // namespace kb

extern "C" int kb200_attn_prompt_fwd(const KB200PromptArgs* a, void* stream) {
  using namespace kb;
  if (!a) return set_error(KB200_ERR_INVALID, "attn_prompt: null arguments");
  if (a->N < 0 || a->Tq < 0 || a->Tk < 0 || a->N > (1 << 20) || a->Tq > 0x7fffff00LL || a->Tk > 0x7fffff00LL || a->Hq < 1 ||
      a->Hkv < 1 || a->Hq % a->Hkv || a->Hq > (1 << 14) || (a->dtype != 0 && a->dtype != 1))
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
  const int64_t G = a->Hq / a->Hkv;
  if ((a->Tq * G / prompt::ROWS + a->N) * a->Hkv > 0x7fffffffLL) return set_error(KB200_ERR_INVALID, "attn_prompt: too many rows");
  // a scale of 0 becomes one too small to matter, so that a masked score stays -inf
  const float sl2 = fmaxf(fabsf(a->softmax_scale) * 1.4426950408889634f, 1e-30f);
  prompt::Params p{a->q, a->k, a->v, a->o, a->lse, a->cu_q, a->cu_k, a->q_token_stride, a->q_head_stride,
                   a->k_token_stride, a->k_head_stride, a->v_token_stride, a->v_head_stride, a->o_token_stride,
                   a->o_head_stride, a->Tq, a->Tk, (int)a->N, (int)a->Hq, (int)a->Hkv, (int)G,
                   sl2, a->softmax_scale < 0.f ? 0x80008000u : 0u, ((1ull << 32) + G - 1) / G, a->causal};
  prompt::Maps maps;
  memset(&maps, 0, sizeof(maps));
  if (a->Tk > 0) {                                           // (without keys nothing is loaded)
    if (int e = prompt::make_map(&maps.k, a->k, p, (int)a->D, a->k_token_stride, a->k_head_stride, a->dtype)) return e;
    if (int e = prompt::make_map(&maps.v, a->v, p, (int)a->D, a->v_token_stride, a->v_head_stride, a->dtype)) return e;
  }
  cudaStream_t st = (cudaStream_t)stream;
  if (a->D == 64) return a->dtype ? prompt::launch<64, true>(maps, p, st) : prompt::launch<64, false>(maps, p, st);
  return a->dtype ? prompt::launch<128, true>(maps, p, st) : prompt::launch<128, false>(maps, p, st);
}
