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
// One CTA, 18 warps (the schedule of the FP8 kernel, attn_fp8_tc.cu):
//   warp 16    TMA producer: K and V tiles into their rings
//   warp 17    MMA issuer:  S = Q_t K_j^T (TMEM S), O_t += P_t V_j (P_t from TMEM, V read
//              MN-major from its TMA tile), order QK_1(j) PV_1(j-1) QK_0(j+1) PV_0(j)
//   warps 0-15 softmax: query tile t = w / 8, 16 rows each, read as 16x256b fragments: four
//              lanes share a row, so a row's maximum takes two shuffles and no other warp
// The row maximum is kept lazily: O and l are rescaled only when it grows by more than
// TAU (log2 units), so P <= 2^(SHIFT + TAU) (inside f16) and most tiles rescale nothing.
// P is rounded to the input type (half a step, as the output is); l sums the unrounded P.
//
// Keys that a row does not see score -inf.  In the tiles that some row does not see
// fully, V rows behind the sequence are zeroed in shared memory, and V is looked over
// for NaN and infinities, since 0 * NaN would reach rows that must not see them; a tile of
// rows that meets one is computed again, row by row, over the visible keys alone.
//
// Every wait is bounded; if one gives up, the CTA drains what is in flight and writes NaN.
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
constexpr int THREADS = 18 * 32;
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
  uint64_t s_full[QT], s_free[QT], p_full[QT], pv_done[QT], o_done, drain;
  uint32_t tmem_base;
  int seq, tile;                             // this CTA's sequence (-1: none) and row tile in it
  int bad_v[QT];
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

template <int D, bool F16>
__global__ void __launch_bounds__(THREADS, 1) attn_prompt_kernel(const __grid_constant__ Maps maps, Params p) {
  using SM = Smem<D>;
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
    }
  } else if (warp == 16) {
    if (lane == 0) {
      tc::mbar_init(&sm.q_full, 16);
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
        tc::mbar_init(&sm.s_free[i], 8);
        tc::mbar_init(&sm.p_full[i], 8);
        tc::mbar_init(&sm.pv_done[i], 1);
        sm.bad_v[i] = 0;
      }
      tc::mbar_init(&sm.o_done, 1);
      tc::mbar_init(&sm.drain, 1);
      sm.abort_flag = 0;
      sm.keep_tmem = 0;
      tc::fence_barrier_init();
      tc::prefetch_tmap(&maps.k);
      tc::prefetch_tmap(&maps.v);
    }
  } else if (warp == 17) {
    tc::tmem_alloc(&sm.tmem_base, 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  const int seq = sm.seq;
  if (seq < 0) {
    if (warp == 17) tc::tmem_dealloc(tmem, 512);
    return;
  }
  const int2 rq = seq_range(p.cu_q, seq, p.Tq), rk = seq_range(p.cu_k, seq, p.Tk);
  const int n = rq.y - rq.x, m = rk.y - rk.x;
  const int64_t row0 = (int64_t)sm.tile * ROWS;              // first row (token * G + head)
  const int64_t nrows = min((int64_t)ROWS, (int64_t)n * p.G - row0);
  // keys that token t of the sequence sees
  auto seen_by = [&](int64_t t) { return p.causal ? (int)min((int64_t)m, max((int64_t)0, t + 1 + m - n)) : m; };
  const int ntiles = (seen_by((row0 + nrows - 1) / p.G) + BN - 1) / BN;
  auto aborted = [&]() { return *((volatile int*)&sm.abort_flag) != 0; };

  if (warp == 16) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0 && ntiles > 0) {
      int kiss = 0, viss = 0;
      for (int j = 0; j < ntiles; ++j) {
        const int sk = j % KS, sv = j % VS, tok = rk.x + j * BN;
        if (j >= KS && !tc::mbar_wait(&sm.k_empty[sk], (j / KS - 1) & 1)) { sm.abort_flag = 1; break; }
        if (aborted()) break;
        tc::mbar_expect_tx(&sm.k_full[sk], ATOMS * BN * 128);
        for (int a = 0; a < ATOMS; ++a) tc::tma_load_3d(sm.k[sk][a], &maps.k, &sm.k_full[sk], a * 64, hk, tok);
        ++kiss;
        if (j >= VS && !tc::mbar_wait(&sm.v_empty[sv], (j / VS - 1) & 1)) { sm.abort_flag = 1; break; }
        if (aborted()) break;
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
  } else if (warp == 17) {
    // ------------------------------------------------------------ MMA issuer
    // The whole warp runs the schedule, so every operand is warp-uniform; one elected lane issues.
    if (ntiles > 0) {
      const bool leader = tc::elect_one();
      constexpr uint32_t IDESC_QK = tc::idesc_f32acc(F16 ? 0 : 1, BM, BN, 0, 0);
      constexpr uint32_t IDESC_PV = tc::idesc_f32acc(F16 ? 0 : 1, BM, D, 0, 1);
      constexpr uint64_t ATOM = BN * 128 / 16;               // descriptor units between 64-channel atoms
      const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
      const uint64_t dq0 = tc::sdesc_sw128_kmajor(sm.q[0][0]);
      const uint64_t dk0 = tc::sdesc_sw128_kmajor(sm.k[0][0]);
      const uint64_t dv0 = tc::sdesc_sw128_mnmajor(sm.v[0][0], BN * 128);
      auto commit = [&](uint64_t* bar) {
        if (leader) tc::tc_commit(bar);
        __syncwarp();
      };
      auto qk = [&](int t, int j) {   // S = Q_t K_j^T
        const uint64_t dq = dq0 + (uint64_t)(t * ATOMS) * ATOM, dk = dk0 + (uint64_t)((j % KS) * ATOMS) * ATOM;
        if (leader) {
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
            tc::mma_bf16(tmem_u + TM_S, dq + (ks >> 2) * ATOM + 2 * (ks & 3), dk + (ks >> 2) * ATOM + 2 * (ks & 3), IDESC_QK,
                         ks > 0 ? 1u : 0u);
          tc::tc_commit(&sm.s_full[t]);
        }
        __syncwarp();
      };
      auto pv = [&](int t, int j) {   // O_t += P_t V_j, 16 keys per instruction
        const uint64_t dv = dv0 + (uint64_t)((j % VS) * ATOMS) * ATOM;
        if (leader) {
#pragma unroll
          for (int ks = 0; ks < BN / 16; ++ks)
            tc::mma_bf16_ts(tmem_u + TM_O + t * 128, tmem_u + TM_P + t * 64 + ks * 8, dv + ks * (16 * 128 / 16), IDESC_PV,
                            (j > 0 || ks > 0) ? 1u : 0u);
          tc::tc_commit(&sm.pv_done[t]);
        }
        __syncwarp();
      };
      // a probe of the next phase goes out before the current group, so its latency overlaps the issue
      auto probe = [&](uint64_t* bar, uint32_t parity) { return tc::mbar_test_wait(bar, parity); };
      auto finish = [&](uint64_t* bar, uint32_t parity, bool pre) {
        const bool w = __all_sync(0xffffffffu, pre || tc::mbar_test_wait_loop(bar, parity));
        if (!w) sm.abort_flag = 1;
        return w;
      };
      bool ok = __all_sync(0xffffffffu, tc::mbar_wait(&sm.q_full, 0) && tc::mbar_wait(&sm.k_full[0], 0));
      if (!ok) sm.abort_flag = 1;
      if (ok) {
        tc::tc_fence_after();
        qk(0, 0);
      }
      bool pre_s0 = probe(&sm.s_free[0], 0);
      for (int j = 0; ok && j < ntiles; ++j) {
        const bool last = j + 1 == ntiles;
        const int kn = (j + 1) % KS, vn = j % VS;
        if (!finish(&sm.s_free[0], j & 1, pre_s0) || aborted()) { ok = false; break; }
        tc::tc_fence_after();
        const bool pre_p1 = j >= 1 ? probe(&sm.p_full[1], (j - 1) & 1) : true;
        qk(1, j);
        commit(&sm.k_empty[j % KS]);
        bool pre_s1 = false, pre_k = true;
        if (j >= 1) {
          if (!finish(&sm.p_full[1], (j - 1) & 1, pre_p1)) { ok = false; break; }
          tc::tc_fence_after();
          pre_s1 = probe(&sm.s_free[1], j & 1);
          if (!last) pre_k = probe(&sm.k_full[kn], ((j + 1) / KS) & 1);
          pv(1, j - 1);
          commit(&sm.v_empty[(j - 1) % VS]);
        } else if (!last) {
          pre_s1 = probe(&sm.s_free[1], j & 1);
          pre_k = probe(&sm.k_full[kn], ((j + 1) / KS) & 1);
        }
        bool pre_p0, pre_v;
        if (!last) {
          if (!finish(&sm.k_full[kn], ((j + 1) / KS) & 1, pre_k)) { ok = false; break; }
          if (!finish(&sm.s_free[1], j & 1, pre_s1)) { ok = false; break; }
          tc::tc_fence_after();
          pre_p0 = probe(&sm.p_full[0], j & 1);
          pre_v = probe(&sm.v_full[vn], (j / VS) & 1);
          qk(0, j + 1);
        } else {
          pre_p0 = probe(&sm.p_full[0], j & 1);
          pre_v = probe(&sm.v_full[vn], (j / VS) & 1);
        }
        if (!finish(&sm.v_full[vn], (j / VS) & 1, pre_v)) { ok = false; break; }
        if (!finish(&sm.p_full[0], j & 1, pre_p0)) { ok = false; break; }
        tc::tc_fence_after();
        pre_s0 = last ? true : probe(&sm.s_free[0], (j + 1) & 1);
        pv(0, j);
      }
      if (ok) {   // PV_1 of the last key tile
        const int j = ntiles - 1;
        if (finish(&sm.p_full[1], j & 1, false)) {
          tc::tc_fence_after();
          pv(1, j);
          commit(&sm.o_done);
        }
      }
      commit(&sm.drain);   // every MMA this warp issued must complete before TMEM is freed
      if (!__all_sync(0xffffffffu, tc::mbar_wait(&sm.drain, 0))) {
        sm.abort_flag = 1;
        sm.keep_tmem = 1;
      }
    }
  } else {
    // ------------------------------------------------------------ softmax (warps 0..15)
    // Q into shared memory: 256 rows of D channels, 16 bytes at a time
    const uint32_t flip = p.flip;                            // 0x80008000: a negative scale, moved into q
    for (int i = tid; ntiles > 0 && i < ROWS * (D / 8); i += 512) {
      const int r = i / (D / 8), c = i % (D / 8);
      uint4 x = make_uint4(0, 0, 0, 0);
      if (r < nrows) {
        const int64_t R = row0 + r, tok = R / p.G;
        x = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p.q) +
                                                 2 * ((rq.x + tok) * p.q_ts + (hk * p.G + (R - tok * p.G)) * p.q_hs + c * 8)));
        x.x ^= flip; x.y ^= flip; x.z ^= flip; x.w ^= flip;
      }
      const int rr = r % BM;
      *reinterpret_cast<uint4*>(&sm.q[r / BM][c / 8][rr * 128 + (((c % 8) ^ (rr & 7)) << 4)]) = x;
    }
    tc::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&sm.q_full);

    const int qt = warp >> 3, w8 = warp & 7;
    const int rbase = (warp & 3) * 32 + (w8 >> 2) * 16;      // this warp's first row == TMEM lane
    const int g = lane >> 2, t4 = lane & 3;
    const uint32_t lane_off = (uint32_t)rbase << 16;
    const uint32_t tS = tmem + TM_S + lane_off, tO = tmem + TM_O + qt * 128 + lane_off, tP = tmem + TM_P + qt * 64 + lane_off;
    const float sl2 = p.scale_log2;
    int lim[2];                                              // keys that rows g, g + 8 see
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = qt * BM + rbase + g + 8 * i;
      lim[i] = r < nrows ? seen_by((row0 + r) / p.G) : 0x7fffffff;
    }
    // key tiles below are seen fully by every row of this query tile
    const int full = qt * BM < nrows ? seen_by((row0 + qt * BM) / p.G) / BN : 0x7fffffff;
    float mref[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    bool ok = true;
    for (int j = 0; j < ntiles; ++j) {
      if (!tc::mbar_wait(&sm.s_full[qt], j & 1)) { sm.abort_flag = 1; ok = false; }
      if (__any_sync(0xffffffffu, !ok || aborted())) { ok = false; break; }
      tc::tc_fence_after();
      uint32_t s[64];                                        // [8-column group][row g: 2, row g + 8: 2]
      tc::tmem_ld16x256b_x16(tS, s);
      tc::tmem_wait_ld();
      warp_arrive(&sm.s_free[qt], lane);
      if (j >= full) {
        const int key0 = j * BN + 2 * t4;
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (key0 + (c >> 2) * 8 + (c & 1) >= lim[(c >> 1) & 1]) s[c] = __float_as_uint(-INFINITY);
        // V of this tile: rows behind the sequence become 0; NaN and infinities are reported
        if (!tc::mbar_wait(&sm.v_full[j % VS], (j / VS) & 1)) { sm.abort_flag = 1; ok = false; }
        if (__any_sync(0xffffffffu, !ok)) break;
        constexpr uint32_t EXP = F16 ? 0x7c007c00u : 0x7f807f80u, ONE = F16 ? 0x04000400u : 0x00800080u;
        uint32_t bad = 0;
        uint8_t* vb = sm.v[j % VS][0];
#pragma unroll 1
        for (int i = w8 * 32 + lane; i < ATOMS * BN * 8; i += 256) {
          uint4* x = reinterpret_cast<uint4*>(vb) + i;       // 8 chunks per 128-byte row
          if (j * BN + ((i >> 3) & (BN - 1)) >= m) {
            *x = make_uint4(0, 0, 0, 0);
          } else {
            const uint4 y = *x;
            bad |= ((y.x & EXP) + ONE) | ((y.y & EXP) + ONE) | ((y.z & EXP) + ONE) | ((y.w & EXP) + ONE);
          }
        }
        if (bad & 0x80008000u) sm.bad_v[qt] = 1;
        tc::fence_proxy_async_smem();
      }
      // maxima of this lane's scores (log2 units); those of the rows, which four lanes share, are
      // only looked up when one passes the reference by TAU
      float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        mx0 = fmaxf(mx0, fmaxf(__uint_as_float(s[4 * c]), __uint_as_float(s[4 * c + 1])));
        mx1 = fmaxf(mx1, fmaxf(__uint_as_float(s[4 * c + 2]), __uint_as_float(s[4 * c + 3])));
      }
      mx0 *= sl2;
      mx1 *= sl2;
      const bool grow = __any_sync(0xffffffffu, mx0 > mref[0] + TAU || mx1 > mref[1] + TAU);
      float a0 = 1.f, a1 = 1.f;
      if (grow) {
#pragma unroll
        for (int w = 1; w < 4; w <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, w));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, w));
        }
        const float n0 = fmaxf(mref[0], mx0), n1 = fmaxf(mref[1], mx1);
        if (n0 != -INFINITY) a0 = ex2(mref[0] - n0);
        if (n1 != -INFINITY) a1 = ex2(mref[1] - n1);
        mref[0] = n0;
        mref[1] = n1;
        l[0] *= a0;
        l[1] *= a1;
      }
      // (no key of the row seen yet: every score here is -inf, and so is x)
      const float b0 = mref[0] == -INFINITY ? 0.f : SHIFT - mref[0], b1 = mref[1] == -INFINITY ? 0.f : SHIFT - mref[1];
      const float2 sc = make_float2(sl2, sl2), bias0 = make_float2(b0, b0), bias1 = make_float2(b1, b1);
      float2 ls0 = make_float2(0.f, 0.f), ls1 = make_float2(0.f, 0.f);
      uint32_t pk[32];
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const float2 x = ffma2(make_float2(__uint_as_float(s[4 * c]), __uint_as_float(s[4 * c + 1])), sc, bias0);
        const float2 y = ffma2(make_float2(__uint_as_float(s[4 * c + 2]), __uint_as_float(s[4 * c + 3])), sc, bias1);
        const float2 e = make_float2(ex2(x.x), ex2(x.y)), f = make_float2(ex2(y.x), ex2(y.y));
        ls0 = fadd2(ls0, e);
        ls1 = fadd2(ls1, f);
        pk[2 * c] = kv::pack16<F16>(e.x, e.y);
        pk[2 * c + 1] = kv::pack16<F16>(f.x, f.y);
      }
      l[0] += ls0.x + ls0.y;
      l[1] += ls1.x + ls1.y;
      // P_t(j) overwrites P_t(j-1) and O_t may be rescaled: PV_t(j-1) must have completed
      if (j >= 1 && !tc::mbar_wait(&sm.pv_done[qt], (j - 1) & 1)) { sm.abort_flag = 1; ok = false; }
      if (__any_sync(0xffffffffu, !ok)) break;
      tc::tc_fence_after();
      tc::tmem_st16x128b_x16(tP, pk);
      if (grow && j >= 1) {
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          uint32_t o[32];
          tc::tmem_ld16x256b_x8(tO + c * 64, o);
          tc::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * ((e & 2) ? a1 : a0));
          tc::tmem_st16x256b_x8(tO + c * 64, o);
        }
      }
      tc::tmem_wait_st();
      warp_arrive(&sm.p_full[qt], lane);
    }
    // ---- epilogue: this warp's 16 rows, through its part of the Q tile (every product has read Q)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    if (ok && ntiles > 0) ok = __all_sync(0xffffffffu, tc::mbar_wait(&sm.o_done, 0));
    if (!ok) sm.abort_flag = 1;
    tc::bar_sync_named(1 + qt, 256);                         // bad_v of the whole query tile
    const bool bad = *((volatile int*)&sm.bad_v[qt]) != 0;
    if (bad) {
      for (int i = 0; i < 16; ++i) {
        const int r = qt * BM + rbase + i;
        if (r >= nrows) break;
        const int64_t R = row0 + r, tok = R / p.G;
        attend_row<D, F16>(p, rq.x + tok, (int)(hk * p.G + (R - tok * p.G)), rk.x, seen_by(tok), lane);
      }
    } else {
      tc::tc_fence_after();
      static_assert(sizeof(sm.q[0]) == 8 * 16 * D * 2, "the staged rows are the Q tile's size");
      const bool dead = aborted();
      uint8_t* stage = sm.q[qt][0] + w8 * 16 * (D * 2);      // 16 rows of D * 2 bytes, chunks rotated by the row
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        uint32_t o[32];
        if (ntiles > 0 && ok) {
          tc::tmem_ld16x256b_x8(tO + c * 64, o);
          tc::tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
        }
        const float f0 = dead ? NAN : l[0] == 0.f ? 0.f : 1.f / l[0], f1 = dead ? NAN : l[1] == 0.f ? 0.f : 1.f / l[1];
#pragma unroll
        for (int k = 0; k < 8; ++k) {                        // 16-byte chunk: 8 channels
          const int ch = c * 8 + k;
          *reinterpret_cast<uint32_t*>(stage + g * (D * 2) + (((ch ^ g) & (D / 8 - 1)) << 4) + t4 * 4) =
              kv::pack16<F16>(__uint_as_float(o[4 * k]) * f0, __uint_as_float(o[4 * k + 1]) * f0);
          *reinterpret_cast<uint32_t*>(stage + (g + 8) * (D * 2) + (((ch ^ g) & (D / 8 - 1)) << 4) + t4 * 4) =
              kv::pack16<F16>(__uint_as_float(o[4 * k + 2]) * f1, __uint_as_float(o[4 * k + 3]) * f1);
        }
      }
      __syncwarp();
#pragma unroll 4
      for (int i = lane; i < 16 * (D / 8); i += 32) {
        const int rr = i / (D / 8), ch = i % (D / 8), r = qt * BM + rbase + rr;
        if (r < nrows) {
          const int64_t R = row0 + r, tok = R / p.G;
          const uint4 x = *reinterpret_cast<const uint4*>(stage + rr * (D * 2) + (((ch ^ (rr & 7)) & (D / 8 - 1)) << 4));
          *reinterpret_cast<uint4*>(reinterpret_cast<char*>(p.o) +
                                    2 * ((rq.x + tok) * p.o_ts + (hk * p.G + (R - tok * p.G)) * p.o_hs + ch * 8)) = x;
        }
      }
      if (p.lse && t4 == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = qt * BM + rbase + g + 8 * i;
          if (r < nrows) {
            const int64_t R = row0 + r, tok = R / p.G;
            p.lse[(rq.x + tok) * p.Hq + hk * p.G + (R - tok * p.G)] =
                l[i] == 0.f ? -INFINITY : (mref[i] - SHIFT + log2f(l[i])) * 0.6931471805599453f;
          }
        }
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 17 && !sm.keep_tmem) {
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
  const int64_t G = a->Hq / a->Hkv;
  if ((a->Tq * G / prompt::ROWS + a->N) * a->Hkv > 0x7fffffffLL) return set_error(KB200_ERR_INVALID, "attn_prompt: too many rows");
  // a scale of 0 becomes one too small to matter, so that a masked score stays -inf
  const float sl2 = fmaxf(fabsf(a->softmax_scale) * 1.4426950408889634f, 1e-30f);
  prompt::Params p{a->q, a->k, a->v, a->o, a->lse, a->cu_q, a->cu_k, a->q_token_stride, a->q_head_stride,
                   a->k_token_stride, a->k_head_stride, a->v_token_stride, a->v_head_stride, a->o_token_stride,
                   a->o_head_stride, a->Tq, a->Tk, (int)a->N, (int)a->Hq, (int)a->Hkv, (int)G,
                   sl2, a->softmax_scale < 0.f ? 0x80008000u : 0u, a->causal};
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
