// attn_prompt.cu -- causal softmax attention over packed prompts with grouped heads, on
// 5th-generation tensor cores (tcgen05 + TMEM + TMA).
//
//   o_i = sum_{j <= i + m - n} softmax_j(scale q_i . k_j) v_j     (n queries at the end of m keys)
//
// Bound: the tensor pipe and the exponentials together.  A tile of 256 rows x 128 keys is
// 4 * 256 * 128 * D flops (2048 cycles at D = 128) and 32768 exponentials (2048 cycles of MUFU).
//
// Measured: 16380 tokens, 24/24 heads of 128: 1.3-1.5 ms, 1.1-1.27 PFLOP/s as the clock goes, of 64 1.01 ms; 8192
// tokens of 24/8 heads of 128 345 us with the tensor pipe active 68 % of the time.
//
// Rows.  The G = Hq / Hkv heads that share a kv head are rows of one matrix: a query tile of 128
// rows holds T = 128 / G tokens (rounded down) with G heads each, row = token * G + head, so a
// CTA reads each key tile once for all of them, and short prompts still fill the tile.  That is a
// TMA box of T tokens x G heads; with G not a divisor of 128 a few rows stay empty.  (G
// over 128: the heads are taken in equal parts of at most 128.)  K and V come in boxes of 64
// channels x 128 tokens of one head; any token and head stride works.
//
// Items.  The kernel is persistent, a CTA per SM.  An item is a tile of rows with the key tiles
// that it sees; K, V and the next item's Q are on their way while one is computed.
//   * Many items: sorted by their number of keys, most first, one launched CTA for each.  A
//     CTA that runs takes over the next CTA that has not started (cluster launch control), so
//     the items go to the SMs as they become free, without a counter in memory.
//   * Few items for the SMs and many keys: the key tiles of all items are laid end to end and
//     every CTA takes an equal share, as in attn_cached.cu; an item that crosses shares leaves
//     fp32 partials (m, l, O), joined in share order by a second kernel.
// Both are found on the device from the offsets: the host need not know the lengths.
//
// One CTA, 12 warps (registers are dealt by warpgroups of four):
//   warps 0-7  softmax: query tile t = w / 4, one row per thread (its 128 scores in registers)
//   warp 8     TMA producer: K and V tiles into their rings
//   warp 9     issues S = Q_t K_j^T, in the order QK_0(j) QK_1(j): the two query tiles share one
//              TMEM score buffer, which a tile gives back as soon as its scores are in registers
//   warp 10    issues O_t += P_t V_j (P_t from TMEM, V read MN-major from its TMA tile)
//   warp 11    finds the items and loads their Q
// What a period of 256 rows x 128 keys takes is the chain QK_0 - load - QK_1 - load: each link
// is 512 cycles of product, the two hand-offs and the load.  So the loads read whole lanes
// (32x32b; the 16-lane shapes run at half the rate) and the two kinds of products have
// an issuer each, so that no QK waits behind a PV's operands.
// The row maximum is kept lazily: O and l are rescaled only when it grows by more than
// TAU (log2 units), so P <= 2^(SHIFT + TAU) and most tiles rescale nothing.  In f16 P uses the type's range, up to
// 2^14 (V is at most 2^16, so O is far from fp32's end); in bf16 it is at most 2^-8, so that O, which is summed
// before it is divided by l, holds 256 keys with V up to the type's end, and 65536 of equal weight.
// P is rounded to the input type (half a step, as the output is); l sums the unrounded P.
//
// Keys that a row does not see score -inf, so their P is 0.  V rows behind the last that a row of the
// item sees are left out of the product, or zeroed in shared memory before it.  A NaN or an infinity in
// V at a key that a row must not see would still reach it as 0 * NaN.  So the warp that issues PV
// looks over the V rows that are hidden from some row of a query tile (as many as it has tokens, in
// the item's last tiles), in shared memory, while it waits for P: what is not finite there is zeroed
// and its keys are noted, and at the item's end the rows that see such a key add its V, as it is in
// memory, to O.  (The look costs 84.4 -> 87.7 us for 6696 tokens in prompts of 1 to 2600, 24/8 heads of
// 128, since the products leave few of shared memory's cycles; done by the softmax warps, by the
// producer or from global memory it cost 88 to 93.)
//
// Every wait is bounded.  A warp whose wait gives up stops, so that the others' waits give up
// too; what is in flight is drained, the status word is set, and the CTA writes NaN into the outputs, o and lse, of
// the items that it has taken and not finished.
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
  int N, Hq, H, G;         // H kv heads times parts, G query heads of each
  int parts, tq;           // parts of a kv head's query heads; tokens of a query tile
  float scale_log2;        // |softmax scale| log2 e; its sign goes into q (flip)
  uint32_t flip;
  int split;               // equal shares of the key tiles (else whole items)
  float* part;             // shares: [2 CTAs][rows][D] partial O, then [2 CTAs][rows][2] (m, l)
  int causal;
  int* status;             // set when a wait gives up, or null
  long long wait_clocks;   // BOUNDED: bound of a wait
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
KB_DEVI void store16(void* base, int64_t i, float x) {
  if constexpr (F16) reinterpret_cast<__half*>(base)[i] = __float2half_rn(x);
  else reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(x);
}

// 0 if the 16-bit pairs looked at so far are all finite: 0 * x is NaN for the others, and stays.
template <bool F16>
KB_DEVI uint32_t not_finite(uint32_t x, uint32_t so_far) {
  if constexpr (F16) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(so_far) : "r"(x), "r"(0u));
  else asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(so_far) : "r"(x), "r"(0u));
  return so_far;
}
// The halves of a 16-bit pair that are not finite, as ones.
template <bool F16>
KB_DEVI uint32_t odd_halves(uint32_t x) {
  constexpr uint32_t INF = F16 ? 0x7c00u : 0x7f80u;
  return ((x & INF) == INF ? 0xffffu : 0u) | ((x >> 16 & INF) == INF ? 0xffff0000u : 0u);
}

constexpr int BM = 128, BN = 128, QT = 2, ROWS = QT * BM;
template <bool F16>
constexpr float SHIFT = F16 ? 6.f : -16.f;   // P = 2^(s - m + SHIFT)
constexpr float TAU = 8.f;
constexpr int THREADS = 12 * 32;
constexpr int SITE = 50;                     // of a wait that gives up, in the status word
// Registers: the launch gives each thread 168 (its 384 threads share the SM's 65536); the softmax
// warpgroups take 208 and the third leaves itself 88, 2 * 208 + 88 = 3 * 168.
constexpr int REGS_SOFTMAX = 208, REGS_OTHERS = 88;
constexpr int SORTED = 64;                   // up to this many sequences the tiles are sorted by their keys
constexpr uint32_t TM_O = 0, TM_S = 256, TM_P = 384;   // TMEM columns: O_t at 128 t, S, P_t at 64 t

struct Maps {
  CUtensorMap q, k, v;
};

constexpr int TABLE = 128;                   // shares: at most this many row tiles
constexpr int SHORT = 8;                     // whole items: one of fewer key tiles is short
constexpr int PAD = 3;                       // shares: what an item costs besides its key tiles, in key tiles
// shares: at least this many key tiles (450 queries over 2365 keys, 4/1 heads of 128: 28.7 us, with eight 34.8;
// 606 keys and 4339 of 4/4 heads: 38 and 39)
constexpr int LEAST = 4;

// The row tiles of all sequences, and the flat length of those before each (key tiles + PAD).
struct Table {
  int before[TABLE + 1];
  uint8_t seq[TABLE], tile[TABLE];
};

struct Item {
  int q0, n, k0, m;                          // packed queries and keys of the sequence
  int tile, hk;                              // row tile in it, kv head
  int j0, j1, all;                           // key tiles [j0, j1) of the `all` that the tile sees
  int slot;                                  // where the partial goes; -1: the item is whole, -2: no more items, -3: no item
};

template <int D>
struct Smem {
  static constexpr int KS = D == 128 ? 3 : 4, VS = D == 128 ? 2 : 4;
  static constexpr int ATOMS = D / 64;       // 64 channels: 128 swizzled bytes
  uint8_t q[QT][ATOMS][BM * 128];
  uint8_t k[KS][ATOMS][BN * 128];
  uint8_t v[VS][ATOMS][BN * 128];
  uint64_t item_full[2], item_free[2];       // an item is published / every warp has read it
  uint64_t answered;
  uint64_t q_full, q_free;
  uint64_t k_full[KS], k_empty[KS], v_full[VS], v_empty[VS];
  uint64_t s_full[QT], s_free[QT], p_full[QT], pv_done[QT], drain[2];
  alignas(16) uint4 answer[2];
  Item item[2];
  Table table;
  uint32_t tmem_base;
  int took[4], taken;                        // whole items: the CTAs whose items this one took last, and how many
  int done[8];                               // items that each softmax warp has finished
  int abort_flag, keep_tmem;
  // For each query tile, keys with a V that is not finite, counted from the first that some row of the item does not see
  // (a row sees fewer than ROWS from there on), and whether there are some; the items with keys take the two in turn.
  uint32_t odd[2][QT][ROWS / 32];
  int any_odd[2][QT];
};

// What is not finite in the rows [r0, r1) of a V tile in shared memory becomes 0, by one warp; row r is key r + key0
// of those that `odd` marks, for query tile `t` and those behind it.  (The two functions are not inlined: they are hardly ever
// called, and in line their code alone cost 5 % of a packed batch's time.)
template <int D, bool F16>
__device__ __noinline__ void take_out(uint4* v, int r0, int r1, int key0, uint32_t (*odd)[ROWS / 32], int t, int lane) {
  for (int r = r0; r < r1; ++r) {            // (a row is 8 chunks of each atom: its channels, in some order)
    bool mine = false;
    if (lane < D / 8) {
      uint4& x = v[(lane >> 3) * BN * 8 + r * 8 + (lane & 7)];
      const uint4 z = make_uint4(odd_halves<F16>(x.x), odd_halves<F16>(x.y), odd_halves<F16>(x.z), odd_halves<F16>(x.w));
      mine = (z.x | z.y | z.z | z.w) != 0;
      if (mine) x = make_uint4(x.x & ~z.x, x.y & ~z.y, x.z & ~z.z, x.w & ~z.w);
    }
    const int k = r + key0;
    if (__any_sync(0xffffffffu, mine) && lane >= t && lane < QT && k < ROWS) odd[lane][k >> 5] |= 1u << (k & 31);
  }
  tc::fence_proxy_async_smem();
  __syncwarp();
}
// Adds to the O of each lane's row, in TMEM, what was taken out at the first `keys` keys of those that `odd` marks.
template <int D, bool F16>
__device__ __noinline__ void put_back(uint32_t tO, const char* v, int64_t v_bytes, int keys, const uint32_t* odd) {
#pragma unroll 1
  for (int i = 0; i < D / 32; ++i) {
    uint32_t o[32];
    tc::tmem_ld32(tO + i * 32, o);
    tc::tmem_wait_ld();
#pragma unroll 1
    for (int k = 0; k < keys; ++k) {
      if (!(odd[k >> 5] >> (k & 31) & 1)) continue;
      const uint4* src = reinterpret_cast<const uint4*>(v + k * v_bytes + i * 64);
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const uint4 x = __ldg(src + z);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = kv::unpack16<F16>(w[e] & odd_halves<F16>(w[e]));
          o[8 * z + 2 * e] = __float_as_uint(__uint_as_float(o[8 * z + 2 * e]) + f.x);
          o[8 * z + 2 * e + 1] = __float_as_uint(__uint_as_float(o[8 * z + 2 * e + 1]) + f.y);
        }
      }
    }
    __syncwarp();
    tc::tmem_st32(tO + i * 32, o);
  }
  tc::tmem_wait_st();
}

// Keys that query `t` of n sees, of m.
KB_DEVI int seen_by(const Params& p, int64_t t, int n, int m) {
  return p.causal ? (int)min((int64_t)m, max((int64_t)0, t + 1 + m - n)) : m;
}
// Key tiles that row tile `tile` sees.
KB_DEVI int key_tiles(const Params& p, int tile, int n, int m) {
  const int64_t last = min((int64_t)n, (int64_t)(tile + 1) * QT * p.tq) - 1;
  return (seen_by(p, last, n, m) + BN - 1) / BN;
}

// Tile number `r` of the order above: sequence and tile in it, by one warp (seq = -1: there are no more).
KB_DEVI void find_tile(const Params& p, int64_t r, int lane, int& seq, int& tile) {
  auto tiles_of = [&](int s, int& level) {   // row tiles of sequence s; level of its first one
    const int2 q = seq_range(p.cu_q, s, p.Tq), k = seq_range(p.cu_k, s, p.Tk);
    const int n = q.y - q.x;
    level = p.causal ? max(k.y - k.x - n, 0) / (QT * p.tq) : 0;
    return (n + QT * p.tq - 1) / (QT * p.tq);
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
  // Many sequences: sequence s owns the numbers from cu_q[s] / tokens of a tile + s on (it has at most
  // n / tokens + 1 tiles, so these do not overlap), found without going through all of them; a number
  // that no tile has gives tile = -1.  A sequence's last tiles come first, but the sequences are taken in order: 70 prompts
  // of 100 tokens and one of 6000, 24/8 heads of 128, take 254-270 us if that is the first and 295-304 if it is the
  // last (61 prompts, sorted: 241).
  const int per = QT * p.tq;
  auto first = [&](int s) { return min(max((int64_t)p.cu_q[s], (int64_t)0), p.Tq) / per + s; };
  seq = kv::warp_last(p.N, lane, [&](int s) { return first(s) <= r; });
  int lv;
  const int nt = tiles_of(seq, lv);
  const int64_t off = r - first(seq);
  tile = off >= 0 && off < nt ? nt - 1 - (int)off : -1;
}

// Fills the table, by one warp; returns the number of row tiles.
KB_DEVI int build_table(const Params& p, Table& tb, int lane) {
  int base = 0;
  for (int s0 = 0; s0 < p.N; s0 += 32) {
    const int s = s0 + lane;
    int nt = 0;
    if (s < p.N) {
      const int2 q = seq_range(p.cu_q, s, p.Tq);
      nt = min(TABLE, (q.y - q.x + QT * p.tq - 1) / (QT * p.tq));
    }
    int inc = nt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    for (int i = 0; i < nt && base + inc - nt + i < TABLE; ++i) {
      tb.seq[base + inc - nt + i] = (uint8_t)s;
      tb.tile[base + inc - nt + i] = (uint8_t)i;
    }
    base = min(TABLE, base + __shfl_sync(0xffffffffu, inc, 31));
  }
  __syncwarp();
  int before = 0;
  for (int f0 = 0; f0 < base; f0 += 32) {
    int cost = 0;
    if (f0 + lane < base) {
      const int s = tb.seq[f0 + lane];
      const int2 q = seq_range(p.cu_q, s, p.Tq), k = seq_range(p.cu_k, s, p.Tk);
      cost = key_tiles(p, tb.tile[f0 + lane], q.y - q.x, k.y - k.x) + PAD;
    }
    int inc = cost;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (f0 + lane < base) tb.before[f0 + lane + 1] = before + inc;
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) tb.before[0] = 0;
  __syncwarp();
  return base;
}
// Flat positions of a share: those of all kv heads, [hk][row tile][key tile + PAD].
KB_DEVI int64_t share_size(const Params& p, int flat, int ctas) {
  return max((int64_t)LEAST, ((int64_t)flat * p.H + ctas - 1) / ctas);
}

// The next CTA of the grid that has not started will not start, and this one does its work: asks
// for it (the answer, 16 bytes, is counted on `bar`), and reads the answer (-1: there is none).
KB_DEVI void take_over_ask(uint4* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];\n"
               ::"r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
}
KB_DEVI int take_over_answer(const uint4* answer) {
  int block;
  asm volatile(
      "{\n .reg .pred p;\n .reg .b128 h;\n ld.shared.b128 h, [%1];\n"
      " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n mov.b32 %0, -1;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, _, _, _}, h;\n}\n"
      : "=r"(block) : "r"(smem_u32(answer)) : "memory");
  return block;
}

// The items of a CTA, one after the other; by one warp, every lane has them.
struct Items {
  int64_t left;
  int tiles, flat, hk, f, x;                 // shares: row tiles, their flat length; the next position
  KB_DEVI void start(const Params& p, Table& tb, int lane) {
    left = 0;
    if (!p.split) return;
    tiles = build_table(p, tb, lane);
    flat = tb.before[tiles];
    if (flat == 0) return;
    const int64_t all = (int64_t)flat * p.H, per = share_size(p, flat, gridDim.x), at = blockIdx.x * per;
    left = min(per, all - at);
    if (left <= 0) return;
    hk = (int)(at / flat);
    const int rem = (int)(at - (int64_t)hk * flat);
    f = 0;
    while (tb.before[f + 1] <= rem) ++f;
    x = rem - tb.before[f];
  }
  // `block`: whole items, the one to take (-1: none).
  KB_DEVI Item next(const Params& p, const Table& tb, int block, int lane) {
    Item it{};
    it.slot = -2;
    int seq, tile;
    if (!p.split) {
      if (block < 0) return it;
      find_tile(p, block / p.H, lane, seq, tile);
      if (seq < 0) return it;
      if (tile < 0) {
        it.slot = -3;
        return it;
      }
      it.hk = block % p.H;
    } else {
      int take, span;
      do {
        if (left <= 0) return it;
        if (f == tiles) {
          f = 0;
          ++hk;
        }
        span = tb.before[f + 1] - tb.before[f];
        take = (int)min((int64_t)(span - x), left);
        left -= take;
        it.j0 = x;
        it.j1 = min(x + take, span - PAD);
        seq = tb.seq[f];
        tile = tb.tile[f];
        it.hk = hk;
        x += take;
        if (x == span) {
          x = 0;
          ++f;
        }
      } while (it.j1 <= it.j0 && !(it.j0 == 0 && span == PAD));   // (an item that sees no key is written too)
    }
    const int2 q = seq_range(p.cu_q, seq, p.Tq), k = seq_range(p.cu_k, seq, p.Tk);
    it.q0 = q.x; it.n = q.y - q.x; it.k0 = k.x; it.m = k.y - k.x;
    it.tile = tile;
    it.all = key_tiles(p, tile, it.n, it.m);
    if (!p.split) it.j1 = it.all;
    it.slot = it.j0 == 0 && it.j1 == it.all ? -1 : 2 * (int)blockIdx.x + (it.j0 > 0 ? 0 : 1);
    return it;
  }
};

// One arrival per warp, after its TMEM reads or writes.
KB_DEVI void warp_arrive(uint64_t* bar, int lane) {
  tc::tc_fence_before();
  __syncwarp();
  if (lane == 0) tc::mbar_arrive(bar);
}

// Which of every 8 pairs of exponentials go to the FMA pipe (measured with none, 1, 2, 3 and 4 of 8;
// 2 of 8 was fastest at both head dims: D = 128, two pieces of prompts, 170, 161, 156, 165 and 166 us; D = 64, 16380
// tokens of 24/24 heads, 1044, 1033, 1013, 1030 and 1120 us).
constexpr int POLY = 0x88;

// (BOUNDED: with the caller's bound of a wait, instead of 4e9 clocks)
template <int D, bool F16, bool BOUNDED>
__global__ void __launch_bounds__(THREADS, 1) attn_prompt_kernel(const __grid_constant__ Maps maps, Params p) {
  using SM = Smem<D>;
  constexpr int KS = SM::KS, VS = SM::VS, ATOMS = SM::ATOMS;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  SM& sm = *reinterpret_cast<SM*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (warp == 8) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        tc::mbar_init(&sm.s_full[i], 1);
        tc::mbar_init(&sm.s_free[i], 4);
        tc::mbar_init(&sm.p_full[i], 4);
        tc::mbar_init(&sm.pv_done[i], 2);
        tc::mbar_init(&sm.drain[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        tc::mbar_init(&sm.item_full[i], 1);
        tc::mbar_init(&sm.item_free[i], 11);
      }
      tc::mbar_init(&sm.answered, 1);
      tc::mbar_init(&sm.q_full, 1);
      tc::mbar_init(&sm.q_free, 1);
      for (int s = 0; s < KS; ++s) {
        tc::mbar_init(&sm.k_full[s], 1);
        tc::mbar_init(&sm.k_empty[s], 1);
      }
      for (int s = 0; s < VS; ++s) {
        tc::mbar_init(&sm.v_full[s], 1);
        tc::mbar_init(&sm.v_empty[s], 1);
      }
      sm.taken = 0;
      for (int i = 0; i < 8; ++i) sm.done[i] = 0;
      sm.abort_flag = 0;
      sm.keep_tmem = 0;
      tc::fence_barrier_init();
      tc::prefetch_tmap(&maps.q);
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
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");   // the join, if any: it waits for this grid's end

  auto wait_for = [&](uint64_t* bar, uint32_t parity) {
    // (a thread suspended in try_wait looks at no clock: short bounds need the polling loop)
    if constexpr (BOUNDED) return tc::mbar_test_wait_loop(bar, parity, p.wait_clocks);
    else return tc::mbar_wait(bar, parity);
  };
  // Item number `c` of the CTA; false: no more (or its wait gave up).
  auto get_item = [&](int c, Item& it, bool& ok) {
    ok = __all_sync(0xffffffffu, wait_for(&sm.item_full[c & 1], (c >> 1) & 1));
    if (!ok) {
      sm.abort_flag = 1;
      return false;
    }
    it = sm.item[c & 1];
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&sm.item_free[c & 1]);
    return it.slot != -2;
  };

  if (warp >= 8) {
    tc::setmaxnreg_dec<REGS_OTHERS>();
    Item it;
    bool ok = true;
    if (warp == 8) {
      // ---------------------------------------------------------- TMA producer
      int g = 0, ks = 0, vs = 0;                             // key tiles so far: ring positions; K and V tiles loaded
      for (int c = 0; get_item(c, it, ok); ++c) {
        for (int j = it.j0; ok && j < it.j1; ++j, ++g) {
          const int sk = g % KS, sv = g % VS, tok = it.k0 + j * BN;
          if (g >= KS) ok = __all_sync(0xffffffffu, wait_for(&sm.k_empty[sk], (g / KS - 1) & 1));
          if (!ok) break;
          if (lane == 0) {
            tc::mbar_expect_tx(&sm.k_full[sk], ATOMS * BN * 128);
            for (int a = 0; a < ATOMS; ++a) tc::tma_load_3d(sm.k[sk][a], &maps.k, &sm.k_full[sk], a * 64, it.hk / p.parts, tok);
          }
          ++ks;
          if (g >= VS) ok = __all_sync(0xffffffffu, wait_for(&sm.v_empty[sv], (g / VS - 1) & 1));
          if (!ok) break;                                    // (K of this tile is under way, V is not)
          if (lane == 0) {
            tc::mbar_expect_tx(&sm.v_full[sv], ATOMS * BN * 128);
            for (int a = 0; a < ATOMS; ++a) tc::tma_load_3d(sm.v[sv][a], &maps.v, &sm.v_full[sv], a * 64, it.hk / p.parts, tok);
          }
          ++vs;
        }
        if (!ok) break;
      }
      if (!ok) sm.abort_flag = 1;
      // before the CTA may exit, every load must have landed (of each slot the last one: a wait for an earlier phase
      // would take the phase after for it)
      bool drained = true;
      for (int i = max(ks - KS, 0); i < ks; ++i) drained &= tc::mbar_wait(&sm.k_full[i % KS], (i / KS) & 1);
      for (int i = max(vs - VS, 0); i < vs; ++i) drained &= tc::mbar_wait(&sm.v_full[i % VS], (i / VS) & 1);
      if (!drained) { sm.abort_flag = 1; sm.keep_tmem = 1; }
    } else if (warp == 11) {
      // ---------------------------------------------------------- items, and their Q
      Items items;
      items.start(p, sm.table, lane);
      int uses = 0, asked = 0, block = blockIdx.x;           // of the Q tile; take-overs; the CTA whose item is next
      bool ahead = false;
      for (int c = 0; ok; ++c) {
        // The next item is taken when every warp has the last one, not earlier than it is needed; or, if that
        // one is short, when every warp has the one before, so that it is there in time (64 sequences of
        // 200 tokens, 24/8 heads: 76.9 us, 78.6 without; 512 + 300 queries over 12345 + 8000 keys, in shares: 134 and 136).
        if (c > 1) ok = __all_sync(0xffffffffu, wait_for(&sm.item_free[c & 1], ((c >> 1) - 1) & 1));
        if (ok && c > 0 && !ahead) ok = __all_sync(0xffffffffu, wait_for(&sm.item_free[(c - 1) & 1], ((c - 1) >> 1) & 1));
        for (bool own = c == 0; ok; own = false) {
          if (!own && !p.split) {
            if (lane == 0) {
              tc::fence_proxy_async_smem();
              tc::mbar_expect_tx(&sm.answered, 16);
              take_over_ask(&sm.answer[asked & 1], &sm.answered);
            }
            __syncwarp();
            ok = __all_sync(0xffffffffu, wait_for(&sm.answered, asked & 1));
            if (!ok && !__all_sync(0xffffffffu, tc::mbar_wait(&sm.answered, asked & 1))) {   // it must land before the exit
              sm.keep_tmem = 1;
              break;
            }
            block = take_over_answer(&sm.answer[asked & 1]);
            ++asked;
            if (!ok) {                                       // (an item that this CTA has taken and will not finish)
              if (lane == 0) {
                sm.took[c & 3] = block;
                sm.taken = c + 1;
              }
              break;
            }
          }
          it = items.next(p, sm.table, block, lane);
          if (it.slot != -3) break;
        }
        if (!ok) break;
        if (lane == 0) {
          sm.took[c & 3] = block;
          sm.taken = c + 1;
          sm.item[c & 1] = it;
          tc::mbar_arrive(&sm.item_full[c & 1]);
        }
        __syncwarp();
        ahead = p.split || it.j1 - it.j0 < SHORT;
        if (it.slot == -2) break;
        if (it.j1 <= it.j0) continue;
        if (uses > 0) ok = __all_sync(0xffffffffu, wait_for(&sm.q_free, (uses - 1) & 1));
        if (!ok) break;
        ++uses;
        if (lane == 0) {                                     // (tokens behind the sequence: rows that are not stored)
          tc::mbar_expect_tx(&sm.q_full, QT * ATOMS * p.tq * p.G * 128);
          for (int t = 0; t < QT; ++t)
            for (int a = 0; a < ATOMS; ++a)
              tc::tma_load_3d(sm.q[t][a], &maps.q, &sm.q_full, a * 64, it.hk * p.G, it.q0 + (it.tile * QT + t) * p.tq);
        }
        __syncwarp();
      }
      if (uses > 0 && !__all_sync(0xffffffffu, tc::mbar_wait(&sm.q_full, (uses - 1) & 1))) {   // Q must land before the exit
        ok = false;
        sm.keep_tmem = 1;
      }
      if (!ok) sm.abort_flag = 1;
    } else {
      // ---------------------------------------------------------- MMA issuers
      // The whole warp runs the schedule, so every operand is warp-uniform; one elected lane issues.
      const bool leader = tc::elect_one();
      constexpr uint64_t ATOM = BN * 128 / 16;               // descriptor units between 64-channel atoms
      const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        const bool w = __all_sync(0xffffffffu, wait_for(bar, parity));
        tc::tc_fence_after();
        return w;
      };
      int g = 0;                                             // key tiles so far
      if (warp == 9) {
        // (bit 13 of the descriptor negates A: the sign of the scale)
        const uint32_t idesc = tc::idesc_f32acc(F16 ? 0 : 1, BM, BN, 0, 0) | (p.flip ? 1u << 13 : 0u);
        const uint64_t dq0 = tc::sdesc_sw128_kmajor(sm.q[0][0]);
        const uint64_t dk0 = tc::sdesc_sw128_kmajor(sm.k[0][0]);
        auto qk = [&](int t, int slot) {                     // S = Q_t K^T
          const uint64_t dq = dq0 + (uint64_t)(t * ATOMS) * ATOM, dk = dk0 + (uint64_t)(slot * ATOMS) * ATOM;
          if (leader) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
              tc::mma_bf16(tmem_u + TM_S, dq + (ks >> 2) * ATOM + 2 * (ks & 3), dk + (ks >> 2) * ATOM + 2 * (ks & 3), idesc,
                           ks > 0 ? 1u : 0u);
            tc::tc_commit(&sm.s_full[t]);
            if (t == 1) tc::tc_commit(&sm.k_empty[slot]);
          }
          __syncwarp();
        };
        int uses = 0;
        for (int c = 0; get_item(c, it, ok); ++c) {
          if (it.j1 <= it.j0) continue;
          ok = wait(&sm.q_full, uses & 1);
          ++uses;
          for (int j = it.j0; ok && j < it.j1; ++j, ++g) {
            ok = wait(&sm.k_full[g % KS], (g / KS) & 1);
            if (ok && g > 0) ok = wait(&sm.s_free[1], (g - 1) & 1);
            if (!ok) break;
            qk(0, g % KS);
            ok = wait(&sm.s_free[0], g & 1);
            if (ok) qk(1, g % KS);
          }
          if (!ok) break;
          if (leader) tc::tc_commit(&sm.q_free);
          __syncwarp();
        }
      } else {
        constexpr uint32_t IDESC_PV = tc::idesc_f32acc(F16 ? 0 : 1, BM, D, 0, 1);
        const uint64_t dv0 = tc::sdesc_sw128_mnmajor(sm.v[0][0], BN * 128);
        int uses = 0;                                        // items with keys so far
        for (int c = 0; get_item(c, it, ok); ++c) {
          // the first key that some row does not see; the first that no row of tile 0 sees, that none sees
          const int hidden = seen_by(p, it.tile * QT * p.tq, it.n, it.m);
          const int beyond0 = seen_by(p, min(it.n, it.tile * QT * p.tq + p.tq) - 1, it.n, it.m);
          const int beyond = seen_by(p, min((int64_t)it.n, (int64_t)(it.tile + 1) * QT * p.tq) - 1, it.n, it.m);
          for (int j = it.j0; ok && j < it.j1; ++j, ++g) {
            const int slot = g % VS;
            ok = wait(&sm.v_full[slot], (g / VS) & 1);
            if (!ok) break;
            uint4* v = reinterpret_cast<uint4*>(sm.v[slot][0]);
            const int r0 = max(hidden - j * BN, 0), r1 = min(beyond - j * BN, BN), steps1 = (r1 + 15) / 16;
            // (at least one, so that O_0 begins from zero)
            const int steps0 = min(max((beyond0 - j * BN + 15) / 16, 1), steps1), mid = min(max(steps0 * 16, r0), r1);
            if (r1 < steps1 * 16) {                          // (the product takes the keys by 16)
              for (int a = 0; a < ATOMS; ++a)
                for (int i = r1 * 8 + lane; i < steps1 * 128; i += 32) v[a * BN * 8 + i] = make_uint4(0, 0, 0, 0);
              tc::fence_proxy_async_smem();
              __syncwarp();
            }
            if (j == it.j0) {                                // (two items on, this warp has had the P of the item
              if (lane < QT * ROWS / 32) (&sm.odd[uses & 1][0][0])[lane] = 0;   // between, and so every softmax warp
              if (lane < QT) sm.any_odd[uses & 1][lane] = 0;                    // has read these)
              __syncwarp();
            }
            const uint64_t dv = dv0 + (uint64_t)(slot * ATOMS) * ATOM;
            for (int t = 0; ok && t < QT; ++t) {             // O_t += P_t V_j, 16 keys per instruction
              const int from = t == 0 ? r0 : mid, to = t == 0 ? mid : r1, steps = t == 0 ? steps0 : steps1;
              if (from < to) {                               // is V finite at the keys that some row of the tile does not see?
                uint32_t x0 = 0, x1 = 0, x2 = 0, x3 = 0;
                for (int a = 0; a < ATOMS; ++a)
#pragma unroll 4
                  for (int i = from * 8 + lane; i < to * 8; i += 32) {
                    const uint4 x = v[a * BN * 8 + i];
                    x0 = not_finite<F16>(x.x, x0); x1 = not_finite<F16>(x.y, x1);
                    x2 = not_finite<F16>(x.z, x2); x3 = not_finite<F16>(x.w, x3);
                  }
                if (__any_sync(0xffffffffu, ((x0 | x1 | x2 | x3) & 0x7fff7fffu) != 0)) {
                  take_out<D, F16>(v, from, to, j * BN - hidden, sm.odd[uses & 1], t, lane);
                  if (lane >= t && lane < QT) sm.any_odd[uses & 1][lane] = 1;
                  __syncwarp();
                }
              }
              // (the softmax publishes an item's first P_t when it has read the O_t before)
              ok = wait(&sm.p_full[t], g & 1);
              if (ok && leader) {
#pragma unroll
                for (int ks = 0; ks < BN / 16; ++ks) {
                  if (ks == steps) break;
                  tc::mma_bf16_ts(tmem_u + TM_O + t * 128, tmem_u + TM_P + t * 64 + ks * 8, dv + ks * (16 * 128 / 16), IDESC_PV,
                                  (j > it.j0 || ks > 0) ? 1u : 0u);
                }
                tc::tc_commit(&sm.pv_done[t]);
                if (t == 1) tc::tc_commit(&sm.v_empty[slot]);
              }
              __syncwarp();
              if (ok && lane == 0) tc::mbar_arrive(&sm.pv_done[t]);   // (counted too: it releases any_odd and odd)
            }
          }
          if (!ok) break;
          uses += it.j1 > it.j0;
        }
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
  } else {
    // ------------------------------------------------------------ softmax
    tc::setmaxnreg_inc<REGS_SOFTMAX>();
    const int qt = warp >> 2, w4 = warp & 3;
    const int row = w4 * 32 + lane, r = qt * BM + row;       // this thread's row; its TMEM lane is `row`
    const int dt = qt * p.tq + row / p.G, hg = row % p.G;    // its token in the tile and head
    const bool in_tile = row < p.tq * p.G;
    const uint32_t lane_off = (uint32_t)(w4 * 32) << 16;
    const uint32_t tS = tmem + TM_S + lane_off, tO = tmem + TM_O + qt * 128 + lane_off, tP = tmem + TM_P + qt * 64 + lane_off;
    const float sl2 = p.scale_log2;
    int g = 0, uses = 0;                                     // key tiles, and items with keys, so far
    bool ok = true;
    Item it;
    for (int c = 0; get_item(c, it, ok); ++c) {
      const int tok = it.tile * QT * p.tq + dt;              // in the sequence
      const bool live = in_tile && tok < it.n;
      const int lim = live ? seen_by(p, tok, it.n, it.m) : 0x7fffffff;   // keys that the row sees
      const int hidden = seen_by(p, it.tile * QT * p.tq, it.n, it.m);    // the first key that some row does not see
      float mref = -INFINITY, l = 0.f;
      for (int j = it.j0; j < it.j1; ++j, ++g) {
        ok = __all_sync(0xffffffffu, wait_for(&sm.s_full[qt], g & 1));
        if (!ok) break;
        tc::tc_fence_after();
        uint32_t s[128];
#pragma unroll
        for (int i = 0; i < 4; ++i) tc::tmem_ld32(tS + i * 32, s + i * 32);
        tc::tmem_wait_ld();
        warp_arrive(&sm.s_free[qt], lane);
        if (j >= hidden / BN) {                              // (the tiles below are seen fully by every row)
          const int end = lim - j * BN;
#pragma unroll
          for (int c0 = 0; c0 < BN; c0 += 32)
            if (__any_sync(0xffffffffu, end < c0 + 32)) {
#pragma unroll
              for (int i = c0; i < c0 + 32; ++i)
                if (i >= end) s[i] = __float_as_uint(-INFINITY);
            }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < BN; i += 8)
#pragma unroll
          for (int z = 0; z < 4; ++z)
            mx[z] = fmaxf(mx[z], fmaxf(__uint_as_float(s[i + 2 * z]), __uint_as_float(s[i + 2 * z + 1])));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2;
        // (rows that are not stored have no say: what they hold must not change how others round)
        const bool grow = __any_sync(0xffffffffu, live && top > mref + TAU);
        float alpha = 1.f;
        if (grow) {
          const float mn = fmaxf(mref, top);
          if (mn != -INFINITY) alpha = ex2(mref - mn);
          mref = mn;
          l *= alpha;
        }
        // (no key of the row seen yet: every score here is -inf, and so is x)
        const float b0 = mref == -INFINITY ? 0.f : SHIFT<F16> - mref;
        const float2 sc = make_float2(sl2, sl2), bias = make_float2(b0, b0);
        float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int e0 = h * 64 + 2 * i;
            const float2 x = ffma2(make_float2(__uint_as_float(s[e0]), __uint_as_float(s[e0 + 1])), sc, bias);
            const float2 e = ((POLY >> (i & 7)) & 1) ? exp2_poly(x) : make_float2(ex2(x.x), ex2(x.y));
            ls[i & 1] = fadd2(ls[i & 1], e);
            pk[i] = kv::pack16<F16>(e.x, e.y);
          }
          if (h == 0) {
            // P_t(j) overwrites P_t(j-1) and O_t may be rescaled: PV_t(j-1) must have completed
            if (g > 0) ok = __all_sync(0xffffffffu, wait_for(&sm.pv_done[qt], (g - 1) & 1));
            tc::tc_fence_after();
          }
          if (ok) tc::tmem_st32(tP + h * 32, pk);
        }
        if (!ok) break;
        l += (ls[0].x + ls[0].y) + (ls[1].x + ls[1].y);
        if (grow && j > it.j0) {
#pragma unroll 1
          for (int i = 0; i < D / 32; ++i) {
            uint32_t o[32];
            tc::tmem_ld32(tO + i * 32, o);
            tc::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tc::tmem_st32(tO + i * 32, o);
          }
        }
        tc::tmem_wait_st();
        warp_arrive(&sm.p_full[qt], lane);
      }
      // ---- the item's end: O_t of this row
      const bool any = it.j1 > it.j0;
      if (ok && any) ok = __all_sync(0xffffffffu, wait_for(&sm.pv_done[qt], (g - 1) & 1));
      if (!ok) break;
      tc::tc_fence_after();
      if (any && sm.any_odd[uses & 1][qt]) {                     // V that was taken out of the product: added where the row sees it
        const char* v = reinterpret_cast<const char*>(p.v) + 2 * (((int64_t)it.k0 + hidden) * p.v_ts + (it.hk / p.parts) * p.v_hs);
        put_back<D, F16>(tO, v, 2 * p.v_ts, live ? lim - hidden : 0, sm.odd[uses & 1][qt]);
      }
      uses += any;
      if (it.slot >= 0) {                                    // a partial: O and l under this row's m
        float* dst = p.part + ((int64_t)it.slot * ROWS + r) * D;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          uint32_t o[32];
          tc::tmem_ld32(tO + i * 32, o);
          tc::tmem_wait_ld();
#pragma unroll
          for (int z = 0; z < 32; z += 4) *reinterpret_cast<uint4*>(dst + i * 32 + z) = make_uint4(o[z], o[z + 1], o[z + 2], o[z + 3]);
        }
        *reinterpret_cast<float2*>(p.part + (int64_t)2 * gridDim.x * ROWS * D + ((int64_t)it.slot * ROWS + r) * 2) =
            make_float2(mref, l);
        if (lane == 0) sm.done[warp] = c + 1;
        continue;
      }
      const float f = l == 0.f ? 0.f : 1.f / l;
      const int64_t gt = (int64_t)it.q0 + tok;
      const int head = it.hk * p.G + hg;
      char* orow = reinterpret_cast<char*>(p.o) + 2 * (gt * p.o_ts + head * p.o_hs);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        uint32_t o[32];
        if (any) {
          tc::tmem_ld32(tO + i * 32, o);
          tc::tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
        }
        if (live) {
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            uint4 x;
            x.x = kv::pack16<F16>(__uint_as_float(o[8 * z + 0]) * f, __uint_as_float(o[8 * z + 1]) * f);
            x.y = kv::pack16<F16>(__uint_as_float(o[8 * z + 2]) * f, __uint_as_float(o[8 * z + 3]) * f);
            x.z = kv::pack16<F16>(__uint_as_float(o[8 * z + 4]) * f, __uint_as_float(o[8 * z + 5]) * f);
            x.w = kv::pack16<F16>(__uint_as_float(o[8 * z + 6]) * f, __uint_as_float(o[8 * z + 7]) * f);
            *reinterpret_cast<uint4*>(orow + 2 * (i * 32 + z * 8)) = x;
          }
        }
      }
      if (p.lse && live) p.lse[gt * p.Hq + head] = l == 0.f ? -INFINITY : (mref - SHIFT<F16> + log2f(l)) * 0.6931471805599453f;
      if (lane == 0) sm.done[warp] = c + 1;
    }
    if (!ok) sm.abort_flag = 1;
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 9 && !sm.keep_tmem) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
  if (sm.abort_flag && warp == 0) {                          // a wait gave up: no result is better than a wrong one
    if (lane == 0 && p.status) atomicCAS(p.status, 0, SITE);
    int first = sm.done[0];
    for (int i = 1; i < 8; ++i) first = min(first, sm.done[i]);
    Items items;
    items.start(p, sm.table, lane);
    // its shares, or the whole items, from the first that some warp has not finished (a warp that takes an item has finished
    // the one before, and the items are found two ahead: at most four)
    for (int c = p.split ? 0 : first; p.split || c < sm.taken; ++c) {
      const Item it = items.next(p, sm.table, p.split ? 0 : sm.took[c & 3], lane);
      if (it.slot == -2 && p.split) break;
      if (it.slot < -1 || c < first) continue;
      for (int i = lane; i < ROWS; i += 32) {
        const int row = i % BM, tok = (it.tile * QT + i / BM) * p.tq + row / p.G;
        if (it.slot >= 0) {
          *reinterpret_cast<float2*>(p.part + (int64_t)2 * gridDim.x * ROWS * D + ((int64_t)it.slot * ROWS + i) * 2) = make_float2(0.f, NAN);
        } else if (row < p.tq * p.G && tok < it.n) {
          const int64_t gt = (int64_t)it.q0 + tok;
          const int head = it.hk * p.G + row % p.G;
          for (int d = 0; d < D; ++d) store16<F16>(p.o, gt * p.o_ts + head * p.o_hs + d, NAN);
          if (p.lse) p.lse[gt * p.Hq + head] = NAN;
        }
      }
    }
  }
}

// Joins the partials of the items that cross shares.  A block per item and 32 rows, a warp per row.
template <int D, bool F16>
__global__ void __launch_bounds__(256) attn_prompt_join_kernel(Params p, int ctas) {
  __shared__ Table tb;
  __shared__ int count;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    const int n = build_table(p, tb, lane);
    if (lane == 0) count = n;
  }
  __syncthreads();
  const int f = blockIdx.x / p.H, hk = blockIdx.x % p.H;
  // (every block waits, those without work too: this grid must not end before the one it follows)
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  if (f >= count) return;
  const int flat = tb.before[count], all = tb.before[f + 1] - tb.before[f] - PAD;
  if (all == 0) return;
  const int64_t per = share_size(p, flat, ctas), begin = (int64_t)hk * flat + tb.before[f];
  const int c0 = (int)(begin / per), c1 = (int)((begin + all - 1) / per);
  if (c0 == c1) return;                                      // finished there
  const int seq = tb.seq[f], tile = tb.tile[f];
  const int2 q = seq_range(p.cu_q, seq, p.Tq);
  const int n = q.y - q.x;
  constexpr int V = D / 32;                                  // channels of a lane
  const float* mlp = p.part + (int64_t)2 * ctas * ROWS * D;
  for (int r = blockIdx.y * 32 + warp; r < blockIdx.y * 32 + 32; r += 8) {
    const int row = r % BM, tok = (tile * QT + r / BM) * p.tq + row / p.G, head = hk * p.G + row % p.G;
    if (row >= p.tq * p.G || tok >= n) continue;
    float mx = -INFINITY, l = 0.f, acc[V];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = 0.f;
    for (int c = c0; c <= c1; ++c) {
      const int64_t row = (2 * (int64_t)c + (c == c0 ? 1 : 0)) * ROWS + r;
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(mlp + row * 2));
      float x[V];
      if constexpr (V == 4) {
        const float4 y = __ldcg(reinterpret_cast<const float4*>(p.part + row * D) + lane);
        x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w;
      } else {
        const float2 y = __ldcg(reinterpret_cast<const float2*>(p.part + row * D) + lane);
        x[0] = y.x; x[1] = y.y;
      }
      // (m = -inf: no visible key, O and l are 0, or all of its scores are NaN, and so are they)
      const float mn = fmaxf(mx, ml.x), f0 = mx == -INFINITY ? 1.f : ex2(mx - mn), f1 = ml.x == -INFINITY ? 1.f : ex2(ml.x - mn);
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = acc[v] * f0 + x[v] * f1;
      l = l * f0 + ml.y * f1;
      mx = mn;
    }
    const int64_t gt = (int64_t)q.x + tok;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    char* orow = reinterpret_cast<char*>(p.o) + 2 * (gt * p.o_ts + head * p.o_hs + lane * V);
    if constexpr (V == 4)
      *reinterpret_cast<uint2*>(orow) = make_uint2(kv::pack16<F16>(acc[0] * inv, acc[1] * inv), kv::pack16<F16>(acc[2] * inv, acc[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(orow) = kv::pack16<F16>(acc[0] * inv, acc[1] * inv);
    if (lane == 0 && p.lse) p.lse[gt * p.Hq + head] = l == 0.f ? -INFINITY : (mx - SHIFT<F16> + log2f(l)) * 0.6931471805599453f;
  }
}

// [T, H, D] 16-bit with the given strides (elements): boxes of 64 channels x `heads` x `tokens`.
static int make_map(CUtensorMap* m, const void* base, int64_t T, int64_t H, int D, int64_t ts, int64_t hs, int heads, int tokens,
                    int f16) {
  tc::EncodeTiledFn fn = tc::encode_tiled_fn();
  if (!fn) return set_error(KB200_ERR_LAUNCH, "attn_prompt: cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)T};
  cuuint64_t strides[2] = {(cuuint64_t)hs * 2, (cuuint64_t)ts * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)tokens};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base),
                        dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(KB200_ERR_INVALID, "attn_prompt: q, k or v cannot be read by TMA (%d)", (int)r);
  return KB200_OK;
}

// How the G query heads of a kv head are taken: in `parts` equal parts of `g` <= 128 heads, `tq`
// tokens to a query tile.
struct Split {
  int64_t parts, g, tq;
};
static Split split_heads(int64_t G) {
  Split s{1, G, 0};
  while (s.g > BM || G % s.parts) {
    ++s.parts;
    s.g = G / s.parts;
  }
  s.tq = BM / s.g;
  return s;
}

// Row tiles that the sequences have at most.
static int64_t most_tiles(int64_t Tq, int64_t N, int64_t tq) { return Tq / (QT * tq) + N; }

// Whether the key tiles are shared out: when whole items would leave SMs idle (up to 3 items for 2
// SMs; beyond that the sorted order balances) and there are enough keys for the partials and the
// second kernel to pay.  (512 + 300 queries over 12345 + 8000 keys, 32/8 heads, 104 items: 135 us in
// shares, 160 us as whole items.)
static bool shares(int64_t Tq, int64_t Tk, int64_t N, int64_t H, const Split& s, int sms) {
  const int64_t tiles = most_tiles(Tq, N, s.tq);
  return tiles <= TABLE && 2 * tiles * H * s.parts <= 3 * sms && Tk >= 2048;
}

template <int D, bool F16>
static int launch(const Maps& maps, const Params& p, int sms, cudaStream_t st) {
  const size_t smem = sizeof(Smem<D>) + 1024;
  static std::atomic<uint64_t> done[2];
  const bool bounded = p.wait_clocks > 0;
  auto* kern = bounded ? attn_prompt_kernel<D, F16, true> : attn_prompt_kernel<D, F16, false>;
  if (int e = allow_smem((const void*)kern, smem, done[bounded])) return e;
  const int64_t items = most_tiles(p.Tq, p.N, p.tq) * p.H;
  const int grid = p.split ? sms : (int)items;
  kern<<<grid, THREADS, smem, st>>>(maps, p);
  if (int e = check_launch("attn_prompt_kernel")) return e;
  if (!p.split) return KB200_OK;
  cudaLaunchAttribute overlap{};
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)items, ROWS / 32);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = &overlap;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, attn_prompt_join_kernel<D, F16>, p, grid);
  return check_launch("attn_prompt_join_kernel");
}

}  // namespace prompt
}  // namespace kb

extern "C" size_t kb200_attn_prompt_workspace_size(int64_t Tq, int64_t Tk, int64_t N, int64_t Hq, int64_t Hkv, int64_t D) {
  using namespace kb;
  if (Tq <= 0 || Tk < 0 || N <= 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || Hq > (1 << 14) || N > (1 << 20) || Tq > 0x7fffff00LL ||
      (D != 64 && D != 128))
    return 0;
  const int sms = sm_count();
  if (!prompt::shares(Tq, Tk, N, Hkv, prompt::split_heads(Hq / Hkv), sms)) return 0;
  return (size_t)2 * sms * prompt::ROWS * (D + 2) * sizeof(float);
}

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
  const prompt::Split sp = prompt::split_heads(a->Hq / a->Hkv);
  // (passing over a number that no tile has takes a CTA 1-2 us: the second limit keeps a run of them, 2^24 / SMs at
  // most, far inside the bounds of the waits)
  if (prompt::most_tiles(a->Tq, a->N, sp.tq) * a->Hkv * sp.parts > 0x7fffffffLL || a->N * a->Hkv * sp.parts > (1 << 24))
    return set_error(KB200_ERR_INVALID, "attn_prompt: too many rows, or sequences times kv heads");
  if (!(fabsf(a->softmax_scale) < INFINITY)) return set_error(KB200_ERR_INVALID, "attn_prompt: softmax_scale=%f", a->softmax_scale);
  if (a->wait_clocks < 0 || a->wait_clocks > 4000000000LL)
    return set_error(KB200_ERR_INVALID, "attn_prompt: wait_clocks=%lld", (long long)a->wait_clocks);
  // a scale of 0 becomes one too small to matter, so that a masked score stays -inf
  const float sl2 = fmaxf(fabsf(a->softmax_scale) * 1.4426950408889634f, 1e-30f);
  const int sms = sm_count();
  const bool split = a->workspace && a->workspace_bytes > 0 && prompt::shares(a->Tq, a->Tk, a->N, a->Hkv, sp, sms);
  if (split && (a->workspace_bytes < kb200_attn_prompt_workspace_size(a->Tq, a->Tk, a->N, a->Hq, a->Hkv, a->D) ||
                !aligned16(a->workspace)))
    return set_error(KB200_ERR_WORKSPACE, "attn_prompt: workspace of %zu bytes given, %zu needed (or none)", a->workspace_bytes,
                     kb200_attn_prompt_workspace_size(a->Tq, a->Tk, a->N, a->Hq, a->Hkv, a->D));
  prompt::Params p{a->q, a->k, a->v, a->o, a->lse, a->cu_q, a->cu_k, a->q_token_stride, a->q_head_stride,
                   a->k_token_stride, a->k_head_stride, a->v_token_stride, a->v_head_stride, a->o_token_stride,
                   a->o_head_stride, a->Tq, a->Tk, (int)a->N, (int)a->Hq, (int)(a->Hkv * sp.parts), (int)sp.g,
                   (int)sp.parts, (int)sp.tq, sl2, a->softmax_scale < 0.f ? 0x80008000u : 0u, split, (float*)a->workspace,
                   a->causal, a->status, a->wait_clocks};
  prompt::Maps maps;
  memset(&maps, 0, sizeof(maps));
  const int D = (int)a->D;
  if (int e = prompt::make_map(&maps.q, a->q, a->Tq, a->Hq, D, a->q_token_stride, a->q_head_stride, p.G, p.tq, a->dtype)) return e;
  maps.k = maps.v = maps.q;
  if (a->Tk > 0) {                                           // (without keys nothing is loaded)
    if (int e = prompt::make_map(&maps.k, a->k, a->Tk, a->Hkv, D, a->k_token_stride, a->k_head_stride, 1, prompt::BN, a->dtype))
      return e;
    if (int e = prompt::make_map(&maps.v, a->v, a->Tk, a->Hkv, D, a->v_token_stride, a->v_head_stride, 1, prompt::BN, a->dtype))
      return e;
  }
  cudaStream_t st = (cudaStream_t)stream;
  if (a->D == 64) return a->dtype ? prompt::launch<64, true>(maps, p, sms, st) : prompt::launch<64, false>(maps, p, sms, st);
  return a->dtype ? prompt::launch<128, true>(maps, p, sms, st) : prompt::launch<128, false>(maps, p, sms, st);
}
