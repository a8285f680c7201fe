// attn_cached.cu -- attention of a few query tokens per sequence over the 8-bit paged
// cache (kv_cache.cuh): the decode step of one token, or Sq drafted tokens at once.
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j,  j < length - Sq + 1 + i
//
// Bound: HBM, 2 D bytes per cached token and kv head.  Rows are the R = Sq * (Hq / Hkv)
// queries that share a kv head, so the cache is read once for all of them.
//
// Split of the work: the groups of 16 (or 32) cached tokens of all (sequence, kv head, row
// block) units are laid end to end and every CTA takes an equal, contiguous share; the
// shares are computed on the device from the lengths, so ragged batches balance without
// the host knowing them.  A unit inside one share is finished there; one that crosses
// shares leaves a partial (m, l, O) per CTA, joined in share order (no atomics: the
// result does not depend on timing) by a second, dependent kernel.
//
// A short unit in a share of several is one warp's alone, without a join (short_unit below).
//
// Every warp has a ring of its own, fills it by 16-byte cp.async (swizzled, so that no load from
// it conflicts) and takes every WK-th group: no warp waits for another inside a unit.  (One
// TMA box per 16 tokens and head ran at 80-100 cycles a box whatever its size, 25 B a cycle
// and SM at D = 128 and half of that at D = 64.)
// Per 16 tokens:
//   S^T = K Q^T  mma.m16n8k16 f16 (16 tokens x 8 rows), codes widened to f16 in
//                registers (exact); the contraction index is permuted so that a lane's
//                operands are 16 consecutive bytes of the page
//   P   = 2^(s - m), running max per row (per warp; the warps join at the end)
//   O^T += V^T P^T, P transposed between the two by movmatrix.  The products of 16
//                tokens are formed from zero and added times their page's V scale in
//                fp32, so pages of very different scales do not cost each other bits.
// Measured: 96 sequences of 2900 tokens, 24/24 heads of 128: 288 us, 5.9 TB/s; 131072 + 100001 tokens, 32/8
// heads: 92 us, 5.2 TB/s; 64 rows (8 queries, 96/12 heads) of 28957 tokens: 82 us, bound by the issue slots of
// its four row blocks.
// bf16 queries are multiplied by a power of two per row into f16's range first (exact
// but for elements 2^-29 below the row's largest).  P is rounded to f16: 2^-11 of itself, and below 2^-22 of the row's
// largest P (where f16's normal numbers end) 2^-33 of that.  So an output is within 2^-11 sum_j p_j |v_j| +
// 2^-33 sum_j |v_j| of the formula: the second term matters where keys of hardly any weight have values 2^20 times
// the others'.  (Those 16 tokens' P brought to f16's top by a power of two per row, where a page's V scale is over 2^8 times
// an earlier one's, took 41.0 us instead of 39.1 for 16 x 6007 tokens, four queries each.)
#include <math.h>
#include <type_traits>
#include "kv_cache.cuh"

namespace kb {
namespace cached {

constexpr float SHIFT = 8.f;       // P = 2^(s - m + SHIFT), s <= m + TAU: below 2^12, inside f16
constexpr float TAU = 4.f;         // O and l are rescaled when the maximum grows by more than this (log2 units)
// V scales are taken times DOWN and O is taken times UP when it is divided by l.  16 tokens' product is at most
// 16 * 2^12 * 448 < 2^25, so without it O would leave fp32 at scales from 2^103 on, and scales reach 2^120; with it
// 2^19 tokens at that scale fit.  The smallest scale, 2^-117, becomes fp32's smallest number: sums keep 2^-17.
constexpr float DOWN = 0x1p-32f, UP = 0x1p32f;

struct Params {
  const void* q;
  void* o;
  float* lse;
  const int32_t *table, *lengths;
  const uint8_t *k_pages, *v_pages;
  const float *k_scale, *v_scale;
  float* part;                     // [2 G][rows][D] partial O, then [2 G][rows][2] (m, l)
  int64_t q_bs, q_ts, q_hs;        // batch, token, head strides of q, elements
  int B, Sq, Hq, H, G, R;          // G = Hq / H query heads per kv head, R = Sq * G
  int rblocks;                     // row blocks per (sequence, kv head)
  int num_pages, max_pages, page;
  int page_log2;
  float scale_log2;                // |softmax scale| log2 e; its sign goes into q (flip)
  uint32_t flip;
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
// The same from zero.  (As an output alone: a zeroed accumulator passed in would cost four moves.)
KB_DEVI void mma_f16_first(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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
// Groups of GT tokens of sequence b, and the length that each of its units takes in the flat
// order: PAD more, positions without work that stand for what a segment costs apart from
// its groups (Q, the join, the stores), so that shares of many short units balance too.
constexpr int PAD = 16;
template <int GT>
KB_DEVI int seq_groups(const Params& p, int b) { return (seq_len(p, b) + GT - 1) / GT; }
template <int GT>
KB_DEVI int seq_span(const Params& p, int b) {
  const int n = seq_groups<GT>(p, b);
  return n ? n + PAD : 0;
}

// Flat position (a sequence takes units * seq_span) -> the sequence that holds
// it and the position where that begins; by one warp.  at < total.
template <int GT>
KB_DEVI void warp_find(const Params& p, int64_t units, int64_t at, int lane, int& b_out, int64_t& begin_out) {
  int64_t base = 0;
  int b0 = 0;
  for (; b0 + 256 < p.B; b0 += 256) {      // many sequences: 256 are passed over at once
    int64_t sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += seq_span<GT>(p, b0 + i * 32 + lane);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (base + units * sum > at) break;
    base += units * sum;
  }
  for (; b0 < p.B; b0 += 32) {
    const int64_t mine = b0 + lane < p.B ? units * seq_span<GT>(p, b0 + lane) : 0;
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

// CTA c works on the flat positions [c * per, (c + 1) * per): a multiple of the consumer warps.
struct Share {
  int64_t total, per;
};
KB_DEVI Share share_of(int64_t units, int64_t sum_spans, int ctas, int wk) {
  Share s;
  s.total = sum_spans * units;
  s.per = (s.total + (int64_t)ctas * wk - 1) / ((int64_t)ctas * wk) * wk;
  return s;
}

// Where 16-byte chunk `c` of token row `r` lies in a slot.  Eight lanes that load together (K: two
// rows, V: every second row, one or two channel chunks) meet eight different chunks of a line.
template <int D>
KB_DEVI uint32_t swz(int r, int c) {
  if constexpr (D == 128) return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
  else return (uint32_t)((r >> 1) * 128 + (((((r & 1) << 2) | c) ^ (((r >> 1) & 3) << 1)) << 4));
}

// Where 16-byte chunk `c` of row `r` of a warp's O lies in the slot it kept: the eight lanes that store
// together (two chunk groups, four rows r = 2 t) meet eight different chunks of a line.
template <int D>
KB_DEVI int o_chunk(int r, int c) {
  const int t = (r >> 1) & 3;
  return r * (D / 4) + (c ^ (D == 128 ? t : (t & 1) | (t & 2) << 1));
}

// The launch shapes.  NT: 8-row tiles of a CTA (rows up to 8: 1, else 2); a group is NT * 16
// tokens.  WK warps, OCC CTAs per SM: as many as the registers allow with little spilling (8 to 188 bytes a thread;
// 16 rows at D = 128 take all 255 registers: with 12 warps of 168, 32 queries of 32 sequences of 4000 tokens
// took 176-180 us and not 130-133).
template <int D, int NT>
struct Shape {
  static constexpr int GT = NT * 16, ROWS = NT * 8;
  static constexpr int WK = 8;
  static constexpr int OCC = D == 128 ? (NT == 1 ? 2 : 1) : (NT == 1 ? 3 : 2);
  static constexpr int STAGES = D == 64 && NT == 1 ? 4 : 3;
  static constexpr int THREADS = WK * 32;
  static constexpr int JOIN = ROWS * D / 4;  // threads of a joining block: four channels of a row each
};

// A unit is short if a warp alone should take it.  Spread over the WK = 8 warps it costs ng / 8 groups and
// about 2 more for the join, in which all warps wait; one warp's alone ng groups and no join, but the
// share's U = per / (ng + PAD) units may not go evenly into the warps, which costs up to ng groups
// once.  So units of up to 4 U groups are taken alone, if there are at least 4 to a share.  (1024
// sequences of 100 tokens, 24/8 heads of 128: 78 us so, 161 us without; 256 of 300: 53 and 68 us.)
KB_DEVI int short_unit(int64_t per) {      // ng <= per / 4 - PAD, ng (ng + PAD) <= 4 per
  const float x = (float)per;
  return (int)fminf(x * 0.25f - PAD, sqrtf(4.f * x + PAD * PAD / 4) - PAD / 2);
}

// A CTA's segments, in order: the groups [g0, g0 + count) of unit (b, h, rb); `ng` are all of
// the unit's.  (Parts of a share that are padding alone are passed over.)
template <int GT, int WK>
struct Walk {
  int64_t left;                        // flat positions still to come
  int b, u, x;                         // the next one: sequence, unit, position in the unit
  int b_of, h, rb, len, ng, g0, count; // (b_of: the segment's sequence)
  int short_ng;                        // units of up to so many groups are short
  int turn, solo;                      // the warp that takes the next short unit; that takes this segment, -1: all do
  KB_DEVI void start(const Params& p, int64_t at, int64_t end, int64_t per, int b_, int64_t begin) {
    left = end - at;
    short_ng = short_unit(per);
    turn = 0;
    b = b_;
    const int span = seq_span<GT>(p, b);
    u = (int)((at - begin) / span);
    x = (int)((at - begin) - (int64_t)u * span);
  }
  // (by a warp, whose lanes all have the same; 32 sequences are looked at for one that is not empty)
  KB_DEVI bool next(const Params& p, int units, int lane, int warp) {
    while (left > 0) {
      if (u == units) {
        u = x = 0;
        uint32_t some = 0;
        for (++b; b < p.B; b += 32) {
          some = __ballot_sync(0xffffffffu, b + lane < p.B && seq_len(p, b + lane) > 0);
          if (some) break;
        }
        if (!some) return false;
        b += __ffs(some) - 1;
      }
      len = seq_len(p, b);
      ng = (len + GT - 1) / GT;
      const bool alone = ng <= short_ng;
      if (alone && x == 0) {           // the other warps' short units of this sequence are passed over at once
        const int k = min(min(warp >= turn ? warp - turn : warp + WK - turn, units - u), (int)min(left, (int64_t)0x7fffffff) / (ng + PAD));
        u += k;
        left -= (int64_t)k * (ng + PAD);
        turn = turn + k >= WK ? turn + k - WK : turn + k;
        if (u == units || left <= 0) continue;
      }
      const int take = (int)min((int64_t)max(ng + PAD - x, 1), left);
      left -= take;
      g0 = x;
      count = min(x + take, ng) - x;
      b_of = b;
      h = u / p.rblocks;
      rb = u - h * p.rblocks;
      x += take;
      if (x >= ng + PAD) {
        x = 0;
        ++u;
      }
      if (count > 0) {
        solo = -1;
        if (alone && count == ng) {
          solo = turn;
          turn = turn + 1 == WK ? 0 : turn + 1;
          if (solo != warp) continue;
        }
        return true;
      }
    }
    return false;
  }
};

// The first of a segment's groups that `warp` takes, and with which it goes on: a short unit is one
// warp's alone; else every WK-th group, beginning so that short segments use all warps in turn.
template <int GT, int WK>
KB_DEVI int first_group(const Walk<GT, WK>& seg, int rot, int warp) {
  if (seg.solo >= 0) return 0;
  return warp >= rot ? warp - rot : warp + WK - rot;
}

// Where the loading side of a warp is: kept in shared memory, since it is touched once per
// batch and the registers are short.
template <int GT, int WK>
struct Feed {
  Walk<GT, WK> seg;
  int rot, first, done;                      // of the segment: rotation, the warp's first group, groups batched
  int step;                                  // tokens from one of the warp's groups to the next
  int live;
  int h, n, tok0;                            // the next batch: head, groups, first token of its first group
};

template <int D, int NT>
struct Smem {
  using S = Shape<D, NT>;
  struct Slot {
    uint8_t k[S::GT * D], v[S::GT * D];      // swizzled page rows
  };
  static_assert(sizeof(Slot) == S::ROWS * D * sizeof(float), "a slot also holds a warp's O");
  Slot slot[S::WK][S::STAGES];
  float ml[S::WK][S::ROWS][2];
  float2 scale[S::WK][S::STAGES][NT];        // page scales (k, v) of 16 tokens each; k < 0: no such page
  Feed<S::GT, S::WK> feed[S::WK];
  Walk<S::GT, S::WK> walk[S::WK];
  Walk<S::GT, S::WK> start;
  int64_t total;
  int held[S::WK];                           // the slot that holds the warp's O, -1: none
};

// The loading side of one warp: its groups in the order of the segments, STAGES ahead of
// their use.  Page ids and scales are read by lanes, a batch of 32 16-token parts at once and
// a batch ahead; a batch lies in one segment.
template <int D, int NT>
struct Loader {
  using S = Shape<D, NT>;
  static constexpr int BATCH = 32 / NT;      // groups of a batch
  Feed<S::GT, S::WK>* feed;
  int n, pos, row;                           // current batch: groups, next one; this lane's part: its first code row, -1: no such page
  int pg2;                                   // the next batch's: its row, or while `pending` the page that it is formed from
  float2 sc, sc2;
  bool pending;                              // sc2 is still to be read
  float2* owed;                              // where the last group's scales are still to be written (null: nowhere)

  // The scales of the group loaded last.  They are written one call later, so that the copies
  // of a group do not wait for them.
  KB_DEVI void pay(int lane) {
    if (owed) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int src = (pos - 1) * NT + j;
        const float2 s = make_float2(__shfl_sync(0xffffffffu, sc.x, src), __shfl_sync(0xffffffffu, sc.y, src));
        if (lane == 0) owed[j] = s;
      }
    }
    owed = nullptr;
  }
  KB_DEVI void next_batch(const Params& p, int units, int warp, int lane) {
    __syncwarp();
    Feed<S::GT, S::WK> f = *feed;
    f.n = 0;
    pg2 = -1;
    pending = false;
    while (f.live) {
      const bool solo = f.seg.solo >= 0;
      const int by = solo ? 1 : S::WK;
      const int mine = f.seg.count > f.first ? (f.seg.count - f.first + by - 1) / by : 0;   // this warp's groups of the segment
      if (f.done < mine) {
        f.n = min(BATCH, mine - f.done);
        f.h = f.seg.h;
        const int gi = f.first + (f.done + lane / NT) * by;
        if (gi < f.seg.count) {
          const int tok = (f.seg.g0 + gi) * S::GT + (lane % NT) * 16;
          if (tok < f.seg.len) pg2 = __ldg(p.table + (int64_t)f.seg.b_of * p.max_pages + (tok >> p.page_log2));
        }
        f.tok0 = (f.seg.g0 + f.first + f.done * by) * S::GT;
        f.step = by * S::GT;
        f.done += f.n;
        pending = true;
        break;
      }
      if (!solo) f.rot = (f.rot + f.seg.count) % S::WK;
      f.done = 0;
      f.live = f.seg.next(p, units, lane, warp);
      f.first = first_group(f.seg, f.rot, warp);
    }
    __syncwarp();
    if (lane == 0) *feed = f;
    __syncwarp();
  }
  KB_DEVI void read_scales(const Params& p, int lane) {
    sc2 = make_float2(-1.f, 0.f);
    if (pg2 >= 0 && pg2 < p.num_pages) {
      const int64_t i = (int64_t)pg2 * p.H + feed->h;
      sc2.x = __ldg(p.k_scale + i);
      sc2.y = __ldg(p.v_scale + i) * DOWN;
      const int tok = feed->tok0 + (lane / NT) * feed->step + (lane % NT) * 16;
      pg2 = (int)i * p.page + (tok & (p.page - 1));   // (below 2^31: the pool's limit)
    } else {
      pg2 = -1;
    }
    pending = false;
  }
  KB_DEVI Loader(Feed<S::GT, S::WK>* at, const Params& p, int units, int warp, int lane) : feed(at), n(0), pos(0), owed(nullptr) {
    next_batch(p, units, warp, lane);
  }
  // The next group into `slot`; always one cp.async group, empty when the work is over.
  KB_DEVI void load(const Params& p, int units, int warp, int lane, typename Smem<D, NT>::Slot& slot, float2* scale) {
    if (pos == n) {
      pay(lane);
      if (pending) read_scales(p, lane);
      n = feed->n;
      row = pg2; sc = sc2;
      pos = 0;
      if (n) next_batch(p, units, warp, lane);
    } else if (pending) {
      read_scales(p, lane);
    }
    float2* now = nullptr;
    if (n) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int from = __shfl_sync(0xffffffffu, row, pos * NT + j);
        if (from >= 0) {
          const uint8_t *ks = p.k_pages + (int64_t)from * D + lane * 16, *vs = p.v_pages + (int64_t)from * D + lane * 16;
          constexpr int RPI = 512 / D;       // rows that the warp's 32 chunks cover
#pragma unroll
          for (int i = 0; i < 16 / RPI; ++i) {
            const uint32_t dst = swz<D>(j * 16 + i * RPI + lane / (D / 16), lane % (D / 16));
            cp_async16(slot.k + dst, ks + i * 512, true);
            cp_async16(slot.v + dst, vs + i * 512, true);
          }
        }
      }
      now = scale;
    }
    cp_async_commit();
    pay(lane);
    pos += n ? 1 : 0;
    owed = now;
  }
};

template <int D, bool F16, int NT>
__global__ void __launch_bounds__(Shape<D, NT>::THREADS, Shape<D, NT>::OCC)
    attn_cached_kernel(Params p) {
  using S = Shape<D, NT>;
  using SM = Smem<D, NT>;
  constexpr int WK = S::WK, STAGES = S::STAGES, GT = S::GT, ROWS = S::ROWS;
  constexpr int MT = D / 16;               // 16-wide tiles of D
  extern __shared__ __align__(128) unsigned char smem_raw[];
  SM& sm = *reinterpret_cast<SM*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t units = (int64_t)p.H * p.rblocks;

  if (warp == 0) {
    int64_t sum = 0;
    for (int b = lane; b < p.B; b += 32) sum += seq_span<GT>(p, b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const Share sh = share_of(units, sum, gridDim.x, WK);
    int b = 0;
    int64_t begin = 0;
    if ((int64_t)blockIdx.x * sh.per < sh.total) warp_find<GT>(p, units, blockIdx.x * sh.per, lane, b, begin);
    if (lane == 0) {
      sm.total = sum;
      if ((int64_t)blockIdx.x * sh.per < sh.total)
        sm.start.start(p, blockIdx.x * sh.per, min((blockIdx.x + 1) * sh.per, sh.total), sh.per, b, begin);
    }
  }
  __syncthreads();
  const Share sh = share_of(units, sm.total, gridDim.x, WK);
  const int64_t at0 = (int64_t)blockIdx.x * sh.per, at1 = min(at0 + sh.per, sh.total);
  // the join may be scheduled as soon as CTAs leave; it waits for all of them before it reads
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  if (at0 >= at1) return;

  // Every warp walks the CTA's segments in the same order.  Group i of a segment goes to
  // warp (i + rot) % WK, so that short segments use all of them in turn.
  {
    Feed<GT, WK> f{};
    f.seg = sm.start;
    if (lane == 0) sm.walk[warp] = f.seg;
    f.live = f.seg.next(p, (int)units, lane, warp);
    f.first = first_group(f.seg, 0, warp);
    if (lane == 0) sm.feed[warp] = f;
  }
  Loader<D, NT> loader(&sm.feed[warp], p, (int)units, warp, lane);
  for (int s = 0; s < STAGES; ++s) loader.load(p, (int)units, warp, lane, sm.slot[warp][s], sm.scale[warp][s]);
  Walk<GT, WK> seg;
  auto next_segment = [&]() {              // the using side's walk, in shared memory too
    __syncwarp();
    seg = sm.walk[warp];
    const bool more = seg.next(p, (int)units, lane, warp);
    __syncwarp();
    if (lane == 0) sm.walk[warp] = seg;
    __syncwarp();
    return more;
  };
  int rot = 0;
  const int g = lane >> 2, t4 = lane & 3;
  int s = 0;                               // this warp's next slot
  constexpr int CH = D / 64;               // 16-byte code chunks per lane and row
  uint32_t raw[NT][CH * 8];                // the segment's Q, read while the one before is joined
  auto load_q = [&]() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = seg.rb * ROWS + n * 8 + g;
      const bool in = r < p.R;
      const char* src = reinterpret_cast<const char*>(p.q);
      if (in) src += 2 * ((int64_t)seg.b_of * p.q_bs + (int64_t)(r / p.G) * p.q_ts + (int64_t)(seg.h * p.G + r % p.G) * p.q_hs +
                          t4 * (CH * 16));
#pragma unroll
      for (int c = 0; c < CH * 2; ++c) {
        const uint4 x = in ? __ldg(reinterpret_cast<const uint4*>(src) + c) : make_uint4(0, 0, 0, 0);
        raw[n][4 * c] = x.x ^ p.flip; raw[n][4 * c + 1] = x.y ^ p.flip; raw[n][4 * c + 2] = x.z ^ p.flip;
        raw[n][4 * c + 3] = x.w ^ p.flip;
      }
    }
  };
  bool live = next_segment();
  if (live) load_q();
  while (live) {
    const bool solo = seg.solo >= 0;
    const int len = seg.len, first = first_group(seg, rot, warp), step = (solo ? 1 : WK) * GT;
    int left = first < seg.count ? solo ? seg.count : (seg.count - first + WK - 1) / WK : 0;   // this warp's groups
    int base = (seg.g0 + first) * GT;
    if (!solo) rot = (rot + seg.count) % WK;

    // Q^T operands: row n = g of each 8-row tile, this lane's D / 4 channels from t4 * D / 4, as
    // f16 under a power of two per row.
    uint32_t qf[NT][CH * 8];
    float qs[NT][2];                       // log2-domain score factors of the rows 2 t4, 2 t4 + 1
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float f = 1.f;
      if constexpr (F16) {
#pragma unroll
        for (int c = 0; c < CH * 8; ++c) qf[n][c] = raw[n][c];
      } else {
        float amax = 0.f;
#pragma unroll
        for (int c = 0; c < CH * 8; ++c) {
          const float2 x = unpack_bf16(raw[n][c]);
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
          const float2 x = unpack_bf16(raw[n][c]);
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
        const int r = seg.rb * ROWS + n * 8 + 2 * t4 + c;
        seen[n][c] = r < p.R ? len - p.Sq + 1 + r / p.G : len;
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
    }
    const int all_seen = len - p.Sq + 1;   // keys below are seen by every row

    int held = -1;
    for (; left > 0; --left, base += step) {
      cp_async_wait<STAGES - 1>();         // the oldest group has landed, for every lane
      __syncwarp();
      const typename SM::Slot& sl = sm.slot[warp][s];
      float sk[NT], sv[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const float2 sc = sm.scale[warp][s][j];
        sk[j] = sc.x;
        sv[j] = sc.y;
      }
      // Groups in which some row does not see some token, or a page is missing, take a body of their
      // own, so that the others' is free of the tests.
      auto body = [&](auto edge_group) {
      constexpr bool EDGE = decltype(edge_group)::value;
      // ---- S^T = K Q^T of the group's 16-token parts
      float acc[NT][NT][4];                // [part][row tile]
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const int r0 = j * 16 + g;
          const uint4 x0 = *reinterpret_cast<const uint4*>(sl.k + swz<D>(r0, t4 * CH + c));
          const uint4 x1 = *reinterpret_cast<const uint4*>(sl.k + swz<D>(r0 + 8, t4 * CH + c));
          const uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t a[4];
            kv::decode4(w0[e], a[0], a[2]);
            kv::decode4(w1[e], a[1], a[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n)
              if (c == 0 && e == 0) mma_f16_first(acc[j][n], a, qf[n][0], qf[n][1]);
              else mma_f16(acc[j][n], a, qf[n][c * 8 + 2 * e], qf[n][c * 8 + 2 * e + 1]);
          }
        }
      }
      // ---- softmax; lane: tokens g, g + 8 of each part, rows 2 t4, 2 t4 + 1.  The rows' maxima
      // are looked up over the warp only when some lane's score passes the reference by TAU.
      uint32_t pf[NT][NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float t0m = -INFINITY, t1m = -INFINITY;
        float f0[NT], f1[NT];              // score factors, kept above 0: a masked -inf stays one
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float* x = acc[j][n];
          f0[j] = fmaxf(sk[j] * qs[n][0], 1e-37f);
          f1[j] = fmaxf(sk[j] * qs[n][1], 1e-37f);
          if (EDGE && sk[j] < 0.f) {       // a missing page
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = -INFINITY;
          }
          if (EDGE) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (base + j * 16 + g + (e >> 1) * 8 >= seen[n][e & 1]) x[e] = -INFINITY;
          }
          t0m = fmaxf(t0m, fmaxf(x[0], x[2]) * f0[j]);
          t1m = fmaxf(t1m, fmaxf(x[1], x[3]) * f1[j]);
        }
        if (__any_sync(0xffffffffu, t0m > m[n][0] + TAU || t1m > m[n][1] + TAU)) {
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) {
            t0m = fmaxf(t0m, __shfl_xor_sync(0xffffffffu, t0m, w));
            t1m = fmaxf(t1m, __shfl_xor_sync(0xffffffffu, t1m, w));
          }
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
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float* x = acc[j][n];
          const float p0 = ex2(fmaf(x[0], f0[j], b0)), p1 = ex2(fmaf(x[1], f1[j], b1)), p2 = ex2(fmaf(x[2], f0[j], b0)),
                      p3 = ex2(fmaf(x[3], f1[j], b1));
          l[n][0] += p0 + p2;
          l[n][1] += p1 + p3;
          pf[j][n][0] = transpose8(kv::pack16<true>(p0, p1));
          pf[j][n][1] = transpose8(kv::pack16<true>(p2, p3));
        }
      }
      // ---- O^T += sv V^T P^T; lane: tokens 2 t4, +1, +8, +9, channels g * D/8 ...
      constexpr int VW = D / 32;           // 32-bit words of channels per lane
#pragma unroll
      for (int part = 0; part < NT; ++part) {
        if (EDGE && sk[part] < 0.f) continue;
        uint32_t vr[4][VW];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = part * 16 + 2 * t4 + (j & 1) + (j >> 1) * 8;
          if constexpr (D == 128) {
            const uint4 x = *reinterpret_cast<const uint4*>(sl.v + swz<D>(r, g));
            vr[j][0] = x.x; vr[j][1] = x.y; vr[j][2] = x.z; vr[j][3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(sl.v + swz<D>(r, g >> 1) + (g & 1) * 8);
            vr[j][0] = x.x; vr[j][1] = x.y;
          }
        }
        bool poison = false;               // a NaN code that some rows must not see
        if (EDGE) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int tok = base + part * 16 + 2 * t4 + (j & 1) + (j >> 1) * 8;
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
            uint32_t a[4];
            kv::decode4(u01, a[0], a[1]);
            kv::decode4(u89, a[2], a[3]);
            if (EDGE && poison) {
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
                float cnt[4], vis[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) vis[e] = base + part * 16 + g + (e >> 1) * 8 < seen[n][e & 1] ? 1.f : 0.f;
                mma_f16_first(cnt, bad, transpose8(kv::pack16<true>(vis[0], vis[1])), transpose8(kv::pack16<true>(vis[2], vis[3])));
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (cnt[e] > 0.f) o[n][2 * w + z][e] = __uint_as_float(0x7fffffffu);
              }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float d[4];
              mma_f16_first(d, a, pf[part][n][0], pf[part][n][1]);
              float* oo = o[n][2 * w + z];
              const float2 s2 = make_float2(sv[part], sv[part]);
              const float2 o01 = ffma2(make_float2(d[0], d[1]), s2, make_float2(oo[0], oo[1]));
              const float2 o23 = ffma2(make_float2(d[2], d[3]), s2, make_float2(oo[2], oo[3]));
              oo[0] = o01.x; oo[1] = o01.y; oo[2] = o23.x; oo[3] = o23.y;
            }
          }
        }
      }
      };
      bool edge = base + GT > all_seen;
#pragma unroll
      for (int j = 0; j < NT; ++j) edge |= sk[j] < 0.f;
      if (edge) body(std::true_type{});
      else body(std::false_type{});
      __syncwarp();
      // the last slot of the segment is kept: it takes the warp's O
      if (left > 1 || step == GT) loader.load(p, (int)units, warp, lane, sm.slot[warp][s], sm.scale[warp][s]);
      else held = s;
      s = s + 1 == STAGES ? 0 : s + 1;
    }
    const Walk<GT, WK> now = sm.walk[warp];      // (the segment again: read back, not kept over the loop)
    const int b = now.b_of, h = now.h, rb = now.rb, g0 = now.g0;
    const bool whole = now.count == now.ng;
    // ---- the warps' partial results join: each one's O in the slot it kept
    if (held >= 0) {
      float4* mo = reinterpret_cast<float4*>(&sm.slot[warp][held]);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = l[n][c];
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
          const int r = n * 8 + 2 * t4 + c;
          if (g == 0) {
            sm.ml[warp][r][0] = m[n][c];
            sm.ml[warp][r][1] = x;
          }
#pragma unroll
          for (int i = 0; i < MT; i += 2)    // channels g * D/8 + 2 i .. + 3
            mo[o_chunk<D>(r, g * (D / 32) + i / 2)] = make_float4(o[n][i][c], o[n][i][2 + c], o[n][i + 1][c], o[n][i + 1][2 + c]);
        }
      }
    }
    if (lane == 0 && step != GT) sm.held[warp] = held;
    live = next_segment();
    if (live) load_q();
    if (step == GT) {
      // ---- this warp has all of the unit
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = l[n][c];
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
          const int rr = rb * ROWS + n * 8 + 2 * t4 + c;
          if (rr >= p.R) continue;
          const float inv = x > 0.f || x != x ? UP / x : 0.f;
          const int64_t orow = ((int64_t)b * p.Sq + rr / p.G) * p.Hq + h * p.G + rr % p.G;
          uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<char*>(p.o) + 2 * (orow * D + g * (D / 8)));
#pragma unroll
          for (int i = 0; i < MT; i += 4)    // channels g * D/8 + 2 i .. + 7
            dst[i / 4] = make_uint4(kv::pack16<F16>(o[n][i][c] * inv, o[n][i][2 + c] * inv),
                                    kv::pack16<F16>(o[n][i + 1][c] * inv, o[n][i + 1][2 + c] * inv),
                                    kv::pack16<F16>(o[n][i + 2][c] * inv, o[n][i + 2][2 + c] * inv),
                                    kv::pack16<F16>(o[n][i + 3][c] * inv, o[n][i + 3][2 + c] * inv));
          if (g == 0 && p.lse) p.lse[orow] = x == 0.f ? -INFINITY : (m[n][c] - SHIFT + log2f(x)) * 0.6931471805599453f;
        }
      continue;
    }
    __syncthreads();
    const int slot = 2 * blockIdx.x + (g0 > 0 ? 0 : 1);   // a share's first segment may end a unit, its last may begin one
    for (int i = tid; i < ROWS * (D / 4); i += WK * 32) {
      const int r = i / (D / 4), c = i % (D / 4);
      if (rb * ROWS + r >= p.R) break;     // rows in order: no more of them
      float mk[WK], mx = -INFINITY;
#pragma unroll
      for (int k = 0; k < WK; ++k) {
        mk[k] = sm.ml[k][r][0];
        if (sm.held[k] >= 0) mx = fmaxf(mx, mk[k]);
      }
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      float ls = 0.f;
#pragma unroll
      for (int k = 0; k < WK; ++k) {
        const int hs = sm.held[k];
        if (hs >= 0) {
          // (m = -inf: no visible key, O and l are 0, or all of its scores are NaN, and so are they)
          const float f = mk[k] == -INFINITY ? 1.f : ex2(mk[k] - mx);
          const float4 x = reinterpret_cast<const float4*>(&sm.slot[k][hs])[o_chunk<D>(r, c)];
          a.x += f * x.x; a.y += f * x.y; a.z += f * x.z; a.w += f * x.w;
          ls += f * sm.ml[k][r][1];
        }
      }
      if (!whole) {
        float* dst = p.part + ((int64_t)slot * ROWS + r) * D + c * 4;
        *reinterpret_cast<float4*>(dst) = a;
        if (c == 0) {
          float* ml = p.part + (int64_t)2 * gridDim.x * ROWS * D + ((int64_t)slot * ROWS + r) * 2;
          ml[0] = mx;
          ml[1] = ls;
        }
      } else {
        const int rr = rb * ROWS + r;
        if (rr < p.R) {
          const float inv = ls > 0.f || ls != ls ? UP / ls : 0.f;
          const int64_t orow = ((int64_t)b * p.Sq + rr / p.G) * p.Hq + h * p.G + rr % p.G;
          uint2 w;
          w.x = kv::pack16<F16>(a.x * inv, a.y * inv);
          w.y = kv::pack16<F16>(a.z * inv, a.w * inv);
          *reinterpret_cast<uint2*>(reinterpret_cast<char*>(p.o) + 2 * (orow * D + c * 4)) = w;
          if (c == 0 && p.lse) p.lse[orow] = ls == 0.f ? -INFINITY : (mx - SHIFT + log2f(ls)) * 0.6931471805599453f;
        }
      }
    }
    __syncthreads();
    if (held >= 0) loader.load(p, (int)units, warp, lane, sm.slot[warp][held], sm.scale[warp][held]);
  }
}

// Joins the partials of the units that cross shares, and writes the empty sequences.  Block c looks
// at the border before share c; the block of a unit's first border joins it.  (So there are as many
// blocks as shares, whatever the number of units.)
template <int D, bool F16, int NT>
__global__ void __launch_bounds__(Shape<D, NT>::JOIN) attn_cached_join_kernel(Params p, int ctas) {
  constexpr int THREADS = Shape<D, NT>::JOIN;
  constexpr int GT = Shape<D, NT>::GT, ROWS = Shape<D, NT>::ROWS;
  const int lane = threadIdx.x & 31;
  const int64_t units = (int64_t)p.H * p.rblocks;
  int64_t sum = 0;
  for (int i = lane; i < p.B; i += 32) sum += seq_span<GT>(p, i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const Share sh = share_of(units, sum, ctas, Shape<D, NT>::WK);
  const int64_t at = (int64_t)blockIdx.x * sh.per;
  int b = 0, u = 0, c0 = 0, c1 = -1;       // the unit, and the CTAs whose shares hold a part of it (none: nothing to join)
  if (blockIdx.x > 0 && at < sh.total) {
    int64_t begin;
    warp_find<GT>(p, units, at, lane, b, begin);
    const int ng = seq_groups<GT>(p, b), span = seq_span<GT>(p, b);
    u = (int)((at - begin) / span);
    const int before = (int)(at - begin - (int64_t)u * span);   // the unit's groups on this side of the border
    if (before > 0 && before < ng && (at - before) / sh.per == blockIdx.x - 1) {
      c0 = (int)blockIdx.x - 1;
      c1 = (int)((at - before + ng - 1) / sh.per);
    }
  }
  // (every block waits, those without work too: this grid must not end before the one it follows)
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const int64_t per_seq = (int64_t)p.Sq * p.Hq;
  for (int i = blockIdx.x; i < p.B; i += gridDim.x)
    if (seq_len(p, i) == 0) {
      for (int64_t e = threadIdx.x; e < per_seq * (D / 8); e += THREADS)
        reinterpret_cast<uint4*>(p.o)[i * per_seq * (D / 8) + e] = make_uint4(0, 0, 0, 0);
      if (p.lse)
        for (int64_t e = threadIdx.x; e < per_seq; e += THREADS) p.lse[i * per_seq + e] = -INFINITY;
    }
  if (c1 < c0) return;
  const int h = u / p.rblocks, rb = u % p.rblocks;
  // Partials in share order: the part that begins the unit is its CTA's last segment (slot 1),
  // the later ones continue it (slot 0).  A chunk's m and l are read together, then its O with
  // all loads in flight: what the join costs is the two latencies.
  constexpr int CHUNK = 32;
  __shared__ float fac[CHUNK][ROWS], run_m[ROWS], run_l[ROWS], scale_old[ROWS];
  const float2* mlp = reinterpret_cast<const float2*>(p.part + (int64_t)2 * ctas * ROWS * D);
  const int r = threadIdx.x / (D / 4), c = threadIdx.x % (D / 4), rr = rb * ROWS + r;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (threadIdx.x < ROWS) {
    run_m[threadIdx.x] = -INFINITY;
    run_l[threadIdx.x] = 0.f;
  }
  __syncthreads();
  for (int k0 = c0; k0 <= c1; k0 += CHUNK) {
    const int n = min(CHUNK, c1 + 1 - k0);
    // the first parts' O is on its way while the factors are formed
    constexpr int EARLY = 8;
    float4 first[EARLY];
    auto part_of = [&](int k) {
      return reinterpret_cast<const float4*>(p.part + ((2 * (int64_t)(k0 + k) + (k0 + k == c0 ? 1 : 0)) * ROWS + r) * D + c * 4);
    };
#pragma unroll
    for (int k = 0; k < EARLY; ++k) first[k] = k < n && rr < p.R ? __ldcg(part_of(k)) : make_float4(0.f, 0.f, 0.f, 0.f);
    // a warp per row, a lane per part: the parts' factors, and that of what is joined so far
    for (int w = threadIdx.x >> 5; w < ROWS; w += THREADS / 32) {
      float2 x = make_float2(-INFINITY, 0.f);
      if (lane < n) x = __ldcg(mlp + (2 * (int64_t)(k0 + lane) + (k0 + lane == c0 ? 1 : 0)) * ROWS + w);
      const float before = run_m[w], mx = fmaxf(before, warp_max(x.x));
      // (m = -inf: no visible key, O and l are 0, or all of its scores are NaN, and so are they)
      const float f = x.x == -INFINITY ? 1.f : ex2(x.x - mx), f0 = before == -INFINITY ? 1.f : ex2(before - mx);
      const float l = warp_sum(f * x.y) + run_l[w] * f0;
      fac[lane][w] = f;
      __syncwarp();
      if (lane == 0) {
        scale_old[w] = f0;
        run_m[w] = mx;
        run_l[w] = l;
      }
    }
    __syncthreads();
    if (rr < p.R) {
      const float f0 = scale_old[r];
      acc.x *= f0; acc.y *= f0; acc.z *= f0; acc.w *= f0;
#pragma unroll
      for (int k = 0; k < EARLY; ++k)
        if (k < n) {
          const float f = fac[k][r];
          const float4 x = first[k];
          acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
        }
#pragma unroll 8
      for (int k = EARLY; k < n; ++k) {
        const float f = fac[k][r];
        const float4 x = __ldcg(part_of(k));
        acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
      }
    }
    __syncthreads();
  }
  if (rr >= p.R) return;
  const float l = run_l[r], inv = l > 0.f || l != l ? UP / l : 0.f;
  const int64_t orow = ((int64_t)b * p.Sq + rr / p.G) * p.Hq + h * p.G + rr % p.G;
  uint2 w;
  w.x = kv::pack16<F16>(acc.x * inv, acc.y * inv);
  w.y = kv::pack16<F16>(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(reinterpret_cast<char*>(p.o) + 2 * (orow * D + c * 4)) = w;
  if (c == 0 && p.lse) p.lse[orow] = l == 0.f ? -INFINITY : (run_m[r] - SHIFT + log2f(l)) * 0.6931471805599453f;
}

// 8-row tiles that a CTA takes of the R = Sq * Hq / Hkv rows: rows above 16 form blocks that
// read the cache again, mostly from L2 (more tiles per warp would not fit the registers).
static int row_tiles(int64_t R) { return R <= 8 ? 1 : 2; }

// CTAs of the main kernel: as many as fit on the GPU at once, no more than can have work.
template <int D, int NT>
static int grid_of(int64_t B, int64_t H, int64_t R, int64_t max_tokens) {
  using S = Shape<D, NT>;
  const int64_t most = (B * H * ((R + S::ROWS - 1) / S::ROWS) * ((max_tokens + S::GT - 1) / S::GT + PAD) + S::WK - 1) / S::WK;
  const int64_t fit = (int64_t)sm_count() * S::OCC;
  return (int)(most < 1 ? 1 : most < fit ? most : fit);
}
static int grid_of(int64_t D, int64_t B, int64_t H, int64_t R, int64_t max_tokens) {
  if (D == 64) return row_tiles(R) == 1 ? grid_of<64, 1>(B, H, R, max_tokens) : grid_of<64, 2>(B, H, R, max_tokens);
  return row_tiles(R) == 1 ? grid_of<128, 1>(B, H, R, max_tokens) : grid_of<128, 2>(B, H, R, max_tokens);
}

template <int D, bool F16, int NT>
static int launch(const Params& p, int grid, cudaStream_t st) {
  using S = Shape<D, NT>;
  const size_t smem = sizeof(Smem<D, NT>);
  auto* kern = attn_cached_kernel<D, F16, NT>;
  static std::atomic<uint64_t> done{0};
  if (int e = allow_smem((const void*)kern, smem, done)) return e;
  kern<<<grid, S::THREADS, smem, st>>>(p);
  if (int e = check_launch("attn_cached_kernel")) return e;
  cudaLaunchAttribute overlap{};
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(S::JOIN);
  cfg.stream = st;
  cfg.attrs = &overlap;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, attn_cached_join_kernel<D, F16, NT>, p, grid);
  return check_launch("attn_cached_join_kernel");
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
  const int grid = grid_of(D, B, Hkv, R, max_pages * page);
  return (size_t)2 * grid * row_tiles(R) * 8 * (D + 2) * sizeof(float);
}

extern "C" int kb200_attn_cached_fwd(const KB200AttnCachedArgs* a, void* stream) {
  using namespace kb;
  if (!a) return set_error(KB200_ERR_INVALID, "attn_cached: null arguments");
  const KB200KvCache* c = &a->cache;
  const int64_t B = a->B, Sq = a->Sq, Hq = a->Hq, max_pages = a->max_pages;
  const bool dtype = a->dtype == 1;
  if (int e = kv::check_cache(c, "attn_cached")) return e;
  if (int e = cached::check_shape(B, Sq, Hq, c->H, max_pages)) return e;
  if (a->dtype != 0 && a->dtype != 1) return set_error(KB200_ERR_INVALID, "attn_cached: dtype=%lld", (long long)a->dtype);
  if (!(fabsf((float)a->softmax_scale) < INFINITY))
    return set_error(KB200_ERR_INVALID, "attn_cached: softmax_scale=%f", a->softmax_scale);
  if (B == 0 || Sq == 0) return KB200_OK;
  if (!a->q || !a->o || !a->lengths || (max_pages > 0 && !a->page_table))
    return set_error(KB200_ERR_INVALID, "attn_cached: null pointer");
  if (!aligned16(a->q) || !aligned16(a->o) || ((a->q_batch_stride | a->q_token_stride | a->q_head_stride) & 7))
    return set_error(KB200_ERR_ALIGN, "attn_cached: q and o rows must be 16-byte aligned");
  const size_t need = kb200_attn_cached_workspace_size(B, Sq, Hq, c->H, c->D, c->page, max_pages);
  if (!a->workspace || a->workspace_bytes < need || !aligned16(a->workspace))
    return set_error(KB200_ERR_WORKSPACE, "attn_cached: workspace of %zu bytes needed, got %zu", need, a->workspace_bytes);
  const int64_t G = Hq / c->H, R = Sq * G;
  const int nt = cached::row_tiles(R), rows = nt * 8;
  const int64_t rblocks = (R + rows - 1) / rows;
  if (B * c->H * rblocks > 0x7fffffffLL) return set_error(KB200_ERR_INVALID, "attn_cached: too many rows");
  cached::Params p{};
  p.q = a->q; p.o = a->o; p.lse = a->lse; p.table = a->page_table; p.lengths = a->lengths;
  p.k_pages = (const uint8_t*)c->k_pages; p.v_pages = (const uint8_t*)c->v_pages;
  p.k_scale = c->k_scale; p.v_scale = c->v_scale; p.part = (float*)a->workspace;
  p.q_bs = a->q_batch_stride; p.q_ts = a->q_token_stride; p.q_hs = a->q_head_stride;
  p.B = (int)B; p.Sq = (int)Sq; p.Hq = (int)Hq; p.H = (int)c->H; p.G = (int)G; p.R = (int)R;
  p.rblocks = (int)rblocks;
  p.num_pages = (int)c->num_pages; p.max_pages = (int)max_pages; p.page = (int)c->page;
  p.page_log2 = c->page == 16 ? 4 : c->page == 32 ? 5 : c->page == 64 ? 6 : 7;
  p.scale_log2 = fabsf((float)a->softmax_scale) * 1.4426950408889634f;
  p.flip = a->softmax_scale < 0.0 ? 0x80008000u : 0u;
  const int grid = cached::grid_of(c->D, B, c->H, R, max_pages * c->page);
  cudaStream_t st = (cudaStream_t)stream;
  if (c->D == 64) {
    if (nt == 1) return dtype ? cached::launch<64, true, 1>(p, grid, st) : cached::launch<64, false, 1>(p, grid, st);
    return dtype ? cached::launch<64, true, 2>(p, grid, st) : cached::launch<64, false, 2>(p, grid, st);
  }
  if (nt == 1) return dtype ? cached::launch<128, true, 1>(p, grid, st) : cached::launch<128, false, 1>(p, grid, st);
  return dtype ? cached::launch<128, true, 2>(p, grid, st) : cached::launch<128, false, 2>(p, grid, st);
}
