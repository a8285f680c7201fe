// kv_cache.cuh -- the 8-bit paged key/value cache: layout and conversions.
//
// A pool holds pages of `page` tokens for every kv head: codes [pages][Hkv][page][D]
// e4m3 and one fp32 scale per (page, head), always a power of two.  A power of two
// costs e4m3 nothing (a scale only places the range; the significand is unchanged),
// dequantised values are exact in bf16, and when a later token of a page needs a
// larger scale the codes already there move by exponent alone: exact, except where
// they reach e4m3's subnormals.
#pragma once
#include "common.cuh"
#include "kb200_internal.h"

namespace kb {
namespace kv {

constexpr int SCALE_EXP_MIN = -117;   // 2^-9 (smallest code) * 2^-117 is a normal bf16 number

// Smallest e with amax <= 448 * 2^e (448 = 1.75 * 2^8), at least SCALE_EXP_MIN; amax finite, >= 0.
KB_DEVI int scale_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, SCALE_EXP_MIN);
}
// 2^e for a normal exponent; 2^-126 below that range (only products that round to zero get there).
KB_DEVI float pow2(int e) { return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23); }
// Exponent of a stored scale (a power of two).
KB_DEVI int exponent_of(float scale) { return (int)((__float_as_uint(scale) >> 23) & 0xff) - 127; }

// Two floats to e4m3 codes (round to nearest even); an infinity becomes NaN, since e4m3 has none.
KB_DEVI uint32_t encode2(float a, float b) {
  if (fabsf(a) == INFINITY) a = __uint_as_float(0x7fffffffu);
  if (fabsf(b) == INFINITY) b = __uint_as_float(0x7fffffffu);
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
// The same for values known not to be infinite.
KB_DEVI uint32_t encode2_finite(float2 f) { return (uint32_t)__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3); }
// The two e4m3 codes in the low half of `c` as f16 pair (exact).
KB_DEVI uint32_t decode2(uint32_t c) {
  uint32_t r;
  asm("{.reg .b16 t;\n cvt.u16.u32 t, %1;\n cvt.rn.f16x2.e4m3x2 %0, t;}\n" : "=r"(r) : "r"(c));
  return r;
}
// The four codes of a word as two f16 pairs.  (Both halves in one statement: the conversion can
// take either half of its register, where extracting them first costs an instruction each.)
KB_DEVI void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{.reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;}\n"
      : "=r"(lo), "=r"(hi) : "r"(w));
}
KB_DEVI float2 half2_to_float2(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// 16-bit activations: F16 selects fp16, else bf16.
template <bool F16>
KB_DEVI float2 unpack16(uint32_t v) {
  if constexpr (F16) return half2_to_float2(v);
  else return unpack_bf16(v);
}
template <bool F16>
KB_DEVI uint32_t pack16(float lo, float hi) {
  if constexpr (F16) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    return pack_bf16(lo, hi);
  }
}

// The last b < B for which below(b) holds (it holds up to some b, at 0 in any case), by one warp: 32
// places are looked at together, so that 1024 sequences cost two loads' latencies and not ten.
template <class F>
KB_DEVI int warp_last(int B, int lane, F below) {
  int lo = 0, n = B;                       // the answer is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32, at = lo + lane * step;
    const uint32_t m = __ballot_sync(0xffffffffu, lane * step < n && (lane == 0 || below(at)));
    const int k = 31 - __clz(m);
    lo += k * step;
    n = min(step, n - k * step);
  }
  return lo;
}
// Index of the sequence whose packed range holds token t: the last b < B with cu[b] <= t.
KB_DEVI int find_sequence(const int32_t* cu, int B, int64_t t, int lane) {
  return warp_last(B, lane, [&](int b) { return cu[b] <= t; });
}

int check_cache(const KB200KvCache* c, const char* what);

}  // namespace kv
}  // namespace kb
