// The 4-bit KV cache: the format of a row and the arithmetic that writes and reads it (sm_100a).
//
// A key or value row of D numbers (D = 32 / 64 / 128 / 256) is held in groups of 32.  A group has a step s and a middle m,
// both bf16, and 32 codes c of four bits; a number reads back as  m + s * (c - 8).  With lo / hi the group's least and
// greatest number:
//   s = bf16((hi - lo) / 15)      m = bf16(lo + 8 s)      c = clamp(round_half_even((x - m) / s), -8, 7) + 8
// The error of a number is at most s / 2 + 2^-8 |m| (the second part is the rounding of m, not more than the bf16 input's
// own).  A group whose step is 0 or below 2^-120 holds its least number 32 times; a group with an infinity or a NaN, or
// one that spreads over 2^120 or more, reads back as NaN (m = NaN, s = 0).
//
// Memory: codes [slots, heads, D / 2] bytes, lower half of a byte first; (m, s) [slots, heads, D / 32] words, m in the
// lower half.  The codes of a row are in the order in which the lanes of the attention kernel take them, so that each of
// them loads its share of a row at once (D = 128: 16 bytes of a key, 8 bytes of a value):
//   keys    [quarter of a group: 4][group][8 codes], four groups at a time:  a lane's word is 8 numbers of one group
//   values  [eighth of a group: 8][group][4 codes]:                          a lane's half word is 4 numbers of one group
#pragma once
#include "common.cuh"

namespace ab {

// Where word (group w, quarter t) of a key row is held; where half word (group g, eighth i) of a value row is held.
template <int D> __host__ __device__ constexpr int kv4_key_word(int w, int t) {
  constexpr int NG = D / 32;
  return NG <= 4 ? t * NG + w : (w >> 2) * 16 + t * 4 + (w & 3);
}
template <int D> __host__ __device__ constexpr int kv4_value_half(int g, int i) { return i * (D / 32) + g; }

// IEEE single arithmetic that keeps subnormal numbers, whatever the flags of the file: the codes are then the ones of the
// formulas above, the same on every machine.
__device__ __forceinline__ float sub_ieee(float a, float b) {
  float r;
  asm("sub.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float add_ieee(float a, float b) {
  float r;
  asm("add.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float fma_ieee(float a, float b, float c) {
  float r;
  asm("fma.rn.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t min_bf162(uint32_t a, uint32_t b) {  // of both halves; a NaN wins
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// The two numbers, cut to 0 .. 15, before the codes that are there already.
__device__ __forceinline__ uint32_t pack_codes(int high, int low, uint32_t behind) {
  uint32_t r;
  asm("cvt.pack.sat.u4.s32.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(high), "r"(low), "r"(behind));
  return r;
}

// Eight numbers of a lane -> their eight codes (lowest number in the lowest half byte) and the (m, s) word of the group,
// which four neighbouring lanes share.  Every lane of the warp takes part.
__device__ __forceinline__ uint32_t kv4_quantise(const Vec8<__nv_bfloat16>& v, uint32_t& meta) {
  // lower half: the least number, upper half: the greatest with its sign turned
  const uint32_t a = min_bf162(min_bf162(v.raw.x, v.raw.y), min_bf162(v.raw.z, v.raw.w)), turn = 0x80008000u;
  const uint32_t b = min_bf162(min_bf162(v.raw.x ^ turn, v.raw.y ^ turn), min_bf162(v.raw.z ^ turn, v.raw.w ^ turn));
  uint32_t ends = min_bf162(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
  ends = min_bf162(ends, __shfl_xor_sync(0xffffffffu, ends, 1));
  ends = min_bf162(ends, __shfl_xor_sync(0xffffffffu, ends, 2));
  const float lo = __uint_as_float(ends << 16), hi = __uint_as_float((ends ^ 0x80000000u) & 0xffff0000u);
  const float spread = sub_ieee(hi, lo);
  if (!(spread < 0x1p120f)) {  // an infinity, a NaN, or too wide
    meta = 0x00007fffu;        // m = NaN, s = 0
    return 0x88888888u;
  }
  // spread / 15, rounded once: a product with 1 / 15 and one correction by its remainder (Markstein)
  const float q = spread * (1.f / 15.f), quotient = fma_ieee(fma_ieee(-q, 15.f, spread), 1.f / 15.f, q);
  uint32_t s_bits = __bfloat16_as_ushort(__float2bfloat16_rn(quotient));
  if (s_bits < 0x0380u) s_bits = 0;  // below 2^-120
  const float s = __uint_as_float(s_bits << 16);
  const float mid = s_bits ? add_ieee(lo, 8.f * s) : lo;
  const uint32_t m_bits = __bfloat16_as_ushort(__float2bfloat16_rn(mid));
  const float m = __uint_as_float(m_bits << 16);
  meta = m_bits | (s_bits << 16);
  if (!s_bits) return 0x88888888u;
  // c' = the nearest whole number to y / s, y = x - m, ties to the even one.  A product with 1 / s is right up to the
  // neighbour; what it leaves of y is exact (|c' s| has 14 bits at most: |y / s| < 40, as two bf16 numbers of size |m|
  // that differ do so by 2^-8 |m|) and says which of the two it is.
  const float inv = 1.f / s, half = 0.5f * s;  // 2^-120 <= s < 2^117: neither is subnormal
  float x[8];
  v.unpack(x);
  uint32_t word = 0;
#pragma unroll
  for (int j = 7; j >= 0; j -= 2) {
    int code[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float y = sub_ieee(x[j - i], m);
      float big = fmaf(y, inv, 12582912.f);  // 1.5 2^23 + c': the whole number in the low bits
      const float rest = fma_ieee(12582912.f - big, s, y);
      const float most = __uint_as_float(__float_as_uint(half) - (__float_as_uint(big) & 1u));  // an odd c' may not have s / 2 left
      if (fabsf(rest) > most) big += __uint_as_float((__float_as_uint(rest) & 0x80000000u) | 0x3f800000u);
      code[i] = (int)__float_as_uint(big) - (0x4b400000 - 8);
    }
    word = pack_codes(code[0], code[1], word);
  }
  return word;
}

// One row per D / 8 lanes: lane `l` of the row brings its numbers 8 l .. 8 l + 7, and the row goes to `codes` / `meta`.
// Every lane of the warp takes part; a lane with `live` false stores nothing.
template <int D>
__device__ __forceinline__ void kv4_store_numbers(bool live, bool key, int l, const Vec8<__nv_bfloat16>& v, uint8_t* codes, uint32_t* meta) {
  constexpr int NG = D / 32;
  uint32_t ms;
  const uint32_t word = kv4_quantise(v, ms);
  // a value row's words are made of two half words that two lanes may hold
  const int base = (threadIdx.x & 31) - l;
  uint32_t out = 0;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int half = 2 * l + e, i = half / NG, g = half % NG;
    const uint32_t w = __shfl_sync(0xffffffffu, word, base + g * 4 + (i >> 1));
    out |= ((i & 1) ? (w >> 16) : (w & 0xffffu)) << (16 * e);
  }
  if (!live) return;
  if (key) reinterpret_cast<uint32_t*>(codes)[kv4_key_word<D>(l >> 2, l & 3)] = word;
  else reinterpret_cast<uint32_t*>(codes)[l] = out;
  if ((l & 3) == 0) meta[l >> 2] = ms;
}

// The same from memory: `src` is the row, not read where `live` is false.
__device__ __forceinline__ Vec8<__nv_bfloat16> kv4_load_numbers(bool live, int l, const __nv_bfloat16* src) {
  Vec8<__nv_bfloat16> v;
  v.raw = make_uint4(0, 0, 0, 0);
  if (live) v.load(src + 8 * l);
  return v;
}
template <int D>
__device__ __forceinline__ void kv4_store_row(bool live, bool key, int l, const __nv_bfloat16* src, uint8_t* codes, uint32_t* meta) {
  kv4_store_numbers<D>(live, key, l, kv4_load_numbers(live, l, src), codes, meta);
}

}  // namespace ab
