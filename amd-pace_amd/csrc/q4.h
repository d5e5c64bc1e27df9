// The 4-bit form of a cache row and its place in a pool (pools with elem_bytes == PACE_KV_ELEM_Q4).
//
// A row of head_dim values is cut into groups of 32 dims.  A group holds a step s and a middle m (halves) and a
// code -8 .. 7 per value (kept as code + 8 in four bits), and stands for s * code + m.  A row is quantised on its
// own, when it is written: nothing is ever requantised, so appends, rollbacks, evictions and forks move or forget
// stored bits like any other pool's.
//   s    = the least half with 15 s >= max - min: the codes' span covers the group, so no value is cut off
//   m    = half(min + 8 s)
//   code = round-half-even((x - m) / s), 0 where s = 0
// 20 bytes per 32 values: 0.3125 of the 16-bit row.
//
// Slab of one (block, KV head), K or V: 8 D bytes of codes, then 2 D bytes of steps and middles.  The codes are ordered
// as the operands of the 16x16x32 matrix-core instruction (see attn_core.h for the lane (n, g) convention): the
// eight codes of a dword are the eight contraction values one lane holds, and a wavefront-wide load is contiguous.
//   K codes   [dim half of 128+][tile 2][g 4][slot 8][step kk] dwords: eight dims 32 kk + 8 g .. of one token
//   K scales  [tile 2][slot 8][kk] dwords: s in the low half, m in the high one
//   V codes   [token half 2][dim tile quad][dim 16][dim tile] dwords: eight tokens of one dim
//   V scales  [kk][token 16] halves: s, then the same of m
// Value e of a dword sits at bit 4 (e / 2) + 16 (e & 1): a shift by 4 i brings values 2 i and 2 i + 1 to the low bits of the
// two 16-bit halves (see q4_codes).
#pragma once
#include "common.h"

namespace pace_kv {

constexpr int kQ4Group = 32;
constexpr float kQ4Clamp = 32768.f;  // values are held at +-2^15, so that s * code + m stays far from a half's overflow

typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

template <int D>
struct Q4 {
  static constexpr int G = D / 32;                       // groups of a row
  static constexpr int KC = G == 8 ? 4 : G;              // K code dwords of one lane-wide load
  static constexpr int KN = G / KC;                      // ... and how many such loads a tile takes
  static constexpr int VC = (2 * G) % 4 == 0 ? 4 : 3;    // V code dwords of one lane-wide load
  static constexpr int VN = 2 * G / VC;
  static constexpr int kCodeBytes = 8 * D;
  static constexpr int kSlabBytes = 10 * D;              // of K, and of V

  // dword index of the codes of dims 32 kk + 8 g .. + 7 of block token (tile, slot)
  __host__ __device__ static constexpr int k_code(int tile, int g, int slot, int kk) {
    return ((((kk / KC) * 2 + tile) * 4 + g) * 8 + slot) * KC + kk % KC;
  }
  __host__ __device__ static constexpr int k_scale(int tile, int slot, int kk) { return 2 * D + (tile * 8 + slot) * G + kk; }
  // dword index of the codes of block tokens 8 half .. + 7 of dim 16 j + dn
  __host__ __device__ static constexpr int v_code(int half, int j, int dn) { return ((half * VN + j / VC) * 16 + dn) * VC + j % VC; }
  // half index of the step of group kk of block token tok; its middle lies 16 G further
  __host__ __device__ static constexpr int v_scale(int kk, int tok) { return 4 * D + kk * 16 + tok; }
};

__host__ __device__ __forceinline__ constexpr int q4_bit(int e) { return 4 * (e >> 1) + 16 * (e & 1); }

// (tile, slot) of block token tok (the same interleave as the 16-bit K slab's)
__host__ __device__ __forceinline__ constexpr int q4_tile(int tok) { return (tok >> 2) & 1; }
__host__ __device__ __forceinline__ constexpr int q4_slot(int tok) { return ((tok >> 3) << 2) | (tok & 3); }

__device__ __forceinline__ uint32_t half_bits(_Float16 h) { return __builtin_bit_cast(uint16_t, h); }
__device__ __forceinline__ _Float16 half_from(uint32_t b) { return __builtin_bit_cast(_Float16, (uint16_t)b); }

// Value e of a code dword as the number it is, -8 .. 7.
__device__ __forceinline__ float q4_code(uint32_t w, int e) { return (float)((int)((w >> q4_bit(e)) & 15u) - 8); }

// The eight codes of a dword as halves -8 .. 7, in element order, by the published way of or-ing small integers into the mantissa
// of a half of 1024 (Kim, Henry, Fahim, Awadalla, "Who Says Elephants Can't Run", 2022).  `and-or` with the bits of 1024 makes
// a pair of halves 1024 + (code + 8) of the low nibbles and 1024 + 16 (code + 8) of the next ones; one packed add or
// multiply-add takes the offset out again, exactly.  One shift per dword and 2 instructions per pair; `or_bits` comes from q4_or_bits().
__device__ __forceinline__ void q4_codes(uint32_t w, uint32_t or_bits, f16x2 (&c)[4]) {
  const f16x2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = w >> (8 * i);
    c[2 * i] = __builtin_bit_cast(f16x2, (x & 0x000f000fu) | or_bits) + f16x2{(_Float16)-1032.f, (_Float16)-1032.f};
    c[2 * i + 1] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (x & 0x00f000f0u) | or_bits), sixteenth, f16x2{(_Float16)-72.f, (_Float16)-72.f});
  }
}
// 0x64006400 in a vector register: an instruction takes one constant from outside them, so that with both the mask and this one
// outside, `and-or` would be two.
__device__ __forceinline__ uint32_t q4_or_bits() {
  uint32_t b = 0x64006400u;
  asm volatile("" : "+v"(b));
  return b;
}

// Quantises a group of 32 bf16 values held by four neighbouring lanes (eight each, lanes 4 k .. 4 k + 3, all active): the group's
// step and middle, and this lane's codes (+ 8) as byte 2 of eight words.
//
// Codes are decided as by arithmetic in double precision, in which the format is defined.  y = x / s + (136 - m / s), one
// multiply-add with the reciprocal, lies in [128, 144): its last place is 2^-16, and as |m / s| <= 64 (else the group takes the
// other way) it is off by less than one: 2^-17 each for the added constant and for the sum, 9 * 2^-23 for the reciprocal.  Adding
// one half to the bits rounds it, the code is then byte 2, and a fraction within two places of a border (6 values in 100 000)
// is decided again.
// a - b == d + q4_rest(a, b, d) exactly, d the rounded difference (the error-free sum of two numbers: Knuth, Moller).
__device__ __forceinline__ float q4_rest(float a, float b, float d) {
  const float back = d - a;
  return (a - (d - back)) - (b + back);
}
template <int PERM>  // the value of another of the four lanes
__device__ __forceinline__ float q4_quad(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), PERM, 0xf, 0xf, true));
}
__device__ __forceinline__ void bf16x8_to_f32(u32x4 raw, float (&x)[8]);
__device__ __forceinline__ void q4_quantise(u32x4 raw, uint32_t (&q)[8], _Float16& s_out, _Float16& m_out) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  float x[8];
  bf16x8_to_f32(raw, x);
  // magnitudes above 2^15 and NaN are rare: looked for on the bit patterns (0x4700 is 2^15), held only where there are any
  u16x2 top = {0, 0};
#pragma unroll
  for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, raw[e] & 0x7fff7fffu));
  if (top[0] > 0x4700 || top[1] > 0x4700) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] == x[e] ? fminf(fmaxf(x[e], -kQ4Clamp), kQ4Clamp) : 0.f;
  }
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) lo = __builtin_elementwise_minimum(lo, x[e]), hi = __builtin_elementwise_maximum(hi, x[e]);
  lo = __builtin_elementwise_minimum(lo, q4_quad<0xb1>(lo)), hi = __builtin_elementwise_maximum(hi, q4_quad<0xb1>(hi));
  lo = __builtin_elementwise_minimum(lo, q4_quad<0x4e>(lo)), hi = __builtin_elementwise_maximum(hi, q4_quad<0x4e>(hi));
  // The least half with 15 s >= hi - lo: the nearest half to the quotient, then one step up or down (halves >= 0 are in the order of
  // their bit patterns).  The width is kept as the sum of the rounded difference and its error, so the comparisons are exact:
  // 15 s - width is small only where it is a short number.
  const float width = hi - lo, rest = q4_rest(hi, lo, width);
  uint32_t sb = half_bits((_Float16)(width * (1.f / 15.f)));
  if (__builtin_fmaf(15.f, (float)half_from(sb), -width) < rest) ++sb;
  else if (sb > 0 && __builtin_fmaf(15.f, (float)half_from(sb - 1), -width) >= rest) --sb;
  const _Float16 s = half_from(sb);
  const float sf = (float)s;
  const _Float16 m = (_Float16)__builtin_fmaf(8.f, sf, lo);
  const float mf = (float)m;
  const float inv = sf > 0.f ? __builtin_amdgcn_rcpf(sf) : 0.f;
  const float add = __builtin_fmaf(-mf, inv, 136.f);
  u16x2 frac = {0xffff, 0xffff};  // how far above a border the values are
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = __float_as_uint(__builtin_amdgcn_fmed3f(__builtin_fmaf(x[e], inv, add), 128.f, 143.f)) + 0x8002u;
#pragma unroll
  for (int i = 0; i < 4; ++i) frac = __builtin_elementwise_min(frac, __builtin_bit_cast(u16x2, __builtin_amdgcn_perm(q[2 * i + 1], q[2 * i], 0x05040100u)));
  if ((frac[0] < 4 || frac[1] < 4 || fabsf(add - 136.f) > 64.f) && sf > 0.f) {
    // Exactly: x - m as a rounded difference and its error (q4_rest), against the border (f + 1/2) s, a number of 16 bits.  The
    // difference of the two is exact where it is small, so its sign is right everywhere.
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = x[e] - mf, f = floorf(fminf(fmaxf(d * inv, -16.f), 16.f));
      float rest = q4_rest(x[e], mf, d);
      if (fabsf(rest) <= 0x1p-54f * fabsf(d)) rest = 0.f;  // (not seen in double precision, in which the format is defined)
      const float over = __builtin_fmaf(-(f + 0.5f), sf, d) + rest;
      const int code = (int)f + (over > 0.f || (over == 0.f && ((int)f & 1)) ? 1 : 0);
      q[e] = (uint32_t)(8 + min(max(code, -8), 7)) << 16;
    }
  }
  s_out = s, m_out = m;
}

// The eight codes in a dword's bits (see above), and as eight bytes.
__device__ __forceinline__ uint32_t q4_pack(const uint32_t (&q)[8]) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= __builtin_amdgcn_perm(q[2 * i + 1], q[2 * i], 0x0c060c02u) << (4 * i);
  return w;
}
__device__ __forceinline__ u32x2 q4_bytes(const uint32_t (&q)[8]) {
  u32x2 r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __builtin_amdgcn_perm(q[4 * h + 1], q[4 * h], 0x0c0c0602u), hi = __builtin_amdgcn_perm(q[4 * h + 3], q[4 * h + 2], 0x06020c0cu);
    r[h] = lo | hi;
  }
  return r;
}

__device__ __forceinline__ void bf16x8_to_f32(u32x4 raw, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) x[2 * e] = bf16_bits_to_f32(raw[e] & 0xffffu), x[2 * e + 1] = __uint_as_float(raw[e] & 0xffff0000u);
}

}  // namespace pace_kv
