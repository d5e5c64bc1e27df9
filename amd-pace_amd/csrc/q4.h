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

// The eight codes of a dword as halves -8 .. 7, in element order.  `and-or` with the bits of 1024 makes a pair of halves 1024 +
// (code + 8) of the low nibbles and 1024 + 16 (code + 8) of the next ones; one packed add or multiply-add takes the
// offset out again, exactly.  One shift per dword and 2 instructions per pair; `or_bits` comes from q4_or_bits().
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

// Quantises a group of 32 values held by four neighbouring lanes (eight each, lanes 4 k .. 4 k + 3): this lane's codes as
// a dword, and the group's step and middle.  All four lanes have to be active together.
//
// Codes are decided as by exact arithmetic: in single precision (x - m) * (1 / s) is off by less than 2^-18 of a step
// for every quotient that is not cut to -8 or 7 anyway, so only a quotient within 2^-16 of a border (a few values in
// 100 000) is divided again in double precision.
__device__ __forceinline__ uint32_t q4_quantise(const float (&x_in)[8], _Float16& s_out, _Float16& m_out) {
  float x[8], lo = kQ4Clamp, hi = -kQ4Clamp;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = x_in[e] == x_in[e] ? fminf(fmaxf(x_in[e], -kQ4Clamp), kQ4Clamp) : 0.f;
    lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]);
  }
  lo = fminf(lo, __shfl_xor(lo, 1, 64)), hi = fmaxf(hi, __shfl_xor(hi, 1, 64));
  lo = fminf(lo, __shfl_xor(lo, 2, 64)), hi = fmaxf(hi, __shfl_xor(hi, 2, 64));
  // the least half with 15 s >= hi - lo: the nearest half to the quotient, then one step up or down (halves >= 0 are in
  // the order of their bit patterns; 15 s and the width are exact in double precision)
  const double width = (double)hi - (double)lo;
  uint32_t sb = half_bits((_Float16)((hi - lo) * (1.f / 15.f)));
  if (15.0 * (double)(float)half_from(sb) < width) ++sb;
  else if (sb > 0 && 15.0 * (double)(float)half_from(sb - 1) >= width) --sb;
  const _Float16 s = half_from(sb);
  const float sf = (float)s;
  const _Float16 m = (_Float16)__builtin_fmaf(8.f, sf, lo);
  const float mf = (float)m;
  const float inv = sf > 0.f ? 1.f / sf : 0.f;
  float q[8];
  bool border = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = (x[e] - mf) * inv;
    q[e] = __builtin_rintf(t);
    border = border || fabsf(t - q[e]) > 0.5f - 0x1p-16f;
  }
  if (border && sf > 0.f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = (float)__builtin_rint(((double)x[e] - (double)mf) / (double)sf);
  }
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) w |= (uint32_t)((int)fminf(fmaxf(q[e], -8.f), 7.f) + 8) << q4_bit(e);
  s_out = s, m_out = m;
  return w;
}

__device__ __forceinline__ void bf16x8_to_f32(u32x4 raw, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) x[2 * e] = bf16_bits_to_f32(raw[e] & 0xffffu), x[2 * e + 1] = __uint_as_float(raw[e] & 0xffff0000u);
}

}  // namespace pace_kv
