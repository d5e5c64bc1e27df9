// Attention over a pool of 4-bit rows, and attention through a window with sinks over a 4-bit or a bf16 pool.
//
// The query rows of one KV head are the q_len * n_rep (token, GQA replica) pairs, 16 to a tile, as in attn_core.h, whose
// operand layouts this file shares: scores of tokens 8 g .. 8 g + 7 of a 32-token unit for query row n sit in lane (n, g),
// which is where the second product wants the weights.
//
// Which tokens: a row at position pos reads t <= pos (or what the mask tensor allows) and, with a window w, only
// t > pos - w or t < kv_start + sinks.  The units some row of a group reads are two runs -- the sinks' and the window's -- and
// only they are walked: a step through a window costs the same at any length.
//
// 4-bit rows: a value is s * code + m with a step and a middle per token and 32 dims.  Codes become halves by one `and-or`
// per pair (1024 + code + 8), one packed add and one packed multiply-add, and both products run on halves, which hold
// the values to 2^-12 (bf16 would keep 2^-9).  Queries are brought into a half's range by a power of two per row, exactly
// except for components 2^-28 below the row's largest; weights lie in (0, 2^15].
// 16-bit rows are bf16 products, weights rounded to bf16, as in the kernels without a window.
#include <algorithm>

#include "attn_core.h"
#include "q4.h"

namespace pace_kv {

struct WalkParams : PagedAttnParams {
  int32_t window, sinks;  // 0: off
  int32_t group_rows;     // query rows of a group
  int32_t slot_rows;      // query rows of a partial result
  // How the groups (sequence, run of query rows) are dealt to workgroups.  shares == 0: one workgroup per group and KV head.  Else
  // the units of all groups of a KV head lie end to end and `shares` workgroups take equal runs of them (at least
  // min_share), so that a batch of any lengths keeps every workgroup busy for the same time; the units of a single group
  // are dealt out part_units at a time, which asks for no sum over lengths.  A group that one
  // workgroup covers alone is finished there; pieces of others become partial results, two per workgroup at most -- the
  // group it starts in the middle of or with, and the one it breaks off -- which walk_merge_kernel joins.
  int32_t shares, min_share, part_units;
};

// The units a group of rows walks: [su0, su0 + n_sink), then [wu0, wu0 + total - n_sink).
struct Walk {
  int su0, n_sink, wu0, total, sink_end;
  __device__ __forceinline__ int unit(int i) const { return i < n_sink ? su0 + i : wu0 + (i - n_sink); }
};

// One past the last token that a row of query token s reads: the causal limit, the sequence's end, the mask's last column.
template <bool HAS_MASK>
__device__ __forceinline__ int walk_end(const WalkParams& p, int len, int s) {
  const int end = HAS_MASK ? min(len, p.mask_len) : len;
  return p.causal ? min(end, len - p.q_len + s + 1) : end;
}

// s_first, s_last: query tokens of the group's first and last row.
template <bool HAS_MASK>
__device__ __forceinline__ Walk walk_of(const WalkParams& p, int len, int start, int s_first, int s_last) {
  Walk w;
  const int end = walk_end<HAS_MASK>(p, len, s_last);
  int low = start;
  w.sink_end = start;
  if (p.window > 0) {
    low = max(start, len - p.q_len + s_first - p.window + 1);
    w.sink_end = start + p.sinks;
  }
  w.wu0 = low / 32;
  const int wu1 = end > low ? (end + 31) / 32 : w.wu0;
  w.su0 = start / 32;
  // (the sinks' last unit may be the window's first, unless the window is empty: a mask may end below it)
  const int sinks = min(w.sink_end, end), su1 = end > low ? min((sinks + 31) / 32, w.wu0) : (sinks + 31) / 32;
  w.n_sink = sinks > start ? max(su1 - w.su0, 0) : 0;
  w.total = w.n_sink + wu1 - w.wu0;
  return w;
}

__device__ __forceinline__ int walk_len(const WalkParams& p, int b) {
  return max(p.seq_lens[b] + p.len_bias + (p.len_bias_dev ? *p.len_bias_dev : 0), 0);
}
__device__ __forceinline__ int walk_start(const WalkParams& p, int b, int len) { return p.kv_start ? min(max(p.kv_start[b], 0), len) : 0; }

// Group j: sequence j / n_qgroups, its row groups from the last to the first (under the causal limit later rows read more, and the
// longest workgroups should not be the last to start).
struct Group {
  int b, r_first, r_last, s_first, s_last, len, start;
  Walk walk;
};
template <bool HAS_MASK>
__device__ __forceinline__ Group walk_group(const WalkParams& p, int j) {
  Group x;
  x.b = j / p.n_qgroups;
  const int qg = p.n_qgroups - 1 - (j - x.b * p.n_qgroups);
  x.r_first = qg * p.group_rows, x.r_last = min(p.q_len * p.n_rep, x.r_first + p.group_rows) - 1;
  x.s_first = x.r_first / p.n_rep, x.s_last = x.r_last / p.n_rep;
  x.len = walk_len(p, x.b), x.start = walk_start(p, x.b, x.len);
  x.walk = walk_of<HAS_MASK>(p, x.len, x.start, x.s_first, x.s_last);
  return x;
}

// Where groups lie in the run of all units: a wave's prefix sums over the groups, 64 at a time.
struct Shares {
  int total, share;
};
__device__ __forceinline__ int walk_share(const WalkParams& p, int total) {
  return max((total + p.shares - 1) / p.shares, p.min_share);  // (unrounded: equal sequences stay whole)
}
__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) v += __shfl_xor(v, o, 64);
  return __builtin_amdgcn_readfirstlane(v);
}
template <bool HAS_MASK>
__device__ __forceinline__ int group_units(const WalkParams& p, int j) { return j < p.batch * p.n_qgroups ? walk_group<HAS_MASK>(p, j).walk.total : 0; }
template <bool HAS_MASK>
__device__ __forceinline__ Shares walk_shares(const WalkParams& p, int lane) {
  const int n = p.batch * p.n_qgroups;
  int mine = 0;
#pragma unroll 4
  for (int j = lane; j < n; j += 64) mine += group_units<HAS_MASK>(p, j);
  Shares s;
  s.total = wave_sum(mine);
  s.share = walk_share(p, s.total);
  return s;
}
// The group that unit `at` of the run (at < total) lies in, and its place there.
template <bool HAS_MASK>
__device__ __forceinline__ void walk_find(const WalkParams& p, int at, int lane, int& j, int& off) {
  int before = 0;
  for (int base = 0;; base += 64) {
    const int units = group_units<HAS_MASK>(p, base + lane);
    int upto = units;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int v = __shfl_up(upto, o, 64);
      if (lane >= o) upto += v;
    }
    const uint64_t hit = __ballot(before + upto > at);
    if (hit != 0 || base + 64 >= p.batch * p.n_qgroups) {
      const int l = hit != 0 ? __builtin_ctzll(hit) : 63;
      j = base + l;
      off = at - before - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(units, l));
      return;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
}

// ---- units of either pool ---------------------------------------------------------------------------------------
template <int N>
struct Dwords {
  typedef uint32_t type __attribute__((ext_vector_type(N), aligned(4)));
};
template <int N>
__device__ __forceinline__ void load_dwords(uint32_t* r, const uint32_t* at) {
  if constexpr (N == 1) {
    r[0] = *at;
  } else {
    const typename Dwords<N>::type v = *reinterpret_cast<const typename Dwords<N>::type*>(at);
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = v[i];
  }
}
template <int N>
__device__ __forceinline__ void load_dwords_once(uint32_t* r, const uint32_t* at) {  // nothing else will read them
  const typename Dwords<N>::type v = __builtin_nontemporal_load(reinterpret_cast<const typename Dwords<N>::type*>(at));
#pragma unroll
  for (int i = 0; i < N; ++i) r[i] = v[i];
}

// Eight K values of one token / eight V values of one dim from a code dword: one multiply-add per pair, rounded once, to half.
__device__ __forceinline__ u32x4 q4_k_operand(uint32_t codes, uint32_t scale, uint32_t or_bits) {
  const f16x2 sm = __builtin_bit_cast(f16x2, scale);
  f16x2 c[4];
  q4_codes(codes, or_bits, c);
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(c[i], f16x2{sm[0], sm[0]}, f16x2{sm[1], sm[1]}));
  return r;
}
__device__ __forceinline__ u32x4 q4_v_operand(uint32_t codes, const uint32_t (&s)[4], const uint32_t (&m)[4], uint32_t or_bits) {
  f16x2 c[4];
  q4_codes(codes, or_bits, c);
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(c[i], __builtin_bit_cast(f16x2, s[i]), __builtin_bit_cast(f16x2, m[i])));
  return r;
}

// Byte offsets of a unit's two blocks in K and in V.  They are products of wave-uniform numbers; left to itself the compiler
// multiplies after the lanes have picked their block, in vector registers at a quarter of the rate.
struct UnitOffsets {
  int64_t ka, kb, va, vb;
};
template <int BITS>
__device__ __forceinline__ UnitOffsets unit_offsets(const WalkParams& p, int idA, int idB) {
  constexpr int64_t SIZE = BITS == 4 ? 1 : 2;
  UnitOffsets u = {idA * p.k_bs * SIZE, idB * p.k_bs * SIZE, idA * p.v_bs * SIZE, idB * p.v_bs * SIZE};
  asm volatile("" : "+s"(u.ka), "+s"(u.kb), "+s"(u.va), "+s"(u.vb));
  return u;
}
// Lane addresses that do not depend on the unit.
struct LaneBase {
  const char *kc, *ks, *vc, *vs;  // 4-bit pools: codes and scales of K and of V; 16-bit pools: kc and vc
};
template <class T>
__device__ __forceinline__ const T* unit_at(const char* base, int64_t off) {
  return reinterpret_cast<const T*>(base + off);
}

// A unit as one wave fetches it for itself.
template <int BITS, int D>
struct WalkUnit;

template <int D>
struct WalkUnit<16, D> {
  UnitRegs<D> r;
  // (the operand layout of load_unit; nothing else reads these bytes in this launch)
  __device__ static __forceinline__ LaneBase base(const WalkParams& p, int kvh, int n, int g) {
    return {reinterpret_cast<const char*>(p.kpool + (int64_t)kvh * p.k_hs + g * 64 + (n & 7) * 8), nullptr,
            reinterpret_cast<const char*>(p.vpool + (int64_t)kvh * p.v_hs + ((g & 1) * 16 + n) * 8), nullptr};
  }
  __device__ __forceinline__ void load(const LaneBase& lb, const UnitOffsets& o, int n, int g) {
    const uint16_t* kp = unit_at<uint16_t>(lb.kc, n >= 8 ? o.kb : o.ka);
    const uint16_t* vp = unit_at<uint16_t>(lb.vc, g >= 2 ? o.vb : o.va);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk) r.k[t][kk] = load16_stream(kp + t * (D * 8) + kk * 256);
#pragma unroll
    for (int j = 0; j < D / 16; ++j) r.v[j] = load16_stream(vp + j * 256);
  }
  __device__ __forceinline__ u32x4 k(int t, int kk) const { return r.k[t][kk]; }
  __device__ __forceinline__ u32x4 v(int j) const { return r.v[j]; }
  __device__ __forceinline__ void drop(const u32x4& keep) {
#pragma unroll
    for (int j = 0; j < D / 16; ++j) r.v[j] &= keep;
  }
};

template <int D>
struct WalkUnit<4, D> {
  using L = Q4<D>;
  uint32_t kc[2][L::G], ks[2][L::G];  // codes and (step, middle) of this lane's token of either tile
  uint32_t vc[2 * L::G];              // codes of this lane's dim of every dim tile
  uint32_t vs[L::G][4], vm[L::G][4];  // steps and middles of this lane's eight tokens, per group of dims
  uint32_t or_bits;
  __device__ static __forceinline__ LaneBase base(const WalkParams& p, int kvh, int n, int g) {
    const char* k = reinterpret_cast<const char*>(p.kpool) + (int64_t)kvh * p.k_hs;
    const char* v = reinterpret_cast<const char*>(p.vpool) + (int64_t)kvh * p.v_hs;
    return {k + 4 * L::k_code(0, g, n & 7, 0), k + 4 * L::k_scale(0, n & 7, 0), v + 4 * L::v_code(g & 1, 0, n), v + 2 * L::v_scale(0, 8 * (g & 1))};
  }
  __device__ __forceinline__ void load(const LaneBase& lb, const UnitOffsets& o, int n, int g) {
    const int64_t ko = n >= 8 ? o.kb : o.ka, vo = g >= 2 ? o.vb : o.va;
    const uint32_t *kc_at = unit_at<uint32_t>(lb.kc, ko), *ks_at = unit_at<uint32_t>(lb.ks, ko);
    const uint32_t *vc_at = unit_at<uint32_t>(lb.vc, vo), *vs_at = unit_at<uint32_t>(lb.vs, vo);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < L::G; i += L::KC) {
        load_dwords_once<L::KC>(kc[t] + i, kc_at + (L::k_code(t, 0, 0, i) - L::k_code(0, 0, 0, 0)));
        load_dwords<L::KC>(ks[t] + i, ks_at + (L::k_scale(t, 0, i) - L::k_scale(0, 0, 0)));
      }
#pragma unroll
    for (int j = 0; j < 2 * L::G; j += L::VC) load_dwords_once<L::VC>(vc + j, vc_at + (L::v_code(0, j, 0) - L::v_code(0, 0, 0)));
#pragma unroll
    for (int kk = 0; kk < L::G; ++kk) {
      load_dwords<4>(vs[kk], vs_at + 8 * kk);
      load_dwords<4>(vm[kk], vs_at + 8 * (kk + L::G));
    }
  }
  __device__ __forceinline__ u32x4 k(int t, int kk) const { return q4_k_operand(kc[t][kk], ks[t][kk], or_bits); }
  __device__ __forceinline__ u32x4 v(int j) const { return q4_v_operand(vc[j], vs[j / 2], vm[j / 2], or_bits); }
  __device__ __forceinline__ void drop(const u32x4&) {}  // (a 4-bit pool holds finite values only)
};

// A wave's quarter of a unit on its way into LDS: KPW of the K operands (tile wave & 1, steps kk0 ..) and VPW of the V operands
// (dim tiles j0 ..).  Where the operands do not divide by four (head size 96) two waves make the same one.
template <int BITS, int D>
struct UnitShare {
  using L = Q4<D>;
  static constexpr int G = D / 32, PW = (G + 1) / 2, VG = (PW + 1) / 2;
  uint32_t kc[BITS == 4 ? PW : 1], ks[BITS == 4 ? PW : 1], vc[BITS == 4 ? PW : 1], vs[BITS == 4 ? VG : 1][4], vm[BITS == 4 ? VG : 1][4];
  u32x4 kr[BITS == 16 ? PW : 1], vr[BITS == 16 ? PW : 1];
  __device__ static __forceinline__ int kk0(int wave) { return min((wave >> 1) * PW, G - PW); }
  __device__ static __forceinline__ int j0(int wave) { return min(wave * PW, 2 * G - PW); }
  __device__ static __forceinline__ LaneBase base(const WalkParams& p, int kvh, int wave, int n, int g) {
    const int t = wave & 1, kk = kk0(wave), j = j0(wave);
    if constexpr (BITS == 16) {
      return {reinterpret_cast<const char*>(p.kpool + (int64_t)kvh * p.k_hs + g * 64 + (n & 7) * 8 + t * (D * 8) + kk * 256), nullptr,
              reinterpret_cast<const char*>(p.vpool + (int64_t)kvh * p.v_hs + ((g & 1) * 16 + n) * 8 + j * 256), nullptr};
    } else {
      const char* k = reinterpret_cast<const char*>(p.kpool) + (int64_t)kvh * p.k_hs;
      const char* v = reinterpret_cast<const char*>(p.vpool) + (int64_t)kvh * p.v_hs;
      return {k + 4 * L::k_code(t, g, n & 7, kk), k + 4 * L::k_scale(t, n & 7, kk), v + 4 * L::v_code(g & 1, j, n), v + 2 * L::v_scale(j / 2, 8 * (g & 1))};
    }
  }
  __device__ __forceinline__ void load(const LaneBase& lb, const UnitOffsets& o, int wave, int n, int g) {
    const int64_t ko = n >= 8 ? o.kb : o.ka, vo = g >= 2 ? o.vb : o.va;
    if constexpr (BITS == 16) {
      const uint16_t *kp = unit_at<uint16_t>(lb.kc, ko), *vp = unit_at<uint16_t>(lb.vc, vo);
#pragma unroll
      for (int i = 0; i < PW; ++i) {
        kr[i] = *reinterpret_cast<const u32x4*>(kp + i * 256);
        vr[i] = *reinterpret_cast<const u32x4*>(vp + i * 256);
      }
    } else {
      load_dwords<PW>(kc, unit_at<uint32_t>(lb.kc, ko));
      load_dwords<PW>(ks, unit_at<uint32_t>(lb.ks, ko));
      const uint32_t* vc_at = unit_at<uint32_t>(lb.vc, vo);
      if constexpr (L::VC % PW == 0) {
        load_dwords<PW>(vc, vc_at);
      } else {
        const int j = j0(wave);
#pragma unroll
        for (int i = 0; i < PW; ++i) vc[i] = vc_at[L::v_code(0, j + i, 0) - L::v_code(0, j, 0)];
      }
      const uint32_t* vs_at = unit_at<uint32_t>(lb.vs, vo);
#pragma unroll
      for (int i = 0; i < VG; ++i) {
        load_dwords<4>(vs[i], vs_at + 8 * i);
        load_dwords<4>(vm[i], vs_at + 8 * (i + G));
      }
    }
  }
  // keep: see WalkUnit<16>::drop
  __device__ __forceinline__ void put(u32x4* stage, int wave, int lane, const u32x4& keep, uint32_t or_bits) const {
    const int t = wave & 1, kk = kk0(wave), j = j0(wave);
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      if constexpr (BITS == 16) {
        stage[(t * G + kk + i) * 64 + lane] = kr[i];
        stage[(2 * G + j + i) * 64 + lane] = vr[i] & keep;
      } else {
        stage[(t * G + kk + i) * 64 + lane] = q4_k_operand(kc[i], ks[i], or_bits);
        stage[(2 * G + j + i) * 64 + lane] = q4_v_operand(vc[i], vs[i / 2], vm[i / 2], or_bits);
      }
    }
  }
};

template <int BITS>
__device__ __forceinline__ f32x4 walk_mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BITS == 4)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// ---- rows -------------------------------------------------------------------------------------------------------
template <int D, int NQT>
struct WalkRows {
  u32x4 q[NQT][D / 32];
  f32x4 o[NQT][D / 16];
  f32x4 sum[NQT];                        // the weights' sum, four times over (a product with ones)
  float m[NQT], m_top[NQT], m_neg[NQT];  // see RowState
  float c[NQT];    // score product -> log2 units
  float cn[NQT];   // score product -> natural units (with a mask tensor)
  int limit[NQT];  // last readable token (-1: no such row, or none)
  int low[NQT];    // with a window: first token of it
  int s[NQT], hq[NQT];  // query token and head
};

// Weights of halves are kept a factor 2^7 up: with the lazy reference they then reach 2^15, and keep their eleven bits
// down to 2^-21 of the row's largest.
template <int BITS>
constexpr float kWeightShift = BITS == 4 ? 7.f : 0.f;

// Query row -> operand registers; 4-bit pools: as halves, times the power of two that brings the row's largest component to
// [2^14, 2^15) (returned as its exponent; the four lanes (n, 0..3) of a row agree).
template <int BITS, int D>
__device__ __forceinline__ int walk_query(u32x4 (&q)[D / 32]) {
  if constexpr (BITS == 16) {
    return 0;
  } else {
    float top = 0.f;
    float x[D / 32][8];
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) {
      bf16x8_to_f32(q[kk], x[kk]);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[kk][e]));
    }
    top = fmaxf(top, xor_lanes(top, 16));
    top = fmaxf(top, xor_lanes(top, 32));
    const int e = (int)((__float_as_uint(top) >> 23) & 255u);
    const int up = (e == 0 || e == 255) ? 0 : min(14 - (e - 127), 120);  // (0 and infinity stay what they are)
    const float f = __uint_as_float((uint32_t)(up + 127) << 23);
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        q[kk][i] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)(x[kk][2 * i] * f), (_Float16)(x[kk][2 * i + 1] * f)});
    return up;
  }
}

// Sets up tile qt's row: query operand, limits, empty softmax state.  Returns the row's last readable token (no row: none).
template <int BITS, int D, int NQT, bool HAS_MASK>
__device__ __forceinline__ int walk_row(const WalkParams& p, WalkRows<D, NQT>& st, int qt, int b, int kvh, int len, int r, int g) {
  const int S = p.q_len;
  const bool valid = r < S * p.n_rep;
  const int s = valid ? r / p.n_rep : 0, hq = kvh * p.n_rep + (valid ? r % p.n_rep : 0), pos = len - S + s;
  st.s[qt] = s, st.hq[qt] = hq;
  st.limit[qt] = valid ? walk_end<HAS_MASK>(p, len, s) - 1 : -1;
  st.low[qt] = p.window > 0 ? pos - p.window + 1 : 0;
  const uint16_t* qp = p.q + (int64_t)b * p.q_sb + (int64_t)hq * p.q_sh + (int64_t)s * p.q_ss + 8 * g;
#pragma unroll
  for (int kk = 0; kk < D / 32; ++kk) st.q[qt][kk] = *reinterpret_cast<const u32x4*>(qp + kk * 32);  // (no such row: the first one's, and zeros)
#pragma unroll
  for (int kk = 0; kk < D / 32; ++kk) st.q[qt][kk] = valid ? st.q[qt][kk] : u32x4{0u, 0u, 0u, 0u};
  const int up = walk_query<BITS, D>(st.q[qt]);
  const float down = __uint_as_float((uint32_t)(127 - up) << 23);
  st.cn[qt] = p.scale * down;
  st.c[qt] = fminf(fmaxf(p.scale_log2 * down, 0x1p-126f), 0x1p126f);  // (not 0 or infinite: it multiplies -inf and 0)
  st.m[qt] = kNegInf, st.m_top[qt] = kNegInf, st.m_neg[qt] = 0.f, st.sum[qt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < D / 16; ++j) st.o[qt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  return valid ? st.limit[qt] : 0x7fffffff;
}

// Element offset of the mask line of row r.
__device__ __forceinline__ int64_t walk_mask_line(const WalkParams& p, int b, int r) {
  return (int64_t)b * p.m_sb + (int64_t)(r < p.q_len * p.n_rep ? r / p.n_rep : 0) * p.m_ss;
}

// A unit that cannot change any row of the wave: every mask value in it is at the floor (weight exactly 0 next to a real score) and
// every row has met a real score.  (Rows that have met floor values only may end as an average and need every unit.)
template <int D, int NQT>
__device__ __forceinline__ bool walk_masked_out(const MaskRegs<NQT>& mr, const WalkRows<D, NQT>& st) {
  bool out = true;
#pragma unroll
  for (int qt = 0; qt < NQT; ++qt) {
    float top = mr.a[qt][0];
#pragma unroll
    for (int c = 1; c < 8; ++c) top = __builtin_elementwise_maximum(top, mr.a[qt][c]);
    out = out && (st.limit[qt] < 0 || (top <= kMaskFloor && st.m[qt] > 0.5f * kMaskFloor));
  }
  return __all(out);
}

// Tokens of the unit at t0 that no row of a group reads (past its end, between the sinks and the window) may hold anything in a
// 16-bit pool: their weight is 0, and 0 times infinity must not be added.  Mask of the lane's eight tokens' V values.
__device__ __forceinline__ u32x4 walk_keep(int t0, int g, int start, int sink_end, int low, int end) {
  u32x4 keep = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int t = t0 + 8 * g + e;
    if ((t < start) | (t >= end) | ((t < low) & (t >= sink_end))) keep[e >> 1] &= (e & 1) ? 0x0000ffffu : 0xffff0000u;
  }
  return keep;
}

// One unit against the rows of a wave, in three steps.  First the scores.  CHUNK operands are asked for together, ahead of the
// products they go into (operands that come from LDS; 1: they are made from registers, in the compiler's own order).
template <int BITS, int D, int NQT, int CHUNK, class K>
__device__ __forceinline__ void walk_scores(K&& k, const WalkRows<D, NQT>& st, f32x4 (&sc)[NQT][2]) {
  constexpr int KK = D / 32;
#pragma unroll
  for (int qt = 0; qt < NQT; ++qt) sc[qt][0] = sc[qt][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 2 * KK; c += CHUNK) {
    u32x4 a[CHUNK];
#pragma unroll
    for (int i = 0; i < CHUNK; ++i)
      if (c + i < 2 * KK) a[i] = k((c + i) / KK, (c + i) % KK);
    if (CHUNK > 1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < CHUNK; ++i)
      if (c + i < 2 * KK)
#pragma unroll
        for (int qt = 0; qt < NQT; ++qt) sc[qt][(c + i) / KK] = walk_mfma<BITS>(a[i], st.q[qt][(c + i) % KK], sc[qt][(c + i) / KK]);
  }
}

// Scores -> weights (operands of the second product).  full (wave-uniform): every row reads all of the unit's 32 tokens.
template <int BITS, int D, int NQT, bool HAS_MASK>
__device__ __forceinline__ void walk_weights(f32x4 (&sc)[NQT][2], WalkRows<D, NQT>& st, u32x4 (&pb)[NQT], bool full, int t0, int start, int sink_end,
                                             int g, const MaskRegs<NQT>& mregs) {
#pragma clang fp contract(off)
  if (HAS_MASK) {
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt)
#pragma unroll
      for (int e = 0; e < 8; ++e) sc[qt][e >> 2][e & 3] = __builtin_fmaf(sc[qt][e >> 2][e & 3], st.cn[qt], mregs.a[qt][e]);
  }
  if (!full) {
    const int base = t0 + 8 * g;  // this lane's first token
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt) {
      const int hi = st.limit[qt] - base, lo = start - base, wl = st.low[qt] - base, se = sink_end - base;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        sc[qt][e >> 2][e & 3] = (e > hi) | (e < lo) | ((e < wl) & (e >= se)) ? kNegInf : sc[qt][e >> 2][e & 3];  // whatever the token holds
    }
  }
#pragma unroll
  for (int qt = 0; qt < NQT; ++qt) {
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = sc[qt][e >> 2][e & 3];
    const float c = HAS_MASK ? kLog2e : st.c[qt];
    // (this maximum hands NaN on, which needs no instruction to quiet its operands; a row with a NaN weight is NaN throughout)
    float mine = s[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mine = __builtin_elementwise_maximum(mine, s[e]);
    if (__any(mine > st.m_top[qt])) {  // the reference follows the maximum lazily, as in softmax_and_output
      const float mx = row_max4(mine);
      const float m_old = st.m[qt], m_new = fmaxf(m_old, mx);
      const float m_use = m_new == kNegInf ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f((m_old - m_use) * c);
      st.m[qt] = m_new;
      const float neg = kWeightShift<BITS> - m_use * c;
      const bool far = fabsf(neg) > kFarLog2 && m_use != kMaskFloor;  // (a weight of a near row stays below 2^15.02)
      st.m_top[qt] = far ? kNegInf : m_new + kLazyLog2 / c;
      st.m_neg[qt] = far ? kWeightShift<BITS> : neg;
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] -= far ? m_use : 0.f;
      st.sum[qt][0] *= alpha;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) st.o[qt][j] *= alpha;
    }
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, st.m_neg[qt]));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (BITS == 4) pb[qt][i] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)w[2 * i], (_Float16)w[2 * i + 1]});
      else pb[qt][i] = pack_bf16x2(w[2 * i], w[2 * i + 1]);
    }
  }
}

// The second product.  The weights are summed by the matrix cores too, as rounded: the same weights then stand above and below the
// fraction, and eight additions per tile are saved where the vector unit is the bound.
template <int BITS, int D, int NQT, int CHUNK, class V>
__device__ __forceinline__ void walk_output(V&& v, WalkRows<D, NQT>& st, const u32x4 (&pb)[NQT]) {
  const uint32_t one2 = BITS == 4 ? 0x3c003c00u : 0x3f803f80u;
#pragma unroll
  for (int qt = 0; qt < NQT; ++qt) st.sum[qt] = walk_mfma<BITS>(u32x4{one2, one2, one2, one2}, pb[qt], st.sum[qt]);
#pragma unroll
  for (int c = 0; c < D / 16; c += CHUNK) {
    u32x4 a[CHUNK];
#pragma unroll
    for (int i = 0; i < CHUNK; ++i)
      if (c + i < D / 16) a[i] = v(c + i);
    if (CHUNK > 1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < CHUNK; ++i)
      if (c + i < D / 16)
#pragma unroll
        for (int qt = 0; qt < NQT; ++qt) st.o[qt][c + i] = walk_mfma<BITS>(a[i], pb[qt], st.o[qt][c + i]);
  }
}

// Running maximum in log2 units (-inf stays -inf).
template <int D, int NQT, bool HAS_MASK>
__device__ __forceinline__ void walk_finish(WalkRows<D, NQT>& st) {
#pragma unroll
  for (int qt = 0; qt < NQT; ++qt) st.m[qt] *= HAS_MASK ? kLog2e : st.c[qt];
}

// A finished row: the output (slot < 0), or a partial result.
template <int D, int NQT>
__device__ __forceinline__ void walk_store(const WalkParams& p, const WalkRows<D, NQT>& st, int qt, int b, int kvh, int slot, int row, int g) {
  const float l = st.sum[qt][0];
  if (slot < 0) {
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);  // a row that read nothing is 0; NaN stays NaN
    uint16_t* op = p.out + (int64_t)b * p.o_sb + (int64_t)st.hq[qt] * p.o_sh + (int64_t)st.s[qt] * p.o_ss + 4 * g;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      const f32x4 o = st.o[qt][j];
      *reinterpret_cast<u32x2*>(op + 16 * j) = u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
    }
  } else {
    const int64_t at = ((int64_t)slot * p.num_kv_heads + kvh) * p.slot_rows + row;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) *reinterpret_cast<f32x4*>(p.part_o + at * D + 16 * j + 4 * g) = st.o[qt][j];
    if (g == 0) *reinterpret_cast<u32x2*>(p.part_ml + 2 * at) = u32x2{__float_as_uint(st.m[qt]), __float_as_uint(l)};
  }
}

// The pieces of groups that a workgroup works on, one after the other (wave-uniform): for (WalkTurns t(...); t.more(); t.next()).
template <bool HAS_MASK>
struct WalkTurns {
  const WalkParams& p;
  int kvh, w, j, off, left;
  bool first;
  __device__ __forceinline__ WalkTurns(const WalkParams& p_, int lane) : p(p_), off(0), left(0), first(true) {
    const uint32_t item = blockIdx.x;
    kvh = (int)(item % (uint32_t)p.num_kv_heads);  // fastest: one head's K / V stay in one XCD's L2
    w = j = (int)(item / (uint32_t)p.num_kv_heads);
    if (p.shares == 0) return;
    j = 0;
    if (p.part_units > 0 && p.batch * p.n_qgroups == 1) {  // one group: nothing to look up
      off = w * p.part_units, left = w == p.shares - 1 ? 1 << 30 : p.part_units;  // (the last one: whatever there is)
      return;
    }
    const Shares s = walk_shares<HAS_MASK>(p, lane);
    const int64_t at = (int64_t)w * s.share;
    if (at >= s.total) return;
    left = min(s.share, s.total - (int)at);
    walk_find<HAS_MASK>(p, (int)at, lane, j, off);
  }
  // Units [begin, end) of group `x`; slot: where a partial result goes, -1: the group is covered in whole.
  __device__ __forceinline__ bool piece(const Group& x, int& begin, int& end, int& slot) {
    begin = off, end = p.shares == 0 ? x.walk.total : (int)min((int64_t)x.walk.total, (int64_t)off + left);
    slot = begin == 0 && end == x.walk.total ? -1 : (first ? 2 * w : 2 * w + 1);
    if (p.shares == 0) return true;
    const int n = max(end - begin, 0);
    left -= n, off = 0, first = first && n == 0;
    return n > 0;
  }
};

// ---------------------------------------------------------------------------------
// Groups of up to 16 query rows (decode; short appends, and prompts too short to fill the GPU otherwise): every wave walks units of
// its own.  NW waves split a workgroup's units (wave w: units w, w + NW, ...), fetch one ahead, and merge through LDS.
//
// Bound: the pool's bytes.  64 sequences x 4096 tokens, 8 KV heads of 128 dims, 4 query heads each: 57 to 59 us for 336 MB of 4-bit
// rows, over one pool or over four in turn, blocks in order or not (5.7 to 5.9 TB/s; a plain read of as much, four buffers in
// turn: 5.5).  Behind a launch that has written half a gigabyte, whose lines are still on their way out of the cache, it
// takes 79 us, and that plain read slows down from 65 to 109.  32 sequences through a window of 4096 tokens over a bf16 pool:
// 83 to 85 us, 6.4 TB/s.  One sequence of 4096 tokens: 10.6 us, the latency of two launches and of four units one after
// another.  Four waves and units in turn rather than one wave per run of units: a workgroup's reads stay close together.
// Two waves for 256 dims, whose state takes a wave's whole register file and its accumulation registers (4 registers spill over
// a 4-bit pool); 64 sequences x 2048, 16 heads of 256: 122 us, 5.5 TB/s.
// Two or three row tiles per wave instead of walk_rows_kernel (36 rows): 123 us against 65 -- one wave per SIMD, and spills.
// ---------------------------------------------------------------------------------
template <int BITS, int D, bool HAS_MASK, int NW, int OCC>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(OCC, 8))) void walk_attn_kernel(const WalkParams p) {
  constexpr int MT = D / 16, ROW_F = D + 2, SLOT_F = 16 * ROW_F;
  __shared__ float merge_buf[(NW / 2) * SLOT_F];
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  WalkTurns<HAS_MASK> turns(p, lane);
  const int kvh = turns.kvh, S = p.q_len, R = S * p.n_rep, n_groups = p.batch * p.n_qgroups;
  // One sequence without a window and padding: its units do not depend on its length, and the first block ids are asked for
  // along with that.
  const bool known = n_groups == 1 && p.window == 0 && p.kv_start == nullptr;
  int early = 0;
  if (known) {
    const int t = 2 * (turns.off + wave + NW * (lane >> 1)) + (lane & 1);
    early = t < p.table_stride ? p.table[t] : 0;
  }
  do {
    const Group x = walk_group<HAS_MASK>(p, turns.j);
    const int b = x.b, len = x.len, start = x.start;
    const Walk walk = x.walk;
    int i_begin, i_end, slot;
    const bool some = turns.piece(x, i_begin, i_end, slot);
    ++turns.j;
    if (!some) continue;  // uniform over the workgroup
    const int32_t* row = p.table + (int64_t)b * p.table_stride;
    const int n_mine = i_end - i_begin > wave ? (i_end - i_begin - wave + NW - 1) / NW : 0;

    // Pool block ids of 32 units of this wave, one per lane; never outside the pool, whatever the table holds.
    auto inside = [&](int id) { return id < 0 ? 0 : (id >= p.num_blocks ? p.num_blocks - 1 : id); };
    auto fetch_ids = [&](int first) {
      const int i = i_begin + wave + NW * (first + (lane >> 1));
      const int t = 2 * walk.unit(i) + (lane & 1);
      return inside(i < i_end && t < p.table_stride ? row[t] : 0);
    };
    int ids = known ? inside(early) : (n_mine > 0 ? fetch_ids(0) : 0);
    const LaneBase base = WalkUnit<BITS, D>::base(p, kvh, n, g);
    constexpr bool TWO = !(D == 256 && (BITS == 16 || HAS_MASK));  // registers for a second unit under way
    WalkUnit<BITS, D> even, odd;
    MaskRaw<1> even_mask, odd_mask;  // mask values travel with the unit, ahead of it
    const int64_t mask_line[1] = {HAS_MASK ? walk_mask_line(p, b, x.r_first + n) : 0};
    if constexpr (BITS == 4) even.or_bits = odd.or_bits = q4_or_bits();
    auto send = [&](WalkUnit<BITS, D>& u, MaskRaw<1>& m, int k) {
      if (HAS_MASK) load_mask_raw<1>(m, p, mask_line, 32 * walk.unit(i_begin + wave + NW * k), g);
      u.load(base, unit_offsets<BITS>(p, __builtin_amdgcn_readlane(ids, 2 * (k & 31)), __builtin_amdgcn_readlane(ids, 2 * (k & 31) + 1)), n, g);
    };
    if (n_mine > 0) send(even, even_mask, 0);

    WalkRows<D, 1> st;
    int min_limit = walk_row<BITS, D, 1, HAS_MASK>(p, st, 0, b, kvh, len, x.r_first + n, g);
#pragma unroll
    for (int o = 1; o < 16; o *= 2) min_limit = min(min_limit, __shfl_xor(min_limit, o, 64));
    min_limit = __builtin_amdgcn_readfirstlane(min_limit);
    const int row_low = p.window > 0 ? len - S + x.s_first - p.window + 1 : 0;  // the first row's window, and the last row's
    const int max_low = p.window > 0 ? len - S + x.s_last - p.window + 1 : 0;
    const int row_end = walk_end<HAS_MASK>(p, len, x.s_last);

    auto take = [&](WalkUnit<BITS, D>& u, const MaskRaw<1>& m, int k) {
      const int t0 = 32 * walk.unit(i_begin + wave + NW * k);
      MaskRegs<1> mregs;
      if (HAS_MASK) {
        mask_regs_from_raw<1>(mregs, m, p);
        if (walk_masked_out<D, 1>(mregs, st)) return;
      }
      const bool full = t0 >= start && t0 + 31 <= min_limit && (t0 >= max_low || t0 + 32 <= walk.sink_end);
      if (BITS == 16 && !full) u.drop(walk_keep(t0, g, start, walk.sink_end, row_low, row_end));
      f32x4 sc[1][2];
      u32x4 pb[1];
      walk_scores<BITS, D, 1, 1>([&](int t, int kk) { return u.k(t, kk); }, st, sc);
      walk_weights<BITS, D, 1, HAS_MASK>(sc, st, pb, full, t0, start, walk.sink_end, g, mregs);
      walk_output<BITS, D, 1, 1>([&](int j) { return u.v(j); }, st, pb);
    };
    // 32 units per set of block ids.  (Every turn of the inner loop fetches: behind a fetch that may or may not have been sent, the
    // compiler would have the wave wait for all that is under way before it uses the unit before it.)
    for (int k0 = 0; k0 < n_mine; k0 += 32) {
      const int k1 = min(k0 + 32, n_mine);
      if (k0 > 0) {
        ids = fetch_ids(k0);
        send(even, even_mask, k0);
      }
      int k = k0;
      if constexpr (TWO) {
        for (; k + 2 < k1; k += 2) {
          send(odd, odd_mask, k + 1);
          take(even, even_mask, k);
          send(even, even_mask, k + 2);
          take(odd, odd_mask, k + 1);
        }
        if (k + 1 < k1) {
          send(odd, odd_mask, k + 1);
          take(even, even_mask, k);
          take(odd, odd_mask, k + 1);
        } else {
          take(even, even_mask, k);
        }
      } else {
        for (; k + 1 < k1; ++k) {
          take(even, even_mask, k);
          send(even, even_mask, k + 1);
        }
        take(even, even_mask, k);
      }
    }
    walk_finish<D, 1, HAS_MASK>(st);
    // Pairwise merge of the waves' states (fixed order: the same bits from call to call).
#pragma unroll
    for (int stride = 1; stride < NW; stride *= 2) {
      float* slot = merge_buf + wave / (2 * stride) * SLOT_F + n * ROW_F;
      const bool sender = (wave & (2 * stride - 1)) == stride, receiver = (wave & (2 * stride - 1)) == 0;
      if (sender) {
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) slot[16 * j + 4 * g + i] = st.o[0][j][i];
        if (g == 0) slot[D] = st.m[0], slot[D + 1] = st.sum[0][0];
      }
      __syncthreads();
      if (receiver) {
        const float m_b = slot[D], l_b = slot[D + 1], m_new = fmaxf(st.m[0], m_b), m_use = m_new == kNegInf ? 0.f : m_new;
        const float wa = __builtin_amdgcn_exp2f(st.m[0] - m_use), wb = __builtin_amdgcn_exp2f(m_b - m_use);
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) st.o[0][j][i] = st.o[0][j][i] * wa + slot[16 * j + 4 * g + i] * wb;
        st.sum[0][0] = st.sum[0][0] * wa + l_b * wb;
        st.m[0] = m_new;
      }
      __syncthreads();
    }
    if (wave == 0 && x.r_first + n < R) walk_store(p, st, 0, b, kvh, slot, n, g);
  } while (p.shares > 0 && turns.left > 0 && turns.j < n_groups);
}

// ---------------------------------------------------------------------------------
// Groups of 64 or 128 query rows (drafted tokens, chunks of a prompt): the four waves of a workgroup own NQT tiles of 16 rows each and walk the
// units together.  Each wave fetches and unpacks a quarter of a unit and puts it into LDS in operand order, so that the
// unpacking is paid once per workgroup; fetches run three units ahead of their use (two in registers, one in LDS), with
// one barrier per unit.  A row's softmax state never leaves its wave.
//
// Bound: issue for the larger part, waiting for the rest.  Matrix and vector instructions of the waves of one SIMD do not overlap;
// by the counters they take, of a SIMD's cycles, 72 % (31 matrix, 42 vector) for 4 sequences x 512 new tokens over 4096 (8 KV
// heads of 128 dims, 4 query heads each: 171 us, 755 TFLOP/s, where a large fp16 matrix product reaches 1294; with every wave
// unpacking for itself 330 us), 51 % (13 and 38) for 32 sequences x 9 drafted tokens over 1000 .. 6000 (64 us, of which the
// merge takes 12, for 118 MB of rows; 36 of the 64 rows a workgroup computes are real), and 57 % (25 and 31) for 2 x 1024
// tokens through a window of 1024 over a bf16 pool (52 us).  The waves spend 20, 36 and 27 % of theirs at counter waits and
// the barrier, so these launches have room left.  Two tiles per wave above 64 rows halve the LDS reads and the unpacking per
// row.  Vector registers spilled with a mask tensor: 25 to 29 of two tiles and 15 to 17 of one at 128 dims, 7 or 8 at 256; every
// form spills 29 to 100 scalar registers.  Workgroups per compute unit under one tile, drafted tokens: 2 / 3 / 4 run
// 79 / 72 / 84 us.  With a mask tensor every unit up to the length is fetched and unpacked, also those that it leaves out for
// all rows: a prompt of 4 x 2048 tokens takes 517 us with the models' causal mask and 201 without it.
// ---------------------------------------------------------------------------------
template <int BITS, int D, int NQT, bool HAS_MASK, int OCC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(OCC, 8))) void walk_rows_kernel(const WalkParams p) {
  constexpr int KK = D / 32, MT = D / 16, OPERANDS = 2 * MT;  // operands of a unit: K's, then V's, 16 bytes per lane each
  __shared__ __attribute__((aligned(16))) u32x4 stage[2][OPERANDS * 64];
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  WalkTurns<HAS_MASK> turns(p, lane);
  const int kvh = turns.kvh, S = p.q_len, R = S * p.n_rep, n_groups = p.batch * p.n_qgroups;
  do {
    const Group x = walk_group<HAS_MASK>(p, turns.j);
    const int b = x.b, len = x.len, start = x.start, r_first = x.r_first;
    const Walk walk = x.walk;
    int i_begin, i_end, slot;
    const bool some = turns.piece(x, i_begin, i_end, slot);
    ++turns.j;
    if (!some) continue;  // uniform over the workgroup
    const int wg_low = p.window > 0 ? len - S + x.s_first - p.window + 1 : 0;  // what no row of the workgroup reads (see walk_keep)
    const int wg_end = walk_end<HAS_MASK>(p, len, x.s_last);

    const int32_t* row = p.table + (int64_t)b * p.table_stride;
    // Pool blocks of 64 units from c0 on, one per lane in each of two registers; never outside the pool.
    auto fetch_id = [&](int i) {
      const int t = 2 * walk.unit(i) + (lane & 1);
      const int id = i < i_end && t < p.table_stride ? row[t] : 0;
      return id < 0 ? 0 : (id >= p.num_blocks ? p.num_blocks - 1 : id);
    };
    int c0 = i_begin, ids_lo = fetch_id(c0 + (lane >> 1)), ids_hi = fetch_id(c0 + 32 + (lane >> 1));
    const LaneBase base = UnitShare<BITS, D>::base(p, kvh, wave, n, g);
    const uint32_t or_bits = q4_or_bits();
    UnitShare<BITS, D> even, odd;
    auto send = [&](UnitShare<BITS, D>& share, int i) {
      const int at = 2 * (i - c0);  // (past the 64 units: whatever block the lane holds; nobody reads that share)
      const int idA = at & 64 ? __builtin_amdgcn_readlane(ids_hi, at & 63) : __builtin_amdgcn_readlane(ids_lo, at & 63);
      const int idB = at & 64 ? __builtin_amdgcn_readlane(ids_hi, (at & 63) + 1) : __builtin_amdgcn_readlane(ids_lo, (at & 63) + 1);
      share.load(base, unit_offsets<BITS>(p, idA, idB), wave, n, g);
    };
    auto put = [&](UnitShare<BITS, D>& share, int i) {  // (past the last unit: whatever the share holds, into a stage nobody reads)
      u32x4 keep = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
      if (BITS == 16) {
        const int t0 = 32 * walk.unit(i);
        if (t0 < start || t0 + 32 > wg_end || t0 < wg_low) keep = walk_keep(t0, g, start, walk.sink_end, wg_low, wg_end);
      }
      share.put(stage[(i - c0) & 1], wave, lane, keep, or_bits);
    };
    send(even, c0);
    send(odd, c0 + 1);

    WalkRows<D, NQT> st;
    const int w_first = r_first + wave * NQT * 16, w_last = min(R, w_first + NQT * 16) - 1;  // this wave's rows
    const bool any_rows = w_first < R;
    int min_limit = 0x7fffffff;
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt) min_limit = min(min_limit, walk_row<BITS, D, NQT, HAS_MASK>(p, st, qt, b, kvh, len, w_first + qt * 16 + n, g));
#pragma unroll
    for (int o = 1; o < 16; o *= 2) min_limit = min(min_limit, __shfl_xor(min_limit, o, 64));
    min_limit = __builtin_amdgcn_readfirstlane(min_limit);
    const int row_low = p.window > 0 ? len - S + w_first / p.n_rep - p.window + 1 : 0;
    const int max_low = p.window > 0 ? len - S + w_last / p.n_rep - p.window + 1 : 0;
    const int row_end = any_rows ? walk_end<HAS_MASK>(p, len, w_last / p.n_rep) : 0;

    // One turn: unit i + 1 of the set goes from `next` into LDS, `next` fetches unit i + 3, unit i is used.  With two tiles per wave LDS
    // reads travel behind vector work: the K operands are asked for before the unpacking, the V operands before the softmax
    // that needs them after it.  (With one tile a third workgroup on the compute unit does that, and registers are kept for
    // it; head size 256 and a mask have none to spare.)  At the barrier every wave has taken what it needs of unit i, and every share of
    // unit i + 1 is in place.
    constexpr bool AHEAD = D <= 128 && NQT == 2 && !HAS_MASK;
    constexpr int CHUNK = AHEAD ? 1 : (NQT == 2 ? 4 : 8);
    MaskRaw<NQT> coming;  // mask values of the next unit: asked for a turn ahead, before that turn's share
    int64_t mask_line[NQT];
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt) mask_line[qt] = HAS_MASK ? walk_mask_line(p, b, w_first + qt * 16 + n) : 0;
    auto turn = [&](UnitShare<BITS, D>& next, int i) {
      const int t0 = 32 * walk.unit(i);
      const u32x4* unit = &stage[(i - c0) & 1][lane];
      u32x4 kop[AHEAD ? 2 : 1][AHEAD ? KK : 1], vop[AHEAD ? MT : 1];
      if constexpr (AHEAD) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) kop[t][kk] = unit[(t * KK + kk) * 64];
      }
      put(next, i + 1);
      bool needed = t0 < row_end && (t0 + 32 > row_low || t0 < walk.sink_end);
      MaskRegs<NQT> mregs;
      if (HAS_MASK) {
        mask_regs_from_raw<NQT>(mregs, coming, p);
        load_mask_raw<NQT>(coming, p, mask_line, 32 * walk.unit(i + 1), g);
        needed = needed && !walk_masked_out<D, NQT>(mregs, st);
      }
      send(next, i + 3);
      if (needed) {
        const bool full = t0 >= start && t0 + 31 <= min_limit && (t0 >= max_low || t0 + 32 <= walk.sink_end);
        f32x4 sc[NQT][2];
        u32x4 pb[NQT];
        walk_scores<BITS, D, NQT, CHUNK>([&](int t, int kk) { return AHEAD ? kop[AHEAD ? t : 0][AHEAD ? kk : 0] : unit[(t * KK + kk) * 64]; }, st, sc);
        if constexpr (AHEAD) {
#pragma unroll
          for (int j = 0; j < MT; ++j) vop[j] = unit[(MT + j) * 64];
        }
        walk_weights<BITS, D, NQT, HAS_MASK>(sc, st, pb, full, t0, start, walk.sink_end, g, mregs);
        walk_output<BITS, D, NQT, CHUNK>([&](int j) { return AHEAD ? vop[AHEAD ? j : 0] : unit[(MT + j) * 64]; }, st, pb);
      }
      __syncthreads();
    };
    // 64 units per set of block ids.  (Every turn of the inner loop fetches, past the last unit block 0 of the pool, which nobody reads:
    // behind a fetch that may or may not have been sent, the compiler would have the wave wait for all that is under way
    // before it uses the share before it.)
    for (; c0 < i_end; c0 += 64) {
      if (c0 > i_begin) {
        ids_lo = fetch_id(c0 + (lane >> 1)), ids_hi = fetch_id(c0 + 32 + (lane >> 1));
        send(even, c0);
        send(odd, c0 + 1);
      }
      const int c1 = min(c0 + 64, i_end);
      put(even, c0);
      if (HAS_MASK) load_mask_raw<NQT>(coming, p, mask_line, 32 * walk.unit(c0), g);
      send(even, c0 + 2);
      __syncthreads();
      int i = c0;
      for (; i + 1 < c1; i += 2) {
        turn(odd, i);
        turn(even, i + 1);
      }
      if (i < c1) turn(odd, i);
    }
    walk_finish<D, NQT, HAS_MASK>(st);
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt)
      if (w_first + qt * 16 + n < R) walk_store(p, st, qt, b, kvh, slot, w_first + qt * 16 + n - r_first, g);
  } while (p.shares > 0 && turns.left > 0 && turns.j < n_groups);
}

// out = sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p over the partial results of a query row.  A wave takes eight at a time, a lane the
// dims 2 lane, 2 lane + 1 (+ 128); WPR waves share a row (partial results in turn, joined through LDS), or a wave takes
// ROWS rows after one look at the lengths.  Rows of groups that
// one workgroup covered are finished already; rows that read nothing belong to no workgroup and become 0 here.
// Bound: latency (a launch, the lengths, then the partial results): some 5 us next to one sequence, up to 10 next to 9216 rows.
template <int D, int WPR, int ROWS>
__global__ __launch_bounds__(256) void walk_merge_kernel(const WalkParams p, int32_t total_rows) {
  constexpr int PASSES = (D + 127) / 128;
  __shared__ float join[WPR > 1 ? WPR : 1][2 * PASSES + 2][WPR > 1 ? 64 : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slice = wave % WPR;
  const int64_t row0 = WPR > 1 ? (int64_t)blockIdx.x : ((int64_t)blockIdx.x * 4 + wave) * ROWS;  // (b, hq, s)
  if (row0 >= total_rows) return;  // (WPR == 1 only: whole waves)
  const int S = p.q_len, n_groups = p.batch * p.n_qgroups;
  const bool one_group = p.part_units > 0 && n_groups == 1;
  int mine, share;  // units of the first 64 groups, one per lane (<true>: without a mask its length is past every sequence's)
  if (one_group) {
    mine = group_units<true>(p, 0), share = p.part_units;
  } else {
    mine = group_units<true>(p, lane);
    int total = mine;
#pragma unroll 4
    for (int i = lane + 64; i < n_groups; i += 64) total += group_units<true>(p, i);
    share = walk_share(p, wave_sum(total));
  }
  int last_j = -1, w0 = 0, n_parts = 0, late = 0;
  for (int64_t row = row0; row < row0 + ROWS && row < total_rows; ++row) {
    const int s = (int)(row % S), hq = (int)(row / S % p.num_q_heads), b = (int)(row / S / p.num_q_heads);
    const int kvh = hq / p.n_rep, r = s * p.n_rep + hq % p.n_rep, qg = r / p.group_rows;
    const int j = b * p.n_qgroups + p.n_qgroups - 1 - qg;
    if (j != last_j) {  // the group's units, and where they begin in the run of all units
      int before = lane < j ? mine : 0;
      for (int i = lane + 64; i < j; i += 64) before += group_units<true>(p, i);
      const int at = one_group ? 0 : wave_sum(before);
      const int units = j < 64 ? __builtin_amdgcn_readlane(mine, j) : group_units<true>(p, j);
      w0 = at / share, n_parts = units > 0 ? min((at + units - 1) / share, p.shares - 1) - w0 + 1 : 0;
      late = at % share != 0 ? 1 : 0;
      last_j = j;
    }
    if (n_parts == 1) continue;  // uniform over the row's waves
    // workgroup w0 + i's piece lies in its first slot, except the first one's if that workgroup began with other groups
    auto place = [&](int i) { return ((int64_t)(2 * (w0 + i) + (i == 0 ? late : 0)) * p.num_kv_heads + kvh) * p.slot_rows + (r - qg * p.group_rows); };
    const int d0 = 2 * lane;
    float acc[PASSES][2], M = kNegInf, L = 0.f;
#pragma unroll
    for (int e = 0; e < PASSES; ++e) acc[e][0] = acc[e][1] = 0.f;
    for (int base = 8 * slice; base < n_parts; base += 8 * WPR) {
      const u32x2 pair = *reinterpret_cast<const u32x2*>(p.part_ml + 2 * place(min(base + (lane & 7), n_parts - 1)));
      u32x2 v[8][PASSES];
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < PASSES; ++e) {
          v[i][e] = u32x2{0u, 0u};
          if (base + i < n_parts && d0 + 128 * e < D) v[i][e] = *reinterpret_cast<const u32x2*>(p.part_o + place(base + i) * D + d0 + 128 * e);
        }
      const float m_mine = base + (lane & 7) < n_parts ? __uint_as_float(pair[0]) : kNegInf;
      float top = m_mine;
      top = fmaxf(top, __shfl_xor(top, 1, 64)), top = fmaxf(top, __shfl_xor(top, 2, 64)), top = fmaxf(top, __shfl_xor(top, 4, 64));
      const float M_new = fmaxf(M, top), m_use = M_new == kNegInf ? 0.f : M_new, old = __builtin_amdgcn_exp2f(M - m_use);
      const float w_mine = __builtin_amdgcn_exp2f(m_mine - m_use);
      M = M_new, L *= old;
#pragma unroll
      for (int e = 0; e < PASSES; ++e) acc[e][0] *= old, acc[e][1] *= old;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (base + i < n_parts) {  // wave-uniform
          const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w_mine), i));
          L += w * __uint_as_float(__builtin_amdgcn_readlane(pair[1], i));
#pragma unroll
          for (int e = 0; e < PASSES; ++e) acc[e][0] += w * __uint_as_float(v[i][e][0]), acc[e][1] += w * __uint_as_float(v[i][e][1]);
        }
      }
    }
    if constexpr (WPR > 1) {
#pragma unroll
      for (int e = 0; e < PASSES; ++e) join[slice][2 * e][lane] = acc[e][0], join[slice][2 * e + 1][lane] = acc[e][1];
      join[slice][2 * PASSES][lane] = M, join[slice][2 * PASSES + 1][lane] = L;
      __syncthreads();
      if (slice != 0) continue;
      float all = kNegInf;
#pragma unroll
      for (int w = 0; w < WPR; ++w) all = fmaxf(all, join[w][2 * PASSES][lane]);
      const float m_use = all == kNegInf ? 0.f : all;
      L = 0.f;
#pragma unroll
      for (int e = 0; e < PASSES; ++e) acc[e][0] = acc[e][1] = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) {
        const float f = __builtin_amdgcn_exp2f(join[w][2 * PASSES][lane] - m_use);
        L += f * join[w][2 * PASSES + 1][lane];
#pragma unroll
        for (int e = 0; e < PASSES; ++e) acc[e][0] += f * join[w][2 * e][lane], acc[e][1] += f * join[w][2 * e + 1][lane];
      }
    }
    const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);
    uint16_t* op = p.out + (int64_t)b * p.o_sb + (int64_t)hq * p.o_sh + (int64_t)s * p.o_ss + d0;
#pragma unroll
    for (int e = 0; e < PASSES; ++e)
      if (d0 + 128 * e < D) *reinterpret_cast<uint32_t*>(op + 128 * e) = pack_bf16x2(acc[e][0] * inv, acc[e][1] * inv);
  }
}

// ---- host -------------------------------------------------------------------------------------------------------
struct WalkShape {
  int nqt;         // 0: walk_attn_kernel; else row tiles per wave of walk_rows_kernel
  int group_rows;  // query rows per group
  int n_qgroups, shares, min_share, part_units;  // see WalkParams
  int slot_rows;   // rows of a partial result
  int64_t units;   // of the longest group
  size_t bytes;    // of partial results
};

constexpr int walk_waves(int head_dim) { return head_dim == 256 ? 2 : 4; }  // of a workgroup of walk_attn_kernel
constexpr int walk_occ(int head_dim) { return head_dim == 256 ? 1 : 2; }
constexpr int rows_occ(int head_dim, int nqt) { return head_dim == 256 || nqt > 1 ? 2 : 3; }

// What the kernels take, by the query rows of a group, in us at 128 dims: per unit of a workgroup that has a compute unit to itself
// (alone), per unit and workgroup of a compute unit that is full, and for every further workgroup of a compute unit to start.
// (Measured over 4-bit pools with 8 KV heads, 4 query heads each: one sequence x 4096 tokens, 128 / 512 new ones, in groups
// of 16: 32 / 91 us, 64: 103 / 104, 128: 129 / 131; 4 sequences x 4608, 512 new ones: 355 / 247 / 190; 64 dims take 0.63 of it.)
struct WalkKind {
  int nqt, group_rows;  // nqt 0: walk_attn_kernel
  double alone, full, start;
};
static WalkKind walk_kind(int kind, int head_dim) {
  if (head_dim == 256) return kind == 0 ? WalkKind{0, 16, 0.75, 0.72, 1.8} : WalkKind{1, 64, 1.1, 0.65, 4.0};
  const double f = 0.27 + 0.73 * head_dim / 128;
  return kind == 0   ? WalkKind{0, 16, 0.165 * f, 0.165 * f, 1.8}
         : kind == 1 ? WalkKind{1, 64, 0.77 * f, 0.43 * f, 4.0}
                     : WalkKind{2, 128, 1.0 * f, 0.65 * f, 8.0};
}

// The shape of a launch in groups of one kind, and an estimate of its time in us.
static WalkShape walk_shape_of(const pace_kv_pool_t* pool, const pace_paged_attn_args_t* a, const WalkKind& kind, double& time) {
  WalkShape s = {};
  const int64_t n_rep = a->num_q_heads / pool->num_kv_heads, rows = a->q_len * n_rep;
  const int D = pool->head_dim, heads = pool->num_kv_heads;
  const bool few = kind.nqt == 0;
  s.nqt = kind.nqt, s.group_rows = kind.group_rows;
  s.n_qgroups = (int)((rows + s.group_rows - 1) / s.group_rows);
  s.slot_rows = (int)std::min<int64_t>(rows, s.group_rows);
  int64_t units = ((int64_t)a->max_seq_len + 31) / 32;  // of the longest group
  if (a->window > 0) {
    const int64_t tokens = std::min<int64_t>(a->q_len, (s.slot_rows - 1) / std::max<int64_t>(n_rep, 1) + 2);
    units = std::min(units, (a->window + (a->causal ? tokens : a->q_len)) / 32 + 2 + a->sinks / 32 + 2);
  }
  s.units = units = std::max<int64_t>(units, 1);
  s.min_share = few ? walk_waves(D) : 1;  // units a workgroup works on side by side
  const int64_t n_groups = (int64_t)a->batch * s.n_qgroups, groups = n_groups * heads, cus = compute_units();
  // One workgroup per compute unit nearly is enough for walk_attn_kernel, whose waves fetch ahead; where its units are shared out it
  // gets two (64 x 500 .. 8000 tokens: 71 us with one, 60 with two).
  const int64_t slots = cus * (few ? 2 : rows_occ(D, s.nqt));
  int64_t shares = 0;
  if (n_groups * units >= (int64_t)1 << 30) {
    time = 1e30;  // (the run of all units is counted in 32 bits; as many groups as that need no sharing)
  } else if (a->partition_tokens > 0) {
    time = 0;
    // A given cut: no run is longer, and nothing is cut if no group is longer.  (The runs of several groups are equal shares here
    // too, so sequences below max_seq_len make them shorter, not fewer.)
    s.part_units = (int)(((int64_t)a->partition_tokens / 32 + s.min_share - 1) / s.min_share * s.min_share);
    if (units > s.part_units) shares = (n_groups * units + s.part_units - 1) / s.part_units;  // (more than there are groups)
    if (!few) s.min_share = std::min(s.part_units, 4);
    if (n_groups > 1) s.part_units = 0;
  } else {
    // A workgroup per group lasts as long as the longest chain of units, or as a compute unit with its workgroups needs: under the causal
    // limit the groups of a fresh prompt have half as many units on average.  Sequences of long contexts may differ in
    // length (only the bound is known here), which leaves compute units idle, unless there are many: up to 128 rows each, contexts
    // of more than 160 units are taken for ragged.  The border lies between the sequences of 4096 tokens that were measured as
    // equal and those of 1000 .. 6000 and 500 .. 8000 that were measured as ragged, and is a guess between them.  It costs equal
    // long sequences the second launch (shared / not, us: 32 x 8000 65 to 70 / 60, 64 x 8000 114 / 107, 128 x 6000 169 / 160, 64 x 6000
    // with 5 tokens 174 / 152) for what it saves ragged ones (64 x 500 .. 8000 57 / 74, 32 x 1000 .. 6000 with 9 tokens 62 / 145).
    const double fresh = a->causal && a->window == 0 ? std::min(a->q_len, a->max_seq_len) / (double)std::max(a->max_seq_len, 1) : 0.0;
    const double average = (double)units * (1.0 - 0.5 * fresh);
    const double ragged = rows <= 128 && a->batch > 1 && units > 160 ? 1.4 : 1.0;
    const int64_t per_cu = (groups + cus - 1) / cus;
    const double own = (7.0 + std::max(units * kind.alone, average * kind.full * (double)per_cu) + kind.start * (double)(per_cu - 1)) * ragged;
    // Equal shares of all units cost a second launch, the start of more pieces, and a trip of the partial results: some 10 us, 4 next to a
    // single group, 12 to 40 where four waves work in step, and 10 more per 9216 rows.  Measured without -> with, 8 KV heads of 128 dims,
    // 4 query heads each, us:
    //   one row, 1 x 512 tokens: 8.6 -> 9.8; 1 x 4096: 28 -> 10.5; 8 x 2000: 17.7 -> 19.8; 33 x 8000: 99 -> 73;
    //     64 x 500 .. 8000: 76 -> 60; 64 x 8000: 113 -> 127; 256 x 100 .. 8000: 154 -> 175; a window of 4096, 32 sequences: 83 -> 91
    //   9 drafted tokens, 32 x 1000 .. 6000: 146 -> 64; 96 x 500 .. 8000: 224 -> 148; 192 x 500 .. 8000: 350 -> 302; 192 x 6000: 535 -> 534
    //   512 tokens, 2 x 8000: 266 -> 223; 4 x 8000: 392 -> 425; 4 x 800 .. 8000: 269 -> 313; a prompt of 1024: 39 -> 68
    const double work = average * kind.full * (double)groups / (double)cus;
    const double shared = 7.0 + 10.0 / 9216 * (double)(rows * a->batch * heads) + (few ? (n_groups == 1 ? 4.0 : 10.0) + work : std::max(40.0, 12.0 + work));
    time = own;
    if (shared < own && units > 8 && groups <= slots * 2) {
      time = shared;
      shares = std::max<int64_t>(slots / heads, 1);
      if (!few) s.min_share = 4;
      if (n_groups == 1) {
        s.part_units = (int)std::max<int64_t>((units + shares - 1) / shares, few ? 4 : 12);
        s.part_units = (s.part_units + s.min_share - 1) / s.min_share * s.min_share;
        shares = (units + s.part_units - 1) / s.part_units;
        if (shares == 1) shares = 0;
      }
    }
  }
  s.shares = (int)shares;
  return s;
}

// Groups of 16 rows (every wave unpacks for itself, four units of a group at a time) leave the shortest chain, groups of 128 the least
// work: the estimates above decide, for a batch of short appends as for a long prompt.  Measured in groups of 16 / 64 / 128:
// a prompt of 256 tokens 9.2 / 12.7 / 16.5 us, of 1024 40 / 31 / 39, 4 of 512 60 / 32 / 33; 9 tokens to 8 x 2000 19 / 35 / 40.
// workspace_bytes: what partial results may take (the units are shared out over no more workgroups than fit).
static WalkShape walk_shape(const pace_kv_pool_t* pool, const pace_paged_attn_args_t* a, size_t workspace_bytes) {
  const int64_t rows = a->q_len * (int64_t)(a->num_q_heads / pool->num_kv_heads);
  const int D = pool->head_dim, heads = pool->num_kv_heads;
  const int largest = rows <= 16 ? 0 : (rows <= 64 || D == 256 ? 1 : 2);
  double best = 0;
  WalkShape s = walk_shape_of(pool, a, walk_kind(largest, D), best);
  for (int kind = largest - 1; kind >= 0; --kind) {  // (given partitions: the largest groups)
    double time = 0;
    const WalkShape t = walk_shape_of(pool, a, walk_kind(kind, D), time);
    if (time < best) s = t, best = time;
  }
  const int64_t n_groups = (int64_t)a->batch * s.n_qgroups;
  const size_t one = (size_t)heads * 2 * s.slot_rows * (D + 2) * sizeof(float);  // of a workgroup per KV head
  if (s.shares > 0 && workspace_bytes / one < (size_t)s.shares) {
    s.shares = (int)(workspace_bytes / one);
    if (s.shares <= n_groups) s.shares = 0;  // (a workgroup per group does as well)
    s.part_units = 0;
    if (s.shares > 0 && n_groups == 1) s.part_units = (int)(((s.units + s.shares - 1) / s.shares + s.min_share - 1) / s.min_share * s.min_share);
  }
  if (s.shares == 0) s.part_units = 0;
  s.bytes = one * (size_t)s.shares;
  return s;
}

size_t walk_workspace_bytes(const pace_kv_pool_t* pool, const pace_paged_attn_args_t* a) {
  if (a->partition_tokens < 0 || a->partition_tokens % 32 != 0) return 0;  // (the launch refuses it)
  return walk_shape(pool, a, ~(size_t)0).bytes;
}

template <int BITS, int D, bool HAS_MASK>
static void launch_walk_kernel(const WalkParams& p, int nqt, hipStream_t s) {
  const dim3 grid((unsigned)p.total_items);
  if (nqt == 0) hipLaunchKernelGGL((walk_attn_kernel<BITS, D, HAS_MASK, walk_waves(D), walk_occ(D)>), grid, dim3(64 * walk_waves(D)), 0, s, p);
  else if (nqt == 1) hipLaunchKernelGGL((walk_rows_kernel<BITS, D, 1, HAS_MASK, rows_occ(D, 1)>), grid, dim3(256), 0, s, p);
  else if constexpr (D != 256) hipLaunchKernelGGL((walk_rows_kernel<BITS, D, 2, HAS_MASK, rows_occ(D, 2)>), grid, dim3(256), 0, s, p);
}

int walk_kernel_name(const pace_kv_pool_t* pool, const pace_paged_attn_args_t* a, char* out, size_t cap) {
  const WalkShape sh = walk_shape(pool, a, a->workspace ? a->workspace_bytes : 0);
  const int bits = pool_is_q4(pool) ? 4 : 16, D = pool->head_dim;
  const char* masked = a->mask ? "true" : "false";
  if (sh.nqt == 0) snprintf(out, cap, "pace_kv::walk_attn_kernel<%d, %d, %s, %d, %d>", bits, D, masked, walk_waves(D), walk_occ(D));
  else snprintf(out, cap, "pace_kv::walk_rows_kernel<%d, %d, %d, %s, %d>", bits, D, sh.nqt, masked, rows_occ(D, sh.nqt));
  return PACE_KV_OK;
}

int launch_walk(const pace_kv_pool_t* pool, const pace_paged_attn_args_t* a, const char* who, hipStream_t stream) {
  if (a->workspace) PACE_REQUIRE(aligned16(a->workspace), "%s: workspace must be 16-byte aligned", who);
  const WalkShape sh = walk_shape(pool, a, a->workspace ? a->workspace_bytes : 0);
  WalkParams p = {};
  p.q = static_cast<const uint16_t*>(a->q);
  p.q_sb = a->q_stride_b, p.q_sh = a->q_stride_h, p.q_ss = a->q_stride_s;
  p.out = static_cast<uint16_t*>(a->out);
  p.o_sb = a->o_stride_b, p.o_sh = a->o_stride_h, p.o_ss = a->o_stride_s;
  p.kpool = static_cast<const uint16_t*>(pool->k), p.vpool = static_cast<const uint16_t*>(pool->v);
  p.k_bs = pool->k_block_stride, p.k_hs = pool->k_head_stride, p.v_bs = pool->v_block_stride, p.v_hs = pool->v_head_stride;
  p.num_blocks = pool->num_blocks, p.num_kv_heads = pool->num_kv_heads;
  p.table = a->block_table, p.table_stride = a->table_stride;
  p.seq_lens = a->seq_lens, p.len_bias = a->seq_len_bias, p.len_bias_dev = a->seq_len_bias_ptr, p.kv_start = a->kv_start;
  p.mask = a->mask, p.mask_is_f32 = a->mask_dtype == PACE_DTYPE_F32, p.mask_len = a->mask ? a->mask_len : 0x7fffffff;
  p.m_sb = a->mask_stride_b, p.m_ss = a->mask_stride_s;
  p.n_rep = a->num_q_heads / pool->num_kv_heads, p.q_len = a->q_len, p.num_q_heads = a->num_q_heads, p.batch = a->batch;
  p.causal = a->causal;
  p.scale = a->scale, p.scale_log2 = a->scale * kLog2e;
  p.window = std::min(a->window, 1 << 30), p.sinks = std::min(a->sinks, 1 << 30);  // (sums with them stay below 2^31)
  p.n_qgroups = sh.n_qgroups, p.group_rows = sh.group_rows, p.slot_rows = sh.slot_rows;
  p.shares = sh.shares, p.min_share = sh.min_share, p.part_units = sh.part_units;
  const size_t rows = (size_t)a->batch * a->num_q_heads * a->q_len;
  PACE_REQUIRE(rows < ((size_t)1 << 31), "%s: too many query rows", who);
  if (sh.shares > 0) {
    p.part_o = static_cast<float*>(a->workspace);
    p.part_ml = p.part_o + (size_t)sh.shares * 2 * pool->num_kv_heads * sh.slot_rows * pool->head_dim;
  }
  p.total_items = (sh.shares > 0 ? (long long)sh.shares : (long long)a->batch * sh.n_qgroups) * pool->num_kv_heads;
  PACE_REQUIRE(p.total_items < (1ll << 31), "%s: grid too large", who);
  if (a->k_new)  // the new tokens first: they are read back from the pool like all others
    if (int rc = pace_kv_append_paged_at(pool, a->k_new, a->v_new, a->new_stride_b, a->new_stride_h, a->new_stride_t, a->batch, a->n_new,
                                         a->block_table, a->table_stride, a->seq_lens, a->seq_len_bias - a->n_new, a->seq_len_bias_ptr, stream))
      return rc;
  const bool masked = a->mask != nullptr, q4 = pool_is_q4(pool);
  for_head_dim(pool->head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (q4) {
      if (masked) launch_walk_kernel<4, D, true>(p, sh.nqt, stream); else launch_walk_kernel<4, D, false>(p, sh.nqt, stream);
    } else {
      if (masked) launch_walk_kernel<16, D, true>(p, sh.nqt, stream); else launch_walk_kernel<16, D, false>(p, sh.nqt, stream);
    }
    // Few groups, many workgroups each: four waves to a row.  More rows than the GPU holds waves: four rows to a wave, one look at the
    // lengths for all (with the attention, one row -> four: 512 tokens to 4096 83 -> 79 us, 9 to 96 x 500 .. 8000 148 -> 143).
    const bool wide = sh.shares > 4 * (int64_t)a->batch * sh.n_qgroups, many = rows >= (size_t)compute_units() * 32;
    if (sh.shares == 0) return;
    if (wide) hipLaunchKernelGGL((walk_merge_kernel<D, 4, 1>), dim3((unsigned)rows), dim3(256), 0, stream, p, (int32_t)rows);
    else if (many) hipLaunchKernelGGL((walk_merge_kernel<D, 1, 4>), dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, stream, p, (int32_t)rows);
    else hipLaunchKernelGGL((walk_merge_kernel<D, 1, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, p, (int32_t)rows);
  });
  PACE_HIP_CHECK(hipGetLastError());
  return PACE_KV_OK;
}

}  // namespace pace_kv
