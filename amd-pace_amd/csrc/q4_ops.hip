// Pools of 4-bit rows: quantise on append, read back as bf16 token rows.  (Blocks are copied by the kernels of kv_ops.hip:
// a slab is moved as it is.)  Both are bound by HBM: per value 2 bytes of bf16 on one side, 5/8 of a byte on the other.
#include "kv_ops.h"
#include "q4.h"

namespace pace_kv {

// ---------------------------------------------------------------------------------
// Append.  One workgroup of 2 D threads takes up to 16 tokens of one (sequence, KV head): thread (token, chunk) reads eight
// dims of K and of V (16 bytes each), four neighbouring threads make a group of 32 and agree on its step and middle in
// registers.  K codes are a token's own dword and are stored from where they are made; a V code dword holds eight
// tokens of one dim, so the codes meet in LDS, one byte each, and every thread puts one dword together.
//   PAGED: the tokens of one destination block.  A V dword has one writer, the block's workgroup: where the append
//   covers only some of its eight tokens the dword is read, changed and written back.
//   by slot: 16 consecutive tokens of the input, wherever their slots lie.  Tokens of one V dword may then sit in two
//   workgroups; a dword not covered in full is changed by atomics on its own bits (each bit has one writer as long as
//   no slot is named twice, so the order does not matter).
// ---------------------------------------------------------------------------------
template <int D, bool PAGED>
__global__ __launch_bounds__(2 * D) void q4_append_kernel(pace_kv_pool_t pool, const uint16_t* __restrict__ k_new,
                                                          const uint16_t* __restrict__ v_new, int64_t sb, int64_t sh, int64_t st,
                                                          int32_t n_tokens, int32_t groups_x, const AppendDest dest) {
  using L = Q4<D>;
  constexpr int CHUNKS = D / 8, BT = PACE_KV_BLOCK_TOKENS, ROW = D + 8;
  __shared__ __attribute__((aligned(8))) uint8_t codes[BT * ROW];  // V codes, token-major
  __shared__ int64_t slot_of[BT];                                  // by slot: the tokens' slots (-1: none)
  const int H = pool.num_kv_heads;
  const int x = (int)(blockIdx.x % (uint32_t)groups_x), h = (int)(blockIdx.x / (uint32_t)groups_x % (uint32_t)H);
  const int64_t b = blockIdx.x / (uint32_t)groups_x / (uint32_t)H;
  const int i = threadIdx.x / CHUNKS, c = threadIdx.x % CHUNKS;  // this thread's token (of 16) and eight dims
  int64_t t;      // token of the input
  int64_t blk;    // destination block
  int off;        // token slot in it
  int first = 0, count = 0;  // PAGED: block tokens first .. first + count - 1 are written
  bool live;
  if (PAGED) {
    const int64_t pos0 = (int64_t)dest.seq_lens[b] + dest.pos_offset + (dest.offset_dev ? *dest.offset_dev : 0);
    const int64_t jb = (pos0 > 0 ? pos0 : 0) / BT + x;
    if (jb >= dest.table_stride) return;  // uniform over the workgroup, like the next two
    const int64_t lo = max(pos0, jb * BT), hi = min(pos0 + n_tokens, jb * BT + BT);
    if (lo >= hi) return;
    blk = dest.table[b * dest.table_stride + jb];
    if (blk < 0 || blk >= pool.num_blocks) return;  // never write outside the pool
    first = (int)(lo - jb * BT), count = (int)(hi - lo);
    off = i;
    t = jb * BT + i - pos0;
    live = i >= first && i < first + count;
  } else {
    t = (int64_t)x * BT + i;
    int64_t slot = t < n_tokens ? dest.slots[b * n_tokens + t] : -1;
    if (slot < 0 || slot / BT >= pool.num_blocks) slot = -1;
    if (c == 0) slot_of[i] = slot;
    live = slot >= 0;
    blk = live ? slot / BT : 0;
    off = live ? (int)(slot % BT) : 0;
  }
  uint8_t* kslab = static_cast<uint8_t*>(pool.k) + blk * pool.k_block_stride + (int64_t)h * pool.k_head_stride;
  uint8_t* vslab = static_cast<uint8_t*>(pool.v) + blk * pool.v_block_stride + (int64_t)h * pool.v_head_stride;
  const int kk = c / 4, g = c % 4;
  if (live) {  // the same for a token's threads, so for every group of four
    const int64_t src = b * sb + (int64_t)h * sh + t * st + c * 8;
    const u32x4 kraw = load16_stream(k_new + src), vraw = load16_stream(v_new + src);
    float xs[8];
    _Float16 s, m;
    bf16x8_to_f32(kraw, xs);
    const uint32_t kw = q4_quantise(xs, s, m);
    uint32_t* k32 = reinterpret_cast<uint32_t*>(kslab);
    k32[L::k_code(q4_tile(off), g, q4_slot(off), kk)] = kw;
    if (g == 0) k32[L::k_scale(q4_tile(off), q4_slot(off), kk)] = half_bits(s) | (half_bits(m) << 16);
    bf16x8_to_f32(vraw, xs);
    const uint32_t vw = q4_quantise(xs, s, m);
    if (g == 0) {
      uint16_t* v16 = reinterpret_cast<uint16_t*>(vslab);
      v16[L::v_scale(kk, off)] = (uint16_t)half_bits(s);
      v16[L::v_scale(kk, off) + 16 * L::G] = (uint16_t)half_bits(m);
    }
    u32x2 bytes = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e) bytes[e >> 2] |= ((vw >> q4_bit(e)) & 15u) << (8 * (e & 3));
    *reinterpret_cast<u32x2*>(&codes[i * ROW + c * 8]) = bytes;
  }
  __syncthreads();
  // This thread's V dword: (token half, dim), dims in the order of the slab, so that a wave's stores are contiguous.
  const int o = threadIdx.x, half = o / D, r = o % D;
  const int dim = 16 * (r / (16 * L::VC) * L::VC + r % L::VC) + r / L::VC % 16;
  if (PAGED) {
    uint32_t* at = reinterpret_cast<uint32_t*>(vslab) + o;
    uint32_t w = 0, mask = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int tok = 8 * half + e;
      if (tok >= first && tok < first + count) w |= (uint32_t)codes[tok * ROW + dim] << q4_bit(e), mask |= 15u << q4_bit(e);
    }
    if (mask == 0xffffffffu) *at = w;
    else if (mask != 0u) *at = (*at & ~mask) | w;
  } else {
    // Every V dword a token of this workgroup lies in, found at its first token here (uniform over the workgroup); the two
    // thread halves take the dwords in turn.
    int turn = 0;
    for (int a = 0; a < BT; ++a) {
      const int64_t key = slot_of[a] < 0 ? -1 : slot_of[a] / 8;
      bool seen = key < 0;
      for (int e = 0; e < a; ++e) seen = seen || (slot_of[e] >= 0 && slot_of[e] / 8 == key);
      if (seen) continue;
      if ((turn++ & 1) != half) continue;
      uint32_t w = 0, mask = 0;
      for (int e = a; e < BT; ++e) {
        if (slot_of[e] < 0 || slot_of[e] / 8 != key) continue;
        const int bit = q4_bit((int)(slot_of[e] % 8));
        w = (w & ~(15u << bit)) | ((uint32_t)codes[e * ROW + dim] << bit);
        mask |= 15u << bit;
      }
      uint32_t* at = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(pool.v) + key / 2 * pool.v_block_stride + (int64_t)h * pool.v_head_stride) +
                     (key % 2) * D + r;
      if (mask == 0xffffffffu) {
        *at = w;
      } else {
        atomicAnd(at, ~mask);
        atomicOr(at, w);
      }
    }
  }
}

// ---------------------------------------------------------------------------------
// Read back.  One workgroup of 2 D threads rebuilds one logical block (16 tokens) of one KV head as token rows: thread
// (token, chunk) makes eight dims of K from one code dword, and eight dims of V from the eight dwords its token has a
// code in, which pass through LDS.
// ---------------------------------------------------------------------------------
template <int D, bool PACKED>
__global__ __launch_bounds__(2 * D) void q4_gather_kernel(pace_kv_pool_t pool, const int32_t* __restrict__ table, int32_t table_stride,
                                                          const int32_t* __restrict__ seq_lens, int32_t len_bias, int32_t n_rep,
                                                          int32_t n_blocks, const GatherOut out) {
  using L = Q4<D>;
  constexpr int CHUNKS = D / 8, BT = PACE_KV_BLOCK_TOKENS;
  __shared__ uint32_t vc[2 * D];
  int j, b, h;
  if (PACKED) {
    packed_entry(out.cu_seqlens, out.batch, pool.num_kv_heads, blockIdx.x, b, h, j);
  } else {
    j = (int)(blockIdx.x % (uint32_t)n_blocks);
    h = (int)(blockIdx.x / (uint32_t)n_blocks % (uint32_t)pool.num_kv_heads);
    b = (int)(blockIdx.x / (uint32_t)n_blocks / (uint32_t)pool.num_kv_heads);
  }
  const int len = seq_lens[b] + len_bias;
  int64_t blk = table[(int64_t)b * table_stride + min(j, table_stride - 1)];
  const int t0 = j * BT;
  const bool live = t0 < len && j < table_stride;  // uniform over the workgroup
  const bool dense_rows = PACKED && out.dense_rows != 0;  // the dense layout from the packed grid
  const int row_end = PACKED ? (dense_rows ? min(len, out.out_len) : len) : out.out_len;
  if (!live && (PACKED || !out.zero_fill || t0 >= row_end)) return;  // nothing to write
  blk = blk < 0 ? 0 : (blk >= pool.num_blocks ? pool.num_blocks - 1 : blk);  // never read outside the pool
  const uint8_t* kslab = static_cast<const uint8_t*>(pool.k) + blk * pool.k_block_stride + (int64_t)h * pool.k_head_stride;
  const uint8_t* vslab = static_cast<const uint8_t*>(pool.v) + blk * pool.v_block_stride + (int64_t)h * pool.v_head_stride;
  const int tok = threadIdx.x / CHUNKS, c = threadIdx.x % CHUNKS, kk = c / 4, g = c % 4;
  const int t = t0 + tok;
  uint32_t kw = 0, ksm = 0;
  float vs = 0.f, vm = 0.f;
  if (live) {
    const uint32_t* k32 = reinterpret_cast<const uint32_t*>(kslab);
    const uint16_t* v16 = reinterpret_cast<const uint16_t*>(vslab);
    vc[threadIdx.x] = reinterpret_cast<const uint32_t*>(vslab)[threadIdx.x];
    kw = k32[L::k_code(q4_tile(tok), g, q4_slot(tok), kk)];
    ksm = k32[L::k_scale(q4_tile(tok), q4_slot(tok), kk)];
    vs = (float)half_from(v16[L::v_scale(kk, tok)]);
    vm = (float)half_from(v16[L::v_scale(kk, tok) + 16 * L::G]);
  }
  __syncthreads();
  if (t >= row_end) return;
  if (PACKED && !dense_rows && out.cu_seqlens[b] + t >= out.total_rows) return;  // never write past the outputs
  u32x4 kv = {0u, 0u, 0u, 0u}, vv = {0u, 0u, 0u, 0u};
  if (t < len) {
    const float ks = (float)half_from(ksm & 0xffffu), km = (float)half_from(ksm >> 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // s * code is exact in single precision, so the sum is rounded once and then once more to bf16
      kv[e] = pack_bf16x2(__builtin_fmaf(q4_code(kw, 2 * e), ks, km), __builtin_fmaf(q4_code(kw, 2 * e + 1), ks, km));
      float x[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const int dim = c * 8 + 2 * e + a;
        x[a] = __builtin_fmaf(q4_code(vc[L::v_code(tok >> 3, dim >> 4, dim & 15)], tok & 7), vs, vm);
      }
      vv[e] = pack_bf16x2(x[0], x[1]);
    }
  } else if (!out.zero_fill) {
    return;
  }
  const int64_t base = (PACKED && !dense_rows) ? (int64_t)out.cu_seqlens[b] * out.stride_t : (int64_t)b * out.stride_b;
  for (int r = 0; r < n_rep; ++r) {
    const int64_t at = base + (int64_t)(h * n_rep + r) * out.stride_h + (int64_t)t * out.stride_t + c * 8;
    store16_stream(out.k + at, kv);
    store16_stream(out.v + at, vv);
  }
}

int launch_q4_append(const char* who, const pace_kv_pool_t* pool, const void* k_new, const void* v_new, int64_t stride_b,
                     int64_t stride_h, int64_t stride_t, int32_t batch, int32_t n_tokens, const AppendDest& dest, bool paged,
                     hipStream_t stream) {
  // PAGED: the most blocks n_tokens consecutive positions can touch; by slot: runs of 16 input tokens
  const int64_t groups = paged ? ((int64_t)n_tokens + PACE_KV_BLOCK_TOKENS - 2) / PACE_KV_BLOCK_TOKENS + 1
                               : ((int64_t)n_tokens + PACE_KV_BLOCK_TOKENS - 1) / PACE_KV_BLOCK_TOKENS;
  const int64_t grid = groups * pool->num_kv_heads * batch;
  PACE_REQUIRE(grid < (int64_t)1 << 31, "%s: grid too large", who);
  const uint16_t* k = static_cast<const uint16_t*>(k_new);
  const uint16_t* v = static_cast<const uint16_t*>(v_new);
  for_head_dim(pool->head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (paged)
      hipLaunchKernelGGL((q4_append_kernel<D, true>), dim3((unsigned)grid), dim3(2 * D), 0, stream, *pool, k, v, stride_b, stride_h, stride_t,
                         n_tokens, (int32_t)groups, dest);
    else
      hipLaunchKernelGGL((q4_append_kernel<D, false>), dim3((unsigned)grid), dim3(2 * D), 0, stream, *pool, k, v, stride_b, stride_h, stride_t,
                         n_tokens, (int32_t)groups, dest);
  });
  PACE_HIP_CHECK(hipGetLastError());
  return PACE_KV_OK;
}

int launch_q4_gather(const char* who, const pace_kv_pool_t* pool, const int32_t* block_table, int32_t table_stride,
                     const int32_t* seq_lens, int32_t seq_len_bias, int32_t n_rep, const GatherOut& out, int64_t n_blocks, int32_t batch,
                     bool packed, hipStream_t stream) {
  const int64_t grid = packed ? ((int64_t)out.total_rows / PACE_KV_BLOCK_TOKENS + batch) * pool->num_kv_heads
                              : n_blocks * pool->num_kv_heads * batch;
  PACE_REQUIRE(grid < (int64_t)1 << 31, "%s: grid too large", who);
  for_head_dim(pool->head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (packed)
      hipLaunchKernelGGL((q4_gather_kernel<D, true>), dim3((unsigned)grid), dim3(2 * D), 0, stream, *pool, block_table, table_stride, seq_lens,
                         seq_len_bias, n_rep, (int32_t)n_blocks, out);
    else
      hipLaunchKernelGGL((q4_gather_kernel<D, false>), dim3((unsigned)grid), dim3(2 * D), 0, stream, *pool, block_table, table_stride, seq_lens,
                         seq_len_bias, n_rep, (int32_t)n_blocks, out);
  });
  PACE_HIP_CHECK(hipGetLastError());
  return PACE_KV_OK;
}

}  // namespace pace_kv
