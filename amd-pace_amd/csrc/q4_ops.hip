// Pools of 4-bit rows: quantise on append, read back as bf16 token rows.  (Blocks are copied by the kernels of kv_ops.hip:
// a slab is moved as it is.)  Both are bound by HBM: per value 2 bytes of bf16 on one side, 5/8 of a byte on the other.
#include "kv_ops.h"
#include "q4.h"

namespace pace_kv {

// ---------------------------------------------------------------------------------
// Append.  A workgroup of 2 D threads takes up to 16 tokens of one (sequence, KV head) at a time: thread (token, chunk) has eight
// dims of K and of V (16 bytes each), four neighbouring threads make a group of 32 and agree on its step and middle in
// registers.  K codes are a token's own dword and are stored from where they are made; a V code dword holds eight
// tokens of one dim, so the codes meet in LDS, one byte each, and every thread puts one dword together.
// ---------------------------------------------------------------------------------
// Quantises one token's eight dims (chunk c) of K and V: K and the scales into the slabs, V codes as bytes to `bytes`.  The threads of
// a token come here together.
template <int D>
__device__ __forceinline__ void q4_store_token(uint8_t* kslab, uint8_t* vslab, int tok, int c, u32x4 kraw, u32x4 vraw, uint8_t* bytes) {
  using L = Q4<D>;
  const int kk = c / 4, g = c % 4;
  uint32_t q[8];
  _Float16 s, m;
  q4_quantise(kraw, q, s, m);
  uint32_t* k32 = reinterpret_cast<uint32_t*>(kslab);
  k32[L::k_code(q4_tile(tok), g, q4_slot(tok), kk)] = q4_pack(q);
  if (g == 0) k32[L::k_scale(q4_tile(tok), q4_slot(tok), kk)] = half_bits(s) | (half_bits(m) << 16);
  q4_quantise(vraw, q, s, m);
  if (g == 0) {
    uint16_t* v16 = reinterpret_cast<uint16_t*>(vslab);
    v16[L::v_scale(kk, tok)] = (uint16_t)half_bits(s);
    v16[L::v_scale(kk, tok) + 16 * L::G] = (uint16_t)half_bits(m);
  }
  *reinterpret_cast<u32x2*>(bytes) = q4_bytes(q);
}
// The dim of V dword r of a token half, in slab order: a wave's dwords are contiguous.
template <int D>
__device__ __forceinline__ int q4_v_dim(int r) {
  constexpr int VC = Q4<D>::VC;
  return 16 * (r / (16 * VC) * VC + r % VC) + r / VC % 16;
}

// By position: one destination block of one (sequence, KV head).  A V dword has one writer, its block's workgroup: where the append
// covers only some of its eight tokens it is read, changed and written back.
// 8 prompts of 4096 tokens, 8 heads of 128, stored (176 MB) and read back (the same): 79 us, 4.5 TB/s, where a plain copy moves
// 5.1.  Two, four or eight blocks per workgroup with the next one's rows under way took 2, 3 and 6 us more: the workgroups
// that share a compute unit hide the loads already.  The store alone: 51 us, 3.5 TB/s.  One token each of 64 sequences,
// stored and read back: 10 us, latency.
template <int D>
__global__ __launch_bounds__(2 * D) void q4_append_paged_kernel(pace_kv_pool_t pool, const uint16_t* __restrict__ k_new,
                                                                const uint16_t* __restrict__ v_new, int64_t sb, int64_t sh, int64_t st,
                                                                int32_t n_tokens, int32_t groups_x, const AppendDest dest) {
  constexpr int CHUNKS = D / 8, BT = PACE_KV_BLOCK_TOKENS, ROW = D + 8;
  __shared__ __attribute__((aligned(8))) uint8_t codes[BT * ROW];  // V codes, token-major
  const uint32_t H = (uint32_t)pool.num_kv_heads;
  const int x = (int)(blockIdx.x % (uint32_t)groups_x), h = (int)(blockIdx.x / (uint32_t)groups_x % H);
  const int64_t b = blockIdx.x / (uint32_t)groups_x / H;
  const int i = threadIdx.x / CHUNKS, c = threadIdx.x % CHUNKS;  // this thread's token (of 16) and eight dims
  const int64_t pos0 = (int64_t)dest.seq_lens[b] + dest.pos_offset + (dest.offset_dev ? *dest.offset_dev : 0);
  const int64_t jb = (pos0 > 0 ? pos0 : 0) / BT + x;
  if (jb >= dest.table_stride) return;  // uniform over the workgroup, like the next two
  const int64_t lo = max(pos0, jb * BT), hi = min(pos0 + n_tokens, jb * BT + BT);
  if (lo >= hi) return;
  const int64_t blk = dest.table[b * dest.table_stride + jb];
  const int first = (int)(lo - jb * BT), past = (int)(hi - jb * BT);
  const bool live = i >= first && i < past;
  // The rows are asked for next to the block id, not behind it.
  u32x4 kraw = {0u, 0u, 0u, 0u}, vraw = {0u, 0u, 0u, 0u};
  if (live) {
    const int64_t src = b * sb + (int64_t)h * sh + (jb * BT + i - pos0) * st + c * 8;
    kraw = load16_stream(k_new + src), vraw = load16_stream(v_new + src);
  }
  if (blk < 0 || blk >= pool.num_blocks) return;  // never write outside the pool
  uint8_t* kslab = static_cast<uint8_t*>(pool.k) + blk * pool.k_block_stride + (int64_t)h * pool.k_head_stride;
  uint8_t* vslab = static_cast<uint8_t*>(pool.v) + blk * pool.v_block_stride + (int64_t)h * pool.v_head_stride;
  uint32_t* const at = reinterpret_cast<uint32_t*>(vslab) + threadIdx.x;  // this thread's V dword: (token half, dim)
  const int half = threadIdx.x / D, dim = q4_v_dim<D>(threadIdx.x % D);
  uint32_t lower = 0, upper = 0;  // which of its bits are written: the same for the whole workgroup
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lower |= e >= first && e < past ? 15u << q4_bit(e) : 0u;
    upper |= 8 + e >= first && 8 + e < past ? 15u << q4_bit(e) : 0u;
  }
  const uint32_t mask = half ? upper : lower;
  uint32_t old = 0;
  if (mask != 0u && mask != 0xffffffffu) old = *at;
  if (live) q4_store_token<D>(kslab, vslab, i, c, kraw, vraw, &codes[i * ROW + c * 8]);
  __syncthreads();
  uint32_t w = 0;
  if (mask == 0xffffffffu) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= (uint32_t)codes[(8 * half + e) * ROW + dim] << q4_bit(e);
    *at = w;
  } else if (mask != 0u) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= (codes[(8 * half + e) * ROW + dim] & 15u) << q4_bit(e);  // (tokens not written: anything)
    *at = (old & ~mask) | (w & mask);
  }
}

// By slot: 16 consecutive tokens of the input, wherever their slots lie.  Tokens of one V dword may then sit in two workgroups; a
// dword not covered in full is changed by atomics on its own bits (each bit has one writer as long as no slot is named
// twice, so the order does not matter).
// 262144 tokens of 8 heads of 128 (1.4 GB) in order: 481 to 492 us, 2.9 TB/s; by position the same takes 364.  What it costs more is
// the V dwords, put together token by token although 16 tokens in order are two whole ones each; 1135 us while every thread
// looked for the dwords token by token in LDS.  In shuffled order, a dword of V changed by two atomics per token: 1393 us.
template <int D>
__global__ __launch_bounds__(2 * D) void q4_append_slots_kernel(pace_kv_pool_t pool, const uint16_t* __restrict__ k_new,
                                                                const uint16_t* __restrict__ v_new, int64_t sb, int64_t sh, int64_t st,
                                                                int32_t n_tokens, int32_t groups_x, const AppendDest dest) {
  constexpr int CHUNKS = D / 8, BT = PACE_KV_BLOCK_TOKENS, ROW = D + 8;
  __shared__ __attribute__((aligned(8))) uint8_t codes[BT * ROW];
  __shared__ int64_t slot_of[BT];  // the tokens' slots (-1: none)
  const uint32_t H = (uint32_t)pool.num_kv_heads;
  const int x = (int)(blockIdx.x % (uint32_t)groups_x), h = (int)(blockIdx.x / (uint32_t)groups_x % H);
  const int64_t b = blockIdx.x / (uint32_t)groups_x / H;
  const int i = threadIdx.x / CHUNKS, c = threadIdx.x % CHUNKS;
  const int64_t t = (int64_t)x * BT + i;
  int64_t slot = t < n_tokens ? dest.slots[b * n_tokens + t] : -1;
  if (slot < 0 || slot / BT >= pool.num_blocks) slot = -1;
  if (c == 0) slot_of[i] = slot;
  if (__syncthreads_or(slot >= 0) == 0) return;
  uint8_t* const k_head = static_cast<uint8_t*>(pool.k) + (int64_t)h * pool.k_head_stride;
  uint8_t* const v_head = static_cast<uint8_t*>(pool.v) + (int64_t)h * pool.v_head_stride;
  if (slot >= 0) {
    const int64_t src = b * sb + (int64_t)h * sh + t * st + c * 8;
    const u32x4 kraw = load16_stream(k_new + src), vraw = load16_stream(v_new + src);
    q4_store_token<D>(k_head + slot / BT * pool.k_block_stride, v_head + slot / BT * pool.v_block_stride, (int)(slot % BT), c, kraw, vraw,
                      &codes[i * ROW + c * 8]);
  }
  __syncthreads();
  // Every V dword a token of this workgroup lies in, at its first token here (every wave finds them by itself, lane a for token a);
  // the two thread halves take the dwords in turn.
  const int lane = threadIdx.x & 63;
  const int64_t mine = slot_of[lane & (BT - 1)] < 0 ? -1 : slot_of[lane & (BT - 1)] / 8;
  uint32_t same = 0;  // the tokens that share this one's dword
#pragma unroll
  for (int e = 0; e < BT; ++e) same |= (uint32_t)(__shfl(mine, e, 64) == mine) << e;
  const uint32_t firsts = (uint32_t)__ballot(lane < BT && mine >= 0 && (same & ((1u << lane) - 1u)) == 0u);
  const int half = threadIdx.x / D, r = threadIdx.x % D, dim = q4_v_dim<D>(r);
  int turn = 0;
  for (uint32_t left = firsts; left != 0u; left &= left - 1u) {  // uniform over the workgroup
    const int a = __builtin_ctz(left);
    const uint32_t tokens = __builtin_amdgcn_readlane(same, a);
    if ((turn++ & 1) != half) continue;
    const int64_t key = slot_of[a] / 8;
    uint32_t w = 0, mask = 0;
    for (uint32_t m = tokens; m != 0u; m &= m - 1u) {
      const int e = __builtin_ctz(m), bit = q4_bit((int)(slot_of[e] % 8));
      w = (w & ~(15u << bit)) | ((uint32_t)codes[e * ROW + dim] << bit);
      mask |= 15u << bit;
    }
    uint32_t* at = reinterpret_cast<uint32_t*>(v_head + key / 2 * pool.v_block_stride) + (key % 2) * D + r;
    if (mask == 0xffffffffu) {
      *at = w;
    } else {
      atomicAnd(at, ~mask);
      atomicOr(at, w);
    }
  }
}

// ---------------------------------------------------------------------------------
// Read back.  One workgroup of 2 D threads rebuilds one logical block (16 tokens) of one KV head as token rows: thread
// (token, chunk) makes eight dims of K from one code dword, and eight dims of V from the eight dwords its token has a
// code in, which pass through LDS.  64 sequences of 128 .. 8192 tokens, 8 heads of 128: 136 us for 700 MB, the 5.1 TB/s of a plain copy.
// ---------------------------------------------------------------------------------
// packed_entry() with the owner found by the lanes of a wave side by side: 64 sequences per memory round trip where the bisection
// takes one per step.  For grids that are on the GPU all at once, whose time is a chain of such trips (one read of 64
// short sequences, nothing of it in a cache: 8.4 us by bisection, 7.5 us this way; 5 sequences: 4.3 us either way); a long
// grid hides them and pays for the vector work (64 sequences of 128 .. 8192 tokens: 134 us by bisection, 158 us this way).
__device__ __forceinline__ void q4_packed_entry(const int32_t* __restrict__ cu, int batch, int H, unsigned entry, int lane, int& b, int& h, int& j) {
  for (int base = 0;; base += 64) {
    const int i = min(base + lane, batch - 1);
    const int from = cu[i], to = cu[i + 1];
    const uint64_t begun = __ballot(base + lane < batch && (int64_t)(from / PACE_KV_BLOCK_TOKENS + i) * H <= (int64_t)entry);
    if (begun == ~0ull && base + 64 < batch) {
      const int next = cu[base + 64];
      if ((int64_t)(next / PACE_KV_BLOCK_TOKENS + base + 64) * H <= (int64_t)entry) continue;  // uniform: the same for every lane
    }
    const int l = 63 - __builtin_clzll(begun);  // sequence `base` has begun: bit 0 is set
    b = base + l;
    const int first = __builtin_amdgcn_readlane(from, l) / PACE_KV_BLOCK_TOKENS + b;
    const int n = __builtin_amdgcn_readlane(to, l) / PACE_KV_BLOCK_TOKENS + b + 1 - first;  // >= 1
    const int r = (int)((int64_t)entry - (int64_t)first * H);
    h = min(r / n, H - 1), j = r % n;
    return;
  }
}

template <int D, bool PACKED>
__global__ __launch_bounds__(2 * D) void q4_gather_kernel(pace_kv_pool_t pool, const int32_t* __restrict__ table, int32_t table_stride,
                                                          const int32_t* __restrict__ seq_lens, int32_t len_bias, int32_t n_rep,
                                                          int32_t n_blocks, int32_t side_by_side, const GatherOut out) {
  using L = Q4<D>;
  constexpr int CHUNKS = D / 8, BT = PACE_KV_BLOCK_TOKENS;
  __shared__ uint32_t vc[2 * D];
  int j, b, h;
  if (PACKED) {
    if (side_by_side) q4_packed_entry(out.cu_seqlens, out.batch, pool.num_kv_heads, blockIdx.x, threadIdx.x & 63, b, h, j);
    else packed_entry(out.cu_seqlens, out.batch, pool.num_kv_heads, blockIdx.x, b, h, j);
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
  const uint16_t* k = static_cast<const uint16_t*>(k_new);
  const uint16_t* v = static_cast<const uint16_t*>(v_new);
  const int64_t rows = (int64_t)pool->num_kv_heads * batch;
  // the most blocks n_tokens consecutive positions can touch; by slot: runs of 16 input tokens
  const int64_t blocks = paged ? ((int64_t)n_tokens + PACE_KV_BLOCK_TOKENS - 2) / PACE_KV_BLOCK_TOKENS + 1
                               : ((int64_t)n_tokens + PACE_KV_BLOCK_TOKENS - 1) / PACE_KV_BLOCK_TOKENS;
  const int64_t grid = blocks * rows;
  PACE_REQUIRE(grid < (int64_t)1 << 31, "%s: grid too large", who);
  for_head_dim(pool->head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (paged)
      hipLaunchKernelGGL((q4_append_paged_kernel<D>), dim3((unsigned)grid), dim3(2 * D), 0, stream, *pool, k, v, stride_b, stride_h, stride_t,
                         n_tokens, (int32_t)blocks, dest);
    else
      hipLaunchKernelGGL((q4_append_slots_kernel<D>), dim3((unsigned)grid), dim3(2 * D), 0, stream, *pool, k, v, stride_b, stride_h, stride_t,
                         n_tokens, (int32_t)blocks, dest);
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
  const int32_t side_by_side = grid <= 8 * (int64_t)compute_units() ? 1 : 0;
  for_head_dim(pool->head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (packed)
      hipLaunchKernelGGL((q4_gather_kernel<D, true>), dim3((unsigned)grid), dim3(2 * D), 0, stream, *pool, block_table, table_stride, seq_lens,
                         seq_len_bias, n_rep, (int32_t)n_blocks, side_by_side, out);
    else
      hipLaunchKernelGGL((q4_gather_kernel<D, false>), dim3((unsigned)grid), dim3(2 * D), 0, stream, *pool, block_table, table_stride, seq_lens,
                         seq_len_bias, n_rep, (int32_t)n_blocks, side_by_side, out);
  });
  PACE_HIP_CHECK(hipGetLastError());
  return PACE_KV_OK;
}

}  // namespace pace_kv
