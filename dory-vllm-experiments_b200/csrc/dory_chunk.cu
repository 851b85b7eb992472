// dory_chunk.cu — attention of a chunk of new tokens over the paged cache
// (dory_chunk_attention; the C ABI is in include/dory_decode.h).
//
// chunk_rows: one warp per (token, head) row.  Lanes take 32 positions at a time for the scores
// (q from shared memory), then HD / 32 dims each for the weighted sum, with a running maximum
// and sum.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <string.h>

#include "dory_common.h"

namespace {

using dory::aligned16;
using dory::fail;

constexpr float kLog2e = 1.4426950408889634f;

struct ChunkArgs {
  const __nv_bfloat16* q;
  const void* kc;
  const void* vc;
  const int32_t* tables;
  const int32_t* query_start;
  const int32_t* seq_lens;
  const void* gate;
  __nv_bfloat16* out;
  uint32_t* err;
  int64_t q_t, q_h, out_t, gate_t, table_stride, sb, so, sh, blocks;
  float scale_log2, k_scale, v_scale;
  int T, S, max_blocks, NH, NKV, G, B, window, gate_dtype;
};

__device__ __forceinline__ float load_gate(const ChunkArgs& a, int64_t i) {
  if (a.gate_dtype == DORY_DTYPE_F32) return static_cast<const float*>(a.gate)[i];
  if (a.gate_dtype == DORY_DTYPE_BF16)
    return __bfloat162float(static_cast<const __nv_bfloat16*>(a.gate)[i]);
  return __half2float(static_cast<const __half*>(a.gate)[i]);
}

__device__ __forceinline__ float e4m3_to_f32(uint8_t b) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(b)));
  return __half2float(__ushort_as_half(static_cast<unsigned short>(h)));
}
template <bool KV8>
__device__ __forceinline__ float cache_value(const void* p, int64_t i) {
  if (KV8) return e4m3_to_f32(static_cast<const uint8_t*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// Rows [t0, t1) of sequence i, whatever the arrays hold: always within [0, T].
__device__ __forceinline__ void rows_of(const ChunkArgs& a, int i, int& t0, int& t1) {
  t0 = min(max(a.query_start[i], 0), a.T);
  t1 = min(max(a.query_start[i + 1], t0), a.T);
}

// The block of a sequence that holds position c, or -1 (reported) outside the cache.
__device__ __forceinline__ int64_t block_of(const ChunkArgs& a, const int32_t* table, int c) {
  const int b = c / a.B;
  const int64_t id = b < a.max_blocks ? table[b] : -1;
  if (id < 0 || id >= a.blocks) {
    atomicOr(a.err, DORY_DEVERR_BLOCK_OOB);
    return -1;
  }
  return id;
}

template <int HD, bool KV8>
__global__ void __launch_bounds__(128) chunk_rows(const ChunkArgs a) {
  __shared__ float sq[4][HD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x, h = blockIdx.y * 4 + warp;
  if (h >= a.NH) return;
  // the row's sequence: the last one that starts at or before it and is not empty
  int seq = -1, t0 = 0, t1 = 0;
  for (int i = 0; i < a.S; ++i) {
    int u0, u1;
    rows_of(a, i, u0, u1);
    if (u0 <= t && t < u1) {
      seq = i;
      t0 = u0;
      t1 = u1;
      break;
    }
  }
  if (seq < 0) return;
  for (int i = lane; i < HD; i += 32)
    sq[warp][i] = __bfloat162float(a.q[t * a.q_t + h * a.q_h + i]);
  __syncwarp();
  const int p = a.seq_lens[seq] - (t1 - t0) + (t - t0);
  const int lo = a.window ? max(0, p + 1 - a.window) : 0;
  const int32_t* table = a.tables + int64_t(seq) * a.table_stride;
  const int64_t head = int64_t(h / a.G) * a.sh;
  float m = -INFINITY, l = 0.0f, acc[HD / 32];
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) acc[i] = 0.0f;
  const float qk = a.scale_log2 * (KV8 ? a.k_scale : 1.0f);
  for (int c0 = lo; c0 <= p; c0 += 32) {
    const int c = c0 + lane;
    float s = -INFINITY;
    int64_t at = -1;
    if (c <= p) {
      const int64_t id = block_of(a, table, c);
      if (id >= 0) {
        at = id * a.sb + int64_t(c % a.B) * a.so + head;
        float dot = 0.0f;
        for (int i = 0; i < HD; ++i) dot += sq[warp][i] * cache_value<KV8>(a.kc, at + i);
        s = dot * qk;
      }
    }
    float top = s;
    for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    const float m_new = fmaxf(m, top), base = m_new == -INFINITY ? 0.0f : m_new;
    const float w = exp2f(s - base), shrink = exp2f(m - base);
    m = m_new;
    l = l * shrink + w;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) acc[i] *= shrink;
    for (int k = 0; k < 32; ++k) {
      const int64_t row = __shfl_sync(0xffffffffu, at, k);
      const float wk = __shfl_sync(0xffffffffu, w, k);
      if (row < 0) continue;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) acc[i] += wk * cache_value<KV8>(a.vc, row + lane + 32 * i);
    }
  }
  for (int k = 16; k; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
  const float inv = l > 0.0f ? (KV8 ? a.v_scale : 1.0f) / l : (l == 0.0f ? 0.0f : l);
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) {
    const int e = h * HD + lane + 32 * i;
    float y = acc[i] * inv;
    if (a.gate) y *= load_gate(a, t * a.gate_t + e);
    a.out[t * a.out_t + e] = __float2bfloat16_rn(y);
  }
}

}  // namespace

extern "C" {

int64_t dory_chunk_params_bytes(void) { return int64_t(sizeof(DoryChunkParams)); }

int64_t dory_chunk_scratch_bytes(int32_t num_heads, int32_t num_kv_heads, int32_t head_dim) {
  if (num_heads < 1 || num_kv_heads < 1 || num_heads % num_kv_heads ||
      num_heads / num_kv_heads > 64 || (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return 0;
  return 256;
}

int32_t dory_chunk_attention(const DoryChunkParams* P, void* stream) {
  if (!P) return fail(DORY_ERR_INVALID_ARGUMENT, "null params");
  const DoryChunkParams& p = *P;
  if (p.num_heads < 1 || p.num_kv_heads < 1 || p.num_heads % p.num_kv_heads)
    return fail(DORY_ERR_INVALID_ARGUMENT, "query heads must be a multiple of KV heads");
  if (p.num_tokens < 0 || p.num_seqs < 0)
    return fail(DORY_ERR_INVALID_ARGUMENT, "negative token or sequence count");
  if (p.window < 0) return fail(DORY_ERR_INVALID_ARGUMENT, "negative window");
  const int G = p.num_heads / p.num_kv_heads;
  if (G > 64) return fail(DORY_ERR_UNSUPPORTED, "%d query heads per KV head (max 64)", G);
  if (p.head_dim != 64 && p.head_dim != 128 && p.head_dim != 256)
    return fail(DORY_ERR_UNSUPPORTED, "head_dim %d (supported: 64, 128, 256)", p.head_dim);
  if (p.block_size < 16 || p.block_size % 16)
    return fail(DORY_ERR_UNSUPPORTED, "block_size %d is not a multiple of 16", p.block_size);
  if (p.kv_dtype != 0 && p.kv_dtype != DORY_DTYPE_BF16 && p.kv_dtype != DORY_DTYPE_FP8_E4M3)
    return fail(DORY_ERR_INVALID_ARGUMENT, "kv_dtype %d (bf16 or fp8 e4m3)", p.kv_dtype);
  const bool kv8 = p.kv_dtype == DORY_DTYPE_FP8_E4M3;
  if (kv8 && p.head_dim == 64)
    return fail(DORY_ERR_UNSUPPORTED, "FP8 caches take 128/256-dim heads");
  if (kv8 && !(p.k_scale > 0.0f && p.v_scale > 0.0f && p.k_scale < 3.4e38f && p.v_scale < 3.4e38f))
    return fail(DORY_ERR_INVALID_ARGUMENT, "FP8 caches need positive, finite k/v scales");
  if (!(p.softmax_scale > 0.0f && p.softmax_scale < 3.4e38f))
    return fail(DORY_ERR_INVALID_ARGUMENT, "softmax_scale must be positive and finite");
  if (p.gate && (p.gate_dtype < 0 || p.gate_dtype > 2))
    return fail(DORY_ERR_INVALID_ARGUMENT, "gate dtype");
  if (p.num_tokens == 0 || p.num_seqs == 0) return DORY_OK;  // nothing is read or written
  if (p.num_cache_blocks < 1 || p.max_blocks < 1)
    return fail(DORY_ERR_INVALID_ARGUMENT, "the cache and the block tables must not be empty");
  if (!p.q || !p.key_cache || !p.value_cache || !p.block_tables || !p.query_start ||
      !p.seq_lens || !p.out || !p.scratch)
    return fail(DORY_ERR_INVALID_ARGUMENT, "null tensor argument");
  const int64_t cache_mask = kv8 ? 15 : 7;
  if (!aligned16(p.q) || !aligned16(p.out) || ((p.q_stride_token | p.q_stride_head) & 7) ||
      (p.out_stride_token & 7))
    return fail(DORY_ERR_ALIGNMENT, "q and out need 16-byte aligned bases and rows");
  if (!aligned16(p.key_cache) || !aligned16(p.value_cache) ||
      ((p.stride_block | p.stride_offset | p.stride_head) & cache_mask))
    return fail(DORY_ERR_ALIGNMENT, "key/value caches need 16-byte aligned bases and strides");
  if (p.gate && (!aligned16(p.gate) || (p.gate_stride_token & 7)))
    return fail(DORY_ERR_ALIGNMENT, "gate needs a 16-byte aligned base and rows");
  const int64_t need = dory_chunk_scratch_bytes(p.num_heads, p.num_kv_heads, p.head_dim);
  if (p.scratch_bytes < need)
    return fail(DORY_ERR_INVALID_ARGUMENT, "scratch too small (%lld < %lld bytes)",
                (long long)p.scratch_bytes, (long long)need);

  ChunkArgs a;
  memset(&a, 0, sizeof(a));
  a.q = static_cast<const __nv_bfloat16*>(p.q);
  a.kc = p.key_cache;
  a.vc = p.value_cache;
  a.tables = p.block_tables;
  a.query_start = p.query_start;
  a.seq_lens = p.seq_lens;
  a.gate = p.gate;
  a.out = static_cast<__nv_bfloat16*>(p.out);
  a.err = static_cast<uint32_t*>(p.scratch);
  a.q_t = p.q_stride_token;
  a.q_h = p.q_stride_head;
  a.out_t = p.out_stride_token;
  a.gate_t = p.gate_stride_token;
  a.table_stride = p.table_stride;
  a.sb = p.stride_block;
  a.so = p.stride_offset;
  a.sh = p.stride_head;
  a.blocks = p.num_cache_blocks;
  a.scale_log2 = p.softmax_scale * kLog2e;
  a.k_scale = p.k_scale;
  a.v_scale = p.v_scale;
  a.T = p.num_tokens;
  a.S = p.num_seqs;
  a.max_blocks = p.max_blocks;
  a.NH = p.num_heads;
  a.NKV = p.num_kv_heads;
  a.G = G;
  a.B = p.block_size;
  a.window = p.window;
  a.gate_dtype = p.gate_dtype;
  const dim3 grid(p.num_tokens, (p.num_heads + 3) / 4);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (kv8) {
    if (p.head_dim == 128) chunk_rows<128, true><<<grid, 128, 0, s>>>(a);
    else chunk_rows<256, true><<<grid, 128, 0, s>>>(a);
  } else if (p.head_dim == 64) chunk_rows<64, false><<<grid, 128, 0, s>>>(a);
  else if (p.head_dim == 128) chunk_rows<128, false><<<grid, 128, 0, s>>>(a);
  else chunk_rows<256, false><<<grid, 128, 0, s>>>(a);
  return dory::launched(cudaSuccess);
}

}  // extern "C"
