// dory_rotary.cu — rotary positions (dory_rotary_embed) and the rotated, normalised append of
// new keys and values to the paged cache (dory_rotary_append); the C ABI is in
// include/dory_decode.h.
//
// Both read every input once and write every output once, with a handful of operations per
// element: HBM bounds a long prompt, the launch and two dependent loads (position, then
// table row) a single token.
//
// rotary_vec: a head's row belongs to head_dim / 16 neighbouring lanes.  Lane l holds two
// 8-element pieces that contain both members of its pairs: dims 8l and rotary_dim / 2 + 8l of
// the half layout, 16l and 16l + 8 of the interleaved one, so in both it needs the angles 8l ..
// 8l + 7 and no exchange between lanes (the norm alone takes log2(head_dim / 16) shuffles).  A
// lane keeps its angles in registers and uses them for up to kHeads heads of its token, whose
// loads are all in flight together.
// rotary_any: one warp per row, a pair per lane, for every size, stride and alignment.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <string.h>

#include "dory_common.h"

namespace {

using dory::aligned16;
using dory::fail;

struct Rows {  // one of q, k, v or an output
  const void* in;
  void* out;
  int64_t in_t, in_h, out_t, out_h;  // strides in elements
};

struct RotaryArgs {
  Rows q, k, v;
  const void* positions;
  const void* cos_sin;
  const void* sqk;
  const int64_t* slots;
  uint8_t* kc;
  uint8_t* vc;
  uint32_t* err;
  int64_t sb, so, sh, cache_slots, max_position;
  float sqk_factor, eps, k_scale, v_scale;
  int T, NH, NKV, D, R, B, heads, groups;  // heads: rows of a token; groups: head groups
  int cs_dtype, pos32, sqk_dtype, inter, norm;
  float sign;
};

// ---- element types ----
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <> __device__ __forceinline__ __half from_f32<__half>(float x) {
  return __float2half_rn(x);
}
__device__ __forceinline__ float load_as_f32(const void* p, int64_t i, int dtype) {
  if (dtype == DORY_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == DORY_DTYPE_BF16) return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_f32(static_cast<const __half*>(p)[i]);
}

// Eight consecutive elements as they lie in memory.
template <typename T> struct Piece { uint4 w[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(const T* p) {
  Piece<T> r;
#pragma unroll
  for (int i = 0; i < int(sizeof(T) / 2); ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack(const Piece<T>& p, float (&x)[8]) {
  T e[8];
  memcpy(e, &p, sizeof(p));
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
}
template <typename T>
__device__ __forceinline__ void store_piece(T* p, const float (&x)[8]) {
  T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
  Piece<T> r;
  memcpy(&r, e, sizeof(r));
#pragma unroll
  for (int i = 0; i < int(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
}
__device__ __forceinline__ void load8(const void* p, int64_t at, int dtype, float (&x)[8]) {
  if (dtype == DORY_DTYPE_F32) unpack(load_piece(static_cast<const float*>(p) + at), x);
  else if (dtype == DORY_DTYPE_BF16)
    unpack(load_piece(static_cast<const __nv_bfloat16*>(p) + at), x);
  else unpack(load_piece(static_cast<const __half*>(p) + at), x);
}

// Two values as the e4m3 bytes a cache of scale `scale` holds: rounded to bf16 first (the
// value a bf16 cache would hold, and the one the decode kernel quantises), divided in FP32,
// then rounded to nearest even and saturated.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi, float scale) {
  lo = __bfloat162float(__float2bfloat16_rn(lo)) / scale;
  hi = __bfloat162float(__float2bfloat16_rn(hi)) / scale;
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ int64_t position_of(const RotaryArgs& a, int t) {
  return a.pos32 ? static_cast<const int32_t*>(a.positions)[t]
                 : static_cast<const int64_t*>(a.positions)[t];
}
__device__ __forceinline__ void report(const RotaryArgs& a, uint32_t bit) {
  if (a.err) atomicOr(a.err, bit);
}
// Byte address of a cache row (K or V head g) of `slot`; elements of `esize` bytes.
__device__ __forceinline__ uint8_t* cache_row(const RotaryArgs& a, uint8_t* base, int64_t slot,
                                              int g, int esize) {
  const int64_t block = slot < INT32_MAX ? uint32_t(slot) / uint32_t(a.B) : slot / a.B;
  return base + (block * a.sb + (slot - block * a.B) * a.so + int64_t(g) * a.sh) * esize;
}

// Row h of a token: 0 .. NH-1 q, then k heads, then (append) v heads.
template <typename T>
__device__ __forceinline__ const T* row_in(const RotaryArgs& a, int t, int h) {
  if (h < a.NH) return static_cast<const T*>(a.q.in) + t * a.q.in_t + h * a.q.in_h;
  h -= a.NH;
  if (h < a.NKV) return static_cast<const T*>(a.k.in) + t * a.k.in_t + h * a.k.in_h;
  return static_cast<const T*>(a.v.in) + t * a.v.in_t + (h - a.NKV) * a.v.in_h;
}

// ------------------------------------------------------------------------------------
// kHeads: heads a lane takes.  8 for long prompts would need more registers than it hides
// latency; 1 spreads a few tokens over as many lanes as there are.
template <typename T, bool APPEND, bool KV8, int kHeads>
__global__ void __launch_bounds__(256) rotary_vec(const RotaryArgs a) {
  const int lanes = a.D / 16;
  const int rows = 256 / lanes;
  const int local = threadIdx.x / lanes, l = threadIdx.x - local * lanes;
  const int64_t row = int64_t(blockIdx.x) * rows + local;
  const bool live = local < rows && row < int64_t(a.T) * a.groups;
  const int t = live ? int(row / a.groups) : 0;
  const int h0 = live ? int(row - int64_t(t) * a.groups) : a.heads;

  const bool turn = l < a.R / 16;
  const bool apart = turn && !a.inter;
  const int oa = apart ? 8 * l : 16 * l, ob = apart ? a.R / 2 + 8 * l : 16 * l + 8;
  Piece<T> xa[kHeads], xb[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = h0 + i * a.groups;
    if (h < a.heads) {
      const T* p = row_in<T>(a, t, h);
      xa[i] = load_piece(p + oa);
      xb[i] = load_piece(p + ob);
    }
  }
  float c[8], s[8];
  bool inside = true;
  int64_t slot = -1;
  if (live) {
    if (APPEND) slot = a.slots[t];
    if (a.R > 0) {
      const int64_t pos = position_of(a, t);
      inside = pos >= 0 && pos < a.max_position;
      if (turn && inside) {
        load8(a.cos_sin, pos * a.R + 8 * l, a.cs_dtype, c);
        load8(a.cos_sin, pos * a.R + a.R / 2 + 8 * l, a.cs_dtype, s);
      }
      if (!inside && h0 == 0 && l == 0 && !(APPEND && slot < 0))
        report(a, DORY_DEVERR_POSITION_OOB);
    }
    if (APPEND && slot >= a.cache_slots) {
      if (h0 == 0 && l == 0) report(a, DORY_DEVERR_SLOT_OOB);
      slot = -1;
    }
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = h0 + i * a.groups;
    const bool here = h < a.heads, is_v = APPEND && h >= a.NH + a.NKV;
    float ya[8], yb[8];
    if (here) {
      unpack(xa[i], ya);
      unpack(xb[i], yb);
      if (!is_v && !inside) {
#pragma unroll
        for (int j = 0; j < 8; ++j) ya[j] = yb[j] = 0.0f;
      } else if (!is_v && turn) {
        if (a.inter) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float a0 = ya[2 * j], a1 = ya[2 * j + 1], b0 = yb[2 * j], b1 = yb[2 * j + 1];
            const float sa = a.sign * s[j], sb = a.sign * s[4 + j];
            ya[2 * j] = a0 * c[j] - a1 * sa;
            ya[2 * j + 1] = a1 * c[j] + a0 * sa;
            yb[2 * j] = b0 * c[4 + j] - b1 * sb;
            yb[2 * j + 1] = b1 * c[4 + j] + b0 * sb;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float x = ya[j], y = yb[j], sj = a.sign * s[j];
            ya[j] = x * c[j] - y * sj;
            yb[j] = y * c[j] + x * sj;
          }
        }
      }
    }
    if constexpr (APPEND) {
      if (a.norm) {  // every lane of the warp takes part: rows never straddle a warp
        float sum = 0.0f;
        if (here && !is_v) {
#pragma unroll
          for (int j = 0; j < 8; ++j) sum += ya[j] * ya[j] + yb[j] * yb[j];
        }
        for (int m = lanes >> 1; m; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
        if (here && !is_v) {
          const float inv = rsqrtf(sum + a.eps);
          float wa[8], wb[8];
          if (h < a.NH) {
            load8(a.sqk, int64_t(h) * a.D + oa, a.sqk_dtype, wa);
            load8(a.sqk, int64_t(h) * a.D + ob, a.sqk_dtype, wb);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float fa = inv, fb = inv;
            if (h < a.NH) {
              const float u = wa[j] * a.sqk_factor, w = wb[j] * a.sqk_factor;
              fa *= u * u;
              fb *= w * w;
            }
            ya[j] *= fa;
            yb[j] *= fb;
          }
        }
      }
    }
    if (!here) continue;
    if (h < a.NH) {
      if constexpr (APPEND) {
        __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.q.out) + t * a.q.out_t + h * a.q.out_h;
        store_piece(o + oa, ya);
        store_piece(o + ob, yb);
      } else {
        T* o = static_cast<T*>(a.q.out) + t * a.q.out_t + h * a.q.out_h;
        store_piece(o + oa, ya);
        store_piece(o + ob, yb);
      }
    } else if constexpr (!APPEND) {
      T* o = static_cast<T*>(a.k.out) + t * a.k.out_t + (h - a.NH) * a.k.out_h;
      store_piece(o + oa, ya);
      store_piece(o + ob, yb);
    } else if (slot >= 0) {
      const int g = is_v ? h - a.NH - a.NKV : h - a.NH;
      uint8_t* o = cache_row(a, is_v ? a.vc : a.kc, slot, g, KV8 ? 1 : 2);
      if constexpr (KV8) {
        const float scale = is_v ? a.v_scale : a.k_scale;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float(&y)[8] = half ? yb : ya;
          uint2 w;
          w.x = to_e4m3x2(y[0], y[1], scale) | to_e4m3x2(y[2], y[3], scale) << 16;
          w.y = to_e4m3x2(y[4], y[5], scale) | to_e4m3x2(y[6], y[7], scale) << 16;
          *reinterpret_cast<uint2*>(o + (half ? ob : oa)) = w;
        }
      } else {
        __nv_bfloat16* b = reinterpret_cast<__nv_bfloat16*>(o);
        store_piece(b + oa, ya);
        store_piece(b + ob, yb);
      }
    }
  }
}

// ------------------------------------------------------------------------------------
// The rotated element i of a row.
template <typename T>
__device__ __forceinline__ float turned(const RotaryArgs& a, const T* x, int i, int64_t pos) {
  if (i >= a.R) return to_f32(x[i]);
  const int half = a.R / 2;
  const int pair = a.inter ? i / 2 : (i < half ? i : i - half);
  const bool first = a.inter ? (i & 1) == 0 : i < half;
  const int i0 = a.inter ? 2 * pair : pair, i1 = a.inter ? 2 * pair + 1 : pair + half;
  const float c = load_as_f32(a.cos_sin, pos * a.R + pair, a.cs_dtype);
  const float s = a.sign * load_as_f32(a.cos_sin, pos * a.R + half + pair, a.cs_dtype);
  return first ? to_f32(x[i0]) * c - to_f32(x[i1]) * s : to_f32(x[i1]) * c + to_f32(x[i0]) * s;
}

template <typename T, bool APPEND, bool KV8>
__global__ void __launch_bounds__(128) rotary_any(const RotaryArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= int64_t(a.T) * a.heads) return;  // a whole warp
  const int t = int(row / a.heads), h = int(row - int64_t(t) * a.heads);
  const bool is_v = APPEND && h >= a.NH + a.NKV;
  const T* x = row_in<T>(a, t, h);
  int64_t pos = 0;
  bool inside = true;
  if (a.R > 0 && !is_v) {
    pos = position_of(a, t);
    inside = pos >= 0 && pos < a.max_position;
    if (!inside && h == 0 && lane == 0 && !(APPEND && a.slots[t] < 0))
      report(a, DORY_DEVERR_POSITION_OOB);
  }
  if constexpr (!APPEND) {
    T* o = h < a.NH ? static_cast<T*>(a.q.out) + t * a.q.out_t + h * a.q.out_h
                    : static_cast<T*>(a.k.out) + t * a.k.out_t + (h - a.NH) * a.k.out_h;
    const int half = a.R / 2;
    for (int pair = lane; pair < half; pair += 32) {  // both members by one lane: in place is fine
      const int i0 = a.inter ? 2 * pair : pair, i1 = a.inter ? 2 * pair + 1 : pair + half;
      const float y0 = inside ? turned(a, x, i0, pos) : 0.0f;
      const float y1 = inside ? turned(a, x, i1, pos) : 0.0f;
      o[i0] = from_f32<T>(y0);
      o[i1] = from_f32<T>(y1);
    }
    for (int i = a.R + lane; i < a.D; i += 32)
      o[i] = inside ? x[i] : from_f32<T>(0.0f);
  } else {
    int64_t slot = a.slots[t];
    if (slot >= a.cache_slots) {
      if (h == 0 && lane == 0) report(a, DORY_DEVERR_SLOT_OOB);
      slot = -1;
    }
    float inv = 1.0f;
    if (a.norm && !is_v) {
      float sum = 0.0f;
      for (int i = lane; i < a.D; i += 32) {
        const float y = inside ? turned(a, x, i, pos) : 0.0f;
        sum += y * y;
      }
      for (int m = 16; m; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
      inv = rsqrtf(sum + a.eps);
    }
    if (h >= a.NH && slot < 0) return;
    const int g = is_v ? h - a.NH - a.NKV : h - a.NH;
    uint8_t* row_out = h < a.NH ? nullptr : cache_row(a, is_v ? a.vc : a.kc, slot, g, KV8 ? 1 : 2);
    for (int i = lane; i < a.D; i += 32) {
      float y = is_v ? to_f32(x[i]) : inside ? turned(a, x, i, pos) : 0.0f;
      if (a.norm && !is_v) {
        float f = inv;
        if (h < a.NH) {
          const float u = load_as_f32(a.sqk, int64_t(h) * a.D + i, a.sqk_dtype) * a.sqk_factor;
          f *= u * u;
        }
        y *= f;
      }
      if (h < a.NH)
        (static_cast<__nv_bfloat16*>(a.q.out) + t * a.q.out_t + h * a.q.out_h)[i] =
            from_f32<__nv_bfloat16>(y);
      else if (KV8)
        row_out[i] = uint8_t(to_e4m3x2(y, 0.0f, is_v ? a.v_scale : a.k_scale));
      else
        reinterpret_cast<__nv_bfloat16*>(row_out)[i] = from_f32<__nv_bfloat16>(y);
    }
  }
}

// ------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------
template <typename T, bool APPEND, bool KV8>
int32_t run(RotaryArgs& a, bool pieces, cudaStream_t stream) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.stream = stream;
  if (!pieces) {
    const int64_t blocks = (int64_t(a.T) * a.heads + 3) / 4;
    if (blocks > INT32_MAX) return fail(DORY_ERR_UNSUPPORTED, "too many tokens for one launch");
    cfg.gridDim = dim3(unsigned(blocks));
    cfg.blockDim = dim3(128);
    return dory::launched(cudaLaunchKernelEx(&cfg, rotary_any<T, APPEND, KV8>, a));
  }
  const int lanes = a.D / 16, rows = 256 / lanes;
  constexpr int kMany = 4;
  // One head a lane until that fills the machine about once (148 SMs x 2,048 threads); then
  // kMany, which share their angles.
  const int per_lane = int64_t(a.T) * a.heads * lanes > 148 * 2048 ? kMany : 1;
  a.groups = (a.heads + per_lane - 1) / per_lane;
  const int64_t blocks = (int64_t(a.T) * a.groups + rows - 1) / rows;
  if (blocks > INT32_MAX) return fail(DORY_ERR_UNSUPPORTED, "too many tokens for one launch");
  cfg.gridDim = dim3(unsigned(blocks));
  cfg.blockDim = dim3(256);
  return dory::launched(
      per_lane == 1 ? cudaLaunchKernelEx(&cfg, rotary_vec<T, APPEND, KV8, 1>, a)
                    : cudaLaunchKernelEx(&cfg, rotary_vec<T, APPEND, KV8, kMany>, a));
}

template <bool APPEND, bool KV8>
int32_t run_type(RotaryArgs& a, int dtype, bool pieces, cudaStream_t stream) {
  if (dtype == DORY_DTYPE_F32) return run<float, APPEND, KV8>(a, pieces, stream);
  if (dtype == DORY_DTYPE_BF16) return run<__nv_bfloat16, APPEND, KV8>(a, pieces, stream);
  return run<__half, APPEND, KV8>(a, pieces, stream);
}

int32_t rotary(const DoryRotaryParams* P, bool append, void* stream) {
  if (!P) return fail(DORY_ERR_INVALID_ARGUMENT, "null params");
  const DoryRotaryParams& p = *P;
  const bool norm = p.flags & DORY_ROTARY_NORM;
  const bool has_q = !append || p.q || p.q_out;
  const bool has_k = append || p.k || p.k_out;
  if (p.num_tokens < 0 || (has_q && p.num_heads < 1) || (has_k && p.num_kv_heads < 1))
    return fail(DORY_ERR_INVALID_ARGUMENT, "token and head counts must be positive");
  if (append ? (p.head_dim != 64 && p.head_dim != 128 && p.head_dim != 256)
             : (p.head_dim < 1 || p.head_dim > 1024))
    return fail(DORY_ERR_UNSUPPORTED, "head_dim %d (supported: %s)", p.head_dim,
                append ? "64, 128, 256" : "1 to 1024");
  if (p.rotary_dim < (append ? 0 : 2) || (p.rotary_dim & 1) || p.rotary_dim > p.head_dim)
    return fail(DORY_ERR_INVALID_ARGUMENT, "rotary_dim %d must be even and at most head_dim %d",
                p.rotary_dim, p.head_dim);
  if (p.io_dtype < 0 || p.io_dtype > 2 || p.cos_sin_dtype < 0 || p.cos_sin_dtype > 2 ||
      p.positions_dtype < 0 || p.positions_dtype > 1 || p.sqk_dtype < 0 || p.sqk_dtype > 2)
    return fail(DORY_ERR_INVALID_ARGUMENT, "q / k / v, cos_sin, positions or sqk dtype");
  if (p.rotary_dim && p.max_position < 1)
    return fail(DORY_ERR_INVALID_ARGUMENT, "max_position must be positive");
  const bool kv8 = p.kv_dtype == DORY_DTYPE_FP8_E4M3;
  if (append) {
    if (p.kv_dtype != 0 && p.kv_dtype != DORY_DTYPE_BF16 && !kv8)
      return fail(DORY_ERR_INVALID_ARGUMENT, "kv_dtype %d (bf16 or fp8 e4m3)", p.kv_dtype);
    if (kv8 && !(p.k_scale > 0.0f && p.v_scale > 0.0f && p.k_scale < 3.4e38f &&
                 p.v_scale < 3.4e38f))
      return fail(DORY_ERR_INVALID_ARGUMENT, "FP8 caches need positive, finite k/v scales");
    if (p.block_size < 1 || p.num_cache_blocks < 1)
      return fail(DORY_ERR_INVALID_ARGUMENT, "the cache needs at least one block");
    if (p.flags & DORY_ROTARY_INVERSE)
      return fail(DORY_ERR_INVALID_ARGUMENT, "the append rotates forwards only");
  } else if (norm) {
    return fail(DORY_ERR_INVALID_ARGUMENT, "the normalisation belongs to the append");
  }
  if (p.num_tokens == 0) return DORY_OK;  // nothing is read: empty tensors may be NULL
  if ((has_q && (!p.q || !p.q_out)) || (has_k && !p.k) || (append && !p.v) ||
      (!append && has_k && !p.k_out) || (p.rotary_dim && (!p.positions || !p.cos_sin)) ||
      (append && (!p.slot_mapping || !p.key_cache || !p.value_cache)) ||
      (norm && has_q && !p.sqk))
    return fail(DORY_ERR_INVALID_ARGUMENT, "null tensor argument");

  RotaryArgs a;
  memset(&a, 0, sizeof(a));
  a.q = Rows{p.q, p.q_out, p.q_stride_token, p.q_stride_head, p.q_out_stride_token,
             p.q_out_stride_head};
  a.k = Rows{p.k, p.k_out, p.k_stride_token, p.k_stride_head, p.k_out_stride_token,
             p.k_out_stride_head};
  a.v = Rows{p.v, nullptr, p.v_stride_token, p.v_stride_head, 0, 0};
  a.positions = p.positions;
  a.cos_sin = p.cos_sin;
  a.sqk = p.sqk;
  a.slots = p.slot_mapping;
  a.kc = static_cast<uint8_t*>(p.key_cache);
  a.vc = static_cast<uint8_t*>(p.value_cache);
  a.err = p.error_word;
  a.sb = p.stride_block;
  a.so = p.stride_offset;
  a.sh = p.stride_head;
  a.cache_slots = append ? p.num_cache_blocks * p.block_size : 0;
  a.max_position = p.max_position;
  a.sqk_factor = p.sqk_factor;
  a.eps = p.eps;
  a.k_scale = p.k_scale;
  a.v_scale = p.v_scale;
  a.T = p.num_tokens;
  a.NH = has_q ? p.num_heads : 0;
  a.NKV = has_k ? p.num_kv_heads : 0;
  a.D = p.head_dim;
  a.R = p.rotary_dim;
  a.B = p.block_size;
  a.heads = a.NH + (append ? 2 : 1) * a.NKV;
  a.groups = a.heads;
  a.cs_dtype = p.cos_sin_dtype;
  a.pos32 = p.positions_dtype;
  a.sqk_dtype = p.sqk_dtype;
  a.inter = p.flags & DORY_ROTARY_INTERLEAVED ? 1 : 0;
  a.norm = norm;
  a.sign = p.flags & DORY_ROTARY_INVERSE ? -1.0f : 1.0f;

  // The 16-byte pieces need whole pieces and aligned rows everywhere; a lane needs 16 dims.
  const int64_t mask = p.io_dtype == DORY_DTYPE_F32 ? 3 : 7;
  bool pieces = p.head_dim % 16 == 0 && p.rotary_dim % 16 == 0;
  auto fits = [&](const Rows& r, bool out16) {
    const int64_t out_mask = out16 ? 7 : mask;
    pieces = pieces && aligned16(r.in) && aligned16(r.out) && !((r.in_t | r.in_h) & mask) &&
             !((r.out_t | r.out_h) & out_mask);
  };
  if (a.NH) fits(a.q, append);
  if (a.NKV) fits(a.k, false);
  if (append) {
    fits(a.v, false);
    pieces = pieces && aligned16(p.key_cache) && aligned16(p.value_cache) &&
             !((a.sb | a.so | a.sh) & 7);
  }
  pieces = pieces && aligned16(p.cos_sin) && aligned16(p.sqk);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!append) return run_type<false, false>(a, p.io_dtype, pieces, s);
  return kv8 ? run_type<true, true>(a, p.io_dtype, pieces, s)
             : run_type<true, false>(a, p.io_dtype, pieces, s);
}

}  // namespace

extern "C" {

int64_t dory_rotary_params_bytes(void) { return int64_t(sizeof(DoryRotaryParams)); }

int32_t dory_rotary_embed(const DoryRotaryParams* params, void* stream) {
  return rotary(params, false, stream);
}

int32_t dory_rotary_append(const DoryRotaryParams* params, void* stream) {
  return rotary(params, true, stream);
}

}  // extern "C"
