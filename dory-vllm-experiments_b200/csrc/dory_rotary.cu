// dory_rotary.cu — rotary positions (dory_rotary_embed) and the rotated, normalised append of
// new keys and values to the paged cache (dory_rotary_append); the C ABI is in
// include/dory_decode.h.
//
// Both read every input once and write every output once, with a handful of operations per
// element: HBM bounds a long rotation (8192 tokens of 32 + 8 heads of 128 bf16 dims: 30.9 us, 85%
// of the measured copy rate), instruction issue and then HBM a long append (37.5 us; 46 with the
// norm, whose sum is FP64, 69%), the launch and two dependent loads (position, then table row) a
// single token (4.3 us).
//
// rotary_vec: a head's row belongs to head_dim / 16 neighbouring lanes.  Lane l holds two
// 8-element pieces that contain both members of its pairs: dims 8l and rotary_dim / 2 + 8l of
// the half layout, 16l and 16l + 8 of the interleaved one, so in both it needs the angles 8l ..
// 8l + 7 and no exchange between lanes (the norm alone takes log2(head_dim / 16) shuffles).  A
// block takes the heads of one token, then of the next: a lane keeps its head, so its share of
// sqk stays in registers, the heads of a token share its angles in L1, and the loads of the next
// two tokens are on their way while this one is worked on.
// rotary_any: one warp per row, a pair per lane, for every size, stride and alignment, with the
// wide kernel's arithmetic to the last bit (the same rotation one element off the 16-byte grid: 142
// us; the append 205, with the norm 329).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <string.h>

#include <type_traits>

#include "dory_common.h"
#include "dory_sm100.cuh"

namespace {

using dory::aligned16;
using dory::fail;
using namespace sm100;  // packed FP32 arithmetic

constexpr int kVecThreads = 384;  // of rotary_vec, in a block at most; two blocks an SM
constexpr int kMaxShared = 227 * 1024;

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
  int T, NH, NKV, D, R, B;
  int heads;  // rows of a token
  int group;  // of them, in a block
  int run;    // tokens of a block
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
__device__ __forceinline__ void unpack(const Piece<__nv_bfloat16>& p, float (&x)[8]) {
  const uint32_t w[4] = {p.w[0].x, p.w[0].y, p.w[0].z, p.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
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
// Offset of a slot's row (head 0) in a cache, in elements.
__device__ __forceinline__ int64_t slot_offset(const RotaryArgs& a, int64_t slot) {
  const int64_t block = slot < INT32_MAX ? uint32_t(slot) / uint32_t(a.B) : slot / a.B;
  return block * a.sb + (slot - block * a.B) * a.so;
}

// The factor that the decode calls and qk_norm_cache normalise a row with, so that a row's bits do
// not depend on the call that appends it: the FP64 sum of squares rounded to FP32, eps added there,
// and 1 / sqrt of that, correctly rounded.  With y near 1 / sqrt(t) and e = 1 - t y^2, 1 / sqrt(t) =
// y / sqrt(1 - e) = y (1 + e / 2 + 3 e^2 / 8 + ..); |e| < 2^-21, so what is left out is below 2^-64.
// A sum beyond FP32 gives 0.  The wider sum and root cost a long append issue slots (8192 tokens: 46
// us; 40 with both in FP32, whose rows differed in their last bits from those of the other calls).
__device__ __forceinline__ float inv_norm(double sum, float eps) {
  const float t = __fadd_rn(__double2float_rn(sum), eps);
  const double y = double(rsqrtf(t)), e = fma(-double(t), y * y, 1.0);
  const float inv = __double2float_rn(fma(y, e * fma(e, 0.375, 0.5), y));
  return isinf(t) ? 0.0f : inv;
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
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
constexpr int kAhead = 3;  // tokens in flight
template <typename T>
constexpr int kElementBytes = 16 * int(sizeof(T));  // of a thread and token

template <typename T, bool APPEND, bool KV8>
__global__ void __launch_bounds__(kVecThreads, 2) rotary_vec(const RotaryArgs a) {
  // Tokens in flight: [token][16 bytes][thread] of elements, a thread reads its own, then
  // [token][warp][table row] of angles, a warp reads its own.
  extern __shared__ uint4 ring[];
  constexpr int kQuads = int(sizeof(T));  // 16-byte words of a thread's 16 elements
  const int lanes = a.D / 16;
  const int local = threadIdx.x / lanes, l = threadIdx.x - local * lanes;
  const int h = blockIdx.y * a.group + local;
  const bool here = local < a.group && h < a.heads;
  const bool is_q = h < a.NH, is_v = APPEND && h >= a.NH + a.NKV;
  const int g = is_q ? h : is_v ? h - a.NH - a.NKV : h - a.NH;  // among its kind
  const bool turn = here && !is_v && l < a.R / 16;
  const bool apart = l < a.R / 16 && !a.inter && !is_v;
  const int oa = apart ? 8 * l : 16 * l, ob = apart ? a.R / 2 + 8 * l : 16 * l + 8;
  const Rows& rows = is_q ? a.q : is_v ? a.v : a.k;
  const T* in = here ? static_cast<const T*>(rows.in) + g * rows.in_h : nullptr;
  const int64_t in_t = rows.in_t;

  const float sign = APPEND ? 1.0f : a.sign;  // the append rotates forwards only
  uint64_t weight[8];  // with the norm, pairs: (sqk * sqk_factor)^2 of the lane's dims, 1 for k
  if constexpr (APPEND) {
#pragma unroll
    for (int j = 0; j < 8; ++j) weight[j] = pair(1.0f, 1.0f);
    if (a.norm && here && is_q) {
      float w[16];
      load8(a.sqk, int64_t(h) * a.D + oa, a.sqk_dtype, reinterpret_cast<float(&)[8]>(w[0]));
      load8(a.sqk, int64_t(h) * a.D + ob, a.sqk_dtype, reinterpret_cast<float(&)[8]>(w[8]));
#pragma unroll
      for (int j = 0; j < 16; ++j) w[j] = w[j] * a.sqk_factor * (w[j] * a.sqk_factor);
#pragma unroll
      for (int j = 0; j < 8; ++j) weight[j] = pair(w[2 * j], w[2 * j + 1]);
    }
  }

  const int first = blockIdx.x * a.run, last = min(first + a.run, a.T);  // this block's tokens
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  const int angle_quads = a.R * (a.cs_dtype == DORY_DTYPE_F32 ? 4 : 2) / 16;
  // Everything that steps with the token or the place in the ring is kept and added to: address
  // arithmetic was half of the instructions, which bound the append (8192 tokens with the norm, then in
  // FP32: 40 us, 53 before).
  const uint32_t place_bytes = kQuads * blockDim.x * 16, angle_bytes = warps * angle_quads * 16;
  const uint32_t own = uint32_t(__cvta_generic_to_shared(ring + threadIdx.x));
  const uint32_t own_angles = uint32_t(__cvta_generic_to_shared(ring)) + kAhead * place_bytes +
                              (threadIdx.x >> 5) * angle_quads * 16;
  const uint32_t piece = blockDim.x * 16;  // between a thread's 16-byte words
  // Positions and slots: a lane reads those of one token in 32 and the warp hands them round, so
  // that they cost a token one shuffle each and the division by the block size nothing.  A
  // position outside the table is -1, a slot that is not written an offset of -1.
  int positions = -1;
  int64_t offsets = -1, offsets_next = -1;
  auto read_ahead = [&](int t) {  // tokens t .. t + 31
    t += lane;
    const bool reports = blockIdx.y == 0 && threadIdx.x < 32 && t < last;
    int64_t slot = 0;
    if constexpr (APPEND) {
      slot = t < last ? a.slots[t] : -1;
      const bool fits = slot >= 0 && slot < a.cache_slots;
      offsets_next = fits ? slot_offset(a, slot) : -1;
      if (reports && slot >= a.cache_slots) report(a, DORY_DEVERR_SLOT_OOB);
    }
    positions = 0;
    if (a.R > 0) {
      const int64_t pos = t < last ? position_of(a, t) : 0;
      const bool inside = uint64_t(pos) < uint64_t(a.max_position);
      positions = inside ? int(pos) : -1;
      if (reports && !inside && slot >= 0) report(a, DORY_DEVERR_POSITION_OOB);
    }
  };
  // Starts the loads of the next token, t, into the ring's place `to`: elements and angles by
  // asynchronous copies, since registers for as many tokens would leave too few threads.
  const T* next_in = in + (here ? first * in_t : 0);
  uint32_t known_bits = 0;  // whether the angles of the tokens asked for last exist
  auto ask = [&](int t, int to) {
    if (((t - first) & 31) == 0) read_ahead(t);
    const int pos = __shfl_sync(0xffffffffu, positions, (t - first) & 31);
    known_bits = 2 * known_bits + (pos >= 0);
    if (t < last) {
      if (here) {
        const uint32_t dst = own + to * place_bytes;
#pragma unroll
        for (int i = 0; i < kQuads / 2; ++i) {
          copy_async(dst + i * piece, next_in + oa + i * (16 / sizeof(T)));
          copy_async(dst + (kQuads / 2 + i) * piece, next_in + ob + i * (16 / sizeof(T)));
        }
        next_in += in_t;
      }
      if (a.R > 0 && pos >= 0) {
        const uint4* row = static_cast<const uint4*>(a.cos_sin) + int64_t(pos) * angle_quads + lane;
        const uint32_t dst = own_angles + to * angle_bytes + lane * 16;
        if (lane < angle_quads) copy_async(dst, row);
        if (lane + 32 < angle_quads) copy_async(dst + 512, row + 32);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

#pragma unroll 1
  for (int i = 0; i < kAhead - 1; ++i) ask(first + i, i);
  int place = 0;
  uint8_t* out = nullptr;  // of q (append), or of any row
  int64_t out_step = 0;
  uint8_t* const cache_head = (is_v ? a.vc : a.kc) + g * a.sh * (KV8 ? 1 : 2);  // of k and v
  if (here && (!APPEND || is_q)) {
    constexpr int kOut = APPEND ? 2 : int(sizeof(T));
    out = static_cast<uint8_t*>(rows.out) + (g * rows.out_h + first * rows.out_t) * kOut;
    out_step = rows.out_t * kOut;
  }
#pragma unroll 1
  for (int t = first; t < last; ++t) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 2) : "memory");
    __syncwarp();  // the warp's angles are there, and its reads of the token before are done
    if (APPEND && ((t - first) & 31) == 0) offsets = offsets_next;
    ask(t + kAhead - 1, place == 0 ? kAhead - 1 : place - 1);
    const bool known = known_bits >> (kAhead - 1) & 1;
    const int64_t offset = APPEND ? __shfl_sync(0xffffffffu, offsets, (t - first) & 31) : 0;
    const uint4* const mine = ring + place * (kQuads * blockDim.x) + threadIdx.x;
    uint64_t y[8];  // the lane's elements in pairs: four of the first piece, four of the second
    {
      Piece<T> xa, xb;
#pragma unroll
      for (int i = 0; i < kQuads / 2; ++i) {
        xa.w[i] = mine[i * blockDim.x];
        xb.w[i] = mine[(kQuads / 2 + i) * blockDim.x];
      }
      float ya[8], yb[8];
      unpack(xa, ya);
      unpack(xb, yb);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[j] = pair(ya[2 * j], ya[2 * j + 1]);
        y[4 + j] = pair(yb[2 * j], yb[2 * j + 1]);
      }
    }
    if (!is_v && !known) {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = 0;
    } else if (turn) {
      float c[8], s[8];
      const uint4* const angles = ring + kAhead * kQuads * blockDim.x +
                                  (place * warps + (threadIdx.x >> 5)) * angle_quads;
      load8(angles, 8 * l, a.cs_dtype, c);
      load8(angles, a.R / 2 + 8 * l, a.cs_dtype, s);
      if (a.inter) {  // a pair is one rotation: (u, w) c + (w, u) (-s, s)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float u, w;
          split(y[j], u, w);
          const float turn_by = sign * s[j];
          y[j] = fma2(pair(w, u), pair(-turn_by, turn_by), mul2(y[j], pair(c[j], c[j])));
        }
      } else {  // two rotations at once
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint64_t u = y[j], w = y[4 + j], c2 = pair(c[2 * j], c[2 * j + 1]);
          const uint64_t s2 = pair(sign * s[2 * j], sign * s[2 * j + 1]);
          y[j] = fma2(mul2(w, pair(-1.0f, -1.0f)), s2, mul2(u, c2));
          y[4 + j] = fma2(u, s2, mul2(w, c2));
        }
      }
    }
    if constexpr (APPEND) {
      if (a.norm) {  // every lane of the warp takes part: rows never straddle a warp
        double sum = 0.0, other = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float u, w;
          split(y[j], u, w);
          sum += double(u) * double(u);
          other += double(w) * double(w);
        }
        sum += other;
        if (lanes > 8) sum += __shfl_xor_sync(0xffffffffu, sum, 8);  // 4, 8 or 16 lanes a row
        if (lanes > 4) sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        if (!is_v && known) {  // zeros stay zeros, whatever eps
          const float inv = inv_norm(sum, a.eps);
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = mul2(weight[j], mul2(y[j], pair(inv, inv)));
        }
      }
    }
    if (here) {
      float ya[8], yb[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        split(y[j], ya[2 * j], ya[2 * j + 1]);
        split(y[4 + j], yb[2 * j], yb[2 * j + 1]);
      }
      if (!APPEND || is_q) {
        using Out = std::conditional_t<APPEND, __nv_bfloat16, T>;
        store_piece(reinterpret_cast<Out*>(out) + oa, ya);
        store_piece(reinterpret_cast<Out*>(out) + ob, yb);
        out += out_step;
      } else if (offset >= 0) {
        uint8_t* o = cache_head + offset * (KV8 ? 1 : 2);
        if constexpr (KV8) {
          const float scale = is_v ? a.v_scale : a.k_scale;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float(&v)[8] = half ? yb : ya;
            uint2 w;
            w.x = to_e4m3x2(v[0], v[1], scale) | to_e4m3x2(v[2], v[3], scale) << 16;
            w.y = to_e4m3x2(v[4], v[5], scale) | to_e4m3x2(v[6], v[7], scale) << 16;
            *reinterpret_cast<uint2*>(o + (half ? ob : oa)) = w;
          }
        } else {
          __nv_bfloat16* b = reinterpret_cast<__nv_bfloat16*>(o);
          store_piece(b + oa, ya);
          store_piece(b + ob, yb);
        }
      }
    }
    if (++place == kAhead) place = 0;
  }
}

// ------------------------------------------------------------------------------------
// The rotated element i of a row: the product and the fused sum that rotary_vec forms, so that a
// row's bits do not depend on its strides.
template <typename T>
__device__ __forceinline__ float turned(const RotaryArgs& a, const T* x, int i, int64_t pos) {
  if (i >= a.R) return to_f32(x[i]);
  const int half = a.R / 2;
  const int pair = a.inter ? i / 2 : (i < half ? i : i - half);
  const bool first = a.inter ? (i & 1) == 0 : i < half;
  const int i0 = a.inter ? 2 * pair : pair, i1 = a.inter ? 2 * pair + 1 : pair + half;
  const float c = load_as_f32(a.cos_sin, pos * a.R + pair, a.cs_dtype);
  const float s = a.sign * load_as_f32(a.cos_sin, pos * a.R + half + pair, a.cs_dtype);
  return first ? __fmaf_rn(-to_f32(x[i1]), s, __fmul_rn(to_f32(x[i0]), c))
               : __fmaf_rn(to_f32(x[i0]), s, __fmul_rn(to_f32(x[i1]), c));
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
      double sum = 0.0;
      for (int i = lane; i < a.D; i += 32) {
        const double y = inside ? turned(a, x, i, pos) : 0.0f;
        sum += y * y;
      }
      for (int m = 16; m; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
      if (inside) inv = inv_norm(sum, a.eps);
    }
    if (h >= a.NH && slot < 0) return;
    const int g = is_v ? h - a.NH - a.NKV : h - a.NH;
    uint8_t* row_out = h < a.NH ? nullptr
                                : (is_v ? a.vc : a.kc) +
                                      (slot_offset(a, slot) + g * a.sh) * (KV8 ? 1 : 2);
    for (int i = lane; i < a.D; i += 32) {
      float y = is_v ? to_f32(x[i]) : inside ? turned(a, x, i, pos) : 0.0f;
      if (a.norm && !is_v) {
        y *= inv;
        if (h < a.NH) {
          const float u = load_as_f32(a.sqk, int64_t(h) * a.D + i, a.sqk_dtype) * a.sqk_factor;
          y = u * u * y;
        }
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
  // A block takes `group` heads of one token after the other: as many blocks as tokens while
  // that leaves SMs idle, then about 2 kVecThreads threads an SM, each with kAhead tokens in flight.
  int device = 0;
  const int sms = dory::device_sms(&device);
  if (sms <= 0) return fail(DORY_ERR_CUDA, "no current CUDA device");
  const int lanes = a.D / 16;
  a.group = kVecThreads / lanes < a.heads ? kVecThreads / lanes : a.heads;
  const int parts = (a.heads + a.group - 1) / a.group;
  a.group = (a.heads + parts - 1) / parts;
  const int threads = (a.group * lanes + 31) / 32 * 32;
  const int64_t resident = int64_t(sms) * (2 * kVecThreads / threads);
  const int64_t blocks = (resident + parts - 1) / parts;
  a.run = int((a.T + blocks - 1) / blocks);
  cfg.gridDim = dim3(unsigned((a.T + a.run - 1) / a.run), unsigned(parts));
  cfg.blockDim = dim3(unsigned(threads));
  const int angles = a.R * (a.cs_dtype == DORY_DTYPE_F32 ? 4 : 2);
  cfg.dynamicSmemBytes = unsigned(kAhead * (threads * kElementBytes<T> + threads / 32 * angles));
  static bool ready[64] = {false};
  if (!ready[device]) {
    const cudaError_t e =
        cudaFuncSetAttribute(rotary_vec<T, APPEND, KV8>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kMaxShared);
    if (e != cudaSuccess)
      return fail(DORY_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    ready[device] = true;
  }
  return dory::launched(cudaLaunchKernelEx(&cfg, rotary_vec<T, APPEND, KV8>, a));
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
             !((a.sb | a.so | a.sh) & 7) && a.sb >= 0 && a.so >= 0;
  }
  // A block's ring is then at most 3 x (384 threads x 64 bytes + 12 warps x 1 KB) = 108 KB.
  const int angle_bytes = p.rotary_dim * (p.cos_sin_dtype == DORY_DTYPE_F32 ? 4 : 2);
  pieces = pieces && aligned16(p.cos_sin) && aligned16(p.sqk) && angle_bytes <= 1024 &&
           p.max_position <= INT32_MAX;
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
