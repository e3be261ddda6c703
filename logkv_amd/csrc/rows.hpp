// Shared pieces of the row attention kernels (rows_stream.hip, rows.hip): element types, row
// counts, launch parameters.
#pragma once

#include "../../include/logkv_rows.h"
#include "common.hpp"

namespace logkv {

constexpr int kRowTile = 32;        // cache rows (or own rows) per tile
constexpr int kRowsPartTail = 4;    // a partial's maximum and sum, padded to 16 bytes
constexpr int kMaxRowSplits = 64;
constexpr float kTileShift = 7.f;   // tiled kernel: P times 2^7 (below 2^15: its base may lag the maximum by 2^8)
constexpr float kLog2e = 1.44269504088896341f;

// Launch parameters beside the caller's arguments. Workspace regions, 256-byte aligned:
// part [lanes, room, nq, dv + kRowsPartTail]: unnormalised sums, then the base-2 maximum and sum;
// scores [lanes, nq, score_st]: raw products q . k of up to 16 queries (weight attention);
// redo: one flag per block of the tiled kernel;
// shares [lanes]: the partials of a lane where lengths decide (null: splits of them);
// lse [lanes, nq]: base-2 log-sum-exp of longer ones (+inf where a query sees nothing).
struct RowsLaunch {
  float* part;
  float* scores;
  float* lse;
  int* redo;      // tiled kernel: per block whether its share is left to the second launch
  int* shares;
  int64_t score_st;
  int64_t bytes;
  int splits;
  int room;       // partials that a lane has memory for
  int cols;       // streamed kernel: 16-query column blocks per wave
  int q_waves;    // tiled kernel: waves with 32 queries each (0: the streamed kernel)
  float shift;    // the partials' sums carry 2^shift
  float bias2;    // bias to base-2 logits: bias_scale log2(e)
  int causal;     // weight attention; otherwise the visible mask
};

RowsLaunch rows_launch(const logkv_rows_args& a, bool causal, void* ws);
int launch_rows_stream(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream);
int launch_rows_tile(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream);
int launch_rows_weight(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream);
int launch_rows_attention(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream);
int launch_evict(const logkv_evict_args& a, hipStream_t stream);

// Cache rows of batch row b, and its queries (each with an own row).
__device__ __forceinline__ int rows_in_use(const logkv_rows_args& a, int b) {
  int64_t n = a.len_add;
  if (a.lengths) n += a.lengths[static_cast<int64_t>(b) * a.len_stride];
  if (a.lengths2) n += *a.lengths2;
  return static_cast<int>(imax64(0, imin64(n, a.cap)));
}
__device__ __forceinline__ int own_rows(const logkv_rows_args& a, int b) {
  return a.counts ? max(0, min(a.counts[b], a.tq)) : a.tq;
}

// A bias in base 2. A finite one stays finite (a mask of the type's lowest value hides a row only
// beside larger logits).
__device__ __forceinline__ float bias_base2(float x, float bias2) {
  const float y = x * bias2;
  return __builtin_isinf(y) && !__builtin_isinf(x) ? __builtin_copysignf(3.402823466e38f, x) : y;
}

// What is added to a base-2 logit so that the largest of them, y(mx), has the exponent `shift`: shift - m, for m the
// rounded maximum. Where m is beyond 2^22 that sum rounds, and so did m: fp16 probabilities would pass their range (a
// bias of -1e8 leaves spacings of 16, and 15 + 1e8 rounds up to 2^16), so the offset goes down as far.
template <bool BIAS>
__device__ __forceinline__ float exponent_offset(float shift, float m, float mx, float c2) {
  float off = shift - m;
#pragma unroll
  for (int i = 0; i < 2; ++i) {   // a step of off is at least half of both roundings
    if ((BIAS ? mx + off : __builtin_fmaf(mx, c2, off)) > shift + 0.5f)
      off = __uint_as_float(__float_as_uint(off) + (off > 0.f ? -1 : 1));
  }
  return off;
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// The 16-bit element types. kShift: probabilities are scaled by 2^kShift (the sums too, so it
// cancels), which keeps fp16 parts out of the subnormals down to 2^-29; kInf: the bits of infinity.
template <int DT>
struct Elem;
template <>
struct Elem<LOGKV_BF16> {
  typedef bf16x8 vec8;
  static constexpr float kShift = 0.f;
  static constexpr uint32_t kInf = 0x7f80u;
  static __device__ __forceinline__ f32x4 mfma16(vec8 x, vec8 y, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint16_t from_f32(float f) { return f32_to_bf16(f); }
  static __device__ __forceinline__ float to_f32(uint16_t u) { return bf16_to_f32(u); }
  // Two packed parts, each rounded to nearest: 8 and 8 bits. (Cut ones would bias the sums against the divisor's.)
  static __device__ __forceinline__ void parts(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    hi = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x0, x1}, bf16x2));
    const f32x2 r = {x0 - __uint_as_float(hi << 16), x1 - __uint_as_float(hi & 0xffff0000u)};
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));
  }
};
template <>
struct Elem<LOGKV_F16> {
  typedef f16x8 vec8;
  static constexpr float kShift = 15.f;
  static constexpr uint32_t kInf = 0x7c00u;
  static __device__ __forceinline__ f32x4 mfma16(vec8 x, vec8 y, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint16_t from_f32(float f) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  }
  static __device__ __forceinline__ float to_f32(uint16_t u) {
    return static_cast<float>(__builtin_bit_cast(_Float16, u));
  }
  // Two packed parts, each rounded to nearest: 11 and 11 bits.
  static __device__ __forceinline__ void parts(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const f16x2 h = __builtin_convertvector(f32x2{x0, x1}, f16x2);
    const f16x2 r = __builtin_convertvector(f32x2{x0 - static_cast<float>(h[0]), x1 - static_cast<float>(h[1])}, f16x2);
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, r);
  }
};

}  // namespace logkv
