// Shared pieces of the row attention kernels (rows_stream.hpp, rows_tile.hpp, rows.hip): element types, row
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
  // Kernels over pages (template PAGED): cache_k / cache_v are pages [pages, G, 1 << page_shift, d] with
  // strides ck_sb of a page, ck_sg, ck_st, and row i of lane row b is slot i % (1 << page_shift) of page
  // table[b table_sb + (i >> page_shift)]; without a table, of page b (rows of an ordinary cache, page_shift 30).
  const int32_t* table;
  int64_t table_sb;
  int page_shift, pages;
  // odd [lanes, room, q_blocks][2][8]: of a share that met infinities or NaNs in V's cache rows (its partials' third tail
  // word), the features (bits) with +infinity and with -infinity, NaN as both; its call rows' note is the fourth word.
  uint32_t* odd;
  int q_blocks;   // of a lane
  int seqs;       // sequences whose queries a lane takes
  int prefix;     // rows that several sequences share: no own rows, every query sees all
};

void rows_plan(const logkv_rows_args& a, int64_t lanes, int64_t nq, RowsLaunch& r);
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

// Queries of a lane, and query qi of lane row b, group g: its row and its token.
template <bool PAGED>
__device__ __forceinline__ int lane_queries(const logkv_rows_args& a, const RowsLaunch& r) {
  const int nq = a.n_heads / a.n_groups * a.tq;
  return PAGED ? nq * r.seqs : nq;
}
template <bool PAGED>
__device__ __forceinline__ const LOGKV_G uint16_t* query_row(const logkv_rows_args& a, const RowsLaunch& r, int b, int g,
                                                             int qi, int& t) {
  const int rep = a.n_heads / a.n_groups;
  if constexpr (PAGED) {
    const int s = qi / (rep * a.tq);
    b = b * r.seqs + s;
    qi -= s * (rep * a.tq);
  }
  t = qi % a.tq;
  return gp(a.q) + b * a.q_sb + (g * rep + qi / a.tq) * a.q_sh + t * a.q_st;
}
template <bool PAGED>
__device__ __forceinline__ int lane_own_rows(const logkv_rows_args& a, const RowsLaunch& r, int b) {
  return PAGED && r.prefix ? 0 : own_rows(a, b);
}

#if defined(__HIP_DEVICE_COMPILE__)
#define LOGKV_C __attribute__((address_space(4)))
#else
#define LOGKV_C
#endif

// Over pages: a lane's rows and tokens by scalar loads (lane row b is the same in all lanes, and what they read is not
// written while a kernel runs).
__device__ __forceinline__ int lane_rows(const logkv_rows_args& a, int b) {
  int64_t n = a.len_add;
  if (a.lengths) n += ((const LOGKV_C int32_t*)a.lengths)[static_cast<int64_t>(b) * a.len_stride];
  if (a.lengths2) n += *(const LOGKV_C int32_t*)a.lengths2;
  return static_cast<int>(imax64(0, imin64(n, a.cap)));
}
__device__ __forceinline__ int lane_tokens(const logkv_rows_args& a, const RowsLaunch& r, int b) {
  if (r.prefix) return 0;
  return a.counts ? max(0, min(((const LOGKV_C int32_t*)a.counts)[b], a.tq)) : a.tq;
}

// Rows of a page that is not there: of zeros.
inline constexpr int kMostFeatures = 256;
static __device__ const uint4 kZeroRow[kMostFeatures / 8] = {};

// The page of row `row` of lane row b, -1 for none.
__device__ __forceinline__ int page_of(const RowsLaunch& r, int b, int row) {
  if (!r.table) return b;
  const int page = gp(r.table)[b * r.table_sb + (row >> r.page_shift)];
  return static_cast<uint32_t>(page) < static_cast<uint32_t>(r.pages) ? page : -1;
}
// Row `row` of the cache rows `base` (group g's, page 0's) that lie on `page`, and the step to the next rows of the page.
__device__ __forceinline__ const LOGKV_G uint16_t* page_row(const RowsLaunch& r, const LOGKV_G uint16_t* base, int64_t sb,
                                                            int64_t st, int page, int row, int64_t& step) {
  step = page < 0 ? 0 : st;
  const LOGKV_G uint16_t* zero = (const LOGKV_G uint16_t*)gp(kZeroRow);
  return page < 0 ? zero : base + page * sb + (row & ((1 << r.page_shift) - 1)) * st;
}

// A value that is the same in all lanes, kept in a scalar register: a launch's arguments would be read again at every
// use in a loop, and each such read waits.
template <typename T>
__device__ __forceinline__ T held(T x) {
  asm volatile("" : "+s"(x));
  return x;
}

// A lane row's pages for the loops of an attention, where the row's index is the same in all lanes: the table's entries
// by scalar loads (it is not written while a kernel reads it).
struct PagedRows {
  const LOGKV_G uint16_t *k, *v;   // the group's rows of page 0
  int64_t k_sb, k_st, v_sb, v_st;
  const LOGKV_C int32_t* line;     // null: of page `b` alone
  int shift, pages, b;

  __device__ __forceinline__ void init(const logkv_rows_args& a, const RowsLaunch& r, int row_b, int g) {
    k = gp(a.cache_k) + g * a.ck_sg, v = gp(a.cache_v) + g * a.cv_sg;
    k_sb = held(a.ck_sb), k_st = held(a.ck_st), v_sb = held(a.cv_sb), v_st = held(a.cv_st);
    b = row_b, shift = held(r.page_shift), pages = held(r.pages);
    line = r.table ? (const LOGKV_C int32_t*)r.table + b * r.table_sb : nullptr;
    line = held(line);
  }
  __device__ __forceinline__ int page(int row) const {
    if (!line) return b;
    const int x = line[row >> shift];
    return static_cast<uint32_t>(x) < static_cast<uint32_t>(pages) ? x : -1;
  }
  // Row `row`, on page p, and the step to its page's next rows: of zeros where there is no page.
  __device__ __forceinline__ const LOGKV_G uint16_t* at(const LOGKV_G uint16_t* base, int64_t sb, int64_t st, int p, int row,
                                                        int64_t& step) const {
    const LOGKV_G uint16_t* there = base + p * sb + (row & ((1 << shift) - 1)) * st;
    step = p < 0 ? 0 : st;
    return p < 0 ? (const LOGKV_G uint16_t*)gp(kZeroRow) : there;
  }
};

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

// Eight elements with zeros in place of infinities and NaNs.
template <int DT>
__device__ __forceinline__ uint4 finite_only(uint4 x) {
  uint32_t* x4[4] = {&x.x, &x.y, &x.z, &x.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = *x4[j] & 0x7fffu, hi = *x4[j] >> 16 & 0x7fffu;
    *x4[j] &= (lo >= Elem<DT>::kInf ? 0u : 0xffffu) | (hi >= Elem<DT>::kInf ? 0u : 0xffff0000u);
  }
  return x;
}

// What V's cache rows [first, end) of a lane hold that is not finite, as a share's words in r.odd: those of rows that a
// query sees (all do, but where the bias is -inf). By all threads of a block, 16 bytes each; `bits`: 16 words of LDS that
// no thread uses any more.
template <int DT, int THREADS>
__device__ __forceinline__ void note_odd_rows(const logkv_rows_args& a, const RowsLaunch& r, int b, int g, int first, int end,
                                              uint32_t* bits, uint32_t* out) {
  const int tid = threadIdx.x, units = a.dv / 8, rows = THREADS / units, row0 = tid / units, u = tid - row0 * units;
  __syncthreads();
  if (tid < 16) bits[tid] = 0;
  __syncthreads();
  uint32_t pos = 0, neg = 0;
  const LOGKV_G uint16_t* base = gp(a.cache_v) + g * a.cv_sg + 8 * u;
  if (row0 < rows) {
#pragma unroll 4
    for (int i = first + row0; i < end; i += rows) {
      int64_t step;
      const uint4 x = *(const LOGKV_G uint4*)page_row(r, base, a.cv_sb, a.cv_st, page_of(r, b, i), i, step);
      bool see = true;
      if (a.bias) {
        const int64_t at = b * a.b_sb + g * a.b_sg + i * a.b_st;
        see = (a.bias_half ? Elem<DT>::to_f32(gp(static_cast<const uint16_t*>(a.bias))[at])
                           : gp(static_cast<const float*>(a.bias))[at]) != -__builtin_inff();
      }
      const uint32_t x4[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t y = x4[j / 2] >> (16 * (j % 2)) & 0xffffu, mag = y & 0x7fffu;
        if (!see || mag < Elem<DT>::kInf) continue;
        if (mag > Elem<DT>::kInf || !(y >> 15)) pos |= 1u << j;
        if (mag > Elem<DT>::kInf || y >> 15) neg |= 1u << j;
      }
    }
    if (pos) atomicOr(bits + u / 4, pos << 8 * (u % 4));
    if (neg) atomicOr(bits + 8 + u / 4, neg << 8 * (u % 4));
  }
  __syncthreads();
  if (tid < 16) out[tid] = bits[tid];
}

}  // namespace logkv
