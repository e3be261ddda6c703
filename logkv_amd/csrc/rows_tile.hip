// Attention over a cache's rows and the call's own rows for many queries per KV group (rows.hip's rule):
// tiles of K and V in LDS, shared by a block's NW waves.
//
// Same mathematics as rows_stream.hip (one pass with a running maximum). QW waves hold 32 queries
// each, in registers for the whole range, and NW / QW groups of them take 32 RB rows each of a
// tile. Per 32 rows:
//   S^T = K Q^T by 32x32x16 matrix products (a lane holds 16 rows of its own query);
//   O^T += V^T P^T, where P^T's operand is the lane's own score registers (operand element j of a
//   16-row step st is row 16 st + 8 (j / 4) + 4 (l / 32) + j % 4) and V is read transposed.
// Bound by the vector unit beside the matrix cores: two waves a SIMD issue a vector operation every
// 4.7 cycles (one wave: 8), and the exponentials, maxima and conversions of 32 rows take about as
// long as their products. So two waves a SIMD, and in each the score products of the next 32 rows
// are interleaved with the exponentials of these, the value products with half of the conversions,
// the next maxima and the staging of the next tile. 32768 rows of 128 features, 8 lanes of 512
// queries: 124 us, 555 TFLOP/s of the 1207 of a large matrix product (one wave a SIMD with 64
// queries was slower: nothing hid its waits); 30720 rows and 2048 new ones, 8 lanes of 4096
// queries: 824 - 876 us, 610 - 650 TFLOP/s, the two units busy 50% and 46% of the cycles, in turn.
// Up to 64 queries: two blocks of four waves a CU (two waves of queries, two of rows): 64 lanes of
// 8192 rows, 52 queries 64 us the call, in one block of eight waves 86.
// P enters the value products as two parts of the cache's type (one part's rounding would equal the
// output's), V as it is. For bf16, one fp16 part of P against V converted to fp16 was faster (a third
// less matrix work and five conversions a pair fewer: 64 tokens x 8 heads over 32768 rows 104 us the
// call against 125, 2048 tokens over 30720 rows 975 - 1030 against 1150) but rounded P to 2^-11 and V
// below 2^-17 to 2^-25. A share with an infinity or NaN in V is done again by a second launch (in one
// kernel the second form's registers spilled in the first's loop, and a reload there waits for every
// load ahead) in a second form that adds such a tile row by row for the queries that see its rows. The
// second launch's blocks read a flag and end: 4.7 us.
// Rows are stored without padding, their 16-byte units permuted by row so that the operand reads
// and the transposed reads meet every bank once. One barrier per tile, the following tiles' rows on
// their way in registers; two buffers of V and, by RowsSchedule, two or three of K.
#include <algorithm>
#include <type_traits>

#include "rows.hpp"
#include "rows_schedule.hpp"

namespace logkv {

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kCols = 1;                 // 32-query column blocks per wave

// Where 16-byte unit u of row r is stored: u ^ swizzle. 16 units a row: four consecutive rows fall
// into distinct 64-byte quarters of the 256-byte bank row, sixteen into distinct units. 8 units a
// row (two rows to the bank row): the same over row pairs.
template <int UNITS>
__device__ __forceinline__ int swizzle(int r) {
  return UNITS == 16 ? (r & 3) << 2 | (r >> 2 & 3) : (r >> 1 & 1) << 2 | (r >> 2 & 3);
}

__device__ __forceinline__ float pair_max32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int DT>
__device__ __forceinline__ f32x16 mfma32(uint4 x, uint4 y, f32x16 c) {
  if constexpr (DT == LOGKV_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
}

// x, not known to be the same from one use to the next: keeps the addresses of rarely taken branches
// from being computed ahead and held in registers through the loop.
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// A place in program order that x is computed before: products and exponentials stay interleaved as
// written (the compiler moves them otherwise, to their next use).
template <typename T>
__device__ __forceinline__ void here(T& x) {
  asm volatile("" : "+v"(x));
}

}  // namespace

// The block's place in a grid of (query blocks, splits, lanes): workgroups go to the 8 XCDs round
// robin, each with an L2 of its own; dispatched block n takes logical block (n % 8) (N / 8) + n / 8,
// so that an XCD runs whole lanes where their number allows it and a lane's rows are fetched into
// one L2.
struct RowsBlock {
  int qb, split, lane;
};
__device__ __forceinline__ RowsBlock rows_block() {
  const int nx = static_cast<int>(gridDim.x), ny = static_cast<int>(gridDim.y), n = nx * ny * static_cast<int>(gridDim.z);
  int lin = static_cast<int>(blockIdx.x) + nx * (static_cast<int>(blockIdx.y) + ny * static_cast<int>(blockIdx.z));
  if (n % 8 == 0) lin = lin % 8 * (n / 8) + lin / 8;
  return RowsBlock{lin % nx, lin / nx % ny, lin / (nx * ny)};
}

__device__ __forceinline__ int wave_total(int x) {
#pragma unroll
  for (int off = kWave / 2; off; off >>= 1) x += __shfl_xor(x, off, kWave);
  return __builtin_amdgcn_readfirstlane(x);
}

// Of sequences of different lengths: the equal number of shares a lane (splits) is dealt out anew, to
// each batch row as many as its tiles take at R a share, for the smallest R that needs no more shares
// than there are and no more than `room` for a row. Found by every wave for itself, a batch row in each
// of its lanes. Changes the block's place and the shares of its lane; false for a block left over.
template <int TR>
__device__ __forceinline__ bool share_by_length(const logkv_rows_args& a, const RowsLaunch& r, RowsBlock& id, int& splits) {
  const int B = a.n_batch, G = a.n_groups, l = lane_id(), i = min(l, B - 1), slots = B * r.splits;
  const int tiles = max(1, (rows_in_use(a, i) + TR - 1) / TR + (own_rows(a, i) + TR - 1) / TR), t = l < B ? tiles : 0;
  if (__ballot(tiles != __builtin_amdgcn_readfirstlane(tiles)) == 0) return true;   // as they are
  int most = t;
#pragma unroll
  for (int off = kWave / 2; off; off >>= 1) most = max(most, __shfl_xor(most, off, kWave));
  most = __builtin_amdgcn_readfirstlane(most);
  int lo = max((wave_total(t) + slots - 1) / slots, (most + r.room - 1) / r.room), hi = (most + r.splits - 1) / r.splits;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (wave_total((t + mid - 1) / mid) <= slots) hi = mid;
    else lo = mid + 1;
  }
  const int mine = (t + lo - 1) / lo;
  int up_to = mine;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int up = __shfl_up(up_to, off, kWave);
    if (l >= off) up_to += up;
  }
  const int slot = id.lane / G * r.splits + id.split;
  const uint64_t later = __ballot(l < B && up_to > slot);
  if (!later) return false;
  const int b = __ffsll(static_cast<unsigned long long>(later)) - 1;
  splits = __builtin_amdgcn_readlane(mine, b);
  id.split = slot - (__builtin_amdgcn_readlane(up_to, b) - splits);
  id.lane = b * G + id.lane % G;
  return true;
}

// What a block's share needs beside its tiles, and what it leaves: per column block a lane's query
// with 16 features of each 32 per register block.
template <int NKS, int NDV>
struct RowsShare {
  int b, g, n, own, np, begin, end;
  int t[kCols];
  uint4 qf[kCols][NKS];
  f32x16 o[kCols][NDV];
  float m[kCols], lsum[kCols];
};

template <int NKS, int NDV>
__device__ __forceinline__ void clear_sums(RowsShare<NKS, NDV>& c) {
#pragma unroll
  for (int k = 0; k < kCols; ++k) {
#pragma unroll
    for (int nb = 0; nb < NDV; ++nb)
#pragma unroll
      for (int i = 0; i < 16; ++i) c.o[k][nb][i] = 0.f;
    c.m[k] = -__builtin_inff();
    c.lsum[k] = 0.f;
  }
}

// A share's tiles in the first form; false where it meets one that it cannot take. NKS 16-wide steps
// of dk, NDV 32-wide blocks of dv.
template <int DT, int NKS, int NDV, int NW, int QW, int RB, bool BIAS>
__device__ __forceinline__ bool rows_tile_share(const logkv_rows_args& a, const RowsLaunch& r, RowsShare<NKS, NDV>& c,
                                                uint8_t* buf, float (*bias_s)[32 * RB * NW / QW], int* flag_s) {
  typedef __attribute__((address_space(3))) s16x4* lds4;
  typedef __attribute__((address_space(3))) const uint8_t* ldsb;
  typedef __attribute__((address_space(3))) const u32x4* ldsq;
  constexpr int kThreads = 64 * NW, RW = NW / QW, TR = 32 * RB * RW;   // row groups, rows per tile
  constexpr int KU = 2 * NKS, VU = 4 * NDV;            // 16-byte units of a staged row
  constexpr int kKTasks = TR * KU / kThreads, kVTasks = TR * VU / kThreads;
  typedef RowsSchedule<RB> Order;
  constexpr int kKBytes = TR * KU * 16, kVBytes = TR * VU * 16, kVBase = Order::kKBuffers * kKBytes;
  const int tid = threadIdx.x, l = lane_id(), h = l >> 5, col = l & 31, rw = wave_id() / QW;
  const int kunits = a.dk / 8, vunits = a.dv / 8, b = c.b, g = c.g, np = c.np, begin = c.begin, end = c.end;
  auto k_tile = [&](int bf) { return reinterpret_cast<uint4*>(buf + bf * kKBytes); };
  auto v_tile = [&](int bf) { return reinterpret_cast<uint4*>(buf + kVBase + bf * kVBytes); };

  // Registers of the tiles on their way: K two tiles ahead of the sums, V one. A thread's units are
  // rows tid / KU + kThreads / KU q of a tile. The loads are issued on one path for every tile (values
  // merged from two would be waited for at the merge): rows past a tile's are its last one, units past
  // dk and dv the last ones. When stored, V's extra rows and K's extra units become zero (extra rows of
  // K are masked in the scores, extra units of V reach only features that are not written out).
  uint4 kx[kKTasks], vx[kVTasks];
  uint16_t bx[2] = {0, 0};
  const int ku = tid % KU, kr0 = tid / KU, vr0 = tid / VU;
  const int ku8 = 8 * min(ku, kunits - 1), vu8 = 8 * min(tid % VU, vunits - 1);
  const LOGKV_G uint16_t* kc = gp(a.cache_k) + b * a.ck_sb + g * a.ck_sg;
  const LOGKV_G uint16_t* vc = gp(a.cache_v) + b * a.cv_sb + g * a.cv_sg;
  const LOGKV_G uint16_t* ko = gp(a.k) + b * a.k_sb + g * a.k_sg;
  const LOGKV_G uint16_t* vo = gp(a.v) + b * a.v_sb + g * a.v_sg;
  auto rows_in = [&](int ti) { return ti < np ? min(TR, c.n - TR * ti) : min(TR, c.own - TR * (ti - np)); };
  auto load_k = [&](int ti) {
    const int t0 = TR * (ti < np ? ti : ti - np), last = rows_in(ti) - 1;
    const int64_t st = ti < np ? a.ck_st : a.k_st;
    const LOGKV_G uint16_t* base = (ti < np ? kc : ko) + t0 * st;
#pragma unroll
    for (int q = 0; q < kKTasks; ++q) kx[q] = *(const LOGKV_G uint4*)(base + min(kr0 + kThreads / KU * q, last) * st + ku8);
    if constexpr (BIAS) {
      // A bias as its 16-bit halves (behind the cache's rows: any 4 bytes, not used).
      const LOGKV_G uint16_t* at = gp(a.q);
      if (ti < np) at = gp(static_cast<const uint16_t*>(a.bias)) + (a.bias_half ? 1 : 2) * (b * a.b_sb + g * a.b_sg + (t0 + min(tid % TR, last)) * a.b_st);
      bx[0] = at[0];
      bx[1] = at[a.bias_half ? 0 : 1];
    }
  };
  auto load_v = [&](int ti) {
    const int t0 = TR * (ti < np ? ti : ti - np), last = rows_in(ti) - 1;
    const int64_t st = ti < np ? a.cv_st : a.v_st;
    const LOGKV_G uint16_t* base = (ti < np ? vc : vo) + t0 * st;
#pragma unroll
    for (int q = 0; q < kVTasks; ++q) vx[q] = *(const LOGKV_G uint4*)(base + min(vr0 + kThreads / VU * q, last) * st + vu8);
  };
  auto store_k = [&](int ti, int bf, int q) {
    const int rr = kr0 + kThreads / KU * q;
    if (kunits < KU && ku >= kunits) kx[q] = make_uint4(0, 0, 0, 0);
    k_tile(bf)[rr * KU + (ku ^ swizzle<KU>(rr))] = kx[q];
    if constexpr (BIAS) {
      if (q == 0 && tid < TR) {
        const float x = a.bias_half ? Elem<DT>::to_f32(bx[0]) : __uint_as_float(bx[0] | static_cast<uint32_t>(bx[1]) << 16);
        bias_s[bf][tid] = ti < np ? bias_base2(x, r.bias2) : 0.f;
      }
    }
  };
  // V stored, its magnitudes gathered in top.
  u16x2 top = {0, 0};
  auto store_v = [&](int ti, int bf, int q) {
    const int rr = vr0 + kThreads / VU * q, rows = rows_in(ti);
    if (rows < TR && rr >= rows) vx[q] = make_uint4(0, 0, 0, 0);
    const uint32_t x4[4] = {vx[q].x, vx[q].y, vx[q].z, vx[q].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, x4[j] & 0x7fff7fffu));
    v_tile(bf)[rr * VU + (tid % VU ^ swizzle<VU>(rr))] = vx[q];
  };
  // Whether tile ti's V holds an infinity or NaN.
  auto store_flags = [&](int ti) {
    const bool odd = __ballot(top[0] >= Elem<DT>::kInf || top[1] >= Elem<DT>::kInf) != 0;
    if (odd && l == 0) flag_s[(ti - begin) % 3] = 1;
    top = u16x2{0, 0};
  };
  clear_sums(c);
  if (begin >= end) return true;
  const float c2 = a.scale * kLog2e;
  const int r0 = 32 * RB * rw;   // this wave's rows of a tile
  if (tid < 3) flag_s[tid] = 0;
  load_k(begin);
  load_v(begin);
#pragma unroll
  for (int q = 0; q < kKTasks; ++q) store_k(begin, 0, q);
  load_k(min(begin + 1, end - 1));
#pragma unroll
  for (int q = 0; q < kKTasks; ++q) store_k(min(begin + 1, end - 1), 1, q);
  __syncthreads();   // the flags are clear, K of the first tiles is stored
#pragma unroll
  for (int q = 0; q < kVTasks; ++q) store_v(begin, 0, q);
  store_flags(begin);
  load_k(min(begin + 2, end - 1));
  load_v(min(begin + 1, end - 1));

  // LDS addresses of this lane's operands in buffer 0: unit h of K's row r0 + l % 32, and of V's transposed reads
  // features l & 16 .. of rows 4 h .. (8 + 4 h .. behind). Other units are reached by exclusive or: the permutation is
  // one, rows begin at multiples of their length, and row + 8 has the permutation's second bit the other way round.
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((ldsb)buf));
  const int rk = r0 + col, i16 = l & 15, rv = r0 + 4 * h + (i16 >> 2), f = (l & 16) + 4 * (i16 & 3);
  const uint32_t k_at = lds0 + 16 * (rk * KU + (h ^ swizzle<KU>(rk)));
  const uint32_t v_at = lds0 + kVBase + 16 * (rv * VU + ((f >> 3) ^ swizzle<VU>(rv))) + 2 * (f & 7);
  // K operand ks of 32-row block kb, V^T operand nb of the 16 rows st (in P's order) of a tile.
  auto k_frag = [&](int bf, int kb, int ks) {
    return __builtin_bit_cast(uint4, *(ldsq)(uintptr_t)(((k_at + bf * kKBytes) ^ (32 * ks)) + kb * 32 * KU * 16));
  };
  auto v_frag = [&](int bf, int st, int nb) {
    const uint32_t at = v_at + bf * kVBytes;
    const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)((at ^ (64 * nb)) + st * 16 * VU * 16)));
    const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)((at ^ (64 * nb + 32)) + (st * 16 + 8) * VU * 16)));
    return make_uint4(x.x, x.y, y.x, y.y);
  };
  // Scores of the next 32 rows, then with their bias and masks; the first half of their products'
  // operands is read ahead.
  constexpr int kHalf = NKS / 2;
  f32x16 next[kCols];
  uint4 kf[kHalf];
  float mx[kCols], arg0[kCols];
#pragma unroll
  for (int k = 0; k < kCols; ++k) arg0[k] = kTileShift;
  // Element i is row r0 + 32 kb + 8 (i / 4) + 4 h + i % 4 of tile ti, whose bias is in buffer bf.
  auto finish_scores = [&](int ti, int kb, int bf) {
    const bool own = ti >= np;
    const int t0 = TR * (own ? ti - np : ti), rows = min(TR, (own ? c.own : c.n) - t0);
    if constexpr (BIAS) {
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(&bias_s[bf][r0 + 32 * kb + 8 * i4 + 4 * h]);
#pragma unroll
        for (int k = 0; k < kCols; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i)   // a row hidden by -inf stays hidden whatever its key holds
            next[k][4 * i4 + i] = x[i] == -__builtin_inff() ? x[i] : __builtin_fmaf(next[k][4 * i4 + i], c2, x[i]);
      }
    }
    if (own || rows < TR) {
#pragma unroll
      for (int k = 0; k < kCols; ++k) {
        const int lim = (own && r.causal ? min(rows, fresh(c.t[k]) + 1 - t0) : rows) - r0 - 32 * kb - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i / 4) + i % 4 >= lim) next[k][i] = -__builtin_inff();
        if (own && !r.causal) {
          // All flags loaded at once, those past the line's end its last one.
          const LOGKV_G uint8_t* line = gp(a.visible) + b * a.vis_sb + fresh(c.t[k]) * a.vis_st;
          const int first = t0 + r0 + 32 * kb + 4 * h;
          uint8_t see[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) see[i] = line[min(first + 8 * (i / 4) + i % 4, a.tq - 1)];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (!see[i]) next[k][i] = -__builtin_inff();
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kCols; ++k) mx[k] = -__builtin_inff();
  };
  // The sums' base moves when a maximum passes it by more than 2^8 (P stays below 2^(8 + kTileShift)):
  // a few times a share instead of at every new maximum.
  auto move_base = [&]() {
    float x[kCols], y[kCols];
    bool past = false;
#pragma unroll
    for (int k = 0; k < kCols; ++k) {
      x[k] = pair_max32(mx[k]);
      y[k] = BIAS ? x[k] : x[k] * c2;
      // The difference, since a sum rounds beside a large maximum; and the exponent as it will be formed.
      past |= y[k] - c.m[k] > 8.f || (BIAS ? x[k] + arg0[k] : __builtin_fmaf(x[k], c2, arg0[k])) > kTileShift + 8.5f;
    }
    if (!__ballot(past)) return;
#pragma unroll
    for (int k = 0; k < kCols; ++k) {
      const float m_new = fmaxf(c.m[k], y[k]), mb = m_new == -__builtin_inff() ? 0.f : m_new;
      const float corr = __builtin_amdgcn_exp2f(c.m[k] - mb);
      c.m[k] = m_new;
      arg0[k] = exponent_offset<BIAS>(kTileShift, mb, x[k], c2);
      c.lsum[k] *= corr;
#pragma unroll
      for (int nb = 0; nb < NDV; ++nb)
#pragma unroll
        for (int i = 0; i < 16; ++i) c.o[k][nb][i] *= corr;
    }
  };
#pragma unroll
  for (int k = 0; k < kCols; ++k)
#pragma unroll
    for (int i = 0; i < 16; ++i) next[k][i] = 0.f;
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    kf[ks % kHalf] = k_frag(0, 0, ks);
#pragma unroll
    for (int k = 0; k < kCols; ++k) next[k] = mfma32<DT>(kf[ks % kHalf], c.qf[k][ks], next[k]);
  }
  finish_scores(begin, 0, 0);
#pragma unroll
  for (int k = 0; k < kCols; ++k)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx[k] = fmaxf(mx[k], next[k][i]);
  move_base();
#pragma unroll
  for (int ks = 0; ks < kHalf; ++ks) kf[ks] = k_frag(RB > 1 ? 0 : 1, RB > 1 ? 1 : 0, ks);

  int k_cur = 0, v_cur = 0;   // the buffers of tile ti
  for (int ti = begin; ti < end; ++ti) {
    const int it = ti - begin, k_next = Order::next_k(k_cur), v_next = Order::next_v(v_cur);
    // V of tile ti and K of tile ti + 1 are stored; V of tile ti - 1 has been read, and K of the tile whose buffer
    // tile ti + 2 takes (RB == 1: of tile ti, of which RB > 1 still reads the later blocks: of tile ti - 1).
    __syncthreads();
    if (flag_s[it % 3]) return false;
    if (tid == 0) flag_s[(it + 2) % 3] = 0;
#pragma unroll
    for (int kb = 0; kb < RB; ++kb) {
      // 32 rows: their exponentials and the first 16 rows' parts among the score products of the next 32,
      // then their value products among the other parts, the maxima of those and, behind a tile's last
      // rows, the staging of the next tiles. (Behind
      // the share's last rows the scores are of what the buffer holds, if anything, and unused.)
      f32x16 s[kCols];
#pragma unroll
      for (int k = 0; k < kCols; ++k) {
        s[k] = next[k];
#pragma unroll
        for (int i = 0; i < 16; ++i) next[k][i] = 0.f;
      }
      const int nbf = kb + 1 < RB ? k_cur : k_next, nkb = kb + 1 < RB ? kb + 1 : 0;
      uint4 vf[NDV];
      if constexpr (RB == 1) {
#pragma unroll
        for (int ks = 0; ks < kHalf; ++ks) kf[ks] = k_frag(nbf, nkb, ks);
      }
#pragma unroll
      for (int nb = 0; nb < NDV; ++nb) vf[nb] = v_frag(v_cur, 2 * kb, nb);
      uint32_t hi[kCols][4], lo[kCols][4], hi1[kCols][4], lo1[kCols][4];   // P of the first and the second 16 rows
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
        for (int k = 0; k < kCols; ++k) {
          next[k] = mfma32<DT>(kf[ks % kHalf], c.qf[k][ks], next[k]);
          if (k == kCols - 1 && ks < kHalf) kf[ks] = k_frag(nbf, nkb, ks + kHalf);
          here(next[k]);
#pragma unroll
          for (int i = 16 / NKS * ks; i < 16 / NKS * (ks + 1); i += 2) {
            const float p0 = __builtin_amdgcn_exp2f(BIAS ? s[k][i] + arg0[k] : __builtin_fmaf(s[k][i], c2, arg0[k]));
            const float p1 = __builtin_amdgcn_exp2f(BIAS ? s[k][i + 1] + arg0[k] : __builtin_fmaf(s[k][i + 1], c2, arg0[k]));
            c.lsum[k] += p0;
            c.lsum[k] += p1;
            if (i < 8) {
              Elem<DT>::parts(p0, p1, hi[k][i / 2], lo[k][i / 2]);
              here(hi[k][i / 2]);
            } else {
              s[k][i] = p0;
              s[k][i + 1] = p1;
            }
            here(c.lsum[k]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      const bool last = kb + 1 == RB, stage_k = last && ti + 2 < end, stage_v = last && ti + 1 < end;
      if (!last || ti + 1 < end) finish_scores(last ? ti + 1 : ti, nkb, nbf);
      constexpr int kSlots = 2 * NDV * kCols;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int nb = 0; nb < NDV; ++nb)
#pragma unroll
          for (int k = 0; k < kCols; ++k) {
            const int j = (st * NDV + nb) * kCols + k;
            c.o[k][nb] = mfma32<DT>(vf[nb], st ? make_uint4(hi1[k][0], hi1[k][1], hi1[k][2], hi1[k][3]) : make_uint4(hi[k][0], hi[k][1], hi[k][2], hi[k][3]), c.o[k][nb]);
            if (st == 0) {
              // The second 16 rows' parts among the first ones' products.
#pragma unroll
              for (int i = 4 / NDV * nb; i < 4 / NDV * (nb + 1); ++i) {
                Elem<DT>::parts(s[k][8 + 2 * i], s[k][9 + 2 * i], hi1[k][i], lo1[k][i]);
                here(hi1[k][i]);
                here(lo1[k][i]);
              }
              __builtin_amdgcn_sched_barrier(0);
            }
            c.o[k][nb] = mfma32<DT>(vf[nb], st ? make_uint4(lo1[k][0], lo1[k][1], lo1[k][2], lo1[k][3]) : make_uint4(lo[k][0], lo[k][1], lo[k][2], lo[k][3]), c.o[k][nb]);
            if (k == kCols - 1 && st == 0) vf[nb] = v_frag(v_cur, 2 * kb + 1, nb);
            here(c.o[k][nb]);
#pragma unroll
            for (int kk = 0; kk < kCols; ++kk) {
#pragma unroll
              for (int i = 16 / kSlots * j; i < 16 / kSlots * (j + 1); ++i) mx[kk] = fmaxf(mx[kk], next[kk][i]);
              here(mx[kk]);
            }
            if constexpr (RB > 1) {
              // After (ti, 0) the products were of (ti, 1), the ones to come are of (ti + 1, 0); after (ti, 1),
              // of (ti + 1, 1).
              if (j < kHalf) kf[j] = k_frag(k_next, kb, j);
            }
            if (stage_v) {
              constexpr int kStores = (kVTasks + kSlots - 1) / kSlots;
#pragma unroll
              for (int q = kStores * j; q < min(kStores * (j + 1), kVTasks); ++q) store_v(ti + 1, v_next, q);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
      if (!last || ti + 1 < end) move_base();
      if (stage_k) {
#pragma unroll
        for (int q = 0; q < kKTasks; ++q) store_k(ti + Order::kAhead, Order::next_k(k_next), q);
      }
      if (stage_v) store_flags(ti + 1);
    }
    load_k(min(ti + 3, end - 1));
    load_v(min(ti + 2, end - 1));
    k_cur = k_next;
    v_cur = v_next;
  }
  return true;
}

// The same in the second form: a tile that is not finite row by row in float32, each row for the
// queries that see it. Plain steps (one buffer, nothing ahead): shares that need it are rare.
template <int DT, int NKS, int NDV, int NW, int QW, int RB, bool BIAS>
__device__ __forceinline__ void rows_tile_share2(const logkv_rows_args& a, const RowsLaunch& r, RowsShare<NKS, NDV>& c,
                                                 uint8_t* buf, float (*bias_s)[32 * RB * NW / QW], int* flag_s) {
  typedef __attribute__((address_space(3))) s16x4* lds4;
  constexpr int kThreads = 64 * NW, RW = NW / QW, TR = 32 * RB * RW, KU = 2 * NKS, VU = 4 * NDV;
  static_assert(NW * 16 * 32 * 4 <= TR * (KU + VU) * 16, "a second tile's place holds 16 rows' probabilities of every wave");
  const int tid = threadIdx.x, w = wave_id(), l = lane_id(), h = l >> 5, col = l & 31, r0 = 32 * RB * (w / QW);
  uint4* ks_ = reinterpret_cast<uint4*>(buf);
  uint4* vs_ = reinterpret_cast<uint4*>(buf + TR * KU * 16);
  float* p_s = reinterpret_cast<float*>(buf + TR * (KU + VU) * 16) + w * 16 * 32;
  clear_sums(c);
  const float c2 = a.scale * kLog2e;
#pragma unroll 1
  for (int ti = c.begin; ti < c.end; ++ti) {
    const bool own = ti >= c.np;
    const int t0 = TR * (own ? ti - c.np : ti), rows = min(TR, (own ? c.own : c.n) - t0);
    const int64_t kst = own ? a.k_st : a.ck_st, vst = own ? a.v_st : a.cv_st;
    const LOGKV_G uint16_t* kr = (own ? gp(a.k) + c.b * a.k_sb + c.g * a.k_sg : gp(a.cache_k) + c.b * a.ck_sb + c.g * a.ck_sg) + t0 * kst;
    const LOGKV_G uint16_t* vr = (own ? gp(a.v) + c.b * a.v_sb + c.g * a.v_sg : gp(a.cache_v) + c.b * a.cv_sb + c.g * a.cv_sg) + t0 * vst;
    __syncthreads();   // the last tile has been read
    if (tid == 0) flag_s[0] = 0;
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < TR * KU; i += kThreads) {
      const int rr = i / KU, u = i % KU;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (8 * u < a.dk) x = *(const LOGKV_G uint4*)(kr + min(rr, rows - 1) * kst + 8 * u);
      ks_[rr * KU + (u ^ swizzle<KU>(rr))] = x;
    }
#pragma unroll 1
    for (int i = tid; i < TR * VU; i += kThreads) {
      const int rr = i / VU, u = i % VU;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (8 * u < a.dv && rr < rows) x = *(const LOGKV_G uint4*)(vr + rr * vst + 8 * u);
      const uint32_t x4[4] = {x.x, x.y, x.z, x.w};
      uint32_t most = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) most = max(most, max(x4[j] & 0x7fffu, x4[j] >> 16 & 0x7fffu));
      if (most >= Elem<DT>::kInf) flag_s[0] = 1;
      vs_[rr * VU + (u ^ swizzle<VU>(rr))] = x;
    }
    if constexpr (BIAS) {
      if (tid < TR) {
        float x = 0.f;
        if (!own) {
          const int64_t at = c.b * a.b_sb + c.g * a.b_sg + (t0 + min(tid, rows - 1)) * a.b_st;
          x = bias_base2(a.bias_half ? Elem<DT>::to_f32(gp(static_cast<const uint16_t*>(a.bias))[at])
                                     : gp(static_cast<const float*>(a.bias))[at], r.bias2);
        }
        bias_s[0][tid] = x;
      }
    }
    __syncthreads();
    const bool finite = flag_s[0] == 0;
#pragma unroll 1
    for (int kb = 0; kb < RB; ++kb) {
#pragma unroll
      for (int k = 0; k < kCols; ++k) {
        f32x16 s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
        const int rk = r0 + 32 * kb + col;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
          s = mfma32<DT>(ks_[rk * KU + ((2 * ks + h) ^ swizzle<KU>(rk))], c.qf[k][ks], s);
          __builtin_amdgcn_sched_barrier(0);
        }
        const int lim = (own && r.causal ? min(rows, c.t[k] + 1 - t0) : rows) - r0 - 32 * kb - 4 * h;
        const LOGKV_G uint8_t* line = gp(a.visible) + c.b * a.vis_sb + c.t[k] * a.vis_st + t0 + r0 + 32 * kb + 4 * h;
        uint32_t seen = 0;
        float mx = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int rr = 8 * (i / 4) + i % 4;
          if constexpr (BIAS) {
            const float x = bias_s[0][r0 + 32 * kb + 4 * h + rr];
            s[i] = x == -__builtin_inff() ? x : __builtin_fmaf(s[i], c2, x);
          }
          bool see = rr < lim;
          if (own && !r.causal && see) see = line[rr] != 0;
          if (!see) s[i] = -__builtin_inff();
          mx = fmaxf(mx, s[i]);
          seen |= (s[i] != -__builtin_inff() ? 1u : 0u) << (rr + 4 * h);
        }
        seen |= __shfl_xor(seen, 32, kWave);
        mx = pair_max32(mx);
        const float m_new = fmaxf(c.m[k], BIAS ? mx : mx * c2);
        const float mb = m_new == -__builtin_inff() ? 0.f : m_new, corr = __builtin_amdgcn_exp2f(c.m[k] - mb);
        const float arg0 = exponent_offset<BIAS>(kTileShift, mb, mx, c2);
        c.m[k] = m_new;
        c.lsum[k] *= corr;
#pragma unroll
        for (int nb = 0; nb < NDV; ++nb)
#pragma unroll
          for (int i = 0; i < 16; ++i) c.o[k][nb][i] *= corr;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[i] = __builtin_amdgcn_exp2f(BIAS ? s[i] + arg0 : __builtin_fmaf(s[i], c2, arg0));
          c.lsum[k] += s[i];
        }
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          if (finite) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) Elem<DT>::parts(s[8 * st + 2 * j], s[8 * st + 2 * j + 1], hi[j], lo[j]);
#pragma unroll
            for (int nb = 0; nb < NDV; ++nb) {
              const int i = l & 15, ra = r0 + 32 * kb + 16 * st + 4 * h + (i >> 2), rb = ra + 8, f = 32 * nb + (l & 16) + 4 * (i & 3);
              const uint16_t* base = reinterpret_cast<const uint16_t*>(vs_);
              const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(base + ra * (8 * VU) + 8 * ((f >> 3) ^ swizzle<VU>(ra)) + (f & 7))));
              const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(base + rb * (8 * VU) + 8 * ((f >> 3) ^ swizzle<VU>(rb)) + (f & 7))));
              const uint4 v = make_uint4(x.x, x.y, y.x, y.y);
              c.o[k][nb] = mfma32<DT>(v, make_uint4(hi[0], hi[1], hi[2], hi[3]), c.o[k][nb]);
              c.o[k][nb] = mfma32<DT>(v, make_uint4(lo[0], lo[1], lo[2], lo[3]), c.o[k][nb]);
              __builtin_amdgcn_sched_barrier(0);
            }
          } else {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int j = 0; j < 8; ++j) p_s[32 * (8 * (j / 4) + 4 * h + j % 4) + col] = s[8 * st + j];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (int j = 0; j < 16; ++j) {
              const int rr = r0 + 32 * kb + 16 * st + j;
              const float pk = p_s[32 * j + col];
              const bool see = seen >> (16 * st + j) & 1;
#pragma unroll
              for (int nb = 0; nb < NDV; ++nb) {
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) {
                  const uint16_t* v = reinterpret_cast<const uint16_t*>(vs_ + rr * VU + ((4 * nb + i4) ^ swizzle<VU>(rr))) + 4 * h;
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    const float x = pk * Elem<DT>::to_f32(v[i]);
                    c.o[k][nb][4 * i4 + i] += see ? x : 0.f;
                  }
                  __builtin_amdgcn_sched_barrier(0);
                }
              }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          }
        }
      }
    }
  }
}

// SECOND: the launch that follows, whose blocks do again what the first left (r.redo, one flag a block).
template <int DT, int NKS, int NDV, int NW, int QW, int RB, bool BIAS, bool SECOND>
__global__ __launch_bounds__(64 * NW, 2) void rows_tile_kernel(logkv_rows_args a, RowsLaunch r) {
  constexpr int kThreads = 64 * NW, RW = NW / QW, TR = 32 * RB * RW, kQueries = 32 * kCols;   // per wave
  constexpr int kTileBytes = TR * 16 * (RowsSchedule<RB>::kKBuffers * 2 * NKS + RowsSchedule<RB>::kVBuffers * 4 * NDV);
  constexpr int kOutBytes = RW > 1 ? NW * kQueries * 32 * NDV * 4 : 0;
  __shared__ __align__(256) uint8_t buf[kTileBytes > kOutBytes ? kTileBytes : kOutBytes];
  __shared__ __align__(16) float bias_s[BIAS ? RowsSchedule<RB>::kKBuffers : 1][TR];
  __shared__ int flag_s[3];
  __shared__ float m_s[NW][kQueries], l_s[NW][kQueries];
  RowsBlock id = rows_block();
  int* redo = r.redo + (static_cast<int64_t>(id.lane) * gridDim.y + id.split) * gridDim.x + id.qb;
  if (SECOND && *redo == 0) return;
  int splits = r.splits;
  if (r.shares) {
    if (!share_by_length<TR>(a, r, id, splits)) {
      if (threadIdx.x == 0) *redo = 0;
      return;
    }
    if (id.split == 0 && id.qb == 0 && threadIdx.x == 0) r.shares[id.lane] = splits;
  }
  const int lane = id.lane, G = a.n_groups, tid = threadIdx.x;
  const int rep = a.n_heads / G, nq = rep * a.tq, w = wave_id(), l = lane_id(), h = l >> 5, col = l & 31;
  RowsShare<NKS, NDV> c;
  c.b = lane / G;
  c.g = lane % G;
  c.n = rows_in_use(a, c.b);
  c.own = own_rows(a, c.b);
  const int q_first = id.qb * kQueries * QW, q_last = min(q_first + kQueries * QW, nq) - 1;
  const int q0 = q_first + kQueries * (w % QW) + col;   // the first column block's query
  // Own rows that some query of the block may see.
  const int t_max = q_first / a.tq == q_last / a.tq ? q_last % a.tq : a.tq - 1;
  const int own_end = r.causal ? min(c.own, t_max + 1) : c.own;
  c.np = (c.n + TR - 1) / TR;
  const int tiles = c.np + (own_end + TR - 1) / TR, share = (tiles + splits - 1) / splits;
  c.begin = min(id.split * share, tiles);
  c.end = min(c.begin + share, tiles);
#pragma unroll
  for (int k = 0; k < kCols; ++k) {
    const int qc = min(q0 + 32 * k, nq - 1);
    c.t[k] = qc % a.tq;
    const LOGKV_G uint16_t* qrow = gp(a.q) + c.b * a.q_sb + (c.g * rep + qc / a.tq) * a.q_sh + c.t[k] * a.q_st;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      c.qf[k][ks] = make_uint4(0, 0, 0, 0);
      if (2 * ks + h < a.dk / 8) c.qf[k][ks] = *(const LOGKV_G uint4*)(qrow + 16 * ks + 8 * h);
    }
  }
  if constexpr (SECOND) {
    rows_tile_share2<DT, NKS, NDV, NW, QW, RB, BIAS>(a, r, c, buf, bias_s, flag_s);
  } else {
    const bool done = rows_tile_share<DT, NKS, NDV, NW, QW, RB, BIAS>(a, r, c, buf, bias_s, flag_s);
    if (tid == 0) *redo = done ? 0 : 1;
    if (!done) return;
  }
#pragma unroll
  for (int k = 0; k < kCols; ++k) {
    c.lsum[k] = pair_sum32(c.lsum[k]);
    if (c.t[k] >= c.own) {   // a query past its batch row's count sees nothing
      c.m[k] = -__builtin_inff();
      c.lsum[k] = 0.f;
#pragma unroll
      for (int nb = 0; nb < NDV; ++nb)
#pragma unroll
        for (int i = 0; i < 16; ++i) c.o[k][nb][i] = 0.f;
    }
  }
  float* part = r.part + (static_cast<int64_t>(lane) * r.room + id.split) * nq * (a.dv + kRowsPartTail);
  if constexpr (RW == 1) {
#pragma unroll
    for (int k = 0; k < kCols; ++k) {
      const int qi = q0 + 32 * k;
      if (qi >= nq) continue;
      float* out = part + static_cast<int64_t>(qi) * (a.dv + kRowsPartTail);
      if (h == 0) *reinterpret_cast<float2*>(out + a.dv) = make_float2(c.m[k], c.lsum[k]);
#pragma unroll
      for (int nb = 0; nb < NDV; ++nb)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          const int d = 32 * nb + 8 * i4 + 4 * h;
          const f32x4 y = {c.o[k][nb][4 * i4], c.o[k][nb][4 * i4 + 1], c.o[k][nb][4 * i4 + 2], c.o[k][nb][4 * i4 + 3]};
          if (d < a.dv) *reinterpret_cast<f32x4*>(out + d) = y;
        }
    }
  } else {
    // The row groups joined in their order.
    constexpr int kLd = 32 * NDV;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kCols; ++k) {
      float* acc = reinterpret_cast<float*>(buf) + (w * kQueries + 32 * k + col) * kLd;
#pragma unroll
      for (int nb = 0; nb < NDV; ++nb)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          const f32x4 y = {c.o[k][nb][4 * i4], c.o[k][nb][4 * i4 + 1], c.o[k][nb][4 * i4 + 2], c.o[k][nb][4 * i4 + 3]};
          *reinterpret_cast<f32x4*>(acc + 4 * ((8 * nb + 2 * i4 + h) ^ (col & 7))) = y;
        }
      if (h == 0) {
        m_s[w][32 * k + col] = c.m[k];
        l_s[w][32 * k + col] = c.lsum[k];
      }
    }
    __syncthreads();
    const int queries = min(kQueries * QW, nq - q_first), units = a.dv / 4 + 1;
    for (int e = tid; e < queries * units; e += kThreads) {
      const int q = e / units, u = e % units, qq = q / kQueries, cc = q % kQueries;
      float mx = -__builtin_inff();
#pragma unroll
      for (int k = 0; k < RW; ++k) mx = fmaxf(mx, m_s[k * QW + qq][cc]);
      const float top = mx == -__builtin_inff() ? 0.f : mx;
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < RW; ++k) {
        const int ww = k * QW + qq;
        const float f = __builtin_amdgcn_exp2f(m_s[ww][cc] - top);
        if (u == units - 1) sum[1] += l_s[ww][cc] * f;
        else sum += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(buf) + (ww * kQueries + cc) * kLd + 4 * (u ^ (cc & 7))) * f;
      }
      if (u == units - 1) sum[0] = mx;
      *reinterpret_cast<f32x4*>(part + static_cast<int64_t>(q_first + q) * (a.dv + kRowsPartTail) + 4 * u) = sum;
    }
  }
}

namespace {

template <int DT, int NKS, int NDV, int NW, int QW, int RB>
void launch_one(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream) {
  const int nq = a.n_heads / a.n_groups * a.tq, queries = 32 * kCols * QW;
  const dim3 grid((nq + queries - 1) / queries, r.splits, a.n_batch * a.n_groups);
  if (a.bias) {
    hipLaunchKernelGGL((rows_tile_kernel<DT, NKS, NDV, NW, QW, RB, true, false>), grid, dim3(64 * NW), 0, stream, a, r);
    hipLaunchKernelGGL((rows_tile_kernel<DT, NKS, NDV, NW, QW, RB, true, true>), grid, dim3(64 * NW), 0, stream, a, r);
  } else {
    hipLaunchKernelGGL((rows_tile_kernel<DT, NKS, NDV, NW, QW, RB, false, false>), grid, dim3(64 * NW), 0, stream, a, r);
    hipLaunchKernelGGL((rows_tile_kernel<DT, NKS, NDV, NW, QW, RB, false, true>), grid, dim3(64 * NW), 0, stream, a, r);
  }
}

template <int DT, int NKS, int NDV>
void launch_width(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream) {
  if (r.q_waves == 2) launch_one<DT, NKS, NDV, 4, 2, 1>(a, r, stream);
  else if (r.q_waves == 4) launch_one<DT, NKS, NDV, 8, 4, 1>(a, r, stream);
  else launch_one<DT, NKS, NDV, 8, 8, 2>(a, r, stream);
}

template <int DT>
void launch_type(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream) {
  if (a.dk <= 64 && a.dv <= 64) launch_width<DT, 4, 2>(a, r, stream);
  else launch_width<DT, 8, 4>(a, r, stream);
}

}  // namespace

int launch_rows_tile(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream) {
  if (a.dtype == LOGKV_BF16) launch_type<LOGKV_BF16>(a, r, stream);
  else launch_type<LOGKV_F16>(a, r, stream);
  return hipGetLastError() == hipSuccess ? LOGKV_OK : LOGKV_ERUNTIME;
}

}  // namespace logkv
