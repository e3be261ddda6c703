// Attention over a cache's rows and the call's own rows for more queries than a wave's columns:
// tiles of K and V in LDS, shared by a block's eight waves.
//
// Same mathematics as rows_stream.hip (one pass with a running maximum). QW waves hold 32 queries
// each (one per lane column, in registers for the whole range), and 8 / QW groups of them take
// 32 RB rows each of a tile:
//   S^T = K Q^T by 32x32x16 matrix products (a lane holds 16 rows of its own query per 32 rows);
//   O^T += V^T P^T, where P^T's operand is the lane's own score registers (operand element j of a
//   16-row step st is row 16 st + 8 (j / 4) + 4 (l / 32) + j % 4) and V is read transposed.
// bf16 caches: V enters the products as fp16, converted as it is staged (times 2^6: exact from 2^-23
// up, below that to 2^-31 absolute), and P as fp16 times 2^15 (11 bits): one product per step, a
// third less matrix work than two bf16 parts of P, and P's error stays an eighth of the output's
// rounding. A share with a tile whose largest magnitude is not in [2^-8, 2^9) is done again in a
// second form: V as bf16, P as two parts. fp16 caches: P as two fp16 parts in both forms, since one
// part's rounding would equal the output's; the second form is for infinities and NaNs in V, which
// it adds row by row for the queries that see them.
// Rows are stored without padding, their 16-byte units permuted by row so that the operand reads
// and the transposed reads meet every bank once. Two buffers, one barrier per tile, the next
// tile's rows on their way in registers.
#include <algorithm>
#include <type_traits>

#include "rows.hpp"

namespace logkv {

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 512;
constexpr float kVScale = 64.f;          // bf16 V as fp16: times 2^6
constexpr float kPShift = 15.f;          // P times 2^15

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

// Two bf16 values as fp16 times 2^6, exact in the range above.
__device__ __forceinline__ uint32_t half_of_bf16(uint32_t x) {
  const f32x2 f = {__uint_as_float(x << 16) * kVScale, __uint_as_float(x & 0xffff0000u) * kVScale};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, f16x2));
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

// What a block's share needs beside its tiles, and what it leaves: a lane's query column with 16
// features of each 32 per register block.
template <int NKS, int NDV>
struct RowsShare {
  int b, g, t, n, own, np, begin, end;
  uint4 qf[NKS];
  f32x16 o[NDV];
  float m, lsum;
};

// A share's tiles. False where the first form (SECOND false) meets a tile that it cannot take.
// NKS 16-wide steps of dk, NDV 32-wide blocks of dv.
template <int DT, int NKS, int NDV, int QW, int RB, bool BIAS, bool SECOND>
__device__ __forceinline__ bool rows_tile_share(const logkv_rows_args& a, const RowsLaunch& r, RowsShare<NKS, NDV>& c,
                                                uint8_t* buf, float (*bias_s)[32 * RB * 8 / QW], int* flag_s) {
  typedef __attribute__((address_space(3))) s16x4* lds4;
  constexpr int RW = 8 / QW, TR = 32 * RB * RW;        // row groups, rows per tile
  constexpr int KU = 2 * NKS, VU = 4 * NDV;            // 16-byte units of a staged row
  constexpr int kKTasks = TR * KU / kThreads, kVTasks = TR * VU / kThreads;
  constexpr int kTileBytes = TR * (KU + VU) * 16;
  constexpr bool kHalfV = DT == LOGKV_BF16 && !SECOND; // V converted to fp16
  constexpr int kPDT = kHalfV ? LOGKV_F16 : DT;        // type of the value products
  constexpr float kVFactor = DT == LOGKV_BF16 && SECOND ? kVScale : 1.f;   // both forms' sums carry V's scale
  static_assert(8 * 16 * 32 * 4 <= kTileBytes, "a tile buffer holds 16 rows' probabilities of every wave");
  const int tid = threadIdx.x, w = wave_id(), l = lane_id(), h = l >> 5, col = l & 31, rw = w / QW;
  const int kunits = a.dk / 8, vunits = a.dv / 8, b = c.b, g = c.g, t = c.t, np = c.np, begin = c.begin, end = c.end;
  const LOGKV_G uint16_t* kc = gp(a.cache_k) + b * a.ck_sb + g * a.ck_sg;
  const LOGKV_G uint16_t* vc = gp(a.cache_v) + b * a.cv_sb + g * a.cv_sg;
  const LOGKV_G uint16_t* ko = gp(a.k) + b * a.k_sb + g * a.k_sg;
  const LOGKV_G uint16_t* vo = gp(a.v) + b * a.v_sb + g * a.v_sg;
  auto k_tile = [&](int bf) { return reinterpret_cast<uint4*>(buf + bf * kTileBytes); };
  auto v_tile = [&](int bf) { return reinterpret_cast<uint4*>(buf + bf * kTileBytes + TR * KU * 16); };

  // Registers of the tile on its way. Rows past the tile's: K repeats the last one (masked in the
  // scores), V is zero; units past dk and dv are zero.
  uint4 kx[kKTasks], vx[kVTasks];
  float bx = 0.f;
  auto load = [&](int ti) {
    const bool of_cache = ti < np;
    const int t0 = TR * (of_cache ? ti : ti - np), rows = min(TR, (of_cache ? c.n : c.own) - t0);
    const int64_t kst = of_cache ? a.ck_st : a.k_st, vst = of_cache ? a.cv_st : a.v_st;
    const LOGKV_G uint16_t* kr = (of_cache ? kc : ko) + t0 * kst;
    const LOGKV_G uint16_t* vr = (of_cache ? vc : vo) + t0 * vst;
#pragma unroll
    for (int q = 0; q < kKTasks; ++q) {
      const int i = tid + kThreads * q, rr = min(i / KU, rows - 1), u = i % KU;
      kx[q] = make_uint4(0, 0, 0, 0);
      if (u < kunits) kx[q] = *(const LOGKV_G uint4*)(kr + rr * kst + 8 * u);
    }
#pragma unroll
    for (int q = 0; q < kVTasks; ++q) {
      const int i = tid + kThreads * q, rr = i / VU, u = i % VU;
      vx[q] = make_uint4(0, 0, 0, 0);
      if (u < vunits && rr < rows) vx[q] = *(const LOGKV_G uint4*)(vr + rr * vst + 8 * u);
    }
    if constexpr (BIAS) {
      if (tid < TR) {
        bx = 0.f;
        if (of_cache) {
          const int64_t at = b * a.b_sb + g * a.b_sg + (t0 + min(tid, rows - 1)) * a.b_st;
          bx = bias_base2(a.bias_half ? Elem<DT>::to_f32(gp(static_cast<const uint16_t*>(a.bias))[at])
                                      : gp(static_cast<const float*>(a.bias))[at]);
        }
      }
    }
  };
  // Flags of a tile's V magnitudes: 1 some at 2^9 (fp16 caches and the second form: not finite) or
  // above, 2 some nonzero, 4 some at 2^-8 or above.
  auto store = [&](int ti, int bf) {
#pragma unroll
    for (int q = 0; q < kKTasks; ++q) {
      const int i = tid + kThreads * q, rr = i / KU, u = i % KU;
      k_tile(bf)[rr * KU + (u ^ swizzle<KU>(rr))] = kx[q];
    }
    u16x2 top = {0, 0};
#pragma unroll
    for (int q = 0; q < kVTasks; ++q) {
      const int i = tid + kThreads * q, rr = i / VU, u = i % VU;
      uint32_t x4[4] = {vx[q].x, vx[q].y, vx[q].z, vx[q].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, x4[j] & 0x7fff7fffu));
        if constexpr (kHalfV) x4[j] = half_of_bf16(x4[j]);
      }
      v_tile(bf)[rr * VU + (u ^ swizzle<VU>(rr))] = make_uint4(x4[0], x4[1], x4[2], x4[3]);
    }
    const int mag = max(static_cast<int>(top[0]), static_cast<int>(top[1]));
    constexpr int kMost = kHalfV ? (127 + 9) << 7 : static_cast<int>(Elem<DT>::kInf), kLeast = (127 - 8) << 7;
    const int bits = (__ballot(mag >= kMost) ? 1 : 0) | (kHalfV ? (__ballot(mag != 0) ? 2 : 0) | (__ballot(mag >= kLeast) ? 4 : 0) : 0);
    if (bits && l == 0) atomicOr(&flag_s[(ti - begin) % 3], bits);
    if constexpr (BIAS) {
      if (tid < TR) bias_s[bf][tid] = bx;
    }
  };
#pragma unroll
  for (int nb = 0; nb < NDV; ++nb)
#pragma unroll
    for (int i = 0; i < 16; ++i) c.o[nb][i] = 0.f;
  c.m = -__builtin_inff();
  c.lsum = 0.f;
  const float c2 = a.scale * kLog2e;
  if (tid < 3) flag_s[tid] = 0;
  __syncthreads();   // the flags are clear
  if (begin < end) {
    load(begin);
    store(begin, 0);
    if (begin + 1 < end) load(begin + 1);
  }
  const int r0 = 32 * RB * rw;   // this wave's rows of a tile
  for (int ti = begin; ti < end; ++ti) {
    const int it = ti - begin, bf = it & 1;
    __syncthreads();   // tile ti is stored, tile ti - 1 has been read
    const int flags = flag_s[it % 3];
    if (!SECOND && ((flags & 1) || (flags & 6) == 2)) return false;
    if (tid == 0) flag_s[(it + 2) % 3] = 0;
    const bool own = ti >= np;
    const int t0 = TR * (own ? ti - np : ti), rows = min(TR, (own ? c.own : c.n) - t0);
    // V^T operand of rows 16 st .. + 15 (in P's order), features 32 nb + l % 32.
    auto load_vt = [&](int nb, int st) {
      const int i = l & 15, ra = r0 + 16 * st + 4 * h + (i >> 2), rb = ra + 8, f = 32 * nb + (l & 16) + 4 * (i & 3);
      const uint16_t* base = reinterpret_cast<const uint16_t*>(v_tile(bf));
      const uint16_t* p0 = base + ra * (8 * VU) + 8 * ((f >> 3) ^ swizzle<VU>(ra)) + (f & 7);
      const uint16_t* p1 = base + rb * (8 * VU) + 8 * ((f >> 3) ^ swizzle<VU>(rb)) + (f & 7);
      const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p0)));
      const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p1)));
      return make_uint4(x.x, x.y, y.x, y.y);
    };
    f32x16 s[RB];
#pragma unroll
    for (int kb = 0; kb < RB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
      for (int kb = 0; kb < RB; ++kb) {
        const int rr = r0 + 32 * kb + col;
        s[kb] = mfma32<DT>(k_tile(bf)[rr * KU + ((2 * ks + h) ^ swizzle<KU>(rr))], c.qf[ks], s[kb]);
      }
    if constexpr (BIAS) {
#pragma unroll
      for (int kb = 0; kb < RB; ++kb)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(&bias_s[bf][r0 + 32 * kb + 8 * i4 + 4 * h]);
#pragma unroll
          for (int i = 0; i < 4; ++i)   // a row hidden by -inf stays hidden whatever its key holds
            s[kb][4 * i4 + i] = x[i] == -__builtin_inff() ? x[i] : __builtin_fmaf(s[kb][4 * i4 + i], c2, x[i]);
        }
    }
    // Masks: element i of block kb is row r0 + 32 kb + 8 (i / 4) + 4 h + i % 4 of the tile.
    if (own || rows < TR) {
      const int lim = (own && r.causal ? min(rows, t + 1 - t0) : rows) - r0 - 4 * h;
#pragma unroll
      for (int kb = 0; kb < RB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int rr = 32 * kb + 8 * (i / 4) + i % 4;
          bool see = rr < lim;
          if (own && !r.causal && see)
            see = gp(a.visible)[b * a.vis_sb + t * a.vis_st + t0 + r0 + 4 * h + rr] != 0;
          if (!see) s[kb][i] = -__builtin_inff();
        }
    }
    float mx = -__builtin_inff();
#pragma unroll
    for (int kb = 0; kb < RB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
    mx = pair_max32(mx);
    const float m_new = fmaxf(c.m, BIAS ? mx : mx * c2);
    const float mb = m_new == -__builtin_inff() ? 0.f : m_new;
    const float corr = __builtin_amdgcn_exp2f(c.m - mb);
    c.m = m_new;
    if (__ballot(corr != 1.f)) {
      c.lsum *= corr;
#pragma unroll
      for (int nb = 0; nb < NDV; ++nb)
#pragma unroll
        for (int i = 0; i < 16; ++i) c.o[nb][i] *= corr;
    }
    uint32_t seen[RB];   // the second form: rows that the query sees
    if constexpr (SECOND) {
#pragma unroll
      for (int kb = 0; kb < RB; ++kb) {
        seen[kb] = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) seen[kb] |= (s[kb][i] != -__builtin_inff() ? 1u : 0u) << (8 * (i / 4) + 4 * h + i % 4);
        seen[kb] |= __shfl_xor(seen[kb], 32, kWave);
      }
    }
    const float arg0 = kPShift - mb;
    float sum = 0.f;
#pragma unroll
    for (int kb = 0; kb < RB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[kb][i] = __builtin_amdgcn_exp2f(BIAS ? s[kb][i] + arg0 : __builtin_fmaf(s[kb][i], c2, arg0));
        sum += s[kb][i];
      }
    c.lsum += sum;
    if (!SECOND || !(flags & 1)) {
#pragma unroll
      for (int st = 0; st < 2 * RB; ++st) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p0 = s[st / 2][8 * (st % 2) + 2 * j], p1 = s[st / 2][8 * (st % 2) + 2 * j + 1];
          if constexpr (kHalfV) hi[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{p0, p1}, f16x2));
          else Elem<DT>::parts(kVFactor * p0, kVFactor * p1, hi[j], lo[j]);
        }
#pragma unroll
        for (int nb = 0; nb < NDV; ++nb) {
          const uint4 v = load_vt(nb, st);
          c.o[nb] = mfma32<kPDT>(v, make_uint4(hi[0], hi[1], hi[2], hi[3]), c.o[nb]);
          if constexpr (!kHalfV) c.o[nb] = mfma32<kPDT>(v, make_uint4(lo[0], lo[1], lo[2], lo[3]), c.o[nb]);
        }
      }
    } else if constexpr (SECOND) {
      // Not finite: row by row in float32, each for the queries that see it. The probabilities pass
      // through the other tile buffer, which holds nothing now.
      float* p_s = reinterpret_cast<float*>(buf + (bf ^ 1) * kTileBytes) + w * 16 * 32;
#pragma unroll
      for (int st = 0; st < 2 * RB; ++st) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int j = 0; j < 8; ++j) p_s[32 * (8 * (j / 4) + 4 * h + j % 4) + col] = kVFactor * s[st / 2][8 * (st % 2) + j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int k = 0; k < 16; ++k) {
          const int rr = r0 + 16 * st + k;
          const float pk = p_s[32 * k + col];
          const bool see = seen[st / 2] >> (16 * (st % 2) + k) & 1;
#pragma unroll
          for (int nb = 0; nb < NDV; ++nb)
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
              const uint16_t* v = reinterpret_cast<const uint16_t*>(v_tile(bf) + rr * VU + ((4 * nb + i4) ^ swizzle<VU>(rr))) + 4 * h;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float x = pk * Elem<DT>::to_f32(v[i]);
                c.o[nb][4 * i4 + i] += see ? x : 0.f;
              }
            }
        }
      }
      __syncthreads();
    }
    if (ti + 1 < end) {
      store(ti + 1, bf ^ 1);
      if (ti + 2 < end) load(ti + 2);
    }
  }
  return true;
}

template <int DT, int NKS, int NDV, int QW, int RB, bool BIAS>
__global__ __launch_bounds__(kThreads, 2) void rows_tile_kernel(logkv_rows_args a, RowsLaunch r) {
  constexpr int RW = 8 / QW, TR = 32 * RB * RW;
  constexpr int kTileBytes = TR * (2 * NKS + 4 * NDV) * 16;
  constexpr int kOutBytes = RW > 1 ? 8 * 32 * 32 * NDV * 4 : 0;
  __shared__ __align__(16) uint8_t buf[2 * kTileBytes > kOutBytes ? 2 * kTileBytes : kOutBytes];
  __shared__ __align__(16) float bias_s[BIAS ? 2 : 1][TR];
  __shared__ int flag_s[3];
  __shared__ float m_s[8][32], l_s[8][32];
  const RowsBlock id = rows_block();
  const int lane = id.lane, G = a.n_groups, tid = threadIdx.x;
  const int rep = a.n_heads / G, nq = rep * a.tq, w = wave_id(), l = lane_id(), h = l >> 5, col = l & 31;
  RowsShare<NKS, NDV> c;
  c.b = lane / G;
  c.g = lane % G;
  c.n = rows_in_use(a, c.b);
  c.own = own_rows(a, c.b);
  const int q_first = id.qb * 32 * QW, q_last = min(q_first + 32 * QW, nq) - 1;
  const int qi = q_first + 32 * (w % QW) + col, qc = min(qi, nq - 1);
  c.t = qc % a.tq;
  // Own rows that some query of the block may see.
  const int t_max = q_first / a.tq == q_last / a.tq ? q_last % a.tq : a.tq - 1;
  const int own_end = r.causal ? min(c.own, t_max + 1) : c.own;
  c.np = (c.n + TR - 1) / TR;
  const int tiles = c.np + (own_end + TR - 1) / TR, share = (tiles + r.splits - 1) / r.splits;
  c.begin = min(id.split * share, tiles);
  c.end = min(c.begin + share, tiles);
  const LOGKV_G uint16_t* qrow = gp(a.q) + c.b * a.q_sb + (c.g * rep + qc / a.tq) * a.q_sh + c.t * a.q_st;
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    c.qf[ks] = make_uint4(0, 0, 0, 0);
    if (2 * ks + h < a.dk / 8) c.qf[ks] = *(const LOGKV_G uint4*)(qrow + 16 * ks + 8 * h);
  }
  if (!rows_tile_share<DT, NKS, NDV, QW, RB, BIAS, false>(a, r, c, buf, bias_s, flag_s)) {
    __syncthreads();
    rows_tile_share<DT, NKS, NDV, QW, RB, BIAS, true>(a, r, c, buf, bias_s, flag_s);
  }
  c.lsum = pair_sum32(c.lsum);
  if (c.t >= c.own || qi >= nq) {   // a query past its batch row's count sees nothing
    c.m = -__builtin_inff();
    c.lsum = 0.f;
#pragma unroll
    for (int nb = 0; nb < NDV; ++nb)
#pragma unroll
      for (int i = 0; i < 16; ++i) c.o[nb][i] = 0.f;
  }
  const float vscale = DT == LOGKV_BF16 ? 1.f / kVScale : 1.f;
  float* part = r.part + (static_cast<int64_t>(lane) * r.splits + id.split) * nq * (a.dv + kRowsPartTail);
  if constexpr (RW == 1) {
    if (qi >= nq) return;
    float* out = part + static_cast<int64_t>(qi) * (a.dv + kRowsPartTail);
    if (h == 0) *reinterpret_cast<float2*>(out + a.dv) = make_float2(c.m, c.lsum);
#pragma unroll
    for (int nb = 0; nb < NDV; ++nb)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const int d = 32 * nb + 8 * i4 + 4 * h;
        f32x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = c.o[nb][4 * i4 + i] * vscale;
        if (d < a.dv) *reinterpret_cast<f32x4*>(out + d) = y;
      }
  } else {
    // The row groups joined in their order.
    constexpr int kLd = 32 * NDV;
    __syncthreads();
    float* acc = reinterpret_cast<float*>(buf) + w * 32 * kLd;
#pragma unroll
    for (int nb = 0; nb < NDV; ++nb)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        f32x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = c.o[nb][4 * i4 + i] * vscale;
        *reinterpret_cast<f32x4*>(acc + col * kLd + 4 * ((8 * nb + 2 * i4 + h) ^ (col & 7))) = y;
      }
    if (h == 0) {
      m_s[w][col] = c.m;
      l_s[w][col] = c.lsum;
    }
    __syncthreads();
    const int queries = min(32 * QW, nq - q_first), units = a.dv / 4 + 1;
    for (int e = tid; e < queries * units; e += kThreads) {
      const int q = e / units, u = e % units, qq = q / 32, cc = q % 32;
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
        else sum += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(buf) + (ww * 32 + cc) * kLd + 4 * (u ^ (cc & 7))) * f;
      }
      if (u == units - 1) sum[0] = mx;
      *reinterpret_cast<f32x4*>(part + static_cast<int64_t>(q_first + q) * (a.dv + kRowsPartTail) + 4 * u) = sum;
    }
  }
}

namespace {

template <int DT, int NKS, int NDV, int QW, int RB>
void launch_one(const logkv_rows_args& a, const RowsLaunch& r, dim3 grid, hipStream_t stream) {
  if (a.bias) hipLaunchKernelGGL((rows_tile_kernel<DT, NKS, NDV, QW, RB, true>), grid, dim3(kThreads), 0, stream, a, r);
  else hipLaunchKernelGGL((rows_tile_kernel<DT, NKS, NDV, QW, RB, false>), grid, dim3(kThreads), 0, stream, a, r);
}

template <int DT, int NKS, int NDV>
void launch_width(const logkv_rows_args& a, const RowsLaunch& r, dim3 grid, hipStream_t stream) {
  if (r.q_waves == 2) launch_one<DT, NKS, NDV, 2, 1>(a, r, grid, stream);
  else if (r.q_waves == 4) launch_one<DT, NKS, NDV, 4, 2>(a, r, grid, stream);
  else launch_one<DT, NKS, NDV, 8, 2>(a, r, grid, stream);
}

template <int DT>
void launch_type(const logkv_rows_args& a, const RowsLaunch& r, dim3 grid, hipStream_t stream) {
  if (a.dk <= 64 && a.dv <= 64) launch_width<DT, 4, 2>(a, r, grid, stream);
  else launch_width<DT, 8, 4>(a, r, grid, stream);
}

}  // namespace

int launch_rows_tile(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream) {
  const int nq = a.n_heads / a.n_groups * a.tq;
  const dim3 grid((nq + 32 * r.q_waves - 1) / (32 * r.q_waves), r.splits, a.n_batch * a.n_groups);
  if (a.dtype == LOGKV_BF16) launch_type<LOGKV_BF16>(a, r, grid, stream);
  else launch_type<LOGKV_F16>(a, r, grid, stream);
  return hipGetLastError() == hipSuccess ? LOGKV_OK : LOGKV_ERUNTIME;
}

}  // namespace logkv
