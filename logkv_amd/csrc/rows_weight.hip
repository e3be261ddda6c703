// Attention weights of more than 16 queries per KV group: with a query's base-2 log-sum-exp L known,
//   weight_j = sum over queries of 2^(s_j c2 - L),  c2 = scale log2(e).
// S = Q K^T by 32x32x16 matrix products with the keys as columns, so a lane sums its own key over
// the queries in registers: a wave holds 32 KB keys' operands for good, and the block's queries pass
// through LDS, a tile of 64, two buffers, the next tile's rows on their way in registers. The products
// of one 32x32 block and the exponentials of the one before are independent and interleaved: both
// take about as long (16 quarter-rate exponentials a lane against eight products of 32 cycles at 128
// features). One wave owns a key: no atomics, a fixed order. 8 lanes of 30720 rows and 2048 new ones,
// 4096 queries of 128 features: 374 - 393 us, 680 - 710 TFLOP/s; the vector unit and the matrix cores are
// busy 49% and 32% of the cycles. 32 keys a wave (twice the reads of Q): 50 us more.
#include <algorithm>
#include <type_traits>

#include "rows.hpp"

namespace logkv {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;

template <int DT>
__device__ __forceinline__ f32x16 mfma32(uint4 x, uint4 y, f32x16 c) {
  if constexpr (DT == LOGKV_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
}

// Where 16-byte unit u of row r is stored: u ^ swizzle, so that 8 rows' reads of one unit meet
// every bank once (8, 16 or 32 units a row).
template <int UNITS>
__device__ __forceinline__ int swizzle(int r) {
  return UNITS == 8 ? (r >> 1 & 1) << 2 | (r >> 2 & 3) : (r & 3) << 2 | (r >> 2 & 3);
}

}  // namespace

// NKS 16-wide steps of dk, KB 32-key blocks per wave, QG groups of waves that share a tile's queries.
template <int DT, int NKS, int KB, int QG>
__global__ __launch_bounds__(kThreads, 2) void rows_weight_kernel(logkv_rows_args a, RowsLaunch r, int cache_blocks) {
  constexpr int kQueries = NKS > 8 ? 32 : 64;   // per staged tile (64 of 256 features spill: 8 lanes, 4096 rows, 400
                                                // queries 200 us the call, 149)
  constexpr int KU = 2 * NKS, kTasks = kQueries * KU / kThreads, kKeyWaves = 4 / QG, kKeys = kKeyWaves * 32 * KB;
  __shared__ __align__(16) uint4 q_s[2][kQueries * KU];
  __shared__ __align__(16) float l_s[2][kQueries];
  __shared__ __align__(16) int t_s[2][kQueries];
  const int lane = blockIdx.y, G = a.n_groups, b = lane / G, g = lane % G, tid = threadIdx.x;
  const int rep = a.n_heads / G, nq = rep * a.tq, units = a.dk / 8;
  const int w = wave_id(), l = lane_id(), col = l & 31, h = l >> 5;
  const int n = rows_in_use(a, b), own = own_rows(a, b);
  // Blocks of the cache's rows, then of the own rows. Fewer queries see a later own block: lanes take them in turned
  // order, or the XCD that a multiple of eight blocks a lane hands all first ones ends last (30720 rows and 2048 new
  // ones: 439 us against 340 on the XCD of the last ones).
  const int x = blockIdx.x, own_blocks = gridDim.x - cache_blocks;
  const bool of_cache = x < cache_blocks;
  const int rows = of_cache ? n : own, b0 = (of_cache ? x : (x - cache_blocks + lane) % own_blocks) * kKeys;
  if (b0 >= rows || own == 0) return;
  const int k0 = b0 + w % kKeyWaves * 32 * KB, q_block = w / kKeyWaves * (kQueries / 32 / QG);   // the wave's first query block of a tile
  const LOGKV_G uint16_t* kr = of_cache ? gp(a.cache_k) + b * a.ck_sb + g * a.ck_sg : gp(a.k) + b * a.k_sb + g * a.k_sg;
  const int64_t kst = of_cache ? a.ck_st : a.k_st;
  uint4 kf[KB][NKS];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      kf[kb][ks] = make_uint4(0, 0, 0, 0);
      if (2 * ks + h < units)
        kf[kb][ks] = *(const LOGKV_G uint4*)(kr + min(k0 + 32 * kb + col, rows - 1) * kst + 16 * ks + 8 * h);
    }
  const LOGKV_G float* lse = gp(r.lse) + static_cast<int64_t>(lane) * nq;
  // Each task's unit of the tile on its way, moved on by a tile without a product or a division.
  static_assert(kThreads % KU == 0, "a thread's tasks share a unit");
  const int unit = tid % KU, step_t = kQueries % a.tq;
  const int64_t step = kQueries / a.tq * a.q_sh + step_t * a.q_st, wrap = a.q_sh - a.tq * a.q_st;
  const LOGKV_G uint16_t* qp[kTasks];
  int pos[kTasks];
#pragma unroll
  for (int k = 0; k < kTasks; ++k) {
    const int qq = (tid + kThreads * k) / KU;
    pos[k] = qq % a.tq;
    qp[k] = gp(a.q) + b * a.q_sb + (g * rep + qq / a.tq) * a.q_sh + pos[k] * a.q_st + 8 * unit;
  }
  int my_t = tid % a.tq;   // of query tid of the tile (tid < kQueries)
  // A key's position for the masks: the cache's rows are before every query.
  const int key0 = of_cache ? 0 : k0 + col, key_step = of_cache ? 0 : 32;
  uint4 qx[kTasks];
  float lx = 0.f;
  int tx = 0;
  // Queries past nq or the row's tokens are stored as zeros before every key (position -1): L = +inf alone would not
  // do, since a key's infinity times zero is NaN.
  auto load = [&](int q0) {
#pragma unroll
    for (int k = 0; k < kTasks; ++k) {
      qx[k] = make_uint4(0, 0, 0, 0);
      if (unit < units && q0 + (tid + kThreads * k) / KU < nq && pos[k] < own) qx[k] = *(const LOGKV_G uint4*)qp[k];
      qp[k] += step;
      pos[k] += step_t;
      if (pos[k] >= a.tq) {
        pos[k] -= a.tq;
        qp[k] += wrap;
      }
    }
    if (tid < kQueries) lx = q0 + tid < nq ? lse[q0 + tid] : __builtin_inff();
    tx = q0 + tid < nq && my_t < own ? my_t : -1;
    my_t += step_t;
    if (my_t >= a.tq) my_t -= a.tq;
  };
  auto store = [&](int bf) {
#pragma unroll
    for (int k = 0; k < kTasks; ++k) {
      const int qq = (tid + kThreads * k) / KU;
      q_s[bf][qq * KU + (unit ^ swizzle<KU>(qq))] = qx[k];
    }
    if (tid < kQueries) {
      l_s[bf][tid] = lx;
      t_s[bf][tid] = tx;
    }
  };
  load(0);
  store(0);
  if (kQueries < nq) load(kQueries);
  float sum[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) sum[kb] = 0.f;
  const float c2 = a.scale * kLog2e;
  const int tiles = (nq + kQueries - 1) / kQueries;
  int t_first = 0;   // position of the tile's first query
  for (int it = 0; it < tiles; ++it) {
    const int bf = it & 1;
    __syncthreads();   // tile it is stored, tile it - 1 has been read
    // Own rows: no query of the tile is as late as the wave's first key.
    const bool none = !of_cache && t_first + kQueries <= a.tq && t_first + kQueries <= k0;
    t_first += step_t;
    if (t_first >= a.tq) t_first -= a.tq;
    // Operand ks of the 32 queries of block qb.
    auto frag = [&](int qb, int ks) {
      const int qq = 32 * qb + col;
      return q_s[bf][qq * KU + ((2 * ks + h) ^ swizzle<KU>(qq))];
    };
    auto tile = [&](auto mask_tag) {
      constexpr bool MASK = decltype(mask_tag)::value;
      constexpr int kBlocks = kQueries / 32 * KB / QG, kShare = 16 / NKS;   // 32x32 blocks; exponentials per product
      uint4 qa[NKS];
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) qa[ks] = frag(q_block, ks);
      f32x16 s, next;
#pragma unroll
      for (int i = 0; i < 16; ++i) next[i] = 0.f;
      f32x4 x[4];
      i32x4 t[4];
#pragma unroll
      for (int blk = 0; blk <= kBlocks; ++blk) {
        // The products of block blk among the exponentials of block blk - 1.
        s = next;
        if (blk > 0) {
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            x[i4] = *reinterpret_cast<const f32x4*>(&l_s[bf][32 * (q_block + (blk - 1) / KB) + 8 * i4 + 4 * h]);
            if constexpr (MASK) t[i4] = *reinterpret_cast<const i32x4*>(&t_s[bf][32 * (q_block + (blk - 1) / KB) + 8 * i4 + 4 * h]);
          }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) next[i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
          if (blk < kBlocks) {
            next = mfma32<DT>(qa[ks], kf[blk % KB][ks], next);
            if (blk % KB == KB - 1 && blk + 1 < kBlocks) qa[ks] = frag(q_block + (blk + 1) / KB, ks);
          }
          if (blk > 0) {
            // Element i is query 32 (q_block + (blk - 1) / KB) + 8 (i / 4) + 4 h + i % 4 against key 32 ((blk - 1) % KB) + col.
#pragma unroll
            for (int i = kShare * ks; i < kShare * (ks + 1); ++i) {
              float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c2, -x[i / 4][i % 4]));
              if (MASK && key0 + key_step * ((blk - 1) % KB) > t[i / 4][i % 4]) p = 0.f;
              sum[(blk - 1) % KB] += p;
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    // Against the cache's rows only padding is masked: past the last query, or in a padded batch.
    if (of_cache && own == a.tq && kQueries * (it + 1) <= nq) tile(std::false_type{});
    else if (!none) tile(std::true_type{});
    if (it + 1 < tiles) {
      store(bf ^ 1);
      if (it + 2 < tiles) load(kQueries * (it + 2));
    }
  }
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) sum[kb] += __shfl_xor(sum[kb], 32, kWave);
  if constexpr (QG > 1) {
    // The groups' sums joined in their order.
    __shared__ float sum_s[4][KB][32];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      if (h == 0) sum_s[w][kb][col] = sum[kb];
    __syncthreads();
    if (w >= kKeyWaves) return;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int k = 1; k < QG; ++k) sum[kb] += sum_s[k * kKeyWaves + w][kb][col];
  }
  LOGKV_G float* wrow = gp(a.weights) + b * a.w_sb + g * a.w_sg;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    const int j = k0 + 32 * kb + col;
    if (h || j >= rows) continue;
    if (of_cache) wrow[j] += sum[kb];
    else if (n + j < a.cap) wrow[n + j] = sum[kb];
  }
}

namespace {

template <int DT, int NKS, int KB, int QG>
void launch_one(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream) {
  constexpr int kKeys = 4 / QG * 32 * KB;
  const int cache_blocks = (a.cap + kKeys - 1) / kKeys;
  const dim3 grid(cache_blocks + (a.tq + kKeys - 1) / kKeys, a.n_batch * a.n_groups);
  hipLaunchKernelGGL((rows_weight_kernel<DT, NKS, KB, QG>), grid, dim3(kThreads), 0, stream, a, r, cache_blocks);
}

template <int DT>
void launch_type(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream) {
  // 64 keys a wave where that leaves two blocks for every CU; two waves to 32 keys, each half of the queries, where
  // four waves of 32 keys would leave less than two blocks (4 lanes of 2048 rows, 2000 queries of 128 features: 78.5 us
  // the call, 85.1 without; 8 lanes of 4096, 666: 66.0 and 66.7).
  const int64_t keys = (static_cast<int64_t>(a.cap) + a.tq) * a.n_batch * a.n_groups;
  const bool many = keys >= 512 * 256, few = keys < 512 * 128;
  if (a.dk <= 64) {
    if (many) launch_one<DT, 4, 2, 1>(a, r, stream);
    else if (few) launch_one<DT, 4, 1, 2>(a, r, stream);
    else launch_one<DT, 4, 1, 1>(a, r, stream);
  } else if (a.dk <= 128) {
    if (many) launch_one<DT, 8, 2, 1>(a, r, stream);
    else if (few) launch_one<DT, 8, 1, 2>(a, r, stream);
    else launch_one<DT, 8, 1, 1>(a, r, stream);
  } else {
    launch_one<DT, 16, 1, 1>(a, r, stream);
  }
}

}  // namespace

int launch_rows_weight(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream) {
  if (a.dtype == LOGKV_BF16) launch_type<LOGKV_BF16>(a, r, stream);
  else launch_type<LOGKV_F16>(a, r, stream);
  return hipGetLastError() == hipSuccess ? LOGKV_OK : LOGKV_ERUNTIME;
}

}  // namespace logkv
