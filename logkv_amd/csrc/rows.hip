// Attention over a cache's rows and the call's own rows: what follows the streamed products
// (rows_stream.hip), and the sizes of a launch.
#include <algorithm>
#include <type_traits>

#include "rows.hpp"

namespace logkv {

namespace {

constexpr int kThreads = 256;
constexpr int kAppendUnits = 4 * kThreads;  // 16-byte units per block of the append

int64_t align256(int64_t x) { return (x + 255) & ~int64_t(255); }

// Partials join under the largest maximum; an empty one has maximum -inf and zero sums, one of NaN
// logits alone -inf and NaN, so a sum of zero (and only that) means that a query sees no row.

// Maximum and sum of a query over its splits' partials; `threads` lanes of a wave (a power of two)
// take every threads-th split and fold theirs by xor.
__device__ __forceinline__ void fold_splits(const float* base, int64_t step, int splits, int dv, int j, int threads,
                                            float& m, float& lsum) {
  m = -__builtin_inff();
  for (int sp = j; sp < splits; sp += threads) m = fmaxf(m, base[sp * step + dv]);
  for (int off = threads / 2; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
  lsum = 0.f;
  const float top = m == -__builtin_inff() ? 0.f : m;
  for (int sp = j; sp < splits; sp += threads)
    lsum += base[sp * step + dv + 1] * __builtin_amdgcn_exp2f(base[sp * step + dv] - top);
  for (int off = threads / 2; off >= 1; off >>= 1) lsum += __shfl_xor(lsum, off, kWave);
}

}  // namespace

// Roles by blockIdx.x, all of one launch:
//  * [0, out_blocks): outputs. TQ threads per query, four features each; the block's other factor
//    is shared by queries and by groups of splits (QPB queries x SG groups), whose sums are
//    joined in group order.
//  * [out_blocks, + weight_blocks): weights of up to 16 queries from the stored products,
//    p = 2^(s c2 - m) / l, COLS score columns a thread.
//  * the rest: the own rows copied behind the cache's rows.
template <int DT, int TQ, int SG, int COLS>
__global__ __launch_bounds__(kThreads) void rows_finish_kernel(logkv_rows_args a, RowsLaunch r, int out_blocks,
                                                               int weight_blocks) {
  typedef Elem<DT> E;
  constexpr int QPB = kThreads / (TQ * SG);
  const int lane = blockIdx.y, G = a.n_groups, b = lane / G, g = lane % G;
  const int rep = a.n_heads / G, nq = rep * a.tq, tid = threadIdx.x;
  const int stride = a.dv + kRowsPartTail;
  const int64_t step = static_cast<int64_t>(nq) * stride;
  const float* lane_part = r.part + static_cast<int64_t>(lane) * r.room * step;
  const int splits = r.shares ? r.shares[lane] : r.splits;
  int blk = blockIdx.x;
  if (blk < out_blocks) {
    __shared__ __align__(16) float acc_s[QPB][SG][4 * TQ];
    __shared__ float m_s[QPB][SG], l_s[QPB][SG];
    const int qs = tid / (TQ * SG), sg = tid / TQ % SG, d = 4 * (tid % TQ);
    const int qi = blk * QPB + qs;
    const bool there = qi < nq && d < a.dv;
    const float* base = lane_part + static_cast<int64_t>(min(qi, nq - 1)) * stride;
    float m = -__builtin_inff(), lsum = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    // Eight splits' loads at a time, joined under the running maximum.
    for (int s0 = sg; s0 < splits; s0 += 8 * SG) {
      float2 ml[8];
      f32x4 x[8];
      float mx = m;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int sp = s0 + k * SG;
        ml[k] = make_float2(-__builtin_inff(), 0.f);
        x[k] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (there && sp < splits) {
          ml[k] = *reinterpret_cast<const float2*>(base + sp * step + a.dv);
          x[k] = *reinterpret_cast<const f32x4*>(base + sp * step + d);
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) mx = fmaxf(mx, ml[k].x);
      const float top = mx == -__builtin_inff() ? 0.f : mx;
      const float corr = __builtin_amdgcn_exp2f(m - top);
      lsum *= corr;
      acc *= corr;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float f = __builtin_amdgcn_exp2f(ml[k].x - top);
        lsum += ml[k].y * f;
        acc += x[k] * f;
      }
      m = mx;
    }
    if constexpr (SG > 1) {
      *reinterpret_cast<f32x4*>(&acc_s[qs][sg][d]) = acc;
      if (d == 0) {
        m_s[qs][sg] = m;
        l_s[qs][sg] = lsum;
      }
      __syncthreads();
      if (sg) return;
      float mx = m;
#pragma unroll
      for (int k = 1; k < SG; ++k) mx = fmaxf(mx, m_s[qs][k]);
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
      float total = 0.f;
      const float top = mx == -__builtin_inff() ? 0.f : mx;
#pragma unroll
      for (int k = 0; k < SG; ++k) {
        const float f = __builtin_amdgcn_exp2f(m_s[qs][k] - top);
        total += l_s[qs][k] * f;
        sum += *reinterpret_cast<const f32x4*>(&acc_s[qs][k][d]) * f;
      }
      m = mx;
      lsum = total;
      acc = sum;
    }
    if (!there) return;
    const bool empty = lsum == 0.f;
    if (r.lse && d == 0)
      r.lse[static_cast<int64_t>(lane) * nq + qi] = empty ? __builtin_inff() : m + __builtin_amdgcn_logf(lsum) - r.shift;
    uint16_t y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = empty ? uint16_t(0) : E::from_f32(acc[k] / lsum);
    LOGKV_G uint16_t* o = gp(a.out) + b * a.o_sb + (g * rep + qi / a.tq) * a.o_sh + qi % a.tq * a.o_st + d;
    *reinterpret_cast<LOGKV_G uint2*>(o) =
        make_uint2(y[0] | static_cast<uint32_t>(y[1]) << 16, y[2] | static_cast<uint32_t>(y[3]) << 16);
    return;
  }
  blk -= out_blocks;
  const int n = rows_in_use(a, b), own = own_rows(a, b);
  if (blk < weight_blocks) {
    __shared__ float qm[16], ql[16];
    const int np = (n + kRowTile - 1) / kRowTile * kRowTile;
    const int c0 = blk * COLS * kThreads;
    if (c0 >= np + own) return;
    {
      const int q = tid / 16;
      if (q < nq) {
        float m, lsum;
        fold_splits(lane_part + static_cast<int64_t>(q) * stride, step, splits, a.dv, tid % 16, 16, m, lsum);
        if (tid % 16 == 0) {
          qm[q] = r.shift - (m == -__builtin_inff() ? 0.f : m);
          ql[q] = lsum == 0.f ? 0.f : 1.f / lsum;
        }
      }
    }
    __syncthreads();
    const int c = c0 + COLS * tid;
    if (c >= np + own) return;
    const float c2 = a.scale * kLog2e;
    typedef float columns __attribute__((ext_vector_type(COLS)));
    float sum[COLS] = {};
    const float* row = r.scores + static_cast<int64_t>(lane) * nq * r.score_st + c;
    LOGKV_G float* wrow = gp(a.weights) + b * a.w_sb + g * a.w_sg;
    float before[COLS];
#pragma unroll
    for (int k = 0; k < COLS; ++k) before[k] = wrow[min(c + k, a.cap - 1)];
    // QB queries' products loaded at once.
    auto add = [&](auto qb) {
      constexpr int QB = decltype(qb)::value;
      for (int q0 = 0; q0 < nq; q0 += QB) {
        columns s[QB];
#pragma unroll
        for (int q = 0; q < QB; ++q) s[q] = *reinterpret_cast<const columns*>(row + min(q0 + q, nq - 1) * r.score_st);
#pragma unroll
        for (int q = 0; q < QB; ++q) {
          if (q0 + q >= nq || ql[q0 + q] == 0.f) continue;   // a query that sees nothing
#pragma unroll
          for (int k = 0; k < COLS; ++k)
            sum[k] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[q][k], c2, qm[q0 + q])) * ql[q0 + q];
        }
      }
    };
    if (nq <= 2) add(std::integral_constant<int, 2>{});
    else add(std::integral_constant<int, 8>{});
#pragma unroll
    for (int k = 0; k < COLS; ++k) {
      if (c + k < n) wrow[c + k] = before[k] + sum[k];
      else if (c + k >= np && c + k < np + own && n + (c + k - np) < a.cap) wrow[n + (c + k - np)] = sum[k];
    }
    return;
  }
  blk -= weight_blocks;
  const int ku = a.dk / 8, vu = a.dv / 8, total = min(own, a.cap - n) * (ku + vu);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int i = blk * kAppendUnits + k * kThreads + tid;
    if (i >= total) return;
    const int t = i / (ku + vu), u = i % (ku + vu);
    if (u < ku)
      *(LOGKV_G uint4*)(gp(a.cache_k) + b * a.ck_sb + g * a.ck_sg + (n + t) * a.ck_st + 8 * u) =
          *(const LOGKV_G uint4*)(gp(a.k) + b * a.k_sb + g * a.k_sg + t * a.k_st + 8 * u);
    else
      *(LOGKV_G uint4*)(gp(a.cache_v) + b * a.cv_sb + g * a.cv_sg + (n + t) * a.cv_st + 8 * (u - ku)) =
          *(const LOGKV_G uint4*)(gp(a.v) + b * a.v_sb + g * a.v_sg + t * a.v_st + 8 * (u - ku));
  }
}

namespace {

template <int DT, int TQ, int SG, int COLS>
void launch_finish(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream) {
  constexpr int kWeightRows = COLS * kThreads;
  const int nq = a.n_heads / a.n_groups * a.tq, qpb = kThreads / (TQ * SG);
  const int out_blocks = (nq + qpb - 1) / qpb;
  const int weight_blocks = r.scores ? static_cast<int>((r.score_st + kWeightRows - 1) / kWeightRows) : 0;
  const int append_blocks = r.causal ? (a.tq * (a.dk / 8 + a.dv / 8) + kAppendUnits - 1) / kAppendUnits : 0;
  hipLaunchKernelGGL((rows_finish_kernel<DT, TQ, SG, COLS>),
                     dim3(out_blocks + weight_blocks + append_blocks, a.n_batch * a.n_groups), dim3(kThreads), 0, stream, a, r,
                     out_blocks, weight_blocks);
}

template <int DT, int TQ, int SG>
void launch_finish_cols(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream) {
  // Four columns a thread where two would make more blocks than stay resident: 64 lanes of 32768 rows 14.1 us (two:
  // 17.8), 64 lanes of 4096 rows 9.1 (8.0).
  if (r.scores && r.score_st * a.n_batch * a.n_groups >= 2048 * 2 * kThreads) launch_finish<DT, TQ, SG, 4>(a, r, stream);
  else launch_finish<DT, TQ, SG, 2>(a, r, stream);
}

template <int DT>
void launch_finish_type(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream) {
  // Groups of splits share a query where eight queries a block would not fill the CUs: 1 x 32768 rows of 8 heads and
  // 512 queries without them 145 us, with them 145 - 152; 4096 rows and 666 queries 55 and 62 us.
  const bool many = r.splits > 8 && static_cast<int64_t>(a.n_batch) * a.n_heads * a.tq < 8 * 256;
  if (a.dv <= 128) {
    if (many) launch_finish_cols<DT, 32, 8>(a, r, stream);
    else launch_finish_cols<DT, 32, 1>(a, r, stream);
  } else {
    if (many) launch_finish_cols<DT, 64, 4>(a, r, stream);
    else launch_finish_cols<DT, 64, 1>(a, r, stream);
  }
}

// Splits of the tiled kernel: rounds of blocks over the CUs, each of a split's tiles and two more
// for its start and end, and for more than one split two tiles' time for the join and the partials.
int tile_splits(const logkv_rows_args& a, int64_t blocks, int q_waves) {
  const int rows = 64, resident = q_waves == 2 ? 512 : 256;
  const int64_t tiles = (a.cap + rows - 1) / rows + (a.tq + rows - 1) / rows;
  int best = 1;
  int64_t best_cost = INT64_MAX;
  for (int64_t s = 1; s <= std::min<int64_t>(kMaxRowSplits, tiles); ++s) {
    const int64_t rounds = (blocks * s + resident - 1) / resident;
    const int64_t cost = 32 * (rounds * ((tiles + s - 1) / s + 2) + (s > 1 ? 2 : 0)) + (s > 1 ? blocks * s / 2 : 0);
    if (cost < best_cost) {
      best_cost = cost;
      best = static_cast<int>(s);
    }
  }
  return best;
}

}  // namespace

RowsLaunch rows_launch(const logkv_rows_args& a, bool causal, void* ws) {
  const int64_t lanes = static_cast<int64_t>(a.n_batch) * a.n_groups, nq = static_cast<int64_t>(a.n_heads / a.n_groups) * a.tq;
  const bool wide = a.dk > 128 || a.dv > 128;
  RowsLaunch r{};
  r.causal = causal ? 1 : 0;
  r.bias2 = (a.bias_scale == 0.f ? 1.f : a.bias_scale) * kLog2e;
  const int64_t tiles = (a.cap + kRowTile - 1) / kRowTile + (a.tq + kRowTile - 1) / kRowTile;
  // More than 32 queries: tiles in LDS. From 17 on too where rows of more than 64 features are many: the streaming
  // kernel's two query blocks spill there, and the tiled kernel pays a launch more. Streaming and tiled, 128 features, 8
  // lanes of 32768 rows, 32 queries: 46.8 and 40.3 us (fp16: 46.4 and 39.8); 64 lanes of 8192, 20: 74.8 and 59.5 (74.4
  // and 57.1); 8 lanes of 2048, 24: 16.3 and 19.2. At 64 features nothing spills: 64 lanes of 16000 rows, 30: 51 and 67.
  const bool rows_pay = nq > 16 && (a.dk > 64 || a.dv > 64) && lanes * a.cap >= 1 << 17;
  if (!wide && (nq > 32 || rows_pay)) {
    r.q_waves = nq <= 64 ? 2 : nq <= 128 ? 4 : 8;
    r.shift = kTileShift;
    r.splits = tile_splits(a, lanes * ((nq + 32 * r.q_waves - 1) / (32 * r.q_waves)), r.q_waves);
  } else {
    // Wide rows' two query blocks spill; read twice instead up to 128 queries: 32 lanes of 16000 rows of 192 and 128
    // features, 24 queries: 155 us, in blocks of 16 queries 114; 8 lanes of 8000 rows of 256, 256 queries: 117 and 123.
    r.cols = nq <= 16 || (wide && nq <= 128) ? 1 : 2;
    r.shift = a.dtype == LOGKV_F16 ? Elem<LOGKV_F16>::kShift : Elem<LOGKV_BF16>::kShift;
    const int64_t q_blocks = (nq + 16 * r.cols - 1) / (16 * r.cols);
    // One share per resident block, none shorter than a tile for each of its waves.
    const int64_t resident = wide ? 256 : 512;
    r.splits = static_cast<int>(std::max<int64_t>(
        1, std::min<int64_t>({kMaxRowSplits, (tiles + 3) / 4, resident / std::max<int64_t>(1, lanes * q_blocks)})));
  }
  uint8_t* base = static_cast<uint8_t*>(ws);
  int64_t off = 0;
  auto take = [&](int64_t floats) {
    float* p = base ? reinterpret_cast<float*>(base + off) : nullptr;
    off += align256(4 * floats);
    return p;
  };
  // Shares by length (rows_tile.hip): a lane may take up to twice the equal number.
  const bool by_length = r.q_waves && r.splits > 1 && a.n_batch > 1 && a.n_batch <= kWave;
  r.room = by_length ? 2 * r.splits : r.splits;
  r.part = take(lanes * r.room * nq * (a.dv + kRowsPartTail));
  if (r.q_waves) r.redo = reinterpret_cast<int*>(take(lanes * r.splits * ((nq + 32 * r.q_waves - 1) / (32 * r.q_waves))));
  if (causal && nq <= 16) {
    r.score_st = tiles * kRowTile;
    r.scores = take(lanes * nq * r.score_st);
  } else if (causal) {
    r.lse = take(lanes * nq);
  }
  if (by_length) {
    r.shares = reinterpret_cast<int*>(take(lanes));
    if (!a.lengths || !a.len_stride) r.shares = nullptr;   // sequences of one length
  }
  r.bytes = off;
  return r;
}

int launch_rows_attention(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream) {
  const int rc = r.q_waves ? launch_rows_tile(a, r, stream) : launch_rows_stream(a, r, stream);
  if (rc) return rc;
  if (a.dtype == LOGKV_BF16) launch_finish_type<LOGKV_BF16>(a, r, stream);
  else launch_finish_type<LOGKV_F16>(a, r, stream);
  if (r.lse) return launch_rows_weight(a, r, stream);
  return hipGetLastError() == hipSuccess ? LOGKV_OK : LOGKV_ERUNTIME;
}

}  // namespace logkv
