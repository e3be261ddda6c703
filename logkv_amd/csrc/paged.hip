// Attention of a batch over a paged cache, with prefixes that several sequences share.
//
// Softmax over [prefix | own pages | the call's rows] splits by rows: each part gives a query an
// unnormalised sum, a maximum and a sum of exponentials, which join under the largest maximum. So a
// prefix's rows are read once for all of its sequences: their queries (sequences x heads of the KV group
// x tokens) are the columns of one product, in the kernel that so many columns take (plan_passes), and a
// sequence's own rows are read in a second pass of few columns. Both passes are the row attention
// kernels over a page table, in one launch where their kernels go together; this file joins their partials.
// An infinity or NaN in V is left out of a pass's products, which would spread it to queries that do not
// see its row. Every query of a lane sees the same cache rows: a share that met some in them looks at its rows
// once more and leaves the features that they are in, and the join adds those. A call with one among 32768 shared
// rows of 128 features takes 76 us, without 32; among 2^19 rows of 64 features 265 and 95. Those of the call's rows,
// which queries see by their place or mask, the join looks for itself: up to tq rows a query, four at a time.
//
// 64 sequences of 32 heads over 16384 shared rows and 2000 of their own (8 KV groups, 128 features): 110 us, 4.2 TB/s. 8
// sequences of 256 tokens x 16 heads over 32768 shared rows: 862 - 912 us, 605 - 640 TFLOP/s. Bound by what bounds the
// passes; few queries by the launches, 9 us of the first and 4 of the join for 4 sequences over 2048 rows.
#include <algorithm>
#include <array>
#include <cmath>

#include "paged.hpp"

namespace logkv {

namespace {

constexpr int kThreads = 256;

int64_t align256(int64_t x) { return (x + 255) & ~int64_t(255); }

}  // namespace

// Values that are infinite or NaN added to the query's features; others are in its sum.
template <int DT>
__device__ __forceinline__ void add_odd(uint2 x, f32x4& y) {
  const uint32_t v[4] = {x.x & 0xffffu, x.x >> 16, x.y & 0xffffu, x.y >> 16};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if ((v[k] & 0x7fffu) >= Elem<DT>::kInf) y[k] += Elem<DT>::to_f32(static_cast<uint16_t>(v[k]));
}

// Those of the call's rows that query t of sequence b sees.
template <int DT>
__device__ __forceinline__ void add_odd_rows(const logkv_rows_args& a, bool causal, int b, int g, int t, int d, f32x4& y) {
  const int own = own_rows(a, b), n = causal ? min(own, t + 1) : own;
  const LOGKV_G uint16_t* base = gp(a.v) + b * a.v_sb + g * a.v_sg + d;
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += 4) {
    uint2 x[4];
    bool see[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = min(i0 + k, n - 1);   // (the last row again adds nothing new)
      x[k] = *(const LOGKV_G uint2*)(base + i * a.v_st);
      see[k] = causal || gp(a.visible)[b * a.vis_sb + t * a.vis_st + i] != 0;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (see[k]) add_odd<DT>(x[k], y);
  }
}

// What the join reads of a pass: the partials of a lane, [room][queries][dv + kRowsPartTail] each.
struct FinishPass {
  const float* part;
  const int* shares;   // partials of a lane, null: `splits` of each
  int splits, room;
  int seqs;            // sequences of a lane, 0: no such pass
  float unit;          // the sums' scale
  const uint32_t* odd; // what a share's note says of its cache rows (RowsLaunch)
  int q_blocks, block_queries;
};
// What every block reads comes first; the own pass itself is for the call's rows that a note is of.
struct FinishArgs {
  FinishPass own, shared;
  uint16_t* out;
  int64_t o_sb, o_sh, o_st;
  const int32_t* counts;
  int n_groups, rep, tq, dv;
  PagedPass own_pass;
};

// TQ threads per query, four features each; the block's other factor is shared by queries and by groups of
// partials (QPB queries x SG groups), joined in group order. A query's partials are its own ones, then its prefix's.
template <int DT, int TQ, int SG>
__global__ __launch_bounds__(kThreads) void paged_finish_kernel(FinishArgs a) {
  typedef Elem<DT> E;
  constexpr int QPB = kThreads / (TQ * SG);
  __shared__ __align__(16) float acc_s[QPB][SG][4 * TQ];
  __shared__ float m_s[QPB][SG], l_s[QPB][SG];
  __shared__ float2 odd_s[QPB][SG];
  const int G = a.n_groups, b = static_cast<int>(blockIdx.y) / G, g = static_cast<int>(blockIdx.y) - b * G;
  const int nq = a.rep * a.tq, tid = threadIdx.x, stride = a.dv + kRowsPartTail;
  const int qs = tid / (TQ * SG), sg = tid / TQ % SG, d = 4 * (tid % TQ);
  const int qi = static_cast<int>(blockIdx.x) * QPB + qs, qc = min(qi, nq - 1), head = qc / a.tq, t = qc - head * a.tq;
  const bool there = qi < nq && d < a.dv;
  const bool live = !a.counts || t < gp(a.counts)[b];   // a query past its sequence's count sees nothing
  // The two passes' partials of this query, and how far the next ones are.
  const int lane = static_cast<int>(blockIdx.y);
  int n_own = a.own.splits, n_shared = 0;
  if (a.own.shares) n_own = gp(a.own.shares)[lane];
  const int64_t own_step = static_cast<int64_t>(nq) * stride;
  const LOGKV_G float* own = gp(a.own.part) + lane * (a.own.room * own_step) + static_cast<int64_t>(qc) * stride;
  const LOGKV_G float* shared = own;
  int64_t shared_step = 0;
  if (a.shared.seqs) {
    const int run = b / a.shared.seqs, run_lane = run * G + g, s = b - run * a.shared.seqs;
    n_shared = a.shared.splits;
    if (a.shared.shares) n_shared = gp(a.shared.shares)[run_lane];
    shared_step = a.shared.seqs * own_step;
    shared = gp(a.shared.part) + run_lane * (a.shared.room * shared_step) + static_cast<int64_t>(s * nq + qc) * stride;
  }
  const int all = live ? n_own + n_shared : 0;
  float m = -__builtin_inff(), lsum = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float odd[2] = {0.f, 0.f};   // the partials' notes: of cache rows, of the call's
  // Eight partials' loads at a time, joined under the running maximum.
  for (int s0 = sg; s0 < all; s0 += 8 * SG) {
    f32x4 ml[8], x[8];
    float mx = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int sp = s0 + k * SG;
      ml[k] = f32x4{-__builtin_inff(), 0.f, 0.f, 0.f};
      x[k] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (there && sp < all) {
        const LOGKV_G float* at = sp < n_own ? own + sp * own_step : shared + (sp - n_own) * shared_step;
        ml[k] = *reinterpret_cast<const LOGKV_G f32x4*>(at + a.dv);
        x[k] = *reinterpret_cast<const LOGKV_G f32x4*>(at + d);
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) mx = fmaxf(mx, ml[k][0]);
    const float top = mx == -__builtin_inff() ? 0.f : mx;
    const float corr = __builtin_amdgcn_exp2f(m - top);
    lsum *= corr;
    acc *= corr;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool of_own = s0 + k * SG < n_own;
      const float f = (of_own ? a.own.unit : a.shared.unit) * __builtin_amdgcn_exp2f(ml[k][0] - top);
      lsum += ml[k][1] * f;
      acc += x[k] * f;
      odd[0] += ml[k][2];
      odd[1] += ml[k][3];
    }
    m = mx;
  }
  if constexpr (SG > 1) {
    *reinterpret_cast<f32x4*>(&acc_s[qs][sg][d]) = acc;
    if (d == 0) {
      m_s[qs][sg] = m;
      l_s[qs][sg] = lsum;
      odd_s[qs][sg] = make_float2(odd[0], odd[1]);
    }
    __syncthreads();
    if (sg) return;
    float mx = m;
#pragma unroll
    for (int k = 1; k < SG; ++k) mx = fmaxf(mx, m_s[qs][k]);
    const float top = mx == -__builtin_inff() ? 0.f : mx;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < SG; ++k) {
      const float f = __builtin_amdgcn_exp2f(m_s[qs][k] - top);
      total += l_s[qs][k] * f;
      if (k) odd[0] += odd_s[qs][k].x, odd[1] += odd_s[qs][k].y;
      sum += *reinterpret_cast<const f32x4*>(&acc_s[qs][k][d]) * f;
    }
    lsum = total;
    acc = sum;
  }
  if (!there) return;
  f32x4 z = {0.f, 0.f, 0.f, 0.f};
  if (lsum != 0.f) z = acc / lsum;
  if (__builtin_expect(odd[0] + odd[1] > 0.f, 0)) {
    uint32_t pos = 0, neg = 0;
    if (odd[0] > 0.f) {
#pragma unroll 1
      for (int sp = 0; sp < all; ++sp) {
        const bool of_own = sp < n_own;
        const LOGKV_G float* at = of_own ? own + sp * own_step : shared + (sp - n_own) * shared_step;
        if (at[a.dv + 2] == 0.f) continue;
        const FinishPass& p = of_own ? a.own : a.shared;
        const int run = of_own ? b : b / a.shared.seqs, q = of_own ? qc : (b - run * a.shared.seqs) * nq + qc;
        const int64_t share = static_cast<int64_t>(run * G + g) * p.room + (of_own ? sp : sp - n_own);
        const LOGKV_G uint32_t* words = gp(p.odd) + (share * p.q_blocks + q / p.block_queries) * 16 + d / 32;
        pos |= words[0] >> d % 32;
        neg |= words[8] >> d % 32;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (pos >> k & 1) z[k] += __builtin_inff();
      if (neg >> k & 1) z[k] -= __builtin_inff();
    }
    if (odd[1] > 0.f) add_odd_rows<DT>(a.own_pass.args, a.own_pass.launch.causal != 0, b, g, t, d, z);
  }
  uint16_t y[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) y[k] = E::from_f32(z[k]);
  LOGKV_G uint16_t* o = gp(a.out) + b * a.o_sb + (g * a.rep + head) * a.o_sh + t * a.o_st + d;
  *reinterpret_cast<LOGKV_G uint2*>(o) =
      make_uint2(y[0] | static_cast<uint32_t>(y[1]) << 16, y[2] | static_cast<uint32_t>(y[3]) << 16);
}

namespace {

template <int DT, int TQ, int SG>
void launch_finish(const PagedLaunch& p, hipStream_t stream) {
  const logkv_rows_args& a = p.own.args;
  const int rep = a.n_heads / a.n_groups, nq = rep * a.tq, qpb = kThreads / (TQ * SG);
  auto pass = [](const RowsLaunch& r) {
    return FinishPass{r.part, r.shares, r.splits, r.room, r.seqs, exp2f(-r.shift), r.odd, r.q_blocks, paged_block_queries(r)};
  };
  const FinishArgs args = {pass(p.own.launch), pass(p.shared.launch), a.out, a.o_sb, a.o_sh, a.o_st, a.counts,
                           a.n_groups, rep, a.tq, a.dv, p.own};
  hipLaunchKernelGGL((paged_finish_kernel<DT, TQ, SG>), dim3((nq + qpb - 1) / qpb, a.n_batch * a.n_groups), dim3(kThreads),
                     0, stream, args);
}

template <int DT>
void launch_finish_type(const PagedLaunch& p, hipStream_t stream) {
  const logkv_rows_args& a = p.own.args;
  // Groups of partials share a query where eight queries a block would not fill the CUs. The whole call without, by this
  // rule and with them always: 8 heads x 4 sequences over 2000 rows 12.9, 11.6 and 11.8 us, one sequence of 16 heads over
  // 30000 32.0, 27.5 and 27.3; 64 sequences of 32 heads over 4000 36.3, 36.5 and 38.8, 128 of 16 heads 51.8, 51.8 and 54.4.
  const bool many = std::max(p.own.launch.splits, p.shared.launch.splits) > 8 &&
                    static_cast<int64_t>(a.n_batch) * a.n_heads * a.tq < 8 * 256;
  if (a.dv <= 64) {
    if (many) launch_finish<DT, 16, 8>(p, stream);
    else launch_finish<DT, 16, 1>(p, stream);
  } else if (a.dv <= 128) {
    if (many) launch_finish<DT, 32, 8>(p, stream);
    else launch_finish<DT, 32, 1>(p, stream);
  } else {
    if (many) launch_finish<DT, 64, 4>(p, stream);
    else launch_finish<DT, 64, 1>(p, stream);
  }
}

int launch_passes(const PagedPass& shared, const PagedPass& own, hipStream_t stream) {
  const logkv_rows_args& a = own.args;
  const int width = std::max(a.dk, a.dv);
  if (a.dtype == LOGKV_BF16)
    return width <= 64    ? launch_paged_bf16_64(shared, own, stream)
           : width <= 128 ? launch_paged_bf16_128(shared, own, stream)
                          : launch_paged_bf16_256(shared, own, stream);
  return width <= 64    ? launch_paged_f16_64(shared, own, stream)
         : width <= 128 ? launch_paged_f16_128(shared, own, stream)
                        : launch_paged_f16_256(shared, own, stream);
}

}  // namespace

// How a call is run: per pass the tiled kernel's query waves (0: the streamed kernel's columns) and the shares of a lane.
struct PagedPlan {
  int own_waves, own_cols, own_splits;
  int shared_waves, shared_cols, shared_splits;
};

// A pass by one of the kernels. A block takes steps of some rows, `us` microseconds each, and block_us to begin and end; a
// step keeps a CU busy for cu_us (the rest overlaps with another block's). Measured on passes alone and together, 128
// features (64: 0.62 of a step): the tiled kernel's 64 rows 2.2 us for 64 queries, 2.1 for 128 and 3.1 for 256; the
// streamed kernel's 32 rows a wave 1.7 us for 16 queries, 3.1 for 32. 256 features: the tiled kernel's 32 rows 2.9 us for
// 128 queries, the streamed kernel's 3.4 us for 16.
struct PassCost {
  int64_t lanes;   // 0: no such pass
  int q_blocks, queries, steps;
  float us, cu_us, block_us, bytes_us;

  PassCost(const PagedPass& p, int q_waves, int cols, int waves) {
    const logkv_rows_args& a = p.args;
    const int width = std::max(a.dk, a.dv);
    const bool wide = width > 128;
    lanes = p.launch.seqs ? static_cast<int64_t>(a.n_batch) * a.n_groups : 0;
    queries = a.n_heads / a.n_groups * a.tq * p.launch.seqs;
    const int block_queries = q_waves ? 32 * q_waves : 16 * cols, step_rows = !q_waves ? 32 * waves : wide ? 32 : 64;
    q_blocks = (queries + block_queries - 1) / block_queries;
    const int rows = a.cap + (p.launch.prefix ? 0 : a.tq);
    steps = std::max(1, (rows + step_rows - 1) / step_rows);
    if (q_waves && wide) {
      us = cu_us = 2.9f;
    } else {
      const float factor = (width <= 64 ? 0.62f : wide ? 2.f : 1.f) * (q_waves == 0 && cols == 2 ? 1.8f : 1.f);
      us = factor * (q_waves == 8 ? 3.1f : q_waves == 4 ? 2.1f : q_waves == 2 ? 2.2f : 1.7f);
      cu_us = factor * (q_waves == 8 ? 3.1f : q_waves == 4 ? 1.8f : q_waves == 2 ? 2.2f : waves == 8 ? 1.7f : 0.85f);
    }
    block_us = q_waves ? 9.f : 5.f;
    // Own rows come from memory, a prefix's for every block of queries after the first mostly from the caches.
    bytes_us = 2.f * (a.dk + a.dv) * lanes * rows * (p.launch.prefix ? q_blocks / 6e6f : 1 / 5e6f);
  }
  int64_t blocks(int s) const { return lanes * q_blocks * s; }
  int steps_of(int s) const { return (steps + s - 1) / s; }
};

// When `slots` places have run n blocks of tn each and then m of tm, each taken by the first place that is free.
double finished(double n, double tn, double m, double tm, int slots) {
  const double rounds = std::floor(n / slots), late = n - rounds * slots, early = slots - late;
  const double start = rounds * tn, start_late = start + tn, end = late > 0 ? start_late : start;
  auto done = [&](double t) {
    return late * std::max(0.0, std::floor((t - start_late) / tm + 1e-6)) + early * std::max(0.0, std::floor((t - start) / tm + 1e-6));
  };
  if (done(end) >= m) return end;
  // The last one ends a number of tm after either start: the first such time that will do.
  const double even = (m * tm + late * start_late + early * start) / slots;
  double best = even + 2 * tm;
  for (const double base : {start, start_late}) {
    const double k0 = std::max(1.0, std::floor((even - base) / tm) - 1);
    for (int i = 0; i < 4; ++i) {
      const double t = base + (k0 + i) * tm;
      if (t < best && done(t) >= m) best = t;
    }
  }
  return std::max(end, best);
}

// The plan of least time for two passes in one launch, whose blocks run side by side: when the last one ends, the CUs' work, memory's time (a tenth of the less of the two beside the other), and the partials' way out and in. 16 shapes of
// 24 to 256 queries over 1024 to 30000 rows ran within 5% (mean) of their best kernels and shares so. Rows wider than 128
// features: both passes by one kernel (the two side by side take more registers than two waves a SIMD have). Rows are
// taken to fill the tables, since the lengths are on the device; where they do not, shares are too few: 24 sequences of 7
// tokens over 8192 shared rows of 64 features with 200 of their own 35 us behind a table cut to them, 134 behind one of
// 32768 rows.
PagedPlan plan_passes(const PagedPass& own, const PagedPass& shared) {
  static constexpr int kShares[] = {1, 2, 3, 4, 6, 8, 10, 12, 14, 16, 18, 20, 22, 24, 28, 32, 40, 48, 56, 64};
  static constexpr int kWaves[] = {0, 2, 4, 8};
  const int width = std::max(own.args.dk, own.args.dv);
  const int nq = own.args.n_heads / own.args.n_groups * own.args.tq, nq_shared = nq * shared.launch.seqs;
  // Two column blocks of wider rows than 64 spill.
  const int cols = width <= 64 && nq_shared > 16 ? 2 : 1;
  const float partial_us = 8.f * (own.args.dv + kRowsPartTail) / 5e6f;
  PagedPlan plan{};
  float best = 3e38f;
  for (int qw : kWaves) {
    if (qw && ((width > 128 && qw != 4) || std::max(nq, nq_shared) <= 16)) continue;
    for (int own_qw : {0, qw}) {
      // The streamed kernel reads rows again for every 16 (64 features: 32) queries: up to 16 times where there is a choice.
      if (width > 128 ? own_qw != qw : own_qw ? nq <= 16 : nq > 16 * 16 * cols) continue;
      const int waves = paged_waves(qw), slots = waves == 8 || width > 128 ? 256 : 512;
      const PassCost x(shared, qw, cols, waves), y(own, own_qw, cols, waves);
      if (!qw && width <= 128 && x.q_blocks > 16) break;
      const float memory = x.bytes_us + y.bytes_us;
      for (int i : kShares) {
        if (i > 1 && (!x.lanes || i > x.steps || x.blocks(i) > 4 * slots)) break;
        for (int j : kShares) {
          if (j > 1 && (j > y.steps || y.blocks(j) > 4 * slots)) break;
          const int sx = x.steps_of(i), sy = y.steps_of(j);
          const float blocks = static_cast<float>(finished(static_cast<double>(x.blocks(i)), x.block_us + sx * x.us,
                                                           static_cast<double>(y.blocks(j)), y.block_us + sy * y.us, slots));
          const float work = (x.blocks(i) * sx * x.cu_us + y.blocks(j) * sy * y.cu_us) / 256 + 4.f;
          const float t = std::max({blocks, work, memory}) + 0.1f * std::min(blocks, memory) +
                          partial_us * (static_cast<float>(x.lanes) * x.queries * i + static_cast<float>(y.lanes) * y.queries * j);
          if (t < best) {
            best = t;
            plan = PagedPlan{own_qw, cols, j, qw, cols, i};
          }
        }
      }
      if (!qw) break;   // both choices are one
    }
  }
  return plan;
}

// Plans by a call's sizes, kept per thread: a search takes about 10 us, a kernel's launch 2.
PagedPlan plan_of(const logkv_paged_args& a, const PagedPass& own, const PagedPass& shared) {
  const std::array<int, 9> key = {a.n_batch, a.n_heads, a.n_groups, a.tq, a.dk, a.dv, a.n_prefixes, own.args.cap, shared.args.cap};
  struct Entry {
    std::array<int, 9> key;
    PagedPlan plan;
  };
  static thread_local std::array<Entry, 64> entries{};
  uint32_t hash = 0;
  for (int x : key) hash = hash * 31 + static_cast<uint32_t>(x);
  Entry& e = entries[(hash ^ hash >> 15) % entries.size()];
  if (e.key != key) e = Entry{key, plan_passes(own, shared)};
  return e.plan;
}

PagedLaunch paged_launch(const logkv_paged_args& a, void* ws) {
  const int width = std::max(a.dk, a.dv);
  PagedLaunch p{};
  logkv_rows_args& x = p.own.args;
  x.q = a.q, x.q_sb = a.q_sb, x.q_sh = a.q_sh, x.q_st = a.q_st;
  x.k = a.k, x.k_sb = a.k_sb, x.k_sg = a.k_sg, x.k_st = a.k_st;
  x.v = a.v, x.v_sb = a.v_sb, x.v_sg = a.v_sg, x.v_st = a.v_st;
  x.cache_k = a.k_pages, x.ck_sb = a.kp_sp, x.ck_sg = a.kp_sg, x.ck_st = a.kp_st;
  x.cache_v = a.v_pages, x.cv_sb = a.vp_sp, x.cv_sg = a.vp_sg, x.cv_st = a.vp_st;
  x.lengths = a.lengths, x.len_stride = a.len_stride, x.len_add = a.len_add;
  x.visible = a.visible, x.vis_sb = a.vis_sb, x.vis_st = a.vis_st, x.counts = a.counts;
  x.out = a.out, x.o_sb = a.o_sb, x.o_sh = a.o_sh, x.o_st = a.o_st;
  x.n_batch = a.n_batch, x.n_heads = a.n_heads, x.n_groups = a.n_groups, x.tq = a.tq, x.dk = a.dk, x.dv = a.dv;
  x.dtype = a.dtype, x.scale = a.scale, x.cap = a.table_len * a.page;
  p.shared.args = x;
  RowsLaunch &o = p.own.launch, &h = p.shared.launch;
  o.seqs = 1;
  o.table = a.table, o.table_sb = a.table_sb, o.page_shift = __builtin_ctz(a.page), o.pages = a.n_pages;
  if (a.n_prefixes) {
    logkv_rows_args& y = p.shared.args;
    y.n_batch = a.n_prefixes;
    y.lengths = a.prefix_lengths, y.lengths2 = a.prefix_lengths2, y.len_stride = a.prefix_stride, y.len_add = a.prefix_add;
    y.counts = nullptr, y.visible = nullptr;
    h.seqs = a.n_batch / a.n_prefixes, h.prefix = 1, h.pages = a.n_pages;
    if (a.prefix_table) {
      h.table = a.prefix_table, h.table_sb = a.prefix_sb, h.page_shift = o.page_shift;
      y.cap = a.prefix_len * a.page;
    } else {
      h.page_shift = 30;
      y.cache_k = a.prefix_k, y.ck_sb = a.pk_sb, y.ck_sg = a.pk_sg, y.ck_st = a.pk_st;
      y.cache_v = a.prefix_v, y.cv_sb = a.pv_sb, y.cv_sg = a.pv_sg, y.cv_st = a.pv_st;
      y.bias = a.bias, y.b_sb = a.b_sb, y.b_sg = a.b_sg, y.b_st = a.b_st, y.bias_half = a.bias_half;
      y.bias_scale = a.bias_scale;
      y.cap = a.prefix_len;
    }
  }
  if (a.n_prefixes || width > 128) {
    const PagedPlan plan = plan_of(a, p.own, p.shared);
    o.q_waves = plan.own_waves, o.cols = plan.own_cols, o.splits = plan.own_splits;
    if (a.n_prefixes) h.q_waves = plan.shared_waves, h.cols = plan.shared_cols, h.splits = plan.shared_splits;
  } else {   // as of contiguous rows
    rows_plan(x, static_cast<int64_t>(x.n_batch) * x.n_groups, static_cast<int64_t>(x.n_heads / x.n_groups) * x.tq, o);
    if (!o.q_waves && width > 64) o.cols = 1;
  }
  uint8_t* base = static_cast<uint8_t*>(ws);
  auto take = [&](int64_t words) {
    float* at = base ? reinterpret_cast<float*>(base + p.bytes) : nullptr;
    p.bytes += align256(4 * words);
    return at;
  };
  for (PagedPass* pass : {&p.own, &p.shared}) {
    RowsLaunch& r = pass->launch;
    const logkv_rows_args& y = pass->args;
    if (!r.seqs) continue;
    const int64_t lanes = static_cast<int64_t>(y.n_batch) * y.n_groups;
    const int64_t nq = static_cast<int64_t>(y.n_heads / y.n_groups) * y.tq * r.seqs;
    r.bias2 = (y.bias_scale == 0.f ? 1.f : y.bias_scale) * kLog2e;
    r.causal = y.visible ? 0 : 1;
    r.shift = r.q_waves ? kTileShift : y.dtype == LOGKV_F16 ? Elem<LOGKV_F16>::kShift : Elem<LOGKV_BF16>::kShift;
    const int block_queries = paged_block_queries(r);
    r.q_blocks = static_cast<int>((nq + block_queries - 1) / block_queries);
    // Shares by length (rows_tile.hpp), as of contiguous rows.
    const bool by_length = r.q_waves && r.splits > 1 && y.n_batch > 1 && y.n_batch <= kWave;
    r.room = by_length ? 2 * r.splits : r.splits;
    r.part = take(lanes * r.room * nq * (y.dv + kRowsPartTail));
    r.odd = reinterpret_cast<uint32_t*>(take(lanes * r.room * r.q_blocks * 16));
    if (by_length) {
      r.shares = reinterpret_cast<int*>(take(lanes));
      if (!y.lengths || !y.len_stride) r.shares = nullptr;   // rows of one length
    }
    const int64_t blocks = lanes * r.splits * r.q_blocks;
    p.blocks += blocks;
    pass->blocks = static_cast<int>(blocks);
  }
  return p;
}

int launch_paged_attention(const logkv_paged_args& a, const PagedLaunch& p, hipStream_t stream) {
  if (int rc = launch_passes(p.shared, p.own, stream)) return rc;
  if (a.dtype == LOGKV_BF16) launch_finish_type<LOGKV_BF16>(p, stream);
  else launch_finish_type<LOGKV_F16>(p, stream);
  return hipGetLastError() == hipSuccess ? LOGKV_OK : LOGKV_ERUNTIME;
}

}  // namespace logkv
