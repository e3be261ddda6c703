// Attention of a batch over a paged cache, with prefixes that several sequences share.
//
// Softmax over [prefix | own pages | the call's rows] splits by rows: each part gives a query an
// unnormalised sum, a maximum and a sum of exponentials, which join under the largest maximum. So a
// prefix's rows are read once for all of its sequences: their queries (sequences x heads of the KV group
// x tokens) are the columns of one product, in the kernel that so many columns take (rows_plan), and a
// sequence's own rows are read in a second pass of few columns. Both passes are the row attention
// kernels over a page table, in one launch where their kernels go together; this file joins their partials.
// An infinity or NaN in V is left out of a pass's products, which would spread it to queries that do not
// see its row, and noted behind the partial's sums; the join then adds those of the rows that a query sees.
#include <algorithm>
#include <cmath>

#include "paged.hpp"

namespace logkv {

namespace {

constexpr int kThreads = 256;

int64_t align256(int64_t x) { return (x + 255) & ~int64_t(255); }

}  // namespace

// Values of row `at` that are infinite or NaN added to the query's features; others are in its sum.
template <int DT>
__device__ __forceinline__ void add_odd(const LOGKV_G uint16_t* at, f32x4& y) {
  const uint2 x = *(const LOGKV_G uint2*)at;
  const uint32_t v[4] = {x.x & 0xffffu, x.x >> 16, x.y & 0xffffu, x.y >> 16};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if ((v[k] & 0x7fffu) >= Elem<DT>::kInf) y[k] += Elem<DT>::to_f32(static_cast<uint16_t>(v[k]));
}

// Those of every row of a lane that query t sees.
template <int DT>
__device__ __forceinline__ void add_odd_rows(const logkv_rows_args& a, const RowsLaunch& r, int b, int g, int t, int d, f32x4& y) {
  const int n = rows_in_use(a, b), own = lane_own_rows<true>(a, r, b);
  const LOGKV_G uint16_t* base = gp(a.cache_v) + g * a.cv_sg + d;
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    const int page = page_of(r, b, i);
    bool see = page >= 0;
    if (a.bias && see) {
      const int64_t at = b * a.b_sb + g * a.b_sg + i * a.b_st;
      const float x = a.bias_half ? Elem<DT>::to_f32(gp(static_cast<const uint16_t*>(a.bias))[at])
                                  : gp(static_cast<const float*>(a.bias))[at];
      see = x != -__builtin_inff();
    }
    int64_t step;
    if (see) add_odd<DT>(page_row(r, base, a.cv_sb, a.cv_st, page, i, step), y);
  }
#pragma unroll 1
  for (int i = 0; i < own; ++i) {
    const bool see = r.causal ? i <= t : gp(a.visible)[b * a.vis_sb + t * a.vis_st + i] != 0;
    if (see) add_odd<DT>(gp(a.v) + b * a.v_sb + g * a.v_sg + i * a.v_st + d, y);
  }
}

// What the join reads of a pass: the partials of a lane, [room][queries][dv + kRowsPartTail] each.
struct FinishPass {
  const float* part;
  const int* shares;   // partials of a lane, null: `splits` of each
  int splits, room;
  int seqs;            // sequences of a lane, 0: no such pass
  float unit;          // the sums' scale
};
// What every block reads comes first; the passes themselves are for the rows of notes.
struct FinishArgs {
  FinishPass own, shared;
  uint16_t* out;
  int64_t o_sb, o_sh, o_st;
  const int32_t* counts;
  int n_groups, rep, tq, dv;
  PagedPass passes[2];
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
  float odd[2] = {0.f, 0.f};   // the partials' notes
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
      odd[0] += of_own ? ml[k][2] : 0.f;
      odd[1] += of_own ? 0.f : ml[k][2];
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
    const PagedPass &p0 = a.passes[0], &p1 = a.passes[1];
    if (odd[0] > 0.f) add_odd_rows<DT>(p0.args, p0.launch, b, g, t, d, z);
    if (odd[1] > 0.f) add_odd_rows<DT>(p1.args, p1.launch, b / a.shared.seqs, g, t, d, z);
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
  auto pass = [](const RowsLaunch& r) { return FinishPass{r.part, r.shares, r.splits, r.room, r.seqs, exp2f(-r.shift)}; };
  const FinishArgs args = {pass(p.own.launch), pass(p.shared.launch), a.out, a.o_sb, a.o_sh, a.o_st, a.counts,
                           a.n_groups, rep, a.tq, a.dv, {p.own, p.shared}};
  hipLaunchKernelGGL((paged_finish_kernel<DT, TQ, SG>), dim3((nq + qpb - 1) / qpb, a.n_batch * a.n_groups), dim3(kThreads),
                     0, stream, args);
}

template <int DT>
void launch_finish_type(const PagedLaunch& p, hipStream_t stream) {
  const logkv_rows_args& a = p.own.args;
  // Groups of partials share a query where eight queries a block would not fill the CUs.
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

// A pass's lanes, query blocks, rows at most, and a step of one of its blocks: the rows that it takes, in microseconds.
struct PassShape {
  int64_t lanes;
  int q_blocks, queries, rows, step_rows;
  float step_us;
  // Blocks of s shares a lane, and a block's time: its steps, and kBlockUs to begin and to end.
  int64_t blocks(int s) const { return lanes * q_blocks * s; }
  float time(int s) const { return kBlockUs + ((rows + step_rows - 1) / step_rows + s - 1) / s * step_us; }
  static constexpr float kBlockUs = 4.f;
};

PassShape shape_of(const PagedPass& p, int waves) {
  const logkv_rows_args& a = p.args;
  const RowsLaunch& r = p.launch;
  const int width = std::max(a.dk, a.dv);
  PassShape x;
  x.lanes = static_cast<int64_t>(a.n_batch) * a.n_groups;
  x.q_blocks = r.q_blocks;
  x.queries = a.n_heads / a.n_groups * a.tq * r.seqs;
  x.rows = a.cap + (r.prefix ? 0 : a.tq);
  x.step_rows = r.q_waves ? 64 : 32 * waves;
  x.step_us = r.q_waves ? (r.q_waves == 8 ? 3.6f : 2.f) : 1.5f;
  if (width <= 64) x.step_us *= 0.6f;
  if (width > 128) x.step_us *= 2.f;
  return x;
}

// Shares of the lanes of two passes in one launch: the ones of least time by what the blocks take side by side, the
// steps of both over the chip, and the partials' way out and in.
void share_out(PagedPass& shared, PagedPass& own, int slots, int waves) {
  const PassShape x = shape_of(shared, waves), y = shape_of(own, waves);
  static constexpr int kShares[] = {1, 2, 3, 4, 6, 8, 10, 12, 14, 16, 20, 24, 28, 32, 40, 48, 56, 64};
  const float partial_us = 8.f * (own.args.dv + kRowsPartTail) / 5e6f;
  float best = 3e38f;
  for (int i : kShares) {
    if (i > 1 && ((i - 1) * x.step_rows >= x.rows || x.blocks(i) > 4 * slots)) break;
    for (int j : kShares) {
      if (j > 1 && ((j - 1) * y.step_rows >= y.rows || y.blocks(j) > 4 * slots)) break;
      const float tx = x.time(i), ty = y.time(j);
      const int64_t n = x.blocks(i) + y.blocks(j);
      float t = std::max(tx, ty);
      if (n > slots) t = std::max(t, (x.blocks(i) * tx + y.blocks(j) * ty) / slots + std::min(tx, ty) / 2);
      t += partial_us * (static_cast<float>(x.lanes) * x.queries * i + static_cast<float>(y.lanes) * y.queries * j);
      if (t < best) {
        best = t;
        shared.launch.splits = i;
        own.launch.splits = j;
      }
    }
  }
}

PagedLaunch paged_launch(const logkv_paged_args& a, void* ws) {
  const int width = std::max(a.dk, a.dv);
  PagedLaunch p{};
  auto plan = [&](PagedPass& pass) {
    RowsLaunch& r = pass.launch;
    const logkv_rows_args& x = pass.args;
    const int64_t nq = static_cast<int64_t>(x.n_heads / x.n_groups) * x.tq * r.seqs;
    r.bias2 = (x.bias_scale == 0.f ? 1.f : x.bias_scale) * kLog2e;
    r.causal = x.visible ? 0 : 1;
    rows_plan(x, static_cast<int64_t>(x.n_batch) * x.n_groups, nq, r);
    if (!r.q_waves && width > 64) r.cols = 1;   // two column blocks of wider rows spill
    r.q_blocks = static_cast<int>(r.q_waves ? (nq + 32 * r.q_waves - 1) / (32 * r.q_waves) : (nq + 16 * r.cols - 1) / (16 * r.cols));
  };
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
  p.own.launch.seqs = 1;
  p.own.launch.table = a.table, p.own.launch.table_sb = a.table_sb;
  p.own.launch.page_shift = __builtin_ctz(a.page), p.own.launch.pages = a.n_pages;
  plan(p.own);
  if (a.n_prefixes) {
    logkv_rows_args& y = p.shared.args;
    RowsLaunch& r = p.shared.launch;
    y.n_batch = a.n_prefixes;
    y.lengths = a.prefix_lengths, y.lengths2 = a.prefix_lengths2, y.len_stride = a.prefix_stride, y.len_add = a.prefix_add;
    y.counts = nullptr, y.visible = nullptr;
    r.seqs = a.n_batch / a.n_prefixes, r.prefix = 1, r.pages = a.n_pages;
    if (a.prefix_table) {
      r.table = a.prefix_table, r.table_sb = a.prefix_sb, r.page_shift = p.own.launch.page_shift;
      y.cap = a.prefix_len * a.page;
    } else {
      r.page_shift = 30;
      y.cache_k = a.prefix_k, y.ck_sb = a.pk_sb, y.ck_sg = a.pk_sg, y.ck_st = a.pk_st;
      y.cache_v = a.prefix_v, y.cv_sb = a.pv_sb, y.cv_sg = a.pv_sg, y.cv_st = a.pv_st;
      y.bias = a.bias, y.b_sb = a.b_sb, y.b_sg = a.b_sg, y.b_st = a.b_st, y.bias_half = a.bias_half;
      y.bias_scale = a.bias_scale;
      y.cap = a.prefix_len;
    }
    plan(p.shared);
    // Passes of one launch have the same threads a block and at most one tiled and one streamed kernel.
    const RowsLaunch &o = p.own.launch, &h = p.shared.launch;
    p.together = o.q_waves && h.q_waves ? o.q_waves == h.q_waves : o.q_waves || h.q_waves || o.cols == h.cols;
    if (p.together) {
      const int q_waves = std::max(o.q_waves, h.q_waves), waves = paged_waves(q_waves);
      share_out(p.shared, p.own, waves == 8 || width > 128 ? 256 : 512, waves);
    }
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
    // Shares by length (rows_tile.hpp), as of contiguous rows.
    const bool by_length = r.q_waves && r.splits > 1 && y.n_batch > 1 && y.n_batch <= kWave;
    r.room = by_length ? 2 * r.splits : r.splits;
    r.part = take(lanes * r.room * nq * (y.dv + kRowsPartTail));
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
  PagedPass none = p.shared;
  none.blocks = 0;
  if (p.together) {
    if (int rc = launch_passes(p.shared, p.own, stream)) return rc;
  } else {
    if (a.n_prefixes) {
      PagedPass alone = p.own;
      alone.blocks = 0;
      if (int rc = launch_passes(p.shared, alone, stream)) return rc;
    }
    if (int rc = launch_passes(none, p.own, stream)) return rc;
  }
  if (a.dtype == LOGKV_BF16) launch_finish_type<LOGKV_BF16>(p, stream);
  else launch_finish_type<LOGKV_F16>(p, stream);
  return hipGetLastError() == hipSuccess ? LOGKV_OK : LOGKV_ERUNTIME;
}

}  // namespace logkv
