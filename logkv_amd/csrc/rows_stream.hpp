// Attention over a cache's rows and the call's own rows, streamed: up to 32 query rows of a KV
// group (16 NC; rows wider than 128 take several such blocks of queries) are the columns of the matrix products while the group's rows pass once from memory.
//
//   s_j = scale q . k_j + bias_j;  out = sum_j 2^(s'_j - m) v_j / sum_j 2^(s'_j - m),  s' = s log2(e)
//
// with the running maximum m of one pass. A block of four waves takes one share of a lane's tiles
// (the cache's 32-row tiles, then the own rows'); its waves walk alternate tiles on their own:
//   S^T = K Q^T by 16x16x32 matrix products (keys x queries: a lane holds 8 keys of its query
//   l % 16 in each of the NC column blocks), K loaded from memory in operand layout;
//   O^T += V^T P^T, V staged row-major in the wave's own LDS and read transposed
//   (ds_read_b64_tr_b16), P as two rounded parts (16 bits for bf16, 22 for fp16).
// The next tile's K and V are on their way while one is computed.
// Bound by HBM: two queries (heads) of one token over 64 lanes of 32768 rows of 2 x 128 bf16 in 213 us,
// 5.04 TB/s with the stored products, the rate of a large copy; loads past the caches took 230 us in the whole call
// against 237 there but 40 against 34 where the rows fit the last cache, and are not used.
// Rows that no query sees (past the rows in use) have V = 0; a tile with an infinity or NaN in V
// takes a form of its own in which an element reaches only the queries that see its row.
#pragma once

#include <algorithm>

#include "rows.hpp"

namespace logkv {

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;   // of a block over contiguous rows

// LDS row stride of a V tile: 8 dwords modulo 32, so the four rows of a transposed read fall into
// distinct banks.
constexpr int v_stride(int blocks) { return 16 * blocks + 16; }

// A block's LDS: per wave a V tile, then its sums; the waves' maxima and sums; per wave and feature, where a tile is not
// finite, the rows (bits) with +infinity, -infinity and NaN (over pages: whether cache rows (1), call rows (2) held one).
template <int NB, int NWV, bool PAGED>
struct StreamLds {
  static constexpr int kTileBytes = kRowTile * v_stride(NB) * 2, kOutBytes = 16 * 16 * NB * 4;
  alignas(16) uint8_t buf[NWV][kTileBytes > kOutBytes ? kTileBytes : kOutBytes];
  float m[NWV][16], l[NWV][16];
  uint32_t odd[NWV][PAGED ? 1 : 3][PAGED ? 1 : 16 * NB];
};

}  // namespace

// A block's share `split` of lane `lane` for its 16 NC queries from q0 on. NS 32-wide steps of dk, NB 16-wide blocks of
// dv, NC 16-query column blocks, NWV waves. Units past dk and dv are zero. PAGED: rows in pages; infinities and NaNs of V
// are left out and noted behind the partials' sums and, by feature, in r.odd, for the launch that joins them.
template <int DT, int NS, int NB, int NC, bool BIAS, bool PAGED, int NWV>
__device__ __forceinline__ void rows_stream_block(const logkv_rows_args& a, const RowsLaunch& r, int split, int lane, int q0,
                                                  StreamLds<NB, NWV, PAGED>& lds) {
  typedef Elem<DT> E;
  typedef typename E::vec8 vec8;
  typedef __attribute__((address_space(3))) s16x4* lds4;
  constexpr int kLd = v_stride(NB), kVLoads = kRowTile * 2 * NB / 64;
  auto& buf = lds.buf;
  auto& m_s = lds.m;
  auto& l_s = lds.l;
  auto& odd_s = lds.odd;
  const int G = a.n_groups, b = lane / G, g = lane % G;
  const int nq = lane_queries<PAGED>(a, r);
  const int units = a.dk / 8, vunits = a.dv / 8;
  const int w = PAGED ? __builtin_amdgcn_readfirstlane(wave_id()) : wave_id(), l = lane_id(), col = l & 15, hq = l >> 4;
  const int n = PAGED ? lane_rows(a, b) : rows_in_use(a, b), own = PAGED ? lane_tokens(a, r, b) : own_rows(a, b);
  const int np = (n + kRowTile - 1) / kRowTile, tiles = np + (own + kRowTile - 1) / kRowTile;
  // The lane's tiles in r.splits equal shares, multiples of the block's waves; shares past the
  // tiles write empty partials.
  const int share = (tiles + NWV * r.splits - 1) / (NWV * r.splits) * NWV;
  const int begin = min(split * share, tiles), end = min(begin + share, tiles);

  // Query columns as B fragments; columns past nq are zero.
  int tq[NC];
  vec8 qf[NC][NS];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int qi = q0 + 16 * c + col;
    const LOGKV_G uint16_t* qrow = query_row<PAGED>(a, r, b, g, min(qi, nq - 1), tq[c]);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (qi < nq && 4 * s + hq < units) x = *(const LOGKV_G uint4*)(qrow + 32 * s + 8 * hq);
      qf[c][s] = __builtin_bit_cast(vec8, x);
    }
  }
  const LOGKV_G uint16_t* kc = gp(a.cache_k) + (PAGED ? 0 : b * a.ck_sb) + g * a.ck_sg;
  const LOGKV_G uint16_t* vc = gp(a.cache_v) + (PAGED ? 0 : b * a.cv_sb) + g * a.cv_sg;
  const LOGKV_G uint16_t* ko = gp(a.k) + b * a.k_sb + g * a.k_sg;
  const LOGKV_G uint16_t* vo = gp(a.v) + b * a.v_sb + g * a.v_sg;
  uint16_t* v_s = reinterpret_cast<uint16_t*>(buf[w]);

  uint4 kx[2][NS], vx[kVLoads];
  float bx[8];
  // Paged: the two 16-row halves of a tile lie on one page each; read a tile ahead of its rows.
  int page[2] = {0, 0};
  PagedRows in_pages;
  if constexpr (PAGED) in_pages.init(a, r, b, g);
  auto pages = [&](int ti) {
    if constexpr (PAGED) {
      if (ti >= np) return;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) page[kb] = in_pages.page(__builtin_amdgcn_readfirstlane(min(kRowTile * ti + 16 * kb, n - 1)));
    }
  };
  // Rows past the tile's: K repeats its last row (masked in the scores), V is zero.
  auto load = [&](int ti) {
    const bool of_cache = ti < np;
    const int t0 = kRowTile * (of_cache ? ti : ti - np), rows = min(kRowTile, (of_cache ? n : own) - t0);
    const int64_t kst = of_cache ? (PAGED ? in_pages.k_st : a.ck_st) : a.k_st, vst = of_cache ? (PAGED ? in_pages.v_st : a.cv_st) : a.v_st;
    const LOGKV_G uint16_t* kr = (of_cache ? kc : ko) + t0 * kst;
    const LOGKV_G uint16_t* vr = (of_cache ? vc : vo) + t0 * vst;
    const LOGKV_G uint16_t* vh[2] = {vr, vr + 16 * vst};   // V's halves, and the steps of their rows
    int64_t vstep[2] = {vst, vst};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const LOGKV_G uint16_t* row = kr + min(16 * kb + col, rows - 1) * kst;
      if constexpr (PAGED) {
        const int first = min(16 * kb, rows - 1);
        int64_t step = kst;
        const LOGKV_G uint16_t* half = kr + first * kst;
        if (of_cache) {
          half = in_pages.at(in_pages.k, in_pages.k_sb, kst, page[kb], t0 + first, step);
          vh[kb] = in_pages.at(in_pages.v, in_pages.v_sb, vst, page[kb], t0 + first, vstep[kb]);
        }
        row = half + (min(16 * kb + col, rows - 1) - first) * step;
      }
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        kx[kb][s] = make_uint4(0, 0, 0, 0);
        if (4 * s + hq < units) kx[kb][s] = *(const LOGKV_G uint4*)(row + 32 * s + 8 * hq);
      }
    }
#pragma unroll
    for (int i = 0; i < kVLoads; ++i) {
      const int e = l + 64 * i, rr = e / (2 * NB), u = e % (2 * NB);
      vx[i] = make_uint4(0, 0, 0, 0);
      if constexpr (PAGED) {
        constexpr int kHalf = kVLoads / 2;
        if (u < vunits && rr < rows) vx[i] = *(const LOGKV_G uint4*)(vh[i / kHalf] + (rr & 15) * vstep[i / kHalf] + 8 * u);
      } else {
        if (u < vunits && rr < rows) vx[i] = *(const LOGKV_G uint4*)(vr + rr * vst + 8 * u);
      }
    }
    if constexpr (BIAS) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int rr = min(16 * (j / 4) + 4 * hq + j % 4, rows - 1);
        bx[j] = 0.f;
        if (of_cache && (!PAGED || a.bias)) {
          const int64_t at = b * a.b_sb + g * a.b_sg + (t0 + rr) * a.b_st;
          const float x = a.bias_half ? E::to_f32(gp(static_cast<const uint16_t*>(a.bias))[at])
                                      : gp(static_cast<const float*>(a.bias))[at];
          bx[j] = bias_base2(x, r.bias2);
        }
      }
    }
  };
  f32x4 o[NC][NB];
  float m[NC], lsum[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    m[c] = -__builtin_inff();
    lsum[c] = 0.f;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) o[c][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float c2 = a.scale * kLog2e;
  uint32_t odd = 0;   // paged: whether this wave left something out of V, of cache rows (1) or call rows (2)
  if (begin + w < end) {
    pages(begin + w);
    load(begin + w);
    pages(min(begin + w + NWV, end - 1));
  }
  for (int ti = begin + w; ti < end; ti += NWV) {
    const bool of_cache = ti < np;
    const int t0 = kRowTile * (of_cache ? ti : ti - np), rows = min(kRowTile, (of_cache ? n : own) - t0);
    f32x4 s[NC][2];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) s[c][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int c = 0; c < NC; ++c) s[c][kb] = E::mfma16(__builtin_bit_cast(vec8, kx[kb][st]), qf[c][st], s[c][kb]);
    u16x2 top = {0, 0};
#pragma unroll
    for (int i = 0; i < kVLoads; ++i) {
      const uint32_t x4[4] = {vx[i].x, vx[i].y, vx[i].z, vx[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, x4[j] & 0x7fff7fffu));
    }
    bool finite = __ballot(top[0] >= E::kInf || top[1] >= E::kInf) == 0;
    if constexpr (PAGED) {
      if (__builtin_expect(!finite, 0)) {
#pragma unroll
        for (int i = 0; i < kVLoads; ++i) vx[i] = finite_only<DT>(vx[i]);
        odd |= of_cache ? 1 : 2;
        finite = true;
      }
    }
    // The wave's own V tile: written and read by this wave only (LDS accesses of a wave complete
    // in order; the fences keep the compiler's order).
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (!PAGED && __builtin_expect(!finite, 0)) {
      for (int e = l; e < 3 * 16 * NB; e += 64) (&odd_s[w][0][0])[e] = 0;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int i = 0; i < kVLoads; ++i) {
        const int e = l + 64 * i, rr = e / (2 * NB), u = e % (2 * NB);
        uint32_t* x4[4] = {&vx[i].x, &vx[i].y, &vx[i].z, &vx[i].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t y = *x4[j / 2] >> (16 * (j % 2)) & 0xffffu, mag = y & 0x7fffu;
          if (mag < E::kInf) continue;
          atomicOr(&odd_s[w][mag > E::kInf ? 2 : y >> 15][8 * u + j], 1u << rr);
          *x4[j / 2] &= j % 2 ? 0xffffu : 0xffff0000u;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kVLoads; ++i) {
      const int e = l + 64 * i, rr = e / (2 * NB), u = e % (2 * NB);
      *reinterpret_cast<uint4*>(v_s + rr * kLd + 8 * u) = vx[i];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if constexpr (BIAS) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j)   // a row hidden by -inf stays hidden whatever its key holds
          s[c][j / 4][j % 4] = bx[j] == -__builtin_inff() ? bx[j] : __builtin_fmaf(s[c][j / 4][j % 4], c2, bx[j]);
    }
    if (ti + NWV < end) {
      load(ti + NWV);
      pages(min(ti + 2 * NWV, end - 1));
    }
    // Masks: element i of block kb is row t0 + 16 kb + 4 hq + i of its region.
    if (!of_cache || rows < kRowTile) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int lim = (!of_cache && r.causal ? min(rows, tq[c] + 1 - t0) : rows) - 4 * hq;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (16 * (j / 4) + j % 4 >= lim) s[c][j / 4][j % 4] = -__builtin_inff();
        if (!of_cache && !r.causal) {
          // All flags loaded at once, those past the line's end its last one.
          const LOGKV_G uint8_t* line = gp(a.visible) + b * a.vis_sb + tq[c] * a.vis_st;
          uint8_t see[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) see[j] = line[min(t0 + 4 * hq + 16 * (j / 4) + j % 4, a.tq - 1)];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (!see[j]) s[c][j / 4][j % 4] = -__builtin_inff();
        }
      }
    }
    if constexpr (NC == 1) {
      if (r.scores && q0 + col < nq) {
        float* row = r.scores + (static_cast<int64_t>(lane) * nq + q0 + col) * r.score_st + kRowTile * ti + 4 * hq;
        *reinterpret_cast<f32x4*>(row) = s[0][0];
        *reinterpret_cast<f32x4*>(row + 16) = s[0][1];
      }
    }
    vec8 pf[NC][2];
    uint32_t seen[NC];   // where a tile is not finite: the rows that the query sees
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      // Online softmax in base 2; the other 24 rows of the tile in the lanes of the same l % 16.
      float mx = -__builtin_inff();
#pragma unroll
      for (int j = 0; j < 8; ++j) mx = fmaxf(mx, s[c][j / 4][j % 4]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
      mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
      const float m_new = fmaxf(m[c], BIAS ? mx : mx * c2);
      const float mb = m_new == -__builtin_inff() ? 0.f : m_new;
      if (__ballot(m_new != m[c])) {
        const float corr = __builtin_amdgcn_exp2f(m[c] - mb);
        lsum[c] *= corr;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) o[c][nb] *= corr;
      }
      m[c] = m_new;
      if (!PAGED && __builtin_expect(!finite, 0)) {
        seen[c] = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          seen[c] |= (s[c][j / 4][j % 4] != -__builtin_inff() ? 1u : 0u) << (16 * (j / 4) + 4 * hq + j % 4);
        seen[c] |= __shfl_xor(seen[c], 16, kWave);
        seen[c] |= __shfl_xor(seen[c], 32, kWave);
      }
      const float arg0 = exponent_offset<BIAS>(E::kShift, mb, mx, c2);
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y0 = s[c][j / 2][2 * (j % 2)], y1 = s[c][j / 2][2 * (j % 2) + 1];
        const float x0 = __builtin_amdgcn_exp2f(BIAS ? y0 + arg0 : __builtin_fmaf(y0, c2, arg0));
        const float x1 = __builtin_amdgcn_exp2f(BIAS ? y1 + arg0 : __builtin_fmaf(y1, c2, arg0));
        lsum[c] += x0 + x1;
        E::parts(x0, x1, hi[j], lo[j]);
      }
      pf[c][0] = __builtin_bit_cast(vec8, make_uint4(hi[0], hi[1], hi[2], hi[3]));
      pf[c][1] = __builtin_bit_cast(vec8, make_uint4(lo[0], lo[1], lo[2], lo[3]));
    }
    // V^T fragments: features 16 nb + col, rows 4 hq .. + 3 and 16 + 4 hq .. + 3 (P's own order).
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const uint16_t* p = v_s + (4 * hq + (col >> 2)) * kLd + 16 * nb + 4 * (col & 3);
      const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p)));
      const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 16 * kLd)));
      const vec8 vf = __builtin_bit_cast(vec8, make_uint4(x.x, x.y, y.x, y.y));
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int c = 0; c < NC; ++c) o[c][nb] = E::mfma16(vf, pf[c][q], o[c][nb]);
    }
    if (!PAGED && __builtin_expect(!finite, 0)) {
      // The infinities and NaNs left out of the products, for the queries that see their rows.
#pragma unroll
      for (int c = 0; c < NC; ++c) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = 16 * nb + 4 * hq + i;
            if (odd_s[w][0][d] & seen[c]) o[c][nb][i] += __builtin_inff();
            if (odd_s[w][1][d] & seen[c]) o[c][nb][i] -= __builtin_inff();
            if (odd_s[w][2][d] & seen[c]) o[c][nb][i] = __builtin_nanf("");
          }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
  // Waves combined in wave order, one column block after the other: [acc[dv], m, l] per query.
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    lsum[c] += __shfl_xor(lsum[c], 16, kWave);
    lsum[c] += __shfl_xor(lsum[c], 32, kWave);
    if (!(PAGED && r.prefix) && tq[c] >= own) {   // a query past its batch row's count sees nothing
      m[c] = -__builtin_inff();
      lsum[c] = 0.f;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) o[c][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __syncthreads();   // the waves' V tiles (c = 0) or the last block's sums are read
    float* acc_w = reinterpret_cast<float*>(buf[w]);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)   // four features a unit, permuted by query: distinct banks
      *reinterpret_cast<f32x4*>(acc_w + col * (16 * NB) + 4 * ((4 * nb + hq) ^ (col & 7))) = o[c][nb];
    if (hq == 0) {
      m_s[w][col] = m[c];
      l_s[w][col] = lsum[c];
    }
    if (PAGED && c == 0 && l == 0) odd_s[w][0][0] = odd;
    __syncthreads();
    const int qb = q0 + 16 * c, queries = min(16, nq - qb);
    float* out = r.part + ((static_cast<int64_t>(lane) * r.room + split) * nq + qb) * (a.dv + kRowsPartTail);
    const int tid = threadIdx.x;
    // An empty share has zero sums; a share of NaN logits alone has no maximum but a NaN sum.
    float mx, f[NWV];
    auto factors = [&](int q) {
      mx = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < NWV; ++i) mx = fmaxf(mx, m_s[i][q]);
      const float base = mx == -__builtin_inff() ? 0.f : mx;
#pragma unroll
      for (int i = 0; i < NWV; ++i) f[i] = __builtin_amdgcn_exp2f(m_s[i][q] - base);
    };
    for (int e = tid; e < queries * 4 * NB; e += 64 * NWV) {
      const int q = e / (4 * NB), u = e % (4 * NB);
      if (4 * u >= a.dv) continue;
      factors(q);
      f32x4 val = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NWV; ++i)
        val += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(buf[i]) + q * (16 * NB) + 4 * (u ^ (q & 7))) * f[i];
      *reinterpret_cast<f32x4*>(out + static_cast<int64_t>(q) * (a.dv + kRowsPartTail) + 4 * u) = val;
    }
    if (tid < queries) {
      factors(tid);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < NWV; ++i) sum += l_s[i][tid] * f[i];
      float* tail = out + static_cast<int64_t>(tid) * (a.dv + kRowsPartTail) + a.dv;
      if constexpr (PAGED) {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < NWV; ++i) any |= odd_s[i][0][0];
        *reinterpret_cast<f32x4*>(tail) = f32x4{mx, sum, any & 1 ? 1.f : 0.f, any & 2 ? 1.f : 0.f};
      } else {
        *reinterpret_cast<float2*>(tail) = make_float2(mx, sum);
      }
    }
  }
  if constexpr (PAGED) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < NWV; ++i) any |= odd_s[i][0][0];
    if (__builtin_expect(any & 1, 0))
      note_odd_rows<DT, 64 * NWV>(a, r, b, g, kRowTile * begin, min(kRowTile * min(end, np), n), reinterpret_cast<uint32_t*>(buf[0]),
                                  r.odd + ((static_cast<int64_t>(lane) * r.room + split) * r.q_blocks + q0 / (16 * NC)) * 16);
  }
}

}  // namespace logkv
