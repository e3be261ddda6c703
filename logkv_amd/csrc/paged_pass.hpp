// The passes of a paged attention as one launch: blocks of the shared prefixes, then blocks of the sequences' own rows,
// each by the tiled (rows_tile.hpp) or the streamed kernel (rows_stream.hpp). Side by side a pass bound by memory and one
// bound by the matrix cores overlap, and a launch is saved: 32 sequences of two heads a group over 8782 shared rows with a
// bias and 512 of their own took 43 us when they were joined, and 51.6 before in launches of their own (with those of the
// second forms, 4.7 us each); 33 us with what came after.
#pragma once

#include "paged.hpp"
#include "rows_stream.hpp"
#include "rows_tile.hpp"

namespace logkv {

namespace {

constexpr int most(int a, int b) { return a > b ? a : b; }

struct PagedPasses {
  PagedPass pass[2];
};

}  // namespace

// NKS 16-wide steps of dk and NDV 32-wide blocks of dv; QW query waves of the tiled kernel (0: none), NC column blocks of
// the streamed one (0: none). A block takes the pass that its index falls into, by the kernel of that pass.
template <int DT, int NKS, int NDV, int QW, int NC, bool BIAS>
__global__ __launch_bounds__(64 * paged_waves(QW), NDV <= 4 || QW ? 2 : 1) void paged_pass_kernel(PagedPasses both) {
  constexpr int NW = paged_waves(QW), NB = 2 * NDV, RB = QW == 8 ? 2 : 1;
  typedef TileLds<NKS, NDV, NW, QW ? QW : 1, RB, BIAS> Tile;
  typedef StreamLds<NB, NW, true> Stream;
  __shared__ __align__(most(alignof(Tile), alignof(Stream))) uint8_t lds[most(QW ? sizeof(Tile) : 0, NC ? sizeof(Stream) : 0)];
  int lin = blockIdx.x;
  const bool own = lin >= both.pass[0].blocks;
  if (own) lin -= both.pass[0].blocks;
  const logkv_rows_args& a = both.pass[own].args;
  const RowsLaunch& r = both.pass[own].launch;
  const int nq = lane_queries<true>(a, r), lanes = a.n_batch * a.n_groups;
  if constexpr (QW > 0) {
    if (NC == 0 || r.q_waves) {
      const int qb = (nq + 32 * kCols * QW - 1) / (32 * kCols * QW);
      rows_tile_block<DT, NKS, NDV, NW, QW, RB, BIAS, false, true>(a, r, rows_block(lin, qb, r.splits, lanes), qb,
                                                                   *reinterpret_cast<Tile*>(lds));
      return;
    }
  }
  if constexpr (NC > 0) {
    const int split = lin % r.splits, lane = lin / r.splits % lanes, q = lin / (r.splits * lanes);
    rows_stream_block<DT, NKS / 2, NB, NC, BIAS, true, NW>(a, r, split, lane, 16 * NC * q, *reinterpret_cast<Stream*>(lds));
  }
}

namespace {

template <int DT, int NKS, int NDV, int QW, int NC>
int launch_passes(const PagedPass& shared, const PagedPass& own, hipStream_t stream) {
  const dim3 grid(shared.blocks + own.blocks), threads(64 * paged_waves(QW));
  const PagedPasses both = {{shared, own}};
  if (shared.blocks && shared.args.bias) hipLaunchKernelGGL((paged_pass_kernel<DT, NKS, NDV, QW, NC, true>), grid, threads, 0, stream, both);
  else hipLaunchKernelGGL((paged_pass_kernel<DT, NKS, NDV, QW, NC, false>), grid, threads, 0, stream, both);
  return hipGetLastError() == hipSuccess ? LOGKV_OK : LOGKV_ERUNTIME;
}

// Of the two passes' kernels: the tiled one's query waves and the streamed one's columns, 0 where no pass takes it.
template <int DT, int NKS, int NDV>
int launch_paged_width(const PagedPass& shared, const PagedPass& own, hipStream_t stream) {
  int qw = 0, nc = 0;
  for (const PagedPass* p : {&shared, &own}) {
    if (!p->blocks) continue;
    if (p->launch.q_waves) qw = p->launch.q_waves;
    else nc = p->launch.cols;
  }
  if constexpr (NDV <= 4) {
    if (nc == 2) {
      if constexpr (NDV <= 2) {
        if (qw == 2) return launch_passes<DT, NKS, NDV, 2, 2>(shared, own, stream);
        if (qw == 4) return launch_passes<DT, NKS, NDV, 4, 2>(shared, own, stream);
        if (qw == 8) return launch_passes<DT, NKS, NDV, 8, 2>(shared, own, stream);
        return launch_passes<DT, NKS, NDV, 0, 2>(shared, own, stream);
      }
    }
    if (nc == 1) {
      if (qw == 2) return launch_passes<DT, NKS, NDV, 2, 1>(shared, own, stream);
      if (qw == 4) return launch_passes<DT, NKS, NDV, 4, 1>(shared, own, stream);
      if (qw == 8) return launch_passes<DT, NKS, NDV, 8, 1>(shared, own, stream);
    } else {
      if (qw == 2) return launch_passes<DT, NKS, NDV, 2, 0>(shared, own, stream);
      if (qw == 4) return launch_passes<DT, NKS, NDV, 4, 0>(shared, own, stream);
      if (qw == 8) return launch_passes<DT, NKS, NDV, 8, 0>(shared, own, stream);
    }
  } else if (qw) {   // of both passes (the streamed kernel takes more registers)
    return launch_passes<DT, NKS, NDV, 4, 0>(shared, own, stream);
  }
  return launch_passes<DT, NKS, NDV, 0, 1>(shared, own, stream);
}

}  // namespace

}  // namespace logkv
