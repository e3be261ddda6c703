// Tiled attention over a cache's contiguous rows (a block's work: rows_tile.hpp).
#include "rows_tile.hpp"

namespace logkv {

// SECOND: the launch that follows, whose blocks do again what the first left.
template <int DT, int NKS, int NDV, int NW, int QW, int RB, bool BIAS, bool SECOND>
__global__ __launch_bounds__(64 * NW, 2) void rows_tile_kernel(logkv_rows_args a, RowsLaunch r) {
  __shared__ TileLds<NKS, NDV, NW, QW, RB, BIAS> lds;
  const int nx = static_cast<int>(gridDim.x), ny = static_cast<int>(gridDim.y), nz = static_cast<int>(gridDim.z);
  const int lin = static_cast<int>(blockIdx.x) + nx * (static_cast<int>(blockIdx.y) + ny * static_cast<int>(blockIdx.z));
  rows_tile_block<DT, NKS, NDV, NW, QW, RB, BIAS, SECOND, false>(a, r, rows_block(lin, nx, ny, nz), nx, lds);
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
