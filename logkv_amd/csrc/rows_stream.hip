// Streamed attention over a cache's contiguous rows (a block's work: rows_stream.hpp).
#include "rows_stream.hpp"

namespace logkv {

template <int DT, int NS, int NB, int NC, bool BIAS>
__global__ __launch_bounds__(64 * kWaves, NB <= 8 && NC * NB <= 16 ? 2 : 1) void rows_stream_kernel(logkv_rows_args a, RowsLaunch r) {
  __shared__ StreamLds<NB, kWaves, false> lds;
  rows_stream_block<DT, NS, NB, NC, BIAS, false, kWaves>(a, r, blockIdx.x, blockIdx.y, 16 * NC * static_cast<int>(blockIdx.z), lds);
}

namespace {

template <int DT, int NS, int NB, int NC>
void launch_one(const logkv_rows_args& a, const RowsLaunch& r, dim3 grid, hipStream_t stream) {
  if (a.bias) hipLaunchKernelGGL((rows_stream_kernel<DT, NS, NB, NC, true>), grid, dim3(64 * kWaves), 0, stream, a, r);
  else hipLaunchKernelGGL((rows_stream_kernel<DT, NS, NB, NC, false>), grid, dim3(64 * kWaves), 0, stream, a, r);
}

template <int DT>
void launch_type(const logkv_rows_args& a, const RowsLaunch& r, dim3 grid, hipStream_t stream) {
  if (a.dk <= 64 && a.dv <= 64) {
    if (r.cols == 1) launch_one<DT, 2, 4, 1>(a, r, grid, stream);
    else launch_one<DT, 2, 4, 2>(a, r, grid, stream);
  } else if (a.dk <= 128 && a.dv <= 128) {
    if (r.cols == 1) launch_one<DT, 4, 8, 1>(a, r, grid, stream);
    else launch_one<DT, 4, 8, 2>(a, r, grid, stream);
  } else {
    if (r.cols == 1) launch_one<DT, 8, 16, 1>(a, r, grid, stream);
    else launch_one<DT, 8, 16, 2>(a, r, grid, stream);
  }
}

}  // namespace

int launch_rows_stream(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream) {
  const int nq = a.n_heads / a.n_groups * a.tq;
  const dim3 grid(r.splits, a.n_batch * a.n_groups, (nq + 16 * r.cols - 1) / (16 * r.cols));
  if (a.dtype == LOGKV_BF16) launch_type<LOGKV_BF16>(a, r, grid, stream);
  else launch_type<LOGKV_F16>(a, r, grid, stream);
  return hipGetLastError() == hipSuccess ? LOGKV_OK : LOGKV_ERUNTIME;
}

}  // namespace logkv
