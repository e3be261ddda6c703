// Tiled attention over a cache's contiguous rows (the kernel: rows_tile.hpp).
#include "rows_tile.hpp"

namespace logkv {

int launch_rows_tile(const logkv_rows_args& a, const RowsLaunch& r, hipStream_t stream) {
  if (a.dtype == LOGKV_BF16) launch_tile_type<LOGKV_BF16, false>(a, r, stream);
  else launch_tile_type<LOGKV_F16, false>(a, r, stream);
  return hipGetLastError() == hipSuccess ? LOGKV_OK : LOGKV_ERUNTIME;
}

}  // namespace logkv
