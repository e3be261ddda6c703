// Tiled attention over rows in pages, or over rows that several sequences share (the kernel: rows_tile.hpp).
#include "paged.hpp"
#include "rows_tile.hpp"

namespace logkv {

int launch_paged_tile(const PagedPass& p, hipStream_t stream) {
  if (p.args.dtype == LOGKV_BF16) launch_tile_type<LOGKV_BF16, true>(p.args, p.launch, stream);
  else launch_tile_type<LOGKV_F16, true>(p.args, p.launch, stream);
  return hipGetLastError() == hipSuccess ? LOGKV_OK : LOGKV_ERUNTIME;
}

}  // namespace logkv
