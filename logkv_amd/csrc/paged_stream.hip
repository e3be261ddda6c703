// Streamed attention over rows in pages, or over rows that several sequences share (the kernel: rows_stream.hpp).
#include "paged.hpp"
#include "rows_stream.hpp"

namespace logkv {

int launch_paged_stream(const PagedPass& p, hipStream_t stream) {
  if (p.args.dtype == LOGKV_BF16) launch_stream_type<LOGKV_BF16, true>(p.args, p.launch, stream);
  else launch_stream_type<LOGKV_F16, true>(p.args, p.launch, stream);
  return hipGetLastError() == hipSuccess ? LOGKV_OK : LOGKV_ERUNTIME;
}

}  // namespace logkv
