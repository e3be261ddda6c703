// Passes over rows of f16 in pages, up to 64 features (the kernel: paged_pass.hpp).
#include "paged_pass.hpp"

namespace logkv {

int launch_paged_f16_64(const PagedPass& shared, const PagedPass& own, hipStream_t stream) {
  return launch_paged_width<LOGKV_F16, 4, 2>(shared, own, stream);
}

}  // namespace logkv
