// Passes over rows of bf16 in pages, up to 64 features (the kernel: paged_pass.hpp).
#include "paged_pass.hpp"

namespace logkv {

int launch_paged_bf16_64(const PagedPass& shared, const PagedPass& own, hipStream_t stream) {
  return launch_paged_width<LOGKV_BF16, 4, 2>(shared, own, stream);
}

}  // namespace logkv
