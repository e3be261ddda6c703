// Rotary positions, appends to a paged cache (rotary.hip) and attention over one (paged.hip).
#pragma once

#include "../../include/logkv_paged.h"
#include "rows.hpp"

namespace logkv {

// The two passes of a paged attention: a lane of `shared` takes the rows of a prefix for the queries of all of its
// sequences, a lane of `own` a sequence's pages and the call's rows. Each leaves partials that one launch joins.
struct PagedPass {
  logkv_rows_args args;
  RowsLaunch launch;
};
struct PagedLaunch {
  PagedPass own, shared;
  int64_t bytes;
};

PagedLaunch paged_launch(const logkv_paged_args& a, void* ws);
int launch_paged_tile(const PagedPass& p, hipStream_t stream);
int launch_paged_stream(const PagedPass& p, hipStream_t stream);
int launch_paged_attention(const logkv_paged_args& a, const PagedLaunch& p, hipStream_t stream);
int launch_rotary(const logkv_rotary_args& a, bool append, hipStream_t stream);

}  // namespace logkv
