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
  int blocks;   // of the pass in a launch, 0: not in it
};
struct PagedLaunch {
  PagedPass own, shared;
  int64_t bytes, blocks;
};

// Blocks of a launch: fewer than 2^32 threads.
constexpr int64_t kMostPagedBlocks = (int64_t(1) << 32) / 512 - 1;

PagedLaunch paged_launch(const logkv_paged_args& a, void* ws);
int launch_paged_attention(const logkv_paged_args& a, const PagedLaunch& p, hipStream_t stream);
// One launch of both passes: of the same threads a block, by at most one form of the tiled and of the streamed kernel.
int launch_paged_bf16_64(const PagedPass& shared, const PagedPass& own, hipStream_t stream);
int launch_paged_bf16_128(const PagedPass& shared, const PagedPass& own, hipStream_t stream);
int launch_paged_bf16_256(const PagedPass& shared, const PagedPass& own, hipStream_t stream);
int launch_paged_f16_64(const PagedPass& shared, const PagedPass& own, hipStream_t stream);
int launch_paged_f16_128(const PagedPass& shared, const PagedPass& own, hipStream_t stream);
int launch_paged_f16_256(const PagedPass& shared, const PagedPass& own, hipStream_t stream);
int launch_rotary(const logkv_rotary_args& a, bool append, hipStream_t stream);

// Queries of a block: of the tiled kernel's waves, or of the streamed kernel's columns.
inline int paged_block_queries(const RowsLaunch& r) { return r.q_waves ? 32 * r.q_waves : 16 * r.cols; }

// Waves of a block: the tiled kernel's of its query waves, four of the streamed kernel alone.
constexpr int paged_waves(int q_waves) { return q_waves > 2 ? 8 : 4; }

}  // namespace logkv
