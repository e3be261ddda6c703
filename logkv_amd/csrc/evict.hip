// Eviction of a cache's rows by accumulated attention weight: per lane the last `recent` rows and
// the heaviest others stay, in their order.
//
// The rows that stay are those with key >= T, T the (keep - recent)-th largest key of the rows that
// are not recent, where the key is the weight's bits in an order that integers keep (ties at T go to
// the lowest index). One block per lane finds T digit by digit (11 + 11 + 10 bits, a histogram in
// LDS each) with the lane's keys in registers, then numbers the rows that stay; a second launch
// copies them, its stores bypassing the caches (224 lanes of 4096 rows of 512 bytes: 189 us a call
// with ordinary stores, 167 us). Bound by HBM: the copy of those lanes takes 153 us, 4.9 TB/s of
// rows read and written; the selection 10 us, and 24 us over 32768 rows a lane: three
// passes and the numbering on one CU a lane (four histograms in turn against equal bins: 26 us).
#include <algorithm>

#include "rows.hpp"

namespace logkv {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kDigit = 2048;       // histogram bins: 11 bits
constexpr int kCopyThreads = 256;
constexpr int kCopyRows = 32;      // kept rows per copy block

__device__ __forceinline__ int rows_of(const logkv_evict_args& a, int b) {
  const int n = a.lengths ? a.lengths[b] : a.len_add;
  return max(0, min(n, a.cap));
}

// Larger weights have larger keys; both zeros have one key, every NaN the largest.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive scan of x over the block in thread order, and the total; every thread calls it.
__device__ __forceinline__ int block_scan(int x, int* wave_sums, int& total) {
  int inc = x;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int up = __shfl_up(inc, off, kWave);
    if (lane_id() >= off) inc += up;
  }
  __syncthreads();   // wave_sums is free
  if (lane_id() == kWave - 1) wave_sums[wave_id()] = inc;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < wave_id()) before += wave_sums[i];
    total += wave_sums[i];
  }
  return before + inc - x;
}

}  // namespace

// Row i * kThreads + tid is thread tid's i-th: PER of them in registers, or (0) read again in every
// pass. The rows that stay are numbered in row order by ballots: a wave's 64 rows of one i are
// consecutive, and a table of counts per (i, wave), in LDS, is scanned by the block (PER 0: per i).
template <int PER>
__global__ __launch_bounds__(kThreads) void evict_select_kernel(logkv_evict_args a) {
  __shared__ int hist[kDigit];
  __shared__ int wave_sums[kWaves];
  __shared__ int count_s[2][(PER ? PER : 1) * kWaves];   // rows above T, rows at T
  __shared__ int found[2];
  const int lane = blockIdx.x, G = a.n_groups, b = lane / G, g = lane % G, tid = threadIdx.x;
  const int n = rows_of(a, b), keep = a.keep;
  LOGKV_G int32_t* kept = gp(a.kept) + static_cast<int64_t>(lane) * keep;
  if (g == 0 && tid == 0) a.out_lengths[b] = min(n, keep);
  if (n <= keep) {
    for (int i = tid; i < keep; i += kThreads) kept[i] = i < n ? i : -1;
    return;
  }
  const int recent = min(a.recent, keep), old = n - recent, need = keep - recent;
  for (int i = tid; i < recent; i += kThreads) kept[need + i] = old + i;
  if (need == 0) return;
  const LOGKV_G float* w = gp(a.weights) + b * a.w_sb + g * a.w_sg;
  const int steps = (old + kThreads - 1) / kThreads;
  uint32_t keys[PER ? PER : 1];
  if constexpr (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) keys[i] = __float_as_uint(w[min(i * kThreads + tid, old - 1)]);
#pragma unroll
    for (int i = 0; i < PER; ++i) keys[i] = weight_key(__uint_as_float(keys[i]));
  }
  // fn(i, key, whether the row exists), every thread of the block together.
  auto each = [&](auto&& fn) {
    if constexpr (PER > 0) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i < steps) fn(i, keys[i], i * kThreads + tid < old);
    } else {
      for (int i = 0; i < steps; ++i) {
        const int64_t row = static_cast<int64_t>(i) * kThreads + tid;
        fn(i, weight_key(w[imin64(row, old - 1)]), row < old);
      }
    }
  };
  uint32_t prefix = 0, mask = 0;   // the digits of T found so far
  int left = need;                 // T is the left-th largest of the keys with those digits
  for (int shift = 21;; shift = shift == 21 ? 10 : 0) {
    const int bins = shift == 0 ? kDigit / 2 : kDigit;
    for (int i = tid; i < kDigit; i += kThreads) hist[i] = 0;
    __syncthreads();
    each([&](int, uint32_t k, bool there) {
      if (there && (k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
    });
    __syncthreads();
    // Bins from the largest on, two per thread: the bin that holds the left-th key.
    const int hi = bins - 1 - 2 * tid, h0 = hi >= 0 ? hist[hi] : 0, h1 = hi >= 1 ? hist[hi - 1] : 0;
    int total;
    const int before = block_scan(h0 + h1, wave_sums, total);
    if (before < left && left <= before + h0 + h1) {
      const bool first = left <= before + h0;
      found[0] = first ? hi : hi - 1;
      found[1] = left - before - (first ? 0 : h0);
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(found[0]) << shift;
    mask |= static_cast<uint32_t>(bins - 1) << shift;
    left = found[1];
    if (shift == 0) break;
  }
  // prefix is T, and the first `left` rows with key T stay.
  const uint64_t below = (1ull << lane_id()) - 1;
  const int wave = wave_id();
  if constexpr (PER > 0) {
    each([&](int i, uint32_t k, bool there) {
      const uint64_t above = __ballot(there && k > prefix), at = __ballot(there && k == prefix);
      if (lane_id() == 0) {
        count_s[0][i * kWaves + wave] = __popcll(above);
        count_s[1][i * kWaves + wave] = __popcll(at);
      }
    });
    __syncthreads();
    // Where each (i, wave)'s rows start among the rows that stay, and how many of its ties do.
    const bool entry = tid < steps * kWaves;
    const int above = entry ? count_s[0][tid] : 0, at = entry ? count_s[1][tid] : 0;
    int total;
    const int ties = max(0, min(at, left - block_scan(at, wave_sums, total)));
    const int start = block_scan(above + ties, wave_sums, total);
    if (entry) {
      count_s[0][tid] = start;
      count_s[1][tid] = ties;
    }
    __syncthreads();
    each([&](int i, uint32_t k, bool there) {
      const bool tie = there && k == prefix;
      const int rank = __popcll(__ballot(tie) & below);
      const bool stays = (there && k > prefix) || (tie && rank < count_s[1][i * kWaves + wave]);
      const uint64_t all = __ballot(stays);
      if (stays) kept[count_s[0][i * kWaves + wave] + __popcll(all & below)] = i * kThreads + tid;
    });
  } else {
    int start = 0, ties_before = 0;
    for (int i = 0; i < steps; ++i) {
      const int64_t row = static_cast<int64_t>(i) * kThreads + tid;
      const bool there = row < old;
      const uint32_t k = weight_key(w[imin64(row, old - 1)]);
      int ties, stay;
      const int tie = there && k == prefix;
      const int rank = ties_before + block_scan(tie, wave_sums, ties);
      const bool stays = (there && k > prefix) || (tie && rank < left);
      const int at = start + block_scan(stays, wave_sums, stay);
      if (stays) kept[at] = static_cast<int32_t>(row);
      ties_before += ties;
      start += stay;
    }
  }
}

// Rows of K and V in 16-byte units, their weights and positions; rows without a source are zero.
__global__ __launch_bounds__(kCopyThreads) void evict_copy_kernel(logkv_evict_args a) {
  __shared__ int src[kCopyRows];
  const int lane = blockIdx.y, G = a.n_groups, b = lane / G, g = lane % G, tid = threadIdx.x;
  const int j0 = blockIdx.x * kCopyRows, rows = min(kCopyRows, a.keep - j0);
  if (tid < rows) {
    const int s = gp(a.kept)[static_cast<int64_t>(lane) * a.keep + j0 + tid];
    src[tid] = s;
    gp(a.out_weights)[b * a.ow_sb + g * a.ow_sg + j0 + tid] = s < 0 ? 0.f : gp(a.weights)[b * a.w_sb + g * a.w_sg + s];
    if (a.out_positions)
      gp(a.out_positions)[b * a.op_sb + g * a.op_sg + j0 + tid] = s < 0 ? -1 : gp(a.positions)[b * a.p_sb + g * a.p_sg + s];
  }
  __syncthreads();
  const int ku = a.dk * a.size / 16, vu = a.dv * a.size / 16, units = ku + vu, items = rows * units;
  const LOGKV_G char* k = reinterpret_cast<const LOGKV_G char*>(gp(static_cast<const char*>(a.cache_k))) + (b * a.ck_sb + g * a.ck_sg) * a.size;
  const LOGKV_G char* v = reinterpret_cast<const LOGKV_G char*>(gp(static_cast<const char*>(a.cache_v))) + (b * a.cv_sb + g * a.cv_sg) * a.size;
  LOGKV_G char* ok = gp(static_cast<char*>(a.out_k)) + (b * a.ok_sb + g * a.ok_sg) * a.size;
  LOGKV_G char* ov = gp(static_cast<char*>(a.out_v)) + (b * a.ov_sb + g * a.ov_sg) * a.size;
  constexpr int kBatch = 4;
  for (int i0 = tid; i0 < items; i0 += kBatch * kCopyThreads) {
    uint4 x[kBatch];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int i = i0 + q * kCopyThreads;
      x[q] = make_uint4(0, 0, 0, 0);
      if (i >= items) continue;
      const int r = i / units, u = i - r * units, s = src[r];
      if (s < 0) continue;
      x[q] = u < ku ? *(const LOGKV_G uint4*)(k + s * a.ck_st * a.size + 16 * u)
                    : *(const LOGKV_G uint4*)(v + s * a.cv_st * a.size + 16 * (u - ku));
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int i = i0 + q * kCopyThreads;
      if (i >= items) continue;
      const int r = i / units, u = i - r * units;
      if (u < ku) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, x[q]), (LOGKV_G u32x4*)(ok + (j0 + r) * a.ok_st * a.size + 16 * u));
      else __builtin_nontemporal_store(__builtin_bit_cast(u32x4, x[q]), (LOGKV_G u32x4*)(ov + (j0 + r) * a.ov_st * a.size + 16 * (u - ku)));
    }
  }
}

int launch_evict(const logkv_evict_args& a, hipStream_t stream) {
  const int lanes = a.n_batch * a.n_groups;
  // Keys in registers up to 32 a thread (32768 rows).
  const int per = (a.cap + kThreads - 1) / kThreads;
  const dim3 grid(lanes), block(kThreads);
  if (per <= 2) hipLaunchKernelGGL(evict_select_kernel<2>, grid, block, 0, stream, a);
  else if (per <= 4) hipLaunchKernelGGL(evict_select_kernel<4>, grid, block, 0, stream, a);
  else if (per <= 8) hipLaunchKernelGGL(evict_select_kernel<8>, grid, block, 0, stream, a);
  else if (per <= 32) hipLaunchKernelGGL(evict_select_kernel<32>, grid, block, 0, stream, a);
  else hipLaunchKernelGGL(evict_select_kernel<0>, grid, block, 0, stream, a);
  hipLaunchKernelGGL(evict_copy_kernel, dim3((a.keep + kCopyRows - 1) / kCopyRows, lanes), dim3(kCopyThreads), 0, stream, a);
  return hipGetLastError() == hipSuccess ? LOGKV_OK : LOGKV_ERUNTIME;
}

}  // namespace logkv
