// Rotary positions, and appends to a paged cache with the rotation on the way.
//
//   (a, b) -> amplitude (a cos t - b sin t, b cos t + a sin t),  t = sign pos f_i
//
// for the pairs i of a head's rotated part; the rest passes through. A block takes TPB tokens of a batch
// row with all of their heads, so that an angle is formed once for every head: as turns, pos (f / 2 pi) in
// 64 bits with the product's rounding error added back, reduced to [-1/2, 1/2] before it is rounded to
// float32 (a float32 product would be off by 2^-8 of a turn at position 65536). Sine and cosine of the
// block's angles wait in LDS behind the block's only barrier. An item is VEC pairs, VEC features that pass
// through, or VEC features of a value; a thread loads its first query's, key's and value's item before it
// forms angles, and then one ahead.
// Bound by HBM for many tokens: 16001 tokens of 40 heads of 128 features 66 us, 4.9 TB/s of the 5.07 of a large copy;
// 8 x 4096 tokens appended with 16 + 8 + 8 heads 119 us, 5.07 TB/s. By the chain length -> table entry -> store for one:
// 5.2 us with its launch, a rotation alone 3.6 (items unrolled into straight code took 16 us: cold instructions).
#include <algorithm>
#include <type_traits>

#include "paged.hpp"

namespace logkv {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 8;      // of a block
constexpr int kMaxAngles = 1024;   // of a block
constexpr int64_t kMostItems = 1024, kLeastBlocks = 1024;   // of a block beyond one token, and of a launch

// What the launch derives from the arguments. Quotients by multiplication: n / d = high32(n * magic),
// exact for n * d < 2^32 (checked by the launch).
struct RotaryPlan {
  int tpb, tiles;         // tokens of a block, blocks of a batch row
  int half, turned;       // pairs of a head, and items of pairs
  int items[3], heads[3]; // of q, k and v: items of a head, heads
  uint32_t by_item[3], by_head[3], by_half;
};

__device__ __forceinline__ int quotient(int n, uint32_t magic, int d) {
  return d == 1 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), magic));
}

template <typename T, int N>
struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack {
  T x[N];
};

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
  return *(const LOGKV_G Pack<T, N>*)gp(p);
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& x) {
  *(LOGKV_G Pack<T, N>*)gp(p) = x;
}

template <int DT>
struct Type {
  typedef uint16_t raw;
  static __device__ __forceinline__ float get(raw x) { return Elem<DT>::to_f32(x); }
  // Rounded to nearest, two at a time by the hardware's conversions.
  template <int N>
  static __device__ __forceinline__ Pack<raw, N> put(const float (&y)[N]) {
    Pack<raw, N> z;
    if constexpr (N == 1) {
      z.x[0] = Elem<DT>::from_f32(y[0]);
    } else {
#pragma unroll
      for (int k = 0; k < N; k += 2) {
        uint32_t two;
        if constexpr (DT == LOGKV_BF16) two = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{y[k], y[k + 1]}, bf16x2));
        else two = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{y[k], y[k + 1]}, f16x2));
        z.x[k] = static_cast<raw>(two), z.x[k + 1] = static_cast<raw>(two >> 16);
      }
    }
    return z;
  }
};
template <>
struct Type<LOGKV_F32> {
  typedef float raw;
  static __device__ __forceinline__ float get(raw x) { return x; }
  template <int N>
  static __device__ __forceinline__ Pack<raw, N> put(const float (&y)[N]) {
    Pack<raw, N> z;
#pragma unroll
    for (int k = 0; k < N; ++k) z.x[k] = y[k];
    return z;
  }
};

}  // namespace

template <int DT, int CT, int VEC, bool APPEND>
__global__ __launch_bounds__(kThreads) void rotary_kernel(logkv_rotary_args a, RotaryPlan p) {
  typedef Type<DT> In;
  typedef typename In::raw raw;
  typedef Type<APPEND ? CT : LOGKV_BF16> Out;   // of an append's pages
  typedef uint16_t cached;
  __shared__ __align__(16) float2 turn_s[kMaxAngles];
  __shared__ int64_t k_at[kMaxTokens], v_at[kMaxTokens];   // rows in the pages, below 0 for none
  const int tid = threadIdx.x;
  const int blk = static_cast<int>(blockIdx.y * gridDim.x + blockIdx.x), b = blk / p.tiles, t0 = (blk - b * p.tiles) * p.tpb;
  if (b >= a.n_batch) return;
  const int here = min(p.tpb, a.tokens - t0);

  // Item e of the block's queries (OF 0), keys (1) or values (2): its token, head, first feature and that of its second
  // vector (-1: it passes through).
  struct Item {
    int token, head, f, second;
  };
  auto item = [&](auto of, int e) {
    constexpr int OF = decltype(of)::value;
    const int row = quotient(e, p.by_item[OF], p.items[OF]), j = e - row * p.items[OF];
    Item x;
    x.token = quotient(row, p.by_head[OF], p.heads[OF]);
    x.head = row - x.token * p.heads[OF];
    x.second = -1;
    if (OF == 2) {
      x.f = VEC * j;
    } else if (j < p.turned) {
      x.f = a.interleaved ? 2 * VEC * j : VEC * j;
      x.second = a.interleaved ? x.f + VEC : x.f + p.half;
    } else {
      x.f = a.rotated + VEC * (j - p.turned);
    }
    return x;
  };
  typedef Pack<raw, VEC> vec;
  // An item's vectors on their way (of an item past the last: nothing).
  auto load = [&](auto of, int e, int n, vec& x0, vec& x1) {
    constexpr int OF = decltype(of)::value;
    if (e >= n) return;
    const Item x = item(of, e);
    const raw* row = OF == 0   ? static_cast<const raw*>(a.q) + b * a.q_sb + x.head * a.q_sh + (t0 + x.token) * a.q_st
                     : OF == 1 ? static_cast<const raw*>(a.k) + b * a.k_sb + x.head * a.k_sh + (t0 + x.token) * a.k_st
                               : static_cast<const raw*>(a.v) + b * a.v_sb + x.head * a.v_sh + (t0 + x.token) * a.v_st;
    x0 = load_pack<raw, VEC>(row + x.f);
    if (OF < 2) x1 = load_pack<raw, VEC>(row + (x.second < 0 ? x.f : x.second));
  };
  std::integral_constant<int, 0> of_q;
  std::integral_constant<int, 1> of_k;
  std::integral_constant<int, 2> of_v;
  const int nq = here * p.heads[0] * p.items[0], nk = here * p.heads[1] * p.items[1];
  const int nv = APPEND ? here * p.heads[2] * p.items[2] : 0;
  // The first item of each kind is loaded before the angles are formed.
  vec q0, q1, k0, k1, v0, v1;
  load(of_q, tid, nq, q0, q1);
  load(of_k, tid, nk, k0, k1);
  if constexpr (APPEND) load(of_v, tid, nv, v0, v1);

  int64_t row0 = 0;   // the row of the batch row's first token
  if constexpr (APPEND) {
    row0 = static_cast<int64_t>(a.len_add) + (a.lengths ? gp(a.lengths)[b] : 0);
    if (tid < here) {
      const int t = t0 + tid;
      const int64_t row = row0 + t;
      int64_t ko = -1, vo = -1;
      if (row >= 0 && row < static_cast<int64_t>(a.table_len) * a.page && (!a.counts || t < gp(a.counts)[b])) {
        const int shift = __builtin_ctz(a.page), slot = static_cast<int>(row) & (a.page - 1);
        const int page = gp(a.table)[b * a.table_sb + (row >> shift)];
        if (static_cast<uint32_t>(page) < static_cast<uint32_t>(a.n_pages)) {
          ko = page * a.kp_sp + slot * a.kp_st;
          vo = page * a.vp_sp + slot * a.vp_st;
        }
      }
      k_at[tid] = ko;
      v_at[tid] = vo;
    }
  }
  for (int e = tid; e < here * p.half; e += kThreads) {
    const int token = quotient(e, p.by_half, p.half), i = e - token * p.half, t = t0 + token;
    int64_t pos;
    if (a.positions) {
      const int64_t at = b * a.pos_sb + t * a.pos_st;
      pos = a.pos_int ? gp(static_cast<const int32_t*>(a.positions))[at] : gp(static_cast<const int64_t*>(a.positions))[at];
    } else {
      pos = a.first + (a.first_dev ? gp(a.first_dev)[b] : 0) + row0 + t;
    }
    const double f = a.freq_float ? static_cast<double>(gp(static_cast<const float*>(a.frequencies))[i])
                                  : gp(static_cast<const double*>(a.frequencies))[i];
    const double turns = f * 0.15915494309189533577, at = static_cast<double>(pos);
    const double u = at * turns, lost = __builtin_fma(at, turns, -u);
    const float x = static_cast<float>((u - __builtin_rint(u)) + lost);
    float sn, cs;
    sincospif(2.f * x, &sn, &cs);
    turn_s[e] = make_float2(a.amplitude * cs, a.amplitude * a.sign * sn);
  }
  __syncthreads();

  auto turn = [&](const Item& x, float (&y0)[VEC], float (&y1)[VEC]) {
    if (x.second < 0) return;
    const float2* at = turn_s + x.token * p.half + (a.interleaved ? x.f / 2 : x.f);
    auto pair = [](float& u, float& v, float2 c) {
      const float r = __builtin_fmaf(u, c.x, -(v * c.y));
      v = __builtin_fmaf(v, c.x, u * c.y);
      u = r;
    };
    if (VEC > 1 && a.interleaved) {
#pragma unroll
      for (int k = 0; k + 1 < VEC; k += 2) {
        pair(y0[k], y0[k + 1], at[k / 2]);
        pair(y1[k], y1[k + 1], at[(VEC + k) / 2]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) pair(y0[k], y1[k], at[k]);
    }
  };
  auto spread = [](const vec& x, float (&y)[VEC]) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) y[k] = In::get(x.x[k]);
  };
  // All items of one kind; the next one's loads are issued before one is finished.
  auto finish = [&](auto of, int n, vec& x0, vec& x1) {
    constexpr int OF = decltype(of)::value;
#pragma unroll 1
    for (int e = tid; e < n; e += kThreads) {
      const vec c0 = x0, c1 = x1;
      load(of, e + kThreads, n, x0, x1);
      const Item x = item(of, e);
      float y0[VEC], y1[VEC];
      spread(c0, y0);
      if constexpr (OF == 2) {
        if (v_at[x.token] >= 0) store_pack(a.v_pages + v_at[x.token] + x.head * a.vp_sg + x.f, Out::put(y0));
      } else {
        spread(c1, y1);
        turn(x, y0, y1);
        auto store = [&](auto* row, auto as) {
          typedef decltype(as) T;
          store_pack(row + x.f, T::put(y0));
          if (x.second >= 0) store_pack(row + x.second, T::put(y1));
        };
        const int t = t0 + x.token;
        if constexpr (OF == 0) {
          store(static_cast<raw*>(a.q_out) + b * a.qo_sb + x.head * a.qo_sh + t * a.qo_st, In());
        } else if constexpr (!APPEND) {
          store(static_cast<raw*>(a.k_out) + b * a.ko_sb + x.head * a.ko_sh + t * a.ko_st, In());
        } else {
          if (a.k_out) store(static_cast<cached*>(a.k_out) + b * a.ko_sb + x.head * a.ko_sh + t * a.ko_st, Out());
          if (k_at[x.token] >= 0) store(a.k_pages + k_at[x.token] + x.head * a.kp_sg, Out());
        }
      }
    }
  };
  finish(of_q, nq, q0, q1);
  finish(of_k, nk, k0, k1);
  if constexpr (APPEND) finish(of_v, nv, v0, v1);
}

namespace {

uint32_t magic_of(int d) { return d > 1 ? static_cast<uint32_t>(((uint64_t(1) << 32) + d - 1) / d) : 0; }

template <int DT, int CT, bool APPEND>
int launch_vec(const logkv_rotary_args& a, hipStream_t stream) {
  constexpr int size = DT == LOGKV_F32 ? 4 : 2;
  // The widest items, up to 16 bytes a vector, that every row's address and the head's parts allow.
  auto allows = [&](int vec) {
    const int64_t in = std::min(16, vec * size), out = vec * (APPEND ? 2 : size);
    auto rows = [&](const void* p, int64_t sb, int64_t sh, int64_t st, int64_t bytes, int64_t each) {
      return !p || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && sb * each % bytes == 0 && sh * each % bytes == 0 &&
                    st * each % bytes == 0);
    };
    return a.rotated % (2 * vec) == 0 && (a.dim - a.rotated) % vec == 0 && (!a.v || a.dim_v % vec == 0) &&
           rows(a.q, a.q_sb, a.q_sh, a.q_st, in, size) && rows(a.q_out, a.qo_sb, a.qo_sh, a.qo_st, in, size) &&
           rows(a.k, a.k_sb, a.k_sh, a.k_st, in, size) &&
           rows(a.k_out, a.ko_sb, a.ko_sh, a.ko_st, std::min<int64_t>(16, out), APPEND ? 2 : size) &&
           rows(a.v, a.v_sb, a.v_sh, a.v_st, in, size) &&
           (!APPEND || (rows(a.k_pages, a.kp_sp, a.kp_sg, a.kp_st, out, 2) && rows(a.v_pages, a.vp_sp, a.vp_sg, a.vp_st, out, 2)));
  };
  const int vec = DT != LOGKV_F32 && allows(8) ? 8 : allows(4) ? 4 : 1;
  RotaryPlan p{};
  p.half = a.rotated / 2;
  p.turned = p.half / vec;
  const int row_items = p.turned + (a.dim - a.rotated) / vec;
  const int items[3] = {row_items, row_items, APPEND ? a.dim_v / vec : 1};
  const int heads[3] = {a.q ? a.n_heads : 0, a.k ? a.n_groups : 0, APPEND ? a.n_groups : 0};
  int64_t token_items = 0, widest = p.half;
  for (int of = 0; of < 3; ++of) {
    p.items[of] = items[of], p.heads[of] = heads[of];
    p.by_item[of] = magic_of(items[of]), p.by_head[of] = magic_of(heads[of]);
    token_items += int64_t(items[of]) * heads[of];
    widest = std::max<int64_t>({widest, items[of], heads[of]});
  }
  p.by_half = magic_of(p.half);
  // As many tokens a block as its angles have room for, where that leaves every CU blocks to overlap. One token a block,
  // this rule and eight always, 8 + 2 heads of 128 features: 1024 tokens 4.9, 4.8 and 6.0 us, 4096 10.0, 6.8 and 7.4, 65536
  // 122, 76 and 76; 32 + 8 heads: 256 tokens 4.7, 4.7 and 7.1, 16000 71, 65 and 65.
  p.tpb = 1;
  while (p.tpb < kMaxTokens && p.tpb < a.tokens && 2 * p.tpb * p.half <= kMaxAngles && p.tpb * token_items < kMostItems &&
         static_cast<int64_t>(a.n_batch) * a.tokens >= 2 * p.tpb * kLeastBlocks)
    p.tpb *= 2;
  // A block's items, and their products in quotient().
  if (p.tpb * token_items * std::max<int64_t>(widest, 1) >= int64_t(1) << 32) return refuse("too many heads for one rotation");
  p.tiles = (a.tokens + p.tpb - 1) / p.tpb;
  const int64_t blocks = static_cast<int64_t>(p.tiles) * a.n_batch;
  constexpr int64_t kLine = int64_t(1) << 20;   // of the grid, whose axes hold fewer than 2^32 threads
  if (blocks > INT32_MAX - kLine) return refuse("too many tokens for one rotation");
  const dim3 grid(static_cast<uint32_t>(std::min(blocks, kLine)), static_cast<uint32_t>((blocks + kLine - 1) / kLine));
  if (vec == 8) {
    if constexpr (DT != LOGKV_F32) hipLaunchKernelGGL((rotary_kernel<DT, CT, 8, APPEND>), grid, dim3(kThreads), 0, stream, a, p);
  } else if (vec == 4) {
    hipLaunchKernelGGL((rotary_kernel<DT, CT, 4, APPEND>), grid, dim3(kThreads), 0, stream, a, p);
  } else {
    hipLaunchKernelGGL((rotary_kernel<DT, CT, 1, APPEND>), grid, dim3(kThreads), 0, stream, a, p);
  }
  return hipGetLastError() == hipSuccess ? LOGKV_OK : LOGKV_ERUNTIME;
}

template <int DT>
int launch_type(const logkv_rotary_args& a, bool append, hipStream_t stream) {
  if (!append) return launch_vec<DT, DT, false>(a, stream);
  if (a.cache_dtype == LOGKV_BF16) return launch_vec<DT, LOGKV_BF16, true>(a, stream);
  return launch_vec<DT, LOGKV_F16, true>(a, stream);
}

}  // namespace

int launch_rotary(const logkv_rotary_args& a, bool append, hipStream_t stream) {
  if (a.dtype == LOGKV_BF16) return launch_type<LOGKV_BF16>(a, append, stream);
  if (a.dtype == LOGKV_F16) return launch_type<LOGKV_F16>(a, append, stream);
  return launch_type<LOGKV_F32>(a, append, stream);
}

}  // namespace logkv
