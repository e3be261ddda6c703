// Rotary positions, and appends to a paged cache with the rotation on the way.
//
//   (a, b) -> amplitude (a cos t - b sin t, b cos t + a sin t),  t = sign pos f_i
//
// for the pairs i of a head's rotated part; the rest passes through. A block takes TPB tokens with all
// of their heads, so that an angle is formed once for every head: as turns, pos (f / 2 pi) in 64 bits
// with the product's rounding error added back, reduced to [-1/2, 1/2] before it is rounded to float32
// (a float32 product would be off by 2^-8 of a turn at position 65536). Sine and cosine of the block's
// angles wait in LDS. An item is VEC pairs, VEC features that pass through, or VEC features of a value;
// threads load a batch of items before they form angles.
// Bound by HBM for many tokens, by the chain length -> table entry -> store for one.
#include <algorithm>

#include "paged.hpp"

namespace logkv {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxAngles = 1024;   // of a block: 4 tokens of 512 rotated features
constexpr int kBatch = 4;          // items of a thread on their way at once

// What the launch derives from the arguments. Quotients by multiplication: n / d = high32(n * magic),
// exact for n * d < 2^32 (checked by the launch).
struct RotaryPlan {
  int tpb;                      // tokens of a block
  int turned, items;            // items of a head: pairs, and in all
  int q_items, k_items, v_items, token_items;   // of a token
  int v_units;                  // items of a value
  uint32_t by_token, by_head, by_value, by_half;
  int half;
};

__device__ __forceinline__ int quotient(int n, uint32_t magic, int d) {
  return d == 1 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), magic));
}

template <int DT>
struct Type {
  typedef uint16_t raw;
  static __device__ __forceinline__ float get(raw x) { return Elem<DT>::to_f32(x); }
  static __device__ __forceinline__ raw put(float x) { return Elem<DT>::from_f32(x); }
};
template <>
struct Type<LOGKV_F32> {
  typedef float raw;
  static __device__ __forceinline__ float get(raw x) { return x; }
  static __device__ __forceinline__ raw put(float x) { return x; }
};

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

}  // namespace

template <int DT, int CT, int VEC, bool APPEND>
__global__ __launch_bounds__(kThreads) void rotary_kernel(logkv_rotary_args a, RotaryPlan p) {
  typedef Type<DT> In;
  typedef Type<CT> Out;
  typedef typename In::raw raw;
  typedef typename Out::raw cached;
  __shared__ __align__(16) float2 turn_s[kMaxAngles];
  __shared__ int64_t pos_s[16], k_at[16], v_at[16];
  const int tid = threadIdx.x;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.tpb, all = static_cast<int64_t>(a.n_batch) * a.tokens;
  const int here = static_cast<int>(imin64(p.tpb, all - first)), total = here * p.token_items;

  // An item: its token, whose features they are (0: q, 1: k, 2: v), its head and its place there.
  struct Item {
    int token, of, head, j;
  };
  auto item = [&](int e) {
    Item x;
    x.token = quotient(e, p.by_token, p.token_items);
    int r = e - x.token * p.token_items;
    x.of = r < p.q_items ? 0 : r < p.q_items + p.k_items ? 1 : 2;
    r -= x.of == 0 ? 0 : x.of == 1 ? p.q_items : p.q_items + p.k_items;
    const int d = x.of == 2 ? p.v_units : p.items;
    x.head = quotient(r, x.of == 2 ? p.by_value : p.by_head, d);
    x.j = r - x.head * d;
    return x;
  };
  auto feature = [&](const Item& x, int& second) {
    // The item's first feature, and that of its second vector.
    if (x.of < 2 && x.j < p.turned) {
      const int f = a.interleaved ? 2 * VEC * x.j : VEC * x.j;
      second = a.interleaved ? f + VEC : f + p.half;
      return f;
    }
    second = -1;
    return x.of < 2 ? a.rotated + VEC * (x.j - p.turned) : VEC * x.j;
  };
  auto batch_row = [&](int token, int& t) {
    const int64_t at = first + token;
    const int b = static_cast<int>(at / a.tokens);
    t = static_cast<int>(at - static_cast<int64_t>(b) * a.tokens);
    return b;
  };
  auto source = [&](const Item& x) {
    int t;
    const int b = batch_row(x.token, t);
    if (x.of == 0) return static_cast<const raw*>(a.q) + b * a.q_sb + x.head * a.q_sh + t * a.q_st;
    if (x.of == 1) return static_cast<const raw*>(a.k) + b * a.k_sb + x.head * a.k_sh + t * a.k_st;
    return static_cast<const raw*>(a.v) + b * a.v_sb + x.head * a.v_sh + t * a.v_st;
  };

  Pack<raw, VEC> x0[kBatch], x1[kBatch];
  auto load = [&](int e0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int e = min(e0 + kThreads * i, total - 1);
      const Item it = item(e);
      int second;
      const int f = feature(it, second);
      const raw* row = source(it);
      x0[i] = load_pack<raw, VEC>(row + f);
      x1[i] = load_pack<raw, VEC>(row + (second < 0 ? f : second));
    }
  };
  load(tid);

  // Positions, and where the tokens' rows are stored.
  if (tid < here) {
    int t;
    const int b = batch_row(tid, t);
    int64_t pos = a.first + t, row = 0;
    if constexpr (APPEND) {
      row = static_cast<int64_t>(a.len_add) + (a.lengths ? gp(a.lengths)[b] : 0) + t;
      pos = a.first + row;
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
    if (a.first_dev) pos += gp(a.first_dev)[b];
    if (a.positions) {
      const int64_t at = b * a.pos_sb + t * a.pos_st;
      pos = a.pos_int ? gp(static_cast<const int32_t*>(a.positions))[at] : gp(static_cast<const int64_t*>(a.positions))[at];
    }
    pos_s[tid] = pos;
  }
  __syncthreads();
  for (int e = tid; e < here * p.half; e += kThreads) {
    const int token = quotient(e, p.by_half, p.half), i = e - token * p.half;
    const double f = a.freq_float ? static_cast<double>(gp(static_cast<const float*>(a.frequencies))[i])
                                  : gp(static_cast<const double*>(a.frequencies))[i];
    const double turns = f * 0.15915494309189533577, n = static_cast<double>(pos_s[token]);
    const double u = n * turns, lost = __builtin_fma(n, turns, -u);
    const float x = static_cast<float>((u - __builtin_rint(u)) + lost);
    float sn, cs;
    sincospif(2.f * x, &sn, &cs);
    turn_s[e] = make_float2(a.amplitude * cs, a.amplitude * a.sign * sn);
  }
  __syncthreads();

  for (int e0 = tid; e0 < total; e0 += kBatch * kThreads) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int e = e0 + kThreads * i;
      if (e >= total) break;
      const Item it = item(e);
      int second, t;
      const int f = feature(it, second), b = batch_row(it.token, t);
      float y0[VEC], y1[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) y0[k] = In::get(x0[i].x[k]), y1[k] = In::get(x1[i].x[k]);
      if (second >= 0) {
        const float2* turn = turn_s + it.token * p.half + VEC * it.j;
        auto turned = [&](float& u, float& w, float2 c) {
          const float r = __builtin_fmaf(u, c.x, -(w * c.y));
          w = __builtin_fmaf(w, c.x, u * c.y);
          u = r;
        };
        if (VEC > 1 && a.interleaved) {
#pragma unroll
          for (int k = 0; k + 1 < VEC; k += 2) {
            turned(y0[k], y0[k + 1], turn[k / 2]);
            turned(y1[k], y1[k + 1], turn[(VEC + k) / 2]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < VEC; ++k) turned(y0[k], y1[k], turn[k]);
        }
      }
      if (it.of == 0 || (!APPEND && it.of == 1)) {
        raw* o = it.of == 0 ? static_cast<raw*>(a.q_out) + b * a.qo_sb + it.head * a.qo_sh + t * a.qo_st
                            : static_cast<raw*>(a.k_out) + b * a.ko_sb + it.head * a.ko_sh + t * a.ko_st;
        Pack<raw, VEC> z;
#pragma unroll
        for (int k = 0; k < VEC; ++k) z.x[k] = In::put(y0[k]);
        store_pack(o + f, z);
        if (second >= 0) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) z.x[k] = In::put(y1[k]);
          store_pack(o + second, z);
        }
      } else if constexpr (APPEND) {
        Pack<cached, VEC> z0, z1;
#pragma unroll
        for (int k = 0; k < VEC; ++k) z0.x[k] = Out::put(y0[k]), z1.x[k] = Out::put(y1[k]);
        if (it.of == 1) {
          if (a.k_out) {
            cached* o = static_cast<cached*>(a.k_out) + b * a.ko_sb + it.head * a.ko_sh + t * a.ko_st;
            store_pack(o + f, z0);
            if (second >= 0) store_pack(o + second, z1);
          }
          if (k_at[it.token] >= 0) {
            cached* o = reinterpret_cast<cached*>(a.k_pages) + k_at[it.token] + it.head * a.kp_sg;
            store_pack(o + f, z0);
            if (second >= 0) store_pack(o + second, z1);
          }
        } else if (v_at[it.token] >= 0) {
          store_pack(reinterpret_cast<cached*>(a.v_pages) + v_at[it.token] + it.head * a.vp_sg + f, z0);
        }
      }
    }
    if (e0 + kBatch * kThreads < total) load(e0 + kBatch * kThreads);
  }
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
  p.items = p.turned + (a.dim - a.rotated) / vec;
  p.q_items = a.q ? a.n_heads * p.items : 0;
  p.k_items = a.k ? a.n_groups * p.items : 0;
  p.v_units = APPEND ? a.dim_v / vec : 0;
  p.v_items = a.n_groups * p.v_units;
  p.token_items = p.q_items + p.k_items + p.v_items;
  const int64_t all = static_cast<int64_t>(a.n_batch) * a.tokens;
  // Four tokens a block where that leaves every CU blocks to overlap.
  p.tpb = all >= 4 * 1024 ? 4 : 1;
  const int64_t most = static_cast<int64_t>(p.tpb) * p.token_items, widest = std::max({p.token_items, p.items, p.v_units, p.half});
  if (most * widest >= int64_t(1) << 32) return refuse("too many heads for one rotation");
  p.by_token = magic_of(p.token_items);
  p.by_head = magic_of(p.items);
  p.by_value = magic_of(p.v_units);
  p.by_half = magic_of(p.half);
  const int64_t blocks = (all + p.tpb - 1) / p.tpb;
  if (blocks > INT32_MAX) return refuse("too many tokens for one rotation");
  const dim3 grid(static_cast<uint32_t>(blocks));
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
