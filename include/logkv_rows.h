/* Attention over a cache's rows and the rows of the call itself, and eviction of cache rows by
 * accumulated attention weight (C ABI of liblogkv_hip.so, gfx950).
 *
 * Conventions are logkv_hip.h's: device pointers, strides in elements, a hipStream_t as void*;
 * an entry point validates, enqueues on the caller's stream, never allocates and never
 * synchronizes; LOGKV_EINVAL leaves every buffer as it was and logkv_last_error() says why.
 *
 * No counterpart in the reference: its LogKV path has neither a mask among the in-flight rows
 * (log_kv_slot_attention takes a dense mask on its slow path, litgpt/log_kv_cache.py:6501-6570)
 * nor an exact cache that is cut by attention weight. */
#ifndef LOGKV_ROWS_H
#define LOGKV_ROWS_H

#include <stdint.h>

#include "logkv_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { LOGKV_BF16 = 0, LOGKV_F16 = 1 };

/* tq queries per head q [n_batch, n_heads, tq, dk] over the first n_b rows of
 * cache_k / cache_v [n_batch, n_groups, cap, dk / dv] and the call's own rows k / v
 * [n_batch, n_groups, tq, dk / dv] (one per query position), head h reading KV group
 * h / (n_heads / n_groups):
 *
 *   s_j = scale q . cache_k_j + bias_scale bias_j   for j < n_b
 *   s_r = scale q . k_r                             for the own rows r that the query sees
 *   out = softmax(s) [cache_v; v]                   (zeros where a query sees no row)
 *
 * n_b = lengths[b * len_stride] + *lengths2 + len_add (absent pointers count as 0), held to
 * [0, cap]. A NaN or infinity in a row that a query does not see does not reach its output.
 * dtype: LOGKV_BF16 or LOGKV_F16 for q, k, v, the cache and out; arithmetic in float32, the
 * probabilities enter the value products as two parts of 8 (bf16) or 11 (fp16) bits each, rounded,
 * whatever the queries' number and the values' size.
 * dk, dv: multiples of 8 up to 256; every row 16-byte aligned (strides multiples of 8); features
 * contiguous. bias (tree attention): float32, or dtype with bias_half, strided; NULL for none;
 * -inf hides a row. bias_scale: a positive factor, 0 for 1. Where float32 holds the logits in steps
 * of 1 or more (beyond 2^22), an output is still a mean of values, but weights are not kept to it.
 * visible (tree attention): uint8 [tq, tq] per batch row (vis_sb 0: one for all), rows vis_st
 * apart: own row r is seen by query t where visible[t, r] is not 0.
 * counts (weight attention, optional): int32 [n_batch]; only the first counts[b] queries and own
 * rows of batch row b exist (the others' outputs are zeros).
 * weights (weight attention): float32 [n_batch, n_groups, cap]. */
typedef struct logkv_rows_args {
  const uint16_t* q;
  int64_t q_sb, q_sh, q_st;
  const uint16_t* k;
  int64_t k_sb, k_sg, k_st;
  const uint16_t* v;
  int64_t v_sb, v_sg, v_st;
  uint16_t* cache_k;
  int64_t ck_sb, ck_sg, ck_st;
  uint16_t* cache_v;
  int64_t cv_sb, cv_sg, cv_st;
  const void* bias;
  int64_t b_sb, b_sg, b_st;
  const int32_t* lengths;
  const int32_t* lengths2;
  const uint8_t* visible;
  int64_t vis_sb, vis_st;
  const int32_t* counts;
  float* weights;
  int64_t w_sb, w_sg;
  uint16_t* out;
  int64_t o_sb, o_sh, o_st;
  int32_t n_batch, n_heads, n_groups, tq, cap, dk, dv, dtype;
  int32_t len_stride, len_add, bias_half;
  float scale, bias_scale;
} logkv_rows_args;

/* Scratch of one call of either attention below. */
int64_t logkv_rows_workspace_bytes(const logkv_rows_args* args);

/* Attention of drafted tokens over a cache: `visible` says which drafted rows a token sees. The
 * cache is only read. */
int logkv_tree_attention(const logkv_rows_args* args, void* workspace, int64_t workspace_bytes, void* stream);

/* Causal attention of new tokens that adds to weights[j], j < n_b, the sum over the group's heads
 * and the queries of row j's probability, sets weights[n_b + r] to own row r's sum, and stores the
 * own rows at cache rows n_b + r (those below cap). Rows of weights and cache behind them are
 * left as they were. Every sum has a fixed order: equal calls give equal bits. */
int logkv_weight_attention(const logkv_rows_args* args, void* workspace, int64_t workspace_bytes, void* stream);

/* Cuts each lane (batch row, KV group) of a cache to at most `keep` rows: of its n = lengths[b]
 * rows (len_add where lengths is NULL; held to [0, cap]) the last `recent` and, of the others, the
 * ones of largest weight (ties: the lowest index; NaN counts as the largest), in their order. With
 * n <= keep all rows stay. Writes, per lane, rows [0, keep) of out_k / out_v (dk / dv features of
 * `size` bytes each, rows contiguous in features, row bytes and strides multiples of 16 bytes),
 * out_weights [lanes, keep], out_positions (int64, optional with positions), kept (int32, the rows'
 * indices) and out_lengths [n_batch] = min(n, keep); rows from min(n, keep) on: zeros, kept and
 * positions -1. Outputs must not overlap the inputs. Strides in elements. */
typedef struct logkv_evict_args {
  const void* cache_k;
  int64_t ck_sb, ck_sg, ck_st;
  const void* cache_v;
  int64_t cv_sb, cv_sg, cv_st;
  const float* weights;
  int64_t w_sb, w_sg;
  const int64_t* positions;
  int64_t p_sb, p_sg;
  const int32_t* lengths;
  void* out_k;
  int64_t ok_sb, ok_sg, ok_st;
  void* out_v;
  int64_t ov_sb, ov_sg, ov_st;
  float* out_weights;
  int64_t ow_sb, ow_sg;
  int64_t* out_positions;
  int64_t op_sb, op_sg;
  int32_t* kept;
  int32_t* out_lengths;
  int32_t n_batch, n_groups, cap, dk, dv, size;
  int32_t len_add, keep, recent;
} logkv_evict_args;

int logkv_evict_rows(const logkv_evict_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LOGKV_ROWS_H */
