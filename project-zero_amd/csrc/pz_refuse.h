// pz_refuse.h -- which calls of the logit rules, the 8-bit LM head and the
// tree attention are refused, and why.  Host only and without a device, so
// that the refusals have a test of their own.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "../../include/pz_sampler.h"

struct PzRefusal {
  int code;         // PZ_OK: the call is taken
  const char* why;  // nullptr then
};
constexpr int PZ_MOST = 1 << 30;  // of ids and list entries, so that 32-bit counters can step past
constexpr int PZ_MOST_HEADS = 1 << 16;  // so that rows and row lengths fit 32 bits
constexpr PzRefusal PZ_TAKEN = {PZ_OK, nullptr};

// Whether a launch of `wgs` workgroups fits: their threads have 32-bit numbers.
inline bool pz_launch_fits(int64_t wgs, int threads) { return wgs <= UINT32_MAX / threads; }

inline bool pz_aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

inline PzRefusal pz_refuse_rules(const float* d_in, long ld_in, const float* d_out, long ld_out,
                                 int B, int V, const pz_logit_rules* r) {
  if (!d_in || !d_out || !r || B < 0 || V <= 0 || ld_in < V || ld_out < V)
    return {PZ_EINVAL, "bad logits/shape"};
  if (V > PZ_MOST || r->H > PZ_MOST || r->n_bias > PZ_MOST)
    return {PZ_ERANGE, "V, H or n_bias above 2^30"};
  if (d_in == d_out && ld_in != ld_out) return {PZ_EINVAL, "in place needs ld_out == ld_in"};
  if (r->H < 0 || (r->H > 0 && !r->d_hist)) return {PZ_EINVAL, "H>0 needs d_hist"};
  if (r->n_bias < 0 || (r->n_bias > 0 && (!r->d_bias_ids || !r->d_bias)))
    return {PZ_EINVAL, "n_bias>0 needs d_bias_ids and d_bias"};
  if (r->n_masks < 0 || (r->n_masks > 0 && !r->d_mask))
    return {PZ_EINVAL, "n_masks>0 needs d_mask"};
  if (r->n_masks > 0 && r->ld_mask < ((long)V + 31) / 32)
    return {PZ_EINVAL, "ld_mask holds less than V bits"};
  if (r->n_masks > 0 && !r->d_mask_row && r->n_masks != B)
    return {PZ_EINVAL, "without d_mask_row there is a mask for each row"};
  return PZ_TAKEN;
}

inline PzRefusal pz_refuse_quant(const void* d_x, int x_type, long ldx, int rows, int n,
                                 const int8_t* d_q, long ldq, const float* d_scale) {
  if (!d_x || !d_q || !d_scale || rows < 0 || n <= 0 || ldx < n || ldq < n)
    return {PZ_EINVAL, "bad rows to quantise"};
  if (x_type != PZ_F32 && x_type != PZ_BF16 && x_type != PZ_F16)
    return {PZ_EINVAL, "x_type is PZ_F32, PZ_BF16 or PZ_F16"};
  if (((uintptr_t)d_x & (x_type == PZ_F32 ? 3 : 1)) != 0)
    return {PZ_EINVAL, "d_x is not aligned to its type"};
  if (!pz_launch_fits(rows, n > 8192 ? 1024 : 256)) return {PZ_ERANGE, "more rows than a launch takes"};
  return PZ_TAKEN;
}

inline PzRefusal pz_refuse_i8(const int8_t* d_w, const float* d_sw, int V, int n,
                              const int8_t* d_x, const float* d_sx, int B, long ldx,
                              int max_batch) {
  if (!d_w || !d_sw || !d_x || !d_sx || V <= 0 || n <= 0 || B < 0 || ldx < n)
    return {PZ_EINVAL, "bad LM head shape"};
  if (n > PZ_I8_MAX_N) return {PZ_ERANGE, "n > PZ_I8_MAX_N: the sum does not fit 32 bits"};
  if (V > PZ_MOST) return {PZ_ERANGE, "V above 2^30"};
  if (B > max_batch) return {PZ_ERANGE, "B > max_batch"};
  return PZ_TAKEN;
}

inline PzRefusal pz_refuse_cache(const pz_kv_cache* c, const void* d_kn, const void* d_vn,
                                 long ld_n, int B, int T) {
  if (!c || !d_kn || !d_vn || B < 0 || T <= 0) return {PZ_EINVAL, "bad nodes"};
  if (T > PZ_TREE_MAX_NODES) return {PZ_ERANGE, "T > PZ_TREE_MAX_NODES"};
  if (c->type != PZ_BF16 && c->type != PZ_F16)
    return {PZ_ENOTSUP, "the cache's type is PZ_BF16 or PZ_F16"};
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return {PZ_ENOTSUP, "head_dim is 64, 128 or 256"};
  if (!c->d_k || !c->d_v || !c->d_blocks || !c->d_len || c->n_kv_heads <= 0 || c->n_blocks <= 0 ||
      c->max_blocks <= 0)
    return {PZ_EINVAL, "bad cache"};
  if (c->block_size < 8 || (c->block_size & (c->block_size - 1)) != 0)
    return {PZ_EINVAL, "block_size is a power of two, at least 8"};
  if (c->n_kv_heads > PZ_MOST_HEADS) return {PZ_ERANGE, "n_kv_heads above 65536"};
  if (!pz_launch_fits((int64_t)B * T, 256))
    return {PZ_ERANGE, "more sequences and nodes than a launch takes"};
  if ((int64_t)c->max_blocks * c->block_size > INT32_MAX - 64)
    return {PZ_ERANGE, "max_blocks * block_size does not fit 32 bits"};
  const long row = (long)c->n_kv_heads * c->head_dim;
  if (c->ld < row || ld_n < row) return {PZ_EINVAL, "a stride is less than n_kv_heads * head_dim"};
  if (c->ld % 8 || ld_n % 8 || !pz_aligned16(c->d_k) || !pz_aligned16(c->d_v) ||
      !pz_aligned16(d_kn) || !pz_aligned16(d_vn))
    return {PZ_EINVAL, "strides are multiples of 8, pointers 16-byte aligned"};
  return PZ_TAKEN;
}

inline PzRefusal pz_refuse_tree(const pz_kv_cache* c, const void* d_kn, const void* d_vn,
                                long ld_n, int B, int T, int n_heads, float scale,
                                const void* d_q, long ld_q, const void* d_out, long ld_out) {
  const PzRefusal r = pz_refuse_cache(c, d_kn, d_vn, ld_n, B, T);
  if (r.code) return r;
  if (n_heads <= 0 || n_heads % c->n_kv_heads)
    return {PZ_EINVAL, "n_heads is a multiple of n_kv_heads"};
  if (n_heads > PZ_MOST_HEADS) return {PZ_ERANGE, "n_heads above 65536"};
  // (the kernels take scale log2(e), which has to be finite, too)
  if (!(scale > 0.0f) || scale > 2.0e38f)
    return {PZ_EINVAL, "scale is positive, at most 2e38"};
  const long row = (long)n_heads * c->head_dim;
  if (!d_q || !d_out || ld_q < row || ld_out < row) return {PZ_EINVAL, "bad q or out"};
  if (ld_q % 8 || ld_out % 8 || !pz_aligned16(d_q) || !pz_aligned16(d_out))
    return {PZ_EINVAL, "strides are multiples of 8, pointers 16-byte aligned"};
  return PZ_TAKEN;
}
