// pz_refuse.h -- which calls of the logit rules, the 8-bit LM head, the attention
// over a paged cache and the beam search are refused, and why.  Host only and
// without a device, so that the refusals have a test of their own.
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
constexpr size_t PZ_TREE_WS = (size_t)64 << 20;  // bytes of tree attention's workspace
constexpr int PZ_MOST_PREFIXES = 1 << 12;  // whose ranges are given
constexpr int PZ_MOST_ROWS = 1 << 15;  // of a sequence in prefix attention, so that its
                                       // results of two parts fit the workspace
constexpr int PZ_MOST_IDS = 1 << 22;   // of a selection, whose lists of one row are in the workspace
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

inline PzRefusal pz_refuse_prefix(const pz_kv_cache* c, const pz_kv_prefix* p, const void* d_kn,
                                  const void* d_vn, long ld_n, int B, int T, int n_heads,
                                  float scale, const void* d_q, long ld_q, const void* d_out,
                                  long ld_out) {
  const PzRefusal r =
      pz_refuse_tree(c, d_kn, d_vn, ld_n, B, T, n_heads, scale, d_q, ld_q, d_out, ld_out);
  if (r.code) return r;
  if (!p || !p->d_blocks || !p->d_len || p->max_blocks <= 0 || p->n_prefixes <= 0)
    return {PZ_EINVAL, "bad prefix"};
  if ((int64_t)p->max_blocks * c->block_size > INT32_MAX - 64)
    return {PZ_ERANGE, "the prefix's max_blocks * block_size does not fit 32 bits"};
  if (!p->d_first && B % p->n_prefixes)
    return {PZ_EINVAL, "without d_first n_prefixes divides B"};
  // (every workgroup looks for its prefix among the ranges, 64 at a time)
  if (p->d_first && p->n_prefixes > PZ_MOST_PREFIXES)
    return {PZ_ERANGE, "n_prefixes above 4096 with d_first"};
  // (two parts of a sequence's rows are in the workspace)
  if ((int64_t)T * n_heads > PZ_MOST_ROWS ||
      2 * (int64_t)T * n_heads * (c->head_dim + 2) * (int64_t)sizeof(float) > (int64_t)PZ_TREE_WS)
    return {PZ_ERANGE, "T * n_heads above 32768, or 32513 with heads of 256"};
  return PZ_TAKEN;
}

inline PzRefusal pz_refuse_rope(const pz_qk_rope* r, const void* d_q, long ld_q, const void* d_k,
                                long ld_k, const void* d_qo, long ld_qo, const void* d_ko,
                                long ld_ko, int n, const int32_t* d_pos) {
  if (!r || n < 0 || r->n_heads < 0 || r->n_kv_heads < 0 || r->n_heads + r->n_kv_heads <= 0)
    return {PZ_EINVAL, "bad heads or tokens"};
  if (r->type != PZ_F32 && r->type != PZ_BF16 && r->type != PZ_F16)
    return {PZ_EINVAL, "type is PZ_F32, PZ_BF16 or PZ_F16"};
  if (r->head_dim <= 0) return {PZ_EINVAL, "bad head_dim"};
  if (r->head_dim > 1024) return {PZ_ENOTSUP, "head_dim above 1024"};
  if (r->n_heads > PZ_MOST_HEADS || r->n_kv_heads > PZ_MOST_HEADS)
    return {PZ_ERANGE, "n_heads or n_kv_heads above 65536"};
  if (r->rot_dim < 0 || r->rot_dim > r->head_dim || r->rot_dim % 2)
    return {PZ_EINVAL, "rot_dim is even, 0 to head_dim"};
  if (r->layout != PZ_ROPE_HALVES && r->layout != PZ_ROPE_PAIRS)
    return {PZ_EINVAL, "layout is PZ_ROPE_HALVES or PZ_ROPE_PAIRS"};
  if (r->rot_dim && (!r->d_freq || !d_pos)) return {PZ_EINVAL, "a rotation needs d_freq and d_pos"};
  if ((r->d_q_norm || r->d_k_norm) && !(r->eps >= 0.0f && r->eps < 3.0e38f))
    return {PZ_EINVAL, "eps is finite and not negative"};
  const uintptr_t odd = r->type == PZ_F32 ? 3 : 1;
  const struct {
    const void *in, *out;
    long ld_in, ld_out;
    int heads;
  } parts[2] = {{d_q, d_qo, ld_q, ld_qo, r->n_heads}, {d_k, d_ko, ld_k, ld_ko, r->n_kv_heads}};
  for (const auto& p : parts) {
    if (!p.heads) continue;
    const long row = (long)p.heads * r->head_dim;
    if (!p.in || !p.out || p.ld_in < row || p.ld_out < row)
      return {PZ_EINVAL, "bad rows: null, or a stride less than heads * head_dim"};
    if (p.in == p.out && p.ld_in != p.ld_out) return {PZ_EINVAL, "in place needs equal strides"};
    if (((uintptr_t)p.in & odd) || ((uintptr_t)p.out & odd))
      return {PZ_EINVAL, "rows are not aligned to their type"};
  }
  if (((uintptr_t)r->d_q_norm | (uintptr_t)r->d_k_norm | (uintptr_t)r->d_freq) & 3)
    return {PZ_EINVAL, "d_q_norm, d_k_norm or d_freq is not aligned to 4 bytes"};
  // (a wave for every head is the most that a launch takes)
  if (!pz_launch_fits((int64_t)n * (r->n_heads + r->n_kv_heads), 64))
    return {PZ_ERANGE, "more tokens and heads than a launch takes"};
  return PZ_TAKEN;
}

// Whether the rotation's kernel with four waves a workgroup takes n tokens of `heads` heads: a
// wave for each is the most that it launches, whose workgroups are rounded up.  (So the three
// largest calls that are taken go to the kernel with one.)
inline bool pz_rope_in_fours(int n, int heads) {
  return pz_launch_fits(((int64_t)n * heads + 3) / 4, 256);
}

inline PzRefusal pz_refuse_select(const float* d_logits, long ld, int n_groups, int W, int V,
                                  const float* d_scores, int K, const int32_t* d_parent,
                                  const int32_t* d_ids, const float* d_scores_out) {
  if (!d_logits || !d_scores || !d_parent || !d_ids || !d_scores_out || n_groups < 0 || V <= 0 ||
      ld < V)
    return {PZ_EINVAL, "bad logits, scores or outputs"};
  if (W <= 0 || K <= 0) return {PZ_EINVAL, "W and K are positive"};
  if (W > PZ_BEAM_MAX_WIDTH) return {PZ_ERANGE, "W > PZ_BEAM_MAX_WIDTH"};
  if (K > PZ_BEAM_MAX_SELECT) return {PZ_ERANGE, "K > PZ_BEAM_MAX_SELECT"};
  if (V > PZ_MOST_IDS) return {PZ_ERANGE, "V above 2^22"};
  if (n_groups > PZ_BEAM_MAX_BEAMS) return {PZ_ERANGE, "n_groups above 2^20"};
  return PZ_TAKEN;
}

inline PzRefusal pz_refuse_reorder(const pz_kv_cache* layers, int n_layers, int n_groups, int W,
                                   const int32_t* d_parent, const int32_t* d_pool, int n_pool,
                                   int ahead, const int32_t* d_blocks_out,
                                   const int32_t* d_len_out) {
  if (!layers || n_layers <= 0 || n_groups < 0 || !d_parent || !d_blocks_out || !d_len_out)
    return {PZ_EINVAL, "bad layers, parents or outputs"};
  if (W <= 0) return {PZ_EINVAL, "W is positive"};
  if (W > PZ_BEAM_MAX_WIDTH) return {PZ_ERANGE, "W > PZ_BEAM_MAX_WIDTH"};
  if (n_pool < 0 || (n_pool > 0 && !d_pool)) return {PZ_EINVAL, "n_pool>0 needs d_pool"};
  if (n_pool > PZ_BEAM_MAX_POOL) return {PZ_ERANGE, "n_pool > PZ_BEAM_MAX_POOL"};
  if (ahead < 0) return {PZ_EINVAL, "ahead is not negative"};
  if ((int64_t)n_groups * W > PZ_BEAM_MAX_BEAMS)
    return {PZ_ERANGE, "n_groups * W > PZ_BEAM_MAX_BEAMS"};
  for (int i = 0; i < n_layers; i++) {
    const pz_kv_cache &c = layers[i], &o = layers[0];
    const PzRefusal r = pz_refuse_cache(&c, c.d_k, c.d_v, c.ld, n_groups * W, 1);
    if (r.code) return r;
    if (c.type != o.type || c.n_kv_heads != o.n_kv_heads || c.head_dim != o.head_dim ||
        c.ld != o.ld || c.n_blocks != o.n_blocks || c.block_size != o.block_size ||
        c.d_blocks != o.d_blocks || c.max_blocks != o.max_blocks || c.d_len != o.d_len)
      return {PZ_EINVAL, "layers differ in more than d_k and d_v"};
  }
  if ((int64_t)W * layers[0].max_blocks > PZ_MOST) return {PZ_ERANGE, "W * max_blocks above 2^30"};
  if (d_blocks_out == layers[0].d_blocks || d_len_out == layers[0].d_len)
    return {PZ_EINVAL, "new tables and lengths are not the old ones"};
  return PZ_TAKEN;
}
