/*
 * jetlong_b200 — C ABI of the drafted-token operators: the step that verifies a TREE of drafted tokens on the
 * bifocal-RoPE cache in one pass.  Conventions (status codes, strides in elements, caller-owned memory, explicit
 * stream, nothing synchronises or allocates) are those of jetlong_b200.h.
 *
 * A tree has `nodes` places per sample.  A node is one drafted token; its parent is an earlier node or the last
 * committed token.  Sample b has lens[b] committed tokens in its cache rows [0, lens[b]); node t is (to be) stored in
 * row lens[b] + t, whatever its depth, and sits at POSITION lens[b] + depth[b][t].
 */
#ifndef JETLONG_B200_TREE_H_
#define JETLONG_B200_TREE_H_

#include "jetlong_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define JL_TREE_MAX_NODES 256

/* ---------------------------------------------------------------------------------------------
 * jl_tree_plan — depth and ancestor mask of every node from its parent links.
 * parents (batch, nodes) int32: -1 for a child of the last committed token, else the index of an EARLIER node.
 * Any other value (by convention -2) marks an absent node, and so does an absent ancestor.
 * depth (batch, nodes) int32: number of ancestors in the tree, -1 for an absent node.
 * mask (batch, nodes, words) 64-bit words, words = (nodes + 63) / 64: bit u of node t is set iff u is t or an
 * ancestor of t; zero for an absent node.  All arrays contiguous.
 * ------------------------------------------------------------------------------------------- */
typedef struct {
  const int32_t* parents;
  int32_t* depth;
  uint64_t* mask;
  int32_t batch, nodes;
} jl_tree_plan_args;

int jl_tree_plan(const jl_tree_plan_args* args, void* cuda_stream);

/* ---------------------------------------------------------------------------------------------
 * jl_tree_append — everything between the q/k/v projections and the attention of a tree step, in one launch: per-head
 * RMSNorm of q and k and RoPE at the nodes' positions, their regrouped copies, and the write of the nodes' keys and
 * values into rows lens[b] + t of the cache.  Same arithmetic and roundings as jl_norm_rope / jl_decode_append, so a
 * drafted token's key has the bits that decoding it would have written.
 * q: (B, T, H, D), k / v: (B, T, Hk, D) with element strides; q_base / q_group: (B, T, H, D) contiguous;
 * k_cache / v_cache: (B, rows, Hk, D) with strides.  q_group and k_group_cache may be NULL (group_size 1);
 * k_group_cache has the strides of k_cache and receives R(floor(p / group_size)) of the new keys.
 * An absent node (depth < 0) gets zero query rows and writes no cache row, and neither does a row past cache_rows.
 * ------------------------------------------------------------------------------------------- */
typedef struct {
  const void* q;
  const void* k;
  const void* v;
  int64_t q_stride_b, q_stride_s, q_stride_h, k_stride_b, k_stride_s, k_stride_h, v_stride_b, v_stride_s, v_stride_h;
  const void* q_weight;     /* (head_dim,) bf16 */
  const void* k_weight;
  float q_eps, k_eps;
  void* q_base;
  void* q_group;            /* may be NULL */
  void* k_cache;
  void* v_cache;
  void* k_group_cache;      /* may be NULL */
  int64_t kc_stride_b, kc_stride_s, kc_stride_h, vc_stride_b, vc_stride_s, vc_stride_h;
  int64_t cache_rows;
  int32_t batch, nodes, heads, kv_heads, head_dim;
  int32_t group_size;
  const float* inv_freq;    /* (head_dim/2,) fp32 device array */
  const int32_t* lens;      /* (batch,) committed tokens, device */
  const int32_t* depth;     /* (batch, nodes), device */
} jl_tree_append_args;

int jl_tree_append(const jl_tree_append_args* args, void* cuda_stream);

/* ---------------------------------------------------------------------------------------------
 * jl_tree_attention — every node against its sample's committed keys and the nodes its mask names, one softmax:
 *   s(t, j) = softmax_scale * (pq - pk > w_0 ? q_group . k_group : q_base . k_base),  pq = lens[b] + depth[b][t],
 *   pk = j for a committed row j < lens[b], lens[b] + depth[b][u] for the node row j = lens[b] + u.
 * q_base / q_group: (B, T, H, D) sharing strides; k_base / k_group / v: (B, rows, Hk, D), k_group with the strides of
 * k_base.  q_group and k_group both NULL: one class, every pair is scored as q_base . k_base.
 * out (B, T, H, D) with strides, lse (B, H, T) fp32 contiguous or NULL.  A row that sees no key (an absent node of
 * an empty cache, a zero mask) is zero with lse = -inf; an absent node (depth < 0) sees nothing.
 * A row with a score of NaN (a query of NaN, say) is NaN, and so is its lse; no other row is.
 * depth[b][t] < nodes.  A value row that an absent node would use may hold anything; the values of present nodes and of
 * committed rows must be finite.  softmax_scale is positive and finite.  batch * kv_heads <= 65535.
 * 0 <= lens[b] <= rows.  Places of the tree that reach past the last row (lens[b] + t >= rows) are absent nodes, whatever depth and mask
 * say of them; a negative length counts as 0, one above rows as rows - nodes.  No row past lens[b] + nodes is read into a result.
 * workspace: jl_tree_attention_workspace_bytes, 16-byte aligned, not initialised by the caller and not kept between
 * calls; two calls that may overlap on the GPU need one each.
 * ------------------------------------------------------------------------------------------- */
typedef struct {
  const void* q_base;
  const void* q_group;
  const void* k_base;
  const void* k_group;
  const void* v;
  int64_t q_stride_b, q_stride_s, q_stride_h, k_stride_b, k_stride_s, k_stride_h, v_stride_b, v_stride_s, v_stride_h;
  const int32_t* lens;
  const int32_t* depth;
  const uint64_t* mask;
  void* out;
  float* lse;
  int64_t o_stride_b, o_stride_s, o_stride_h;
  int32_t batch, nodes, heads, kv_heads, head_dim, rows;
  int64_t w_0;
  float softmax_scale;
  int32_t reserved;
  void* workspace;
  size_t workspace_bytes;
} jl_tree_attention_args;

size_t jl_tree_attention_workspace_bytes(int32_t batch, int32_t nodes, int32_t heads, int32_t kv_heads, int32_t rows);
int jl_tree_attention(const jl_tree_attention_args* args, void* cuda_stream);

/* ---------------------------------------------------------------------------------------------
 * jl_tree_keep — after a path has been chosen: cache row lens[b] + i becomes what row lens[b] + path[b][i] was, in place, in
 * one launch.  path (batch, kept) int32 node indices, root first; a path ends at the first entry that is not larger than
 * the one before it (-1 pads shorter ones) or whose row is outside the cache.  Rows past the path stay as they are.
 * Node path[b][i] of a path has depth i, so positions do not change and rotated keys stay valid where they land.
 * k_cache / v_cache: (B, rows, Hk, D) with strides; k_group_cache has the strides of k_cache.  Each may be NULL.
 * ------------------------------------------------------------------------------------------- */
typedef struct {
  void* k_cache;
  void* v_cache;
  void* k_group_cache;
  int64_t kc_stride_b, kc_stride_s, kc_stride_h, vc_stride_b, vc_stride_s, vc_stride_h;
  int64_t cache_rows;
  const int32_t* path;
  const int32_t* lens;
  int32_t batch, kept, kv_heads, head_dim;
} jl_tree_keep_args;

int jl_tree_keep(const jl_tree_keep_args* args, void* cuda_stream);

/* Diagnostic (synchronises the device): non-zero if a bounded wait (1 s) inside jl_tree_attention has given up on the
 * current device since the last call; reading a raised status clears it.  The results since the last call are then invalid. */
int jl_tree_status(void);

#ifdef __cplusplus
}
#endif
#endif /* JETLONG_B200_TREE_H_ */
