// A tree of drafted tokens on the bifocal cache: ancestor masks from parent links, the fused "norm -> RoPE -> cache
// write" of the drafted nodes, and the C entry points of the three tree operators.
#include "tc_common.cuh"
#include "../../include/jetlong_b200_tree.h"

namespace jl {

namespace {

// One thread per node walks its parent links.  Every link must go to an EARLIER node, so a walk ends after at most
// `nodes` steps whatever the input holds; a link that does not is an absent node.
__global__ void __launch_bounds__(JL_TREE_MAX_NODES) tree_plan_kernel(const int32_t* parents, int32_t* depth, uint64_t* mask, int nodes) {
  __shared__ int par[JL_TREE_MAX_NODES];
  const int b = blockIdx.x, t = threadIdx.x;
  const int64_t base = static_cast<int64_t>(b) * nodes;
  tc::wait_prerequisites();
  tc::launch_dependents();
  if (t < nodes) par[t] = parents[base + t];
  __syncthreads();
  if (t >= nodes) return;
  uint64_t w[JL_TREE_MAX_NODES / 64] = {};
  int cur = t, d = -1;
  bool present = true;
  for (;;) {
    const int up = par[cur];
    if (up < -1 || up >= cur) { present = false; break; }
#pragma unroll
    for (int i = 0; i < JL_TREE_MAX_NODES / 64; ++i)
      if ((cur >> 6) == i) w[i] |= uint64_t(1) << (cur & 63);
    ++d;
    if (up < 0) break;
    cur = up;
  }
  depth[base + t] = present ? d : -1;
  const int words = (nodes + 63) / 64;
#pragma unroll
  for (int i = 0; i < JL_TREE_MAX_NODES / 64; ++i)
    if (i < words) mask[(base + t) * words + i] = present ? w[i] : 0;
}

struct AppendParams {
  const __nv_bfloat16 *q, *k, *v, *qw, *kw;
  int64_t qs_b, qs_s, qs_h, ks_b, ks_s, ks_h, vs_b, vs_s, vs_h;
  float q_eps, k_eps;
  __nv_bfloat16 *q_base, *q_group, *kc, *vc, *kg;
  int64_t kcs_b, kcs_s, kcs_h, vcs_b, vcs_s, vcs_h, cache_rows;
  int batch, nodes, heads, kv_heads, group_size;
  const float* inv_freq;
  const int32_t *lens, *depth;
};

// A warp takes two of a node's rows of 128 values (query heads, then key heads, then value heads): it loads them together and forms
// the node's angles once for both.  Bound by the sine and cosine (exact ones, with range reduction) and by latency: 8 x 64 nodes of
// 32 + 8 + 8 heads 12.4 us with the plan, 14.4 with one row a warp; 5 nodes of 16 + 8 + 8 heads 6.2 either way, 8.3 with eight rows.
constexpr int kAppendRows = 2;
__global__ void __launch_bounds__(128) tree_append_kernel(const AppendParams p) {
  tc::wait_prerequisites();
  tc::launch_dependents();
  const int lane = threadIdx.x & 31;
  const int keys0 = p.heads, values0 = p.heads + p.kv_heads, per_node = p.heads + 2 * p.kv_heads, warps = (per_node + kAppendRows - 1) / kAppendRows;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (item >= static_cast<int64_t>(p.batch) * p.nodes * warps) return;
  const int64_t node = item / warps;
  const int h0 = static_cast<int>(item % warps) * kAppendRows;
  const int b = static_cast<int>(node / p.nodes), t = static_cast<int>(node % p.nodes);
  const int d = p.depth[node];
  const int64_t len = p.lens[b];
  if (d < 0) {                                          // an absent node: zero query rows, no cache row
    for (int h = h0; h < min(h0 + kAppendRows, p.heads); ++h) {
      const int64_t q_off = (node * p.heads + h) * kHeadDim;
      *reinterpret_cast<uint2*>(p.q_base + q_off + 4 * lane) = make_uint2(0u, 0u);
      if (p.q_group != nullptr) *reinterpret_cast<uint2*>(p.q_group + q_off + 4 * lane) = make_uint2(0u, 0u);
    }
    return;
  }
  const int64_t row = len + t, pos = len + d;
  const bool store = len >= 0 && row < p.cache_rows;
  uint32_t x0[kAppendRows], x1[kAppendRows];            // values 2 lane, 2 lane + 1 of both halves; of a value head 4 lane .. 4 lane + 3
#pragma unroll
  for (int j = 0; j < kAppendRows; ++j) {
    const int h = h0 + j;
    if (h >= per_node) break;
    const __nv_bfloat16* x = h < keys0     ? p.q + b * p.qs_b + t * p.qs_s + h * p.qs_h
                             : h < values0 ? p.k + b * p.ks_b + t * p.ks_s + (h - keys0) * p.ks_h
                                           : p.v + b * p.vs_b + t * p.vs_s + (h - values0) * p.vs_h;
    const bool value = h >= values0;
    x0[j] = *reinterpret_cast<const uint32_t*>(x + (value ? 4 * lane : 2 * lane));
    x1[j] = *reinterpret_cast<const uint32_t*>(x + (value ? 4 * lane + 2 : 64 + 2 * lane));
  }
  float sb0 = 0.f, cb0 = 0.f, sb1 = 0.f, cb1 = 0.f, sd0 = 0.f, cd0 = 0.f, sd1 = 0.f, cd1 = 0.f;
  if (h0 < values0) {
    const float f0 = p.inv_freq[2 * lane], f1 = p.inv_freq[2 * lane + 1];
    const float tb = static_cast<float>(pos);
    sincosf(__fmul_rn(tb, f0), &sb0, &cb0);
    sincosf(__fmul_rn(tb, f1), &sb1, &cb1);
    if (p.q_group != nullptr || p.kg != nullptr) {
      const float td = static_cast<float>(pos / p.group_size - pos);
      sincosf(__fmul_rn(td, f0), &sd0, &cd0);
      sincosf(__fmul_rn(td, f1), &sd1, &cd1);
    }
  }
#pragma unroll
  for (int j = 0; j < kAppendRows; ++j) {
    const int h = h0 + j;
    if (h >= per_node || (h >= keys0 && !store)) break;
    if (h >= values0) {                                 // plain copy into the cache row
      *reinterpret_cast<uint2*>(p.vc + b * p.vcs_b + row * p.vcs_s + (h - values0) * p.vcs_h + 4 * lane) = make_uint2(x0[j], x1[j]);
      continue;
    }
    const bool is_q = h < keys0;
    const __nv_bfloat16* w = is_q ? p.qw : p.kw;
    const float2 w_lo = unpack_bf16x2(*reinterpret_cast<const uint32_t*>(w + 2 * lane));
    const float2 w_hi = unpack_bf16x2(*reinterpret_cast<const uint32_t*>(w + 64 + 2 * lane));
    float bl0, bl1, bh0, bh1;
    norm_rope_head(unpack_bf16x2(x0[j]), unpack_bf16x2(x1[j]), w_lo, w_hi, is_q ? p.q_eps : p.k_eps, sb0, cb0, sb1, cb1, bl0, bl1, bh0, bh1);
    const int64_t q_off = (node * p.heads + h) * kHeadDim, k_off = b * p.kcs_b + row * p.kcs_s + (h - keys0) * p.kcs_h;
    __nv_bfloat16* dst = is_q ? p.q_base + q_off : p.kc + k_off;
    *reinterpret_cast<uint32_t*>(dst + 2 * lane) = pack_bf16x2(bl0, bl1);
    *reinterpret_cast<uint32_t*>(dst + 64 + 2 * lane) = pack_bf16x2(bh0, bh1);
    __nv_bfloat16* grp = is_q ? p.q_group : p.kg;
    if (grp == nullptr) continue;
    grp += is_q ? q_off : k_off;
    *reinterpret_cast<uint32_t*>(grp + 2 * lane) = pack_bf16x2(bl0 * cd0 - bh0 * sd0, bl1 * cd1 - bh1 * sd1);
    *reinterpret_cast<uint32_t*>(grp + 64 + 2 * lane) = pack_bf16x2(bh0 * cd0 + bl0 * sd0, bh1 * cd1 + bl1 * sd1);
  }
}

struct KeepParams {
  __nv_bfloat16 *kc, *vc, *kg;
  int64_t kcs_b, kcs_s, kcs_h, vcs_b, vcs_s, vcs_h, cache_rows;
  const int32_t *path, *lens;
  int kept, kv_heads;
};

// One thread per 16 bytes of a cache row's (buffer, head) carries its column along the path.  Entries rise, so entry j is at
// least j and a row that has been overwritten is never read again: 8 rows are loaded together, then stored.  Bound by the
// latency of one launch and two dependent reads: 1.8 us for 6 nodes of 8 heads in three buffers, 2.0 us for 8 samples.
// grid x: 128 threads over kv_heads * 16 columns, y: sample, z: buffer.
__global__ void __launch_bounds__(128) tree_keep_kernel(const KeepParams p) {
  __shared__ int path[JL_TREE_MAX_NODES];
  __shared__ int n_sh;
  const int b = blockIdx.y, which = blockIdx.z;
  tc::wait_prerequisites();
  tc::launch_dependents();
  for (int i = threadIdx.x; i < p.kept; i += 128) path[i] = p.path[static_cast<int64_t>(b) * p.kept + i];
  const int64_t len = p.lens[b];
  if (threadIdx.x == 0) n_sh = p.kept;
  __syncthreads();
  for (int i = threadIdx.x; i < p.kept; i += 128)                    // the first entry that ends the path
    if (path[i] <= (i > 0 ? path[i - 1] : -1) || len < 0 || len + path[i] >= p.cache_rows) atomicMin(&n_sh, i);
  __syncthreads();
  const int n = n_sh, col = blockIdx.x * 128 + threadIdx.x, h = col >> 4;
  __nv_bfloat16* base = which == 0 ? p.kc : which == 1 ? p.vc : p.kg;
  if (h >= p.kv_heads || base == nullptr) return;
  const int64_t ss = which == 1 ? p.vcs_s : p.kcs_s;
  base += b * (which == 1 ? p.vcs_b : p.kcs_b) + len * ss + h * (which == 1 ? p.vcs_h : p.kcs_h) + (col & 15) * 8;
  for (int i0 = 0; i0 < n; i0 += 8) {
    uint4 x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j < n) x[j] = *reinterpret_cast<const uint4*>(base + path[i0 + j] * ss);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j < n) *reinterpret_cast<uint4*>(base + (i0 + j) * ss) = x[j];
  }
}

int launch_tree_keep(const jl_tree_keep_args* a, cudaStream_t stream) {
  if (a->head_dim != kHeadDim) return fail(JL_ERR_UNSUPPORTED, "jl_tree_keep: head_dim must be 128, got %d", a->head_dim);
  if (a->batch < 0 || a->batch > 65535 || a->kept < 0 || a->kept > JL_TREE_MAX_NODES || a->kv_heads < 1 || a->cache_rows < 0)
    return fail(JL_ERR_BAD_ARG, "jl_tree_keep: sizes out of range");
  if (a->batch == 0 || a->kept == 0) return JL_OK;
  if (a->path == nullptr || a->lens == nullptr) return fail(JL_ERR_BAD_ARG, "jl_tree_keep: NULL pointer");
  if ((reinterpret_cast<uintptr_t>(a->path) | reinterpret_cast<uintptr_t>(a->lens)) & 3) return fail(JL_ERR_BAD_ARG, "jl_tree_keep: misaligned pointer");
  if ((reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache) | reinterpret_cast<uintptr_t>(a->k_group_cache)) & 15)
    return fail(JL_ERR_BAD_ARG, "jl_tree_keep: caches must be 16-byte aligned");
  const int64_t st[] = {a->kc_stride_b, a->kc_stride_s, a->kc_stride_h, a->vc_stride_b, a->vc_stride_s, a->vc_stride_h};
  const int64_t size[] = {a->batch, a->cache_rows, a->kv_heads};
  for (int i = 0; i < 6; ++i) {
    if (st[i] % 8 != 0) return fail(JL_ERR_BAD_ARG, "jl_tree_keep: strides must be multiples of 8 elements");
    if (size[i % 3] > 1 && st[i] <= 0) return fail(JL_ERR_UNSUPPORTED, "jl_tree_keep: a cache dimension larger than 1 needs a positive stride");
  }
  const int rc = check_device_arch();
  if (rc != JL_OK) return rc;
  KeepParams p{};
  p.kc = static_cast<__nv_bfloat16*>(a->k_cache); p.vc = static_cast<__nv_bfloat16*>(a->v_cache); p.kg = static_cast<__nv_bfloat16*>(a->k_group_cache);
  p.kcs_b = a->kc_stride_b; p.kcs_s = a->kc_stride_s; p.kcs_h = a->kc_stride_h;
  p.vcs_b = a->vc_stride_b; p.vcs_s = a->vc_stride_s; p.vcs_h = a->vc_stride_h;
  p.cache_rows = a->cache_rows; p.path = a->path; p.lens = a->lens; p.kept = a->kept; p.kv_heads = a->kv_heads;
  if (launch_dependent(tree_keep_kernel, dim3((a->kv_heads * 16 + 127) / 128, a->batch, 3), dim3(128), 0, stream, p) != cudaSuccess)
    return check_launch("jl_tree_keep");
  return JL_OK;
}

int launch_tree_plan(const jl_tree_plan_args* a, cudaStream_t stream) {
  if (a->batch < 0 || a->nodes < 1 || a->nodes > JL_TREE_MAX_NODES)
    return fail(JL_ERR_BAD_ARG, "jl_tree_plan: need batch >= 0 and 1 <= nodes <= %d, got %d and %d", JL_TREE_MAX_NODES, a->batch, a->nodes);
  if (a->batch == 0) return JL_OK;                      // empty arrays may be NULL
  if (a->parents == nullptr || a->depth == nullptr || a->mask == nullptr) return fail(JL_ERR_BAD_ARG, "jl_tree_plan: NULL pointer");
  if ((reinterpret_cast<uintptr_t>(a->parents) | reinterpret_cast<uintptr_t>(a->depth)) & 3 || reinterpret_cast<uintptr_t>(a->mask) & 7)
    return fail(JL_ERR_BAD_ARG, "jl_tree_plan: misaligned pointer");
  const int rc = check_device_arch();
  if (rc != JL_OK) return rc;
  if (launch_dependent(tree_plan_kernel, dim3(a->batch), dim3((a->nodes + 31) / 32 * 32), 0, stream, a->parents, a->depth, a->mask, a->nodes) != cudaSuccess)
    return check_launch("jl_tree_plan");
  return JL_OK;
}

int launch_tree_append(const jl_tree_append_args* a, cudaStream_t stream) {
  if (a->head_dim != kHeadDim) return fail(JL_ERR_UNSUPPORTED, "jl_tree_append: head_dim must be 128, got %d", a->head_dim);
  if (a->batch < 0 || a->nodes < 1 || a->nodes > JL_TREE_MAX_NODES || a->heads < 1 || a->kv_heads < 1 || a->cache_rows < 0)
    return fail(JL_ERR_BAD_ARG, "jl_tree_append: sizes out of range");
  if (a->batch == 0) return JL_OK;                      // empty arrays may be NULL
  if (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->q_weight == nullptr || a->k_weight == nullptr || a->q_base == nullptr ||
      a->k_cache == nullptr || a->v_cache == nullptr || a->inv_freq == nullptr || a->lens == nullptr || a->depth == nullptr)
    return fail(JL_ERR_BAD_ARG, "jl_tree_append: NULL pointer");
  if ((a->q_group != nullptr || a->k_group_cache != nullptr) && a->group_size < 1)
    return fail(JL_ERR_BAD_ARG, "jl_tree_append: group_size must be >= 1");
  const int64_t st[] = {a->q_stride_b, a->q_stride_s, a->q_stride_h, a->k_stride_b, a->k_stride_s, a->k_stride_h,
                        a->v_stride_b, a->v_stride_s, a->v_stride_h, a->kc_stride_b, a->kc_stride_s, a->kc_stride_h,
                        a->vc_stride_b, a->vc_stride_s, a->vc_stride_h};
  for (int64_t v : st)
    if (v % 4 != 0) return fail(JL_ERR_BAD_ARG, "jl_tree_append: strides must be multiples of 4 elements");
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v) |
                         reinterpret_cast<uintptr_t>(a->q_base) | reinterpret_cast<uintptr_t>(a->q_group) |
                         reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache) |
                         reinterpret_cast<uintptr_t>(a->k_group_cache) | reinterpret_cast<uintptr_t>(a->q_weight) |
                         reinterpret_cast<uintptr_t>(a->k_weight);
  if (ptrs & 7) return fail(JL_ERR_BAD_ARG, "jl_tree_append: pointers must be 8-byte aligned");
  if (misaligned(4, a->inv_freq, a->lens, a->depth)) return fail(JL_ERR_BAD_ARG, "jl_tree_append: inv_freq, lens and depth must be 4-byte aligned");
  const int64_t cache_size[] = {a->batch, a->cache_rows, a->kv_heads, a->batch, a->cache_rows, a->kv_heads};
  for (int i = 0; i < 6; ++i)
    if (cache_size[i] > 1 && st[9 + i] <= 0) return fail(JL_ERR_UNSUPPORTED, "jl_tree_append: a cache dimension larger than 1 needs a positive stride");
  const int rc = check_device_arch();
  if (rc != JL_OK) return rc;
  AppendParams p{};
  p.q = static_cast<const __nv_bfloat16*>(a->q); p.k = static_cast<const __nv_bfloat16*>(a->k);
  p.v = static_cast<const __nv_bfloat16*>(a->v);
  p.qw = static_cast<const __nv_bfloat16*>(a->q_weight); p.kw = static_cast<const __nv_bfloat16*>(a->k_weight);
  p.qs_b = a->q_stride_b; p.qs_s = a->q_stride_s; p.qs_h = a->q_stride_h;
  p.ks_b = a->k_stride_b; p.ks_s = a->k_stride_s; p.ks_h = a->k_stride_h;
  p.vs_b = a->v_stride_b; p.vs_s = a->v_stride_s; p.vs_h = a->v_stride_h;
  p.q_eps = a->q_eps; p.k_eps = a->k_eps;
  p.q_base = static_cast<__nv_bfloat16*>(a->q_base); p.q_group = static_cast<__nv_bfloat16*>(a->q_group);
  p.kc = static_cast<__nv_bfloat16*>(a->k_cache); p.vc = static_cast<__nv_bfloat16*>(a->v_cache);
  p.kg = static_cast<__nv_bfloat16*>(a->k_group_cache);
  p.kcs_b = a->kc_stride_b; p.kcs_s = a->kc_stride_s; p.kcs_h = a->kc_stride_h;
  p.vcs_b = a->vc_stride_b; p.vcs_s = a->vc_stride_s; p.vcs_h = a->vc_stride_h;
  p.cache_rows = a->cache_rows;
  p.batch = a->batch; p.nodes = a->nodes; p.heads = a->heads; p.kv_heads = a->kv_heads;
  p.group_size = a->group_size > 0 ? a->group_size : 1;
  p.inv_freq = a->inv_freq; p.lens = a->lens; p.depth = a->depth;
  const int64_t blocks = (static_cast<int64_t>(a->batch) * a->nodes * ((a->heads + 2 * a->kv_heads + kAppendRows - 1) / kAppendRows) + 3) / 4;
  if (blocks > 0x7fffffff) return fail(JL_ERR_UNSUPPORTED, "jl_tree_append: too many rows for one launch");
  if (launch_dependent(tree_append_kernel, dim3(static_cast<unsigned>(blocks)), dim3(128), 0, stream, p) != cudaSuccess) return check_launch("jl_tree_append");
  return JL_OK;
}

}  // namespace

int launch_tree_attention(const jl_tree_attention_args* a, cudaStream_t stream);
int tree_status();
size_t tree_attention_workspace_bytes(int32_t batch, int32_t nodes, int32_t heads, int32_t kv_heads, int32_t rows);

static int validate_tree_attention(const jl_tree_attention_args* a) {
  if (a->head_dim != kHeadDim) return fail(JL_ERR_UNSUPPORTED, "jl_tree_attention: head_dim must be 128, got %d", a->head_dim);
  if (a->batch < 0 || a->heads < 1 || a->kv_heads < 1) return fail(JL_ERR_BAD_ARG, "jl_tree_attention: batch/heads/kv_heads out of range");
  if (a->nodes < 1 || a->nodes > JL_TREE_MAX_NODES)
    return fail(JL_ERR_BAD_ARG, "jl_tree_attention: nodes must be in [1, %d], got %d", JL_TREE_MAX_NODES, a->nodes);
  if (a->heads % a->kv_heads != 0) return fail(JL_ERR_BAD_ARG, "jl_tree_attention: heads must be divisible by kv_heads");
  if (a->heads / a->kv_heads > 128) return fail(JL_ERR_UNSUPPORTED, "jl_tree_attention: at most 128 query heads per kv head");
  if (a->rows < a->nodes) return fail(JL_ERR_BAD_ARG, "jl_tree_attention: the cache (%d rows) does not hold the %d nodes", a->rows, a->nodes);
  if (a->w_0 < 0) return fail(JL_ERR_BAD_ARG, "jl_tree_attention: w_0 must be >= 0");
  // the running maximum is taken of the unscaled scores
  if (!(a->softmax_scale > 0.f) || isinf(a->softmax_scale)) return fail(JL_ERR_BAD_ARG, "jl_tree_attention: softmax_scale must be positive and finite");
  if ((a->q_group == nullptr) != (a->k_group == nullptr))
    return fail(JL_ERR_BAD_ARG, "jl_tree_attention: q_group and k_group come together or not at all");
  if (a->batch == 0) return JL_OK;                      // empty arrays may be NULL
  if (a->q_base == nullptr || a->k_base == nullptr || a->v == nullptr || a->out == nullptr || a->lens == nullptr || a->depth == nullptr ||
      a->mask == nullptr)
    return fail(JL_ERR_BAD_ARG, "jl_tree_attention: NULL pointer");
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(a->q_base) | reinterpret_cast<uintptr_t>(a->q_group) |
                         reinterpret_cast<uintptr_t>(a->k_base) | reinterpret_cast<uintptr_t>(a->k_group) |
                         reinterpret_cast<uintptr_t>(a->v) | reinterpret_cast<uintptr_t>(a->out);
  if (ptrs & 15) return fail(JL_ERR_BAD_ARG, "jl_tree_attention: pointers must be 16-byte aligned");
  if (misaligned(4, a->lens, a->depth, a->lse) || misaligned(8, a->mask))
    return fail(JL_ERR_BAD_ARG, "jl_tree_attention: lens, depth and lse must be 4-byte aligned, mask 8-byte");
  const int64_t st[] = {a->q_stride_b, a->q_stride_s, a->q_stride_h, a->k_stride_b, a->k_stride_s, a->k_stride_h,
                        a->v_stride_b, a->v_stride_s, a->v_stride_h, a->o_stride_b, a->o_stride_s, a->o_stride_h};
  for (int64_t x : st)
    if (x % 8 != 0) return fail(JL_ERR_BAD_ARG, "jl_tree_attention: strides must be multiples of 8 elements (16 bytes)");
  const int64_t size[] = {a->batch, a->nodes, a->heads, a->batch, a->rows, a->kv_heads, a->batch, a->rows, a->kv_heads, a->batch, a->nodes, a->heads};
  for (int i = 0; i < 12; ++i)
    if (size[i] > 1 && st[i] <= 0) return fail(JL_ERR_UNSUPPORTED, "jl_tree_attention: a dimension larger than 1 needs a positive stride");
  return JL_OK;
}

}  // namespace jl

extern "C" {

int jl_tree_plan(const jl_tree_plan_args* args, void* cuda_stream) {
  if (args == nullptr) return jl::fail(JL_ERR_BAD_ARG, "jl_tree_plan: args is NULL");
  return jl::launch_tree_plan(args, static_cast<cudaStream_t>(cuda_stream));
}

int jl_tree_append(const jl_tree_append_args* args, void* cuda_stream) {
  if (args == nullptr) return jl::fail(JL_ERR_BAD_ARG, "jl_tree_append: args is NULL");
  return jl::launch_tree_append(args, static_cast<cudaStream_t>(cuda_stream));
}

size_t jl_tree_attention_workspace_bytes(int32_t batch, int32_t nodes, int32_t heads, int32_t kv_heads, int32_t rows) {
  return jl::tree_attention_workspace_bytes(batch, nodes, heads, kv_heads, rows);
}

int jl_tree_attention(const jl_tree_attention_args* args, void* cuda_stream) {
  if (args == nullptr) return jl::fail(JL_ERR_BAD_ARG, "jl_tree_attention: args is NULL");
  int rc = jl::validate_tree_attention(args);
  if (rc != JL_OK) return rc;
  if (args->batch == 0) return JL_OK;
  rc = jl::check_device_arch();
  if (rc != JL_OK) return rc;
  return jl::launch_tree_attention(args, static_cast<cudaStream_t>(cuda_stream));
}

int jl_tree_keep(const jl_tree_keep_args* args, void* cuda_stream) {
  if (args == nullptr) return jl::fail(JL_ERR_BAD_ARG, "jl_tree_keep: args is NULL");
  return jl::launch_tree_keep(args, static_cast<cudaStream_t>(cuda_stream));
}

int jl_tree_status(void) { return jl::tree_status(); }

}  // extern "C"
