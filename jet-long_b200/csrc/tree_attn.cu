// Attention of a tree of drafted tokens over the bifocal cache.
//
// One block per (node, head, sample): its warps take the keys in turn, one key per step with 4 dimensions a lane, and
// keep a running (maximum, sum, output) in fp32; the warps' states are merged through shared memory.
#include "jl_common.cuh"
#include "../../include/jetlong_b200_tree.h"

namespace jl {

namespace {

constexpr int kWarps = 8;

__global__ void __launch_bounds__(kWarps * 32) tree_attention_kernel(const jl_tree_attention_args a) {
  const int t = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = h / (a.heads / a.kv_heads);
  const int T = a.nodes, words = (T + 63) / 64;
  const int len = min(max(a.lens[b], 0), a.rows - T);
  const int64_t node = static_cast<int64_t>(b) * T + t;
  const int d = a.depth[node];
  auto row4 = [&](const void* base, int64_t off) {
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(base) + off + 4 * lane);
    const float2 x = unpack_bf16x2(u.x), y = unpack_bf16x2(u.y);
    return make_float4(x.x, x.y, y.x, y.y);
  };
  const int64_t q_off = b * a.q_stride_b + t * a.q_stride_s + h * a.q_stride_h;
  const float4 qb = row4(a.q_base, q_off), qg = a.q_group != nullptr ? row4(a.q_group, q_off) : qb;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  const int n = d < 0 ? 0 : len + T;
  for (int j = warp; j < n; j += kWarps) {
    int pk = j;
    if (j >= len) {
      const int u = j - len;
      if (!((a.mask[node * words + (u >> 6)] >> (u & 63)) & 1)) continue;
      pk = len + a.depth[static_cast<int64_t>(b) * T + u];
    }
    const bool far = a.q_group != nullptr && len + d - pk > a.w_0;
    const float4 k = row4(far ? a.k_group : a.k_base, b * a.k_stride_b + j * a.k_stride_s + kvh * a.k_stride_h);
    const float4 q = far ? qg : qb;
    float s = q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    s *= a.softmax_scale;
    const float4 v = row4(a.v, b * a.v_stride_b + j * a.v_stride_s + kvh * a.v_stride_h);
    const float mn = fmaxf(m, s), f = expf(m - mn), e = expf(s - mn);
    m = mn;
    l = l * f + e;
    o.x = o.x * f + e * v.x; o.y = o.y * f + e * v.y; o.z = o.z * f + e * v.z; o.w = o.w * f + e * v.w;
  }
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][kHeadDim];
  *reinterpret_cast<float4*>(&so[warp][4 * lane]) = o;
  if (lane == 0) { sm[warp] = m; sl[warp] = l; }
  __syncthreads();
  if (threadIdx.x >= kHeadDim) return;
  float M = -INFINITY, L = 0.f, acc = 0.f;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm[w]);
  for (int w = 0; w < kWarps && M != -INFINITY; ++w) {
    const float f = expf(sm[w] - M);
    L += sl[w] * f;
    acc += so[w][threadIdx.x] * f;
  }
  static_cast<__nv_bfloat16*>(a.out)[b * a.o_stride_b + t * a.o_stride_s + h * a.o_stride_h + threadIdx.x] =
      __float2bfloat16(L > 0.f ? acc / L : 0.f);
  if (threadIdx.x == 0 && a.lse != nullptr)
    a.lse[(static_cast<int64_t>(b) * a.heads + h) * T + t] = L > 0.f ? M + logf(L) : -INFINITY;
}

}  // namespace

size_t tree_attention_workspace_bytes(int32_t, int32_t, int32_t, int32_t, int32_t) { return 16; }

int launch_tree_attention(const jl_tree_attention_args* a, cudaStream_t stream) {
  if (a->batch > 65535 || a->heads > 65535) return fail(JL_ERR_UNSUPPORTED, "jl_tree_attention: batch and heads must be at most 65535");
  tree_attention_kernel<<<dim3(a->nodes, a->heads, a->batch), kWarps * 32, 0, stream>>>(*a);
  return check_launch("jl_tree_attention");
}

}  // namespace jl
