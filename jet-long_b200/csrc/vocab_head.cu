// The vocabulary head without logits: softmax statistics of hidden @ weight^T, and the gradients of the cross-entropy
// loss, formed piece by piece of the vocabulary.
//
//   z = h W^T,  lse = log sum exp z,  nll = lse - z_y,  dz = g (exp(z - lse) - onehot(y)),  dh = dz W,  dW = dz^T h
//
// Scores: one product whose epilogue reduces every 64 x 64 tile of z to (maximum, sum, argmax) per row; a second
// kernel folds the tiles' partials.  Gradients: for each piece of the vocabulary the product is formed again, its
// epilogue stores dz of the piece in bf16, and two more products take it to dW (final for the piece) and dh
// (accumulated in fp32 over the pieces).
#include "jl_common.cuh"
#include "../../include/jetlong_b200_head.h"

namespace jl {

namespace {

constexpr int kTile = 64, kStep = 16;

// element (r, c) of a row-major or transposed bf16 operand
struct Operand {
  const __nv_bfloat16* p;
  int64_t sr, sc;
  __device__ float at(int64_t r, int64_t c) const { return __bfloat162float(p[r * sr + c * sc]); }
};

// acc = A[m0 : m0 + 64, 0 : K] B[n0 : n0 + 64, 0 : K]^T of one 64 x 64 tile, 4 x 4 per thread (256 threads)
__device__ __forceinline__ void tile_product(const Operand& A, const Operand& B, int64_t m0, int64_t n0, int64_t M, int64_t N, int64_t K,
                                             float (&acc)[4][4]) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int64_t k0 = 0; k0 < K; k0 += kStep) {
    for (int i = threadIdx.x; i < kTile * kStep; i += 256) {
      const int r = i / kStep, c = i % kStep;
      sa[c][r] = m0 + r < M && k0 + c < K ? A.at(m0 + r, k0 + c) : 0.f;
      sb[c][r] = n0 + r < N && k0 + c < K ? B.at(n0 + r, k0 + c) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
}

struct Partial {
  float m, s;
  int arg;
  float pad;
};

__global__ void __launch_bounds__(256) scores_kernel(Operand h, Operand w, int64_t N, int V, int K, const int64_t* labels, Partial* part,
                                                     float* picked, int tiles) {
  __shared__ float z[kTile][kTile + 1];
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kTile, n0 = static_cast<int64_t>(blockIdx.x) * kTile;
  float acc[4][4] = {};
  tile_product(h, w, m0, n0, N, V, K, acc);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) z[ty * 4 + i][tx * 4 + j] = acc[i][j];
  __syncthreads();
  const int64_t row = m0 + threadIdx.x;
  if (threadIdx.x >= kTile || row >= N) return;
  const int n = static_cast<int>(min(static_cast<int64_t>(kTile), V - n0));
  Partial p{z[threadIdx.x][0], 0.f, static_cast<int>(n0), 0.f};
  for (int j = 1; j < n; ++j)
    if (z[threadIdx.x][j] > p.m) { p.m = z[threadIdx.x][j]; p.arg = static_cast<int>(n0) + j; }
  for (int j = 0; j < n; ++j) p.s += expf(z[threadIdx.x][j] - p.m);
  part[row * tiles + blockIdx.x] = p;
  if (labels != nullptr && labels[row] >= n0 && labels[row] < n0 + n) picked[row] = z[threadIdx.x][labels[row] - n0];
}

// one warp per row folds the tiles' partials
__global__ void __launch_bounds__(128) scores_fold_kernel(const Partial* part, const float* picked, int tiles, int64_t N, int V,
                                                          const int64_t* labels, int64_t ignore, float* nll, float* lse, int64_t* top) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= N) return;
  float m = -INFINITY, s = 0.f;
  int arg = 0x7fffffff;
  for (int i = lane; i < tiles; i += 32) {
    const Partial p = part[row * tiles + i];
    if (p.m > m || (p.m == m && p.arg < arg)) arg = p.arg;
    const float mn = fmaxf(m, p.m);
    s = (m == -INFINITY ? 0.f : s * expf(m - mn)) + p.s * expf(p.m - mn);
    m = mn;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, off), os = __shfl_xor_sync(0xffffffffu, s, off);
    const int oa = __shfl_xor_sync(0xffffffffu, arg, off);
    if (om > m || (om == m && oa < arg)) arg = oa;
    const float mn = fmaxf(m, om);
    s = (m == -INFINITY ? 0.f : s * expf(m - mn)) + (om == -INFINITY ? 0.f : os * expf(om - mn));
    m = mn;
  }
  if (lane != 0) return;
  const float l = m + logf(s);
  if (lse != nullptr) lse[row] = l;
  if (top != nullptr) top[row] = arg;
  if (nll != nullptr) {
    const int64_t y = labels[row];
    nll[row] = y == ignore ? 0.f : (y >= 0 && y < V ? l - picked[row] : __int_as_float(0x7fc00000));
  }
}

// sum of nll and number of counted rows, in a fixed order (one block)
__global__ void __launch_bounds__(1024) loss_sum_kernel(const float* nll, const int64_t* labels, int64_t ignore, int64_t N, float* sum, float* count) {
  __shared__ float ss[32], sc[32];
  float s = 0.f, c = 0.f;
  for (int64_t i = threadIdx.x; i < N; i += 1024) {
    if (nll != nullptr) s += nll[i];
    c += labels[i] != ignore ? 1.f : 0.f;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, off);
    c += __shfl_xor_sync(0xffffffffu, c, off);
  }
  if ((threadIdx.x & 31) == 0) { ss[threadIdx.x >> 5] = s; sc[threadIdx.x >> 5] = c; }
  __syncthreads();
  if (threadIdx.x != 0) return;
  s = c = 0.f;
  for (int i = 0; i < 32; ++i) { s += ss[i]; c += sc[i]; }
  if (sum != nullptr) *sum = s;
  if (count != nullptr) *count = c;
}

struct GradRow {
  const int64_t* labels;
  int64_t ignore;
  const float *lse, *grad, *count;
  int64_t grad_stride;
  // One scalar for all rows is applied to the fp32 results: dz itself is then p - onehot, whose large values next to -1
  // round to bf16 with little error (scaled by 1 / 4014, say, every one of them would take the same error of 0.3 %).
  __device__ float row_factor(int64_t row) const { return grad_stride != 0 ? grad[row] : 1.f; }
  __device__ float scale() const {
    if (grad_stride != 0) return 1.f;
    return count == nullptr ? *grad : *count > 0.f ? *grad / *count : 0.f;
  }
};

__global__ void __launch_bounds__(256) dz_kernel(Operand h, Operand w, int64_t N, int V, int K, int v0, int piece, GradRow g, __nv_bfloat16* dz, int ld) {
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kTile, n0 = static_cast<int64_t>(blockIdx.x) * kTile;
  float acc[4][4] = {};
  w.p += v0 * w.sr;
  tile_product(h, w, m0, n0, N, piece, K, acc);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = m0 + ty * 4 + i;
    if (row >= N) continue;
    const int64_t y = g.labels[row];
    const bool used = y != g.ignore;
    float c = g.row_factor(row);
    if (used && (y < 0 || y >= V)) c = __int_as_float(0x7fc00000);
    const float l = g.lse[row];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t col = n0 + tx * 4 + j;
      if (col >= ld) continue;
      const float p = expf(acc[i][j] - l) - (v0 + col == y ? 1.f : 0.f);
      dz[row * ld + col] = __float2bfloat16(used && col < piece ? c * p : 0.f);
    }
  }
}

// C = A B^T; fp32 accumulation into acc32 (first: overwrite) or a bf16 result
__global__ void __launch_bounds__(256) product_kernel(Operand A, Operand B, int64_t M, int64_t N, int64_t K, float* acc32, int first, __nv_bfloat16* out,
                                                      int64_t ld, GradRow g) {
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * kTile, n0 = static_cast<int64_t>(blockIdx.y) * kTile;
  float acc[4][4] = {};
  tile_product(A, B, m0, n0, M, N, K, acc);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = m0 + ty * 4 + i, c = n0 + tx * 4 + j;
      if (r >= M || c >= N) continue;
      if (out != nullptr) out[r * ld + c] = __float2bfloat16(acc[i][j] * g.scale());
      else acc32[r * ld + c] = acc[i][j] + (first ? 0.f : acc32[r * ld + c]);
    }
}

__global__ void __launch_bounds__(256) round_kernel(const float* x, __nv_bfloat16* out, int64_t n, GradRow g) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) out[i] = __float2bfloat16(x[i] * g.scale());
}

constexpr int kPiece = 8192;       // vocabulary rows per piece of the gradient pass

size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

int validate(const char* op, const void* hidden, const void* weight, int64_t hs, int64_t ws, int64_t rows, int32_t hd, int32_t vocab) {
  if (rows < 0 || hd < 1 || vocab < 1) return fail(JL_ERR_BAD_ARG, "%s: sizes out of range", op);
  if (rows > (int64_t(1) << 22)) return fail(JL_ERR_UNSUPPORTED, "%s: at most %lld rows", op, 1ll << 22);
  if (hd % 8 != 0) return fail(JL_ERR_UNSUPPORTED, "%s: the hidden size must be a multiple of 8, got %d", op, hd);
  if (hidden == nullptr || weight == nullptr) return fail(JL_ERR_BAD_ARG, "%s: NULL pointer", op);
  if ((reinterpret_cast<uintptr_t>(hidden) | reinterpret_cast<uintptr_t>(weight)) & 15)
    return fail(JL_ERR_BAD_ARG, "%s: hidden and weight must be 16-byte aligned", op);
  if (hs % 8 != 0 || ws % 8 != 0 || hs < hd || ws < hd)
    return fail(JL_ERR_BAD_ARG, "%s: row strides must be multiples of 8 elements and at least the hidden size", op);
  return JL_OK;
}

}  // namespace

static size_t scores_bytes(int64_t rows, int32_t vocab) {
  const int64_t tiles = (vocab + kTile - 1) / kTile;
  return up256(rows * tiles * sizeof(Partial)) + up256(rows * sizeof(float)) * 2;
}

static size_t grads_bytes(int64_t rows, int32_t hd, int32_t vocab) {
  const int64_t piece = vocab < kPiece ? (vocab + 7) / 8 * 8 : kPiece;
  return up256(rows * piece * 2) + up256(rows * static_cast<size_t>(hd) * 4);
}

static int launch_scores(const jl_head_scores_args* a, cudaStream_t stream) {
  int rc = validate("jl_head_scores", a->hidden, a->weight, a->hidden_stride, a->weight_stride, a->rows, a->hidden_size, a->vocab);
  if (rc != JL_OK) return rc;
  if (a->labels == nullptr && (a->nll != nullptr || a->loss_sum != nullptr || a->loss_count != nullptr))
    return fail(JL_ERR_BAD_ARG, "jl_head_scores: nll and the loss need labels");
  if (a->workspace == nullptr || a->workspace_bytes < scores_bytes(a->rows, a->vocab))
    return fail(JL_ERR_WORKSPACE, "jl_head_scores: workspace of %zu bytes needed, %zu given", scores_bytes(a->rows, a->vocab), a->workspace_bytes);
  if (reinterpret_cast<uintptr_t>(a->workspace) & 15) return fail(JL_ERR_BAD_ARG, "jl_head_scores: workspace not 16-byte aligned");
  rc = check_device_arch();
  if (rc != JL_OK) return rc;
  const int tiles = (a->vocab + kTile - 1) / kTile;
  Partial* part = static_cast<Partial*>(a->workspace);
  float* picked = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + up256(a->rows * static_cast<int64_t>(tiles) * sizeof(Partial)));
  float* nll = a->nll != nullptr || a->loss_sum == nullptr ? a->nll : reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(picked) + up256(a->rows * sizeof(float)));
  const Operand h{static_cast<const __nv_bfloat16*>(a->hidden), a->hidden_stride, 1}, w{static_cast<const __nv_bfloat16*>(a->weight), a->weight_stride, 1};
  if (a->rows > 0) {
    scores_kernel<<<dim3(tiles, static_cast<unsigned>((a->rows + kTile - 1) / kTile)), 256, 0, stream>>>(h, w, a->rows, a->vocab, a->hidden_size, a->labels, part, picked, tiles);
    scores_fold_kernel<<<static_cast<unsigned>((a->rows + 3) / 4), 128, 0, stream>>>(part, picked, tiles, a->rows, a->vocab, a->labels, a->ignore_index, nll, a->lse, a->top);
  }
  if (a->loss_sum != nullptr || a->loss_count != nullptr)
    loss_sum_kernel<<<1, 1024, 0, stream>>>(nll, a->labels, a->ignore_index, a->rows, a->loss_sum, a->loss_count);
  return check_launch("jl_head_scores");
}

static int launch_grads(const jl_head_grads_args* a, cudaStream_t stream) {
  int rc = validate("jl_head_grads", a->hidden, a->weight, a->hidden_stride, a->weight_stride, a->rows, a->hidden_size, a->vocab);
  if (rc != JL_OK) return rc;
  if (a->labels == nullptr || a->lse == nullptr || a->grad == nullptr) return fail(JL_ERR_BAD_ARG, "jl_head_grads: NULL pointer");
  if (a->grad_stride != 0 && a->grad_stride != 1) return fail(JL_ERR_BAD_ARG, "jl_head_grads: grad_stride must be 0 or 1");
  if ((reinterpret_cast<uintptr_t>(a->d_hidden) | reinterpret_cast<uintptr_t>(a->d_weight)) & 15)
    return fail(JL_ERR_BAD_ARG, "jl_head_grads: d_hidden and d_weight must be 16-byte aligned");
  const size_t need = grads_bytes(a->rows, a->hidden_size, a->vocab);
  if (a->workspace == nullptr || a->workspace_bytes < need)
    return fail(JL_ERR_WORKSPACE, "jl_head_grads: workspace of %zu bytes needed, %zu given", need, a->workspace_bytes);
  if (reinterpret_cast<uintptr_t>(a->workspace) & 15) return fail(JL_ERR_BAD_ARG, "jl_head_grads: workspace not 16-byte aligned");
  rc = check_device_arch();
  if (rc != JL_OK) return rc;
  const int64_t N = a->rows, H = a->hidden_size, V = a->vocab;
  if (N == 0) {
    if (a->d_weight != nullptr && cudaMemsetAsync(a->d_weight, 0, V * H * 2, stream) != cudaSuccess) return check_launch("jl_head_grads");
    return JL_OK;
  }
  const int ld = static_cast<int>(V < kPiece ? (V + 7) / 8 * 8 : kPiece);
  __nv_bfloat16* dz = static_cast<__nv_bfloat16*>(a->workspace);
  float* dh32 = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + up256(N * static_cast<size_t>(ld) * 2));
  const Operand h{static_cast<const __nv_bfloat16*>(a->hidden), a->hidden_stride, 1}, w{static_cast<const __nv_bfloat16*>(a->weight), a->weight_stride, 1};
  const GradRow g{a->labels, a->ignore_index, a->lse, a->grad, a->grad_count, a->grad_stride};
  auto cdiv = [](int64_t x, int64_t y) { return static_cast<unsigned>((x + y - 1) / y); };
  for (int64_t v0 = 0; v0 < V; v0 += kPiece) {
    const int piece = static_cast<int>(V - v0 < kPiece ? V - v0 : kPiece);
    dz_kernel<<<dim3(cdiv(ld, kTile), cdiv(N, kTile)), 256, 0, stream>>>(h, w, N, a->vocab, a->hidden_size, static_cast<int>(v0), piece, g, dz, ld);
    if (a->d_hidden != nullptr) {
      const Operand A{dz, ld, 1}, B{w.p + v0 * w.sr, 1, w.sr};
      product_kernel<<<dim3(cdiv(N, kTile), cdiv(H, kTile)), 256, 0, stream>>>(A, B, N, H, piece, dh32, v0 == 0, nullptr, H, g);
    }
    if (a->d_weight != nullptr) {
      const Operand A{dz, 1, ld}, B{h.p, 1, h.sr};
      product_kernel<<<dim3(cdiv(piece, kTile), cdiv(H, kTile)), 256, 0, stream>>>(A, B, piece, H, N, nullptr, 0, static_cast<__nv_bfloat16*>(a->d_weight) + v0 * H, H, g);
    }
  }
  if (a->d_hidden != nullptr) round_kernel<<<cdiv(N * H, 256), 256, 0, stream>>>(dh32, static_cast<__nv_bfloat16*>(a->d_hidden), N * H, g);
  return check_launch("jl_head_grads");
}

}  // namespace jl

extern "C" {

size_t jl_head_scores_workspace_bytes(int64_t rows, int32_t hidden_size, int32_t vocab) {
  return rows < 0 || hidden_size < 1 || vocab < 1 ? 0 : jl::scores_bytes(rows, vocab) + 256;
}

int jl_head_scores(const jl_head_scores_args* args, void* cuda_stream) {
  if (args == nullptr) return jl::fail(JL_ERR_BAD_ARG, "jl_head_scores: args is NULL");
  return jl::launch_scores(args, static_cast<cudaStream_t>(cuda_stream));
}

size_t jl_head_grads_workspace_bytes(int64_t rows, int32_t hidden_size, int32_t vocab) {
  return rows < 0 || hidden_size < 1 || vocab < 1 ? 0 : jl::grads_bytes(rows, hidden_size, vocab) + 256;
}

int jl_head_grads(const jl_head_grads_args* args, void* cuda_stream) {
  if (args == nullptr) return jl::fail(JL_ERR_BAD_ARG, "jl_head_grads: args is NULL");
  return jl::launch_grads(args, static_cast<cudaStream_t>(cuda_stream));
}

}  // extern "C"
