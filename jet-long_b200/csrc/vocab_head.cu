// The vocabulary head without logits: softmax statistics of hidden @ weight^T, and the gradients of the cross-entropy
// loss, formed piece by piece of the vocabulary.
//
//   z = h W^T,  lse = log sum exp z,  nll = lse - z_y,  dz = exp(z - lse) - onehot(y),  dh = g dz W,  dW = g dz^T h
//
// All products run on one persistent tcgen05 kernel (head_gemm_kernel) whose epilogue is what differs:
//   scores  z tile -> per row (maximum, sum of exponentials, argmax, logit of the label); a fold kernel joins the tiles
//   few     the same with the weight's rows as the rows of the product, for up to 32 rows of hidden states
//   dz      z tile -> exp(z - lse) - onehot in bf16, one piece of the vocabulary at a time; at the label exp(-nll) - 1
//   dh      dz W accumulated in fp32 over the pieces (bulk reductions in L2), rounded once at the end
//   dW      dz^T h, final for the piece
// The score and dz products read hidden and weight along their rows (K-major); dh reads weight and dW reads dz and
// hidden across them (MN-major), so nothing is transposed in memory.  Of a loss over more than 256 rows only those that count
// are multiplied: they are packed first, and the products take their extents from the number on the device.
//
// Few rows are bound by the weight's bytes: 49 rows x 4096 x 151936 205 us after a pause (6.1 TB/s), in a loop 218 to 241, where the
// power cap holds the clock at 1.30 GHz.  Many are bound by the tensor pipe at the capped clock: scores of 8191 rows x 4096
// 7.2 ms in a loop (1416 TFLOP/s), 6.3 after a pause (1620); loss and gradients of 4096 rows x 2560 9.7 and 8.4 ms (1310 and 1515),
// four products where three would do if the logits were kept.
#include <cmath>
#include <type_traits>

#include "tc_common.cuh"
#include "../../include/jetlong_b200_head.h"

namespace jl {

namespace {

using namespace tc;

__device__ int g_head_status = 0;            // raised when a bounded wait gave up

constexpr int kBK = 64;                      // K step: one 128-byte swizzle row of bf16
constexpr int kMaxBN = 256;
constexpr int kABytes = 128 * kBK * 2;       // a CTA's 128 rows of A
constexpr int kTmemCols = 512, kMaxAccs = 4;  // accumulators take turns
constexpr int kEpiWarps = 8;                 // two per quarter of the accumulator's rows, each with half of the columns
constexpr int kGemmThreads = 128 + 32 * kEpiWarps;
constexpr int kRegsLow = 72, kRegsHigh = 216;     // 128 x 72 + 256 x 216 = the launch total 384 x 168
constexpr int kRingBytes = 196608;           // operand ring: as many stages of A and B rows, 64 deep, as fit
constexpr int kMaxStages = 10;
constexpr int kStagingBytes = kEpiWarps * 4096;      // per epilogue warp a box of 32 rows x 128 bytes
constexpr int kSms = 148;

constexpr int kFewRows = 32;                 // up to here the rows are the columns of the score product

enum { kEpiScores = 0, kEpiDz = 1, kEpiF32 = 2, kEpiBf16 = 3, kEpiFew16 = 4, kEpiFew32 = 5 };

struct GradScale {            // scalar factor of both gradients, applied to their fp32 sums
  const float *grad, *count;
  int per_row;
  // dz itself stays p - onehot, whose values next to -1 round to bf16 with little error; scaled by 1 / 4014, say, all of
  // them would take the same error of 0.3 %.
  __device__ float get() const {
    if (per_row) return 1.f;
    return count == nullptr ? *grad : *count > 0.f ? *grad / *count : 0.f;
  }
};

struct GemmParams {
  int64_t M, N;               // result extents (rows of A, rows of B)
  // Of the rows of hidden states in the product only this many are in use, NULL: all.  They start at row0 of all rows in use.
  const int32_t* rows_used;
  int64_t row0;
  int m_tiles, n_tiles, splits, k_blocks, kb_per_split, bn;
  int group_m;                // > 0: m fastest inside groups of this many m tiles; 0: n fastest
  int behind, alone_rounds;   // see TileWalk
  int m_step;                 // rows of A from one tile to the next
  int a_bytes, tx_bytes, stage_bytes, stages;      // of the operand ring, per CTA: A's place, what a stage loads, a stage
  // scores
  float2* part;               // [row][n tile][half] (few rows: [row][m tile]) (maximum, sum of exponentials relative to it, less 1)
  int* part_arg;              // the same or NULL
  float* picked;              // [row] logit of the label
  // dz
  const float *lse, *nll;
  const float* row_grad;      // NULL or one factor per row
  const __nv_bfloat16* hidden;      // copy_counted()'s operands
  __nv_bfloat16* counted;     // NULL: no copy
  int64_t hidden_stride;
  int row_len;
  // both
  const int64_t* labels;      // may be NULL for scores
  int64_t ignore, vocab, v0;  // column 0 of the product is vocabulary entry v0
  // dh: bulk reduction into what is there instead of a store
  int reduce;
  GradScale scale;
};

struct alignas(64) GemmMaps { CUtensorMap a, b, out; };

struct GemmSmem {
  alignas(1024) uint8_t ring[kRingBytes];
  alignas(1024) uint8_t staging[kStagingBytes];
  uint64_t full[kMaxStages], empty[kMaxStages], acc_full[kMaxAccs], acc_free[kMaxAccs];
  uint32_t tmem_base;
  int failed;
};
constexpr int kGemmSmemBytes = sizeof(GemmSmem) + 1024;

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t leader_bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(smem_u32(dst)), "l"(map), "r"(leader_bar), "r"(x), "r"(y) : "memory");
}
// 64 columns of a matrix that lies in blocks of 64 columns: rows from y on of block z
template <int kPair>
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint32_t bar, int y, int z) {
  if (kPair == 2)
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(0), "r"(y), "r"(z) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(0), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int x, int y, int z, bool reduce) {
  if (reduce)
    asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];"
                 ::"l"(map), "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];"
                 ::"l"(map), "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

#define JL_TMEM_LD16(taddr, r)                                                                                             \
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"     \
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), \
                 "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr))

struct TileCoord { int m, n, split; };
__device__ __forceinline__ TileCoord tile_coord(const GemmParams& p, int t) {
  TileCoord c;
  const int per = p.m_tiles * p.n_tiles;
  c.split = t / per;
  int r = t - c.split * per;
  if (p.group_m > 0) {
    const int grp = r / (p.group_m * p.n_tiles), m0 = grp * p.group_m, size = min(p.group_m, p.m_tiles - m0);
    r -= m0 * p.n_tiles;
    c.n = r / size;
    c.m = m0 + r - c.n * size;
  } else {
    c.m = r / p.n_tiles;
    c.n = r - c.m * p.n_tiles;
  }
  return c;
}

// Cost of a tile in K blocks: its own, and about three for a short tile's hand-over.
__host__ __device__ inline int64_t tile_cost(const GemmParams& p) { return p.kb_per_split + 3; }
__host__ __device__ inline int64_t tiles_of(const GemmParams& p) { return static_cast<int64_t>(p.m_tiles) * p.n_tiles * p.splits; }

// Shares of the second product of a launch, so that the workers that carry one tile more of the first end with the others.
__host__ __device__ inline void balance(const GemmParams& first, GemmParams& second) {
  const int64_t W = kSms / 2, n0 = tiles_of(first), n1 = tiles_of(second), c0 = tile_cost(first), c1 = tile_cost(second);
  const int64_t l = n0 / W, rem = n0 % W;
  int64_t late = ((n0 * c0 + n1 * c1) / W - (l + 1) * c0) / c1;            // rounds of the workers with l + 1 tiles
  if (late < 0) late = 0;
  int64_t rounds = (n1 - rem * late + W - rem - 1) / (W - rem);
  if (rounds < late) rounds = late = (n1 + W - 1) / W;
  second.behind = static_cast<int>(rem);
  second.alone_rounds = static_cast<int>(rounds - late);
}

// Persistent walk of a worker over the tiles of one product.  The first `behind` workers of a launch carry one tile more of the
// product before this one: the others do `alone_rounds` rounds without them, so that all end together.
struct TileWalk {
  int worker, workers, behind, alone, rounds;
  int n, round;
  __device__ __forceinline__ TileWalk(const GemmParams& p, int w, int ws)
      : worker(w), workers(ws), behind(p.behind), alone(p.alone_rounds), n(p.m_tiles * p.n_tiles * p.splits), round(w < p.behind ? p.alone_rounds : 0) {}
  __device__ __forceinline__ bool next(int& tile) {
    tile = round < alone ? round * (workers - behind) + worker - behind : alone * (workers - behind) + (round - alone) * workers + worker;
    ++round;
    return tile < n;
  }
};

// The ring and the accumulators go on from one product of a launch to the next.
struct PipeState {
  int slot, i;                        // next stage, tiles done
  uint32_t parity;
  __device__ __forceinline__ void next(int stages) {
    if (++slot == stages) { slot = 0; parity ^= 1u; }
  }
};

// Operand kinds of a product C = A B^T: which of A and B are read across their rows (MN-major), and what becomes of C.
template <int kPair_, bool kAMn_, bool kBMn_, int kEpi_>
struct Product {
  static constexpr int kPair = kPair_, kEpi = kEpi_;
  static constexpr bool kAMn = kAMn_, kBMn = kBMn_;
  static constexpr bool kABlocked = kEpi_ == kEpiF32 || kEpi_ == kEpiBf16;     // A is dz
  // K blocks that an accumulator takes before it is handed over.  The tensor cores cut every sum off instead of rounding it: over
  // the 256 steps of K = 4096 a logit lost 2^-24 of its size 256 times, up to 1e-5 in all, and so did the losses.  Scores
  // therefore take K in parts that are added in fp32 registers.  Error of the loss / time of 8191 rows x 4096 with parts of 256,
  // 512, 1024 and all of K: 2e-7 / 8.0 ms, 3.5e-7 / 7.5, 8e-7 / 7.25, 4e-6 / 7.1; a few rows are bound by the weight's bytes and
  // take parts of 256, up to 32 rows parts of 128, up to 16 of 64 (error of one row's lse with 64, 128, 256: 0.7e-7, 1.4e-7, 2.6e-7;
  // time of 151936 x 2048 in a loop 102.4, 102.3, 98.4 us, after a pause 98 with all; 32 rows x 4096: 225, 218, 207 us).
  // Results that are rounded to bf16 need none of this: in dz a probability may be off by 1e-4 of itself, and the label's p - 1, where
  // that would be all there is, is taken from the loss.
  static constexpr int kAccs = kEpi_ >= kEpiFew16 ? 4 : 2, kAccCols = kTmemCols / kAccs;
  static constexpr bool kFew = kEpi_ == kEpiFew16 || kEpi_ == kEpiFew32, kParts = kEpi_ == kEpiScores || kFew;
  static constexpr int kPart = !kParts ? 1 << 30 : kEpi_ == kEpiFew16 ? 1 : kEpi_ == kEpiFew32 ? 2 : kPair_ == 1 ? 4 : 8;
};

template <class P>
__device__ __forceinline__ void produce(const GemmMaps& maps, const GemmParams& p, GemmSmem& sm, int rank, int worker, int workers, PipeState& st) {
  constexpr int kPair = P::kPair;
  const int b_rows = p.bn / kPair;
  TileWalk walk(p, worker, workers);
  for (int t; walk.next(t);) {
    const TileCoord c = tile_coord(p, t);
    const int m0 = (c.m * kPair + rank) * p.m_step, n0 = c.n * p.bn + rank * b_rows;
    const int kb0 = c.split * p.kb_per_split, kb1 = min(kb0 + p.kb_per_split, p.k_blocks);
    for (int kb = kb0; kb < kb1; ++kb, st.next(p.stages)) {
      const int s = st.slot;
      mbar_wait(&sm.empty[s], st.parity ^ 1u, sm);
      if (*reinterpret_cast<volatile int*>(&sm.failed)) return;
      if (rank == 0) mbar_expect_tx(&sm.full[s], kPair * p.tx_bytes);
      const uint32_t bar = kPair == 2 ? pair::leader_addr(&sm.full[s]) : smem_u32(&sm.full[s]);
      uint8_t* sa = sm.ring + s * p.stage_bytes;
      uint8_t* sb = sa + p.a_bytes;
      auto load = [&](void* dst, const CUtensorMap* map, int x, int y) {
        if (kPair == 2) tma_load_2d_pair(dst, map, bar, x, y);
        else tma_load_2d(dst, map, bar, x, y);
      };
      auto load_a = [&](void* dst, int x, int y) {           // dz lies in blocks of 64 columns: (column in the block, row, block)
        if (P::kABlocked) tma_load_3d<kPair>(dst, &maps.a, bar, y, x >> 6);
        else load(dst, &maps.a, x, y);
      };
      if (P::kAMn) {
        load_a(sa, m0, kb * kBK);
        load_a(sa + 8192, m0 + 64, kb * kBK);
      } else {
        load_a(sa, kb * kBK, m0);
      }
      if (P::kBMn) {
        for (int ch = 0; ch < b_rows / 64; ++ch) load(sb + ch * 8192, &maps.b, n0 + ch * 64, kb * kBK);
      } else {
        load(sb, &maps.b, kb * kBK, n0);
      }
    }
  }
}

template <class P>
__device__ __forceinline__ void issue(const GemmParams& p, GemmSmem& sm, uint32_t tmem, uint32_t leader, int worker, int workers, PipeState& st) {
  constexpr int kPair = P::kPair;
  const uint32_t idesc = instr_desc(128 * kPair, p.bn, P::kBMn) | (P::kAMn ? 1u << 15 : 0u);
  const uint32_t ring = smem_u32(sm.ring);
  TileWalk walk(p, worker, workers);
  for (int t; walk.next(t);) {
    const TileCoord c = tile_coord(p, t);
    const int kb0 = c.split * p.kb_per_split, kb1 = min(kb0 + p.kb_per_split, p.k_blocks);
    uint32_t acc = 0;
    for (int kb = kb0; kb < kb1; ++kb, st.next(p.stages)) {
      const bool first = kb == kb0 || (P::kParts && (kb - kb0) % P::kPart == 0);
      const bool last = kb + 1 == kb1 || (P::kParts && (kb + 1 - kb0) % P::kPart == 0);
      if (first) {
        mbar_wait(&sm.acc_free[st.i % P::kAccs], ((st.i / P::kAccs) & 1) ^ 1, sm);
        acc = tmem + (st.i % P::kAccs) * P::kAccCols;
      }
      const int s = st.slot;
      mbar_wait(&sm.full[s], st.parity, sm);
      if (*reinterpret_cast<volatile int*>(&sm.failed)) return;
      tc_fence_after();
      const uint32_t sa = ring + s * p.stage_bytes, sb = sa + p.a_bytes;
      // K-major rows are 128 bytes in 8-row swizzle atoms; MN-major: 64 elements x 8 k-rows per atom, 8 KB per 64 elements
      const uint64_t ad = P::kAMn ? smem_desc(sa, 8192, 1024) : smem_desc(sa, 16, 1024);
      const uint64_t bd = P::kBMn ? smem_desc(sb, 8192, 1024) : smem_desc(sb, 16, 1024);
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const uint64_t ao = static_cast<uint64_t>((P::kAMn ? kk * 2048 : kk * 32) >> 4);
          const uint64_t bo = static_cast<uint64_t>((P::kBMn ? kk * 2048 : kk * 32) >> 4);
          if (kPair == 2) pair::mma2_ss(acc, ad + ao, bd + bo, idesc, !first || kk > 0);
          else mma_ss(acc, ad + ao, bd + bo, idesc, !first || kk > 0);
        }
        if (kPair == 2) pair::commit_both(&sm.empty[s]);
        else mma_commit(&sm.empty[s]);
        if (last) {
          if (kPair == 2) pair::commit_both(&sm.acc_full[st.i % P::kAccs]);
          else mma_commit(&sm.acc_full[st.i % P::kAccs]);
        }
      }
      __syncwarp();
      if (last) ++st.i;
    }
  }
}

template <class P>
__device__ __forceinline__ void finish(const GemmMaps& maps, const GemmParams& p, GemmSmem& sm, uint32_t tmem, int ew, int lane, int rank, int worker,
                                       int workers, PipeState& st) {
  constexpr int kPair = P::kPair, kEpi = P::kEpi;
  const int quad = ew & 3, half = ew >> 2;         // rows quad * 32 .. of the accumulator, first or second half of its columns
  const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
  uint8_t* const stage = sm.staging + ew * 4096;
  const uint32_t free_bar = kPair == 2 ? pair::leader_addr(&sm.acc_free[0]) : smem_u32(&sm.acc_free[0]);
  const float scale = kEpi == kEpiBf16 ? p.scale.get() : 1.f;
  // 32 rows x 128 bytes of results: 16-byte chunk `ch` of this thread's row
  auto chunk_ptr = [&](int ch) { return reinterpret_cast<uint4*>(stage + lane * 128 + ((ch ^ (lane & 7)) << 4)); };
  auto begin_box = [&]() {
    if (lane == 0) bulk_wait_read<0>();          // the box before has left the buffer
    __syncwarp();
  };
  auto end_box = [&](int x, int64_t row_w, int z, bool reduce) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
      if (row_w < p.M && x < p.N) {
        if (kEpi == kEpiDz) tma_store_3d(&maps.out, stage, 0, static_cast<int>(row_w), x >> 6, false);      // blocks of 64 columns
        else tma_store_3d(&maps.out, stage, x, static_cast<int>(row_w), z, reduce);
      }
      bulk_commit();
    }
  };
  auto hand_back = [&]() {                         // this warp has read the accumulator
    tc_fence_before();
    __syncwarp();
    if (lane == 0) asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(free_bar + 8 * (st.i % P::kAccs)) : "memory");
    ++st.i;
  };
  TileWalk walk(p, worker, workers);
  for (int t; walk.next(t);) {
    const TileCoord c = tile_coord(p, t);
    const int64_t row_w = (static_cast<int64_t>(c.m) * kPair + rank) * 128 + quad * 32, row = row_w + lane;
    const int n0 = c.n * p.bn;

    if constexpr (P::kFew) {
      // The tile is m_step vocabulary entries by up to 32 rows.  Its logits are summed over the parts of K in registers (a thread has
      // an entry and 16 of the rows) and go through shared memory to a warp per row.
      float* const zs = reinterpret_cast<float*>(sm.ring + kRingBytes + kStagingBytes - p.N * 512);      // [row][128 entries], behind the ring
      const int c_lo = half * 16;
      const bool mine = half == 0 || kEpi == kEpiFew32;      // up to 16 rows the second half of the warps only reduces
      float z[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) z[j] = 0.f;
      for (int kb = 0; mine && kb < p.k_blocks; kb += P::kPart) {
        mbar_wait(&sm.acc_full[st.i % P::kAccs], (st.i / P::kAccs) & 1, sm);
        tc_fence_after();
        uint32_t x[16];
        JL_TMEM_LD16(tmem + (st.i % P::kAccs) * P::kAccCols + lane_base + c_lo, x);
        JL_TMEM_WAIT_LD16(x, 0);
#pragma unroll
        for (int j = 0; j < 16; ++j) z[j] += __uint_as_float(x[j]);
        hand_back();
      }
      const int64_t v0 = static_cast<int64_t>(c.m) * p.m_step;
      const int valid = static_cast<int>(p.M - v0 < p.m_step ? p.M - v0 : p.m_step);
      asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");      // the tile before has been read
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (mine && c_lo + j < p.N) zs[(c_lo + j) * 128 + quad * 32 + lane] = quad * 32 + lane < valid ? z[j] : -INFINITY;
      asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
      for (int r = ew; r < p.N; r += kEpiWarps) {
        const float4 x = *reinterpret_cast<const float4*>(zs + r * 128 + 4 * lane);
        float m = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
        const float m_use = m == -INFINITY ? 0.f : m;
        const float e[4] = {fast_exp2((x.x - m_use) * kLog2e), fast_exp2((x.y - m_use) * kLog2e), fast_exp2((x.z - m_use) * kLog2e),
                            fast_exp2((x.w - m_use) * kLog2e)};
        float less = 0.f;
        int ones = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ones += __popc(__ballot_sync(0xffffffffu, e[j] == 1.f));
          less += e[j] == 1.f ? 0.f : e[j];
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) less += __shfl_xor_sync(0xffffffffu, less, off);
        const int64_t at = static_cast<int64_t>(r) * p.m_tiles + c.m;
        if (p.part_arg != nullptr) {
          const int first = x.x == m ? 0 : x.y == m ? 1 : x.z == m ? 2 : x.w == m ? 3 : 128;
          const int arg = __reduce_min_sync(0xffffffffu, 4 * lane + first);
          if (lane == 0) p.part_arg[at] = arg < valid ? static_cast<int>(v0) + arg : 0x7fffffff;
        }
        if (lane == 0) {
          p.part[at] = make_float2(m, less + static_cast<float>(ones - 1));
          const int64_t y = p.labels != nullptr ? p.labels[r] - v0 : -1;
          if (y >= 0 && y < valid) p.picked[r] = zs[r * 128 + y];
        }
      }
    } else if constexpr (kEpi == kEpiScores) {
      // columns [c_lo, c_lo + width) of the tile, up to 128 of them in registers, summed over the parts of K
      const int c_lo = half == 0 ? 0 : (p.bn / 2 + 15) / 16 * 16, width = half == 0 ? (p.bn / 2 + 15) / 16 * 16 : p.bn - c_lo;
      float z[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) z[j] = (j & ~15) < width ? 0.f : -INFINITY;      // blocks of 16 past the half are not read
      for (int part = 0; part * P::kPart < p.k_blocks; ++part) {
        const uint32_t acc = tmem + (st.i % P::kAccs) * P::kAccCols + lane_base + c_lo;
        mbar_wait(&sm.acc_full[st.i % P::kAccs], (st.i / P::kAccs) & 1, sm);
        tc_fence_after();
#pragma unroll
        for (int ch = 0; ch < 8; ++ch) {
          if (ch * 16 < width) {
            uint32_t x[16];
            JL_TMEM_LD16(acc + ch * 16, x);
            JL_TMEM_WAIT_LD16(x, 0);
#pragma unroll
            for (int j = 0; j < 16; ++j) z[ch * 16 + j] += __uint_as_float(x[j]);
          }
        }
        hand_back();
      }
      const int64_t rest = p.N - n0 - c_lo;
      const int valid = static_cast<int>(rest < 0 ? 0 : rest < width ? rest : width);
      if (valid < width) {                             // the vocabulary ends in here
#pragma unroll
        for (int j = 0; j < 128; ++j)
          if (j >= valid) z[j] = -INFINITY;
      }
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 64; ++j) m4[j & 3] = max3(m4[j & 3], z[2 * j], z[2 * j + 1]);
      const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
      const float m_use = m == -INFINITY ? 0.f : m;
      const int64_t y64 = p.labels != nullptr && row < p.M ? p.labels[row] - p.v0 - n0 - c_lo : -1;
      const int y = y64 >= 0 && y64 < valid ? static_cast<int>(y64) : -1;
      float s4[4] = {0.f, 0.f, 0.f, 0.f}, z_y = 0.f;
      int arg = 0x7fffffff;
      if (__any_sync(0xffffffffu, y >= 0)) {
#pragma unroll
        for (int j = 0; j < 128; ++j) z_y = y == j ? z[j] : z_y;
      }
      if (p.part_arg != nullptr) {
#pragma unroll
        for (int j = 127; j >= 0; --j) arg = z[j] == m && j < valid ? j : arg;
      }
      // (z - m) first: exact for the logits that count, whatever their size
      int ones = 0;
#pragma unroll
      for (int j = 0; j < 128; ++j) {
        const float e = fast_exp2((z[j] - m_use) * kLog2e);
        ones += e == 1.f ? 1 : 0;
        s4[j & 3] += e == 1.f ? 0.f : e;
      }
      if (row < p.M) {
        const int64_t at = (row * p.n_tiles + c.n) * 2 + half;
        p.part[at] = make_float2(m, (s4[0] + s4[1]) + (s4[2] + s4[3]) + static_cast<float>(ones - 1));
        if (p.part_arg != nullptr) p.part_arg[at] = arg == 0x7fffffff ? arg : n0 + c_lo + arg;
        if (y >= 0) p.picked[row] = z_y;
      }
    } else {
      const uint32_t acc = tmem + (st.i % P::kAccs) * P::kAccCols + lane_base;
      mbar_wait(&sm.acc_full[st.i % P::kAccs], (st.i / P::kAccs) & 1, sm);
      tc_fence_after();
      float lse = 0.f, factor = 0.f, dz_y = 0.f;
      int y = -1;
      if constexpr (kEpi == kEpiDz) {
        if (row < p.M) {
          const int64_t label = p.labels[row];
          lse = p.lse[row];
          if (label != p.ignore) {
            factor = p.row_grad != nullptr ? p.row_grad[row] : 1.f;
            if (label < 0 || label >= p.vocab) factor = __int_as_float(0x7fc00000);
            const int64_t rel = label - p.v0 - n0;
            y = rel >= 0 && rel < p.bn ? static_cast<int>(rel) : -1;
            // p - 1 = e^-nll - 1.  exp(z - lse) - 1 would cancel: this z is cut off over all of K, and a row with 1 - p = 1e-6 got
            // a hundred times its gradient.
            if (y >= 0) dz_y = expm1f(-p.nll[row]);
          }
        }
      }
      const bool used = kEpi != kEpiDz || factor != 0.f;
      constexpr int kCols = kEpi == kEpiF32 ? 32 : 64;             // columns of one 128-byte box; bn is a multiple of 64 here
      for (int c0 = half * kCols; c0 < p.bn; c0 += 2 * kCols) {      // the two warps of a row quarter take the boxes in turn
        begin_box();
        for (int hc = 0; hc < kCols / 32; ++hc) {
          const int cc = c0 + hc * 32;
          uint32_t z[32];
          JL_TMEM_LD32(acc + cc, z, 0);
          JL_TMEM_WAIT_LD32(z, 0);
          if constexpr (kEpi == kEpiDz) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float pr = y == cc + j ? dz_y : fast_exp2((__uint_as_float(z[j]) - lse) * kLog2e);
              z[j] = used ? __float_as_uint(pr * factor) : 0u;      // a row that does not count is zero whatever it holds
            }
            if (n0 + cc + 32 > p.N) {                              // the piece's last block of 64 columns is stored whole
#pragma unroll
              for (int j = 0; j < 32; ++j) z[j] = n0 + cc + j < p.N ? z[j] : 0u;
            }
          }
          if constexpr (kEpi == kEpiF32) {
#pragma unroll
            for (int v = 0; v < 8; ++v) *chunk_ptr(v) = make_uint4(z[4 * v], z[4 * v + 1], z[4 * v + 2], z[4 * v + 3]);
          } else {
            auto pk = [&](int j) { return pack_bf16x2(__uint_as_float(z[j]) * scale, __uint_as_float(z[j + 1]) * scale); };
#pragma unroll
            for (int v = 0; v < 4; ++v) *chunk_ptr(hc * 4 + v) = make_uint4(pk(8 * v), pk(8 * v + 2), pk(8 * v + 4), pk(8 * v + 6));
          }
        }
        end_box(n0 + c0, row_w, kEpi == kEpiF32 ? c.split : 0, kEpi == kEpiF32 && p.reduce);
      }
      hand_back();
    }
  }
}

// The rows of hidden states with zeros for those that do not count, one warp of every CTA a row at a time: d logits of such a row are
// zero, and 0 * NaN in the weight's gradient is not.  Warp 3 does it while the dz product runs, where it has nothing else to do.
__device__ __forceinline__ void copy_counted(const GemmParams& p, int lane) {
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
    const bool counts = p.labels[row] != p.ignore;
    const uint4* src = reinterpret_cast<const uint4*>(p.hidden + row * p.hidden_stride);
    uint4* dst = reinterpret_cast<uint4*>(p.counted + row * p.row_len);
    for (int c = lane; c < p.row_len / 8; c += 32) dst[c] = counts ? src[c] : make_uint4(0u, 0u, 0u, 0u);
  }
}

// The product's extents for the rows in use.  One row is kept where a result is due whatever the number (it counts for nothing).
template <class P>
__device__ __forceinline__ GemmParams in_use(const GemmParams& p) {
  GemmParams q = p;
  if (P::kPair == 2 && p.rows_used != nullptr) {               // (single CTAs have one row tile at most)
    int64_t n = *p.rows_used - p.row0;
    if (n < (P::kParts ? 0 : 1)) n = P::kParts ? 0 : 1;
    if (P::kAMn) {
      const int kb = static_cast<int>((n + kBK - 1) / kBK);
      q.k_blocks = q.kb_per_split = kb < p.k_blocks ? kb : p.k_blocks;
    } else {
      const int m = static_cast<int>((n + 128 * P::kPair - 1) / (128 * P::kPair));
      q.m_tiles = m < p.m_tiles ? m : p.m_tiles;
    }
  }
  return q;
}

// C tiles (128 * kPair rows x bn columns), fp32 accumulation in tensor memory, of one product or of two that need nothing of each
// other, the second filling the SMs that the first leaves.  kPair = 2: a cluster of two CTAs works on one tile with cta_group::2
// MMAs, each CTA loading its own 128 rows of A and half of the rows of B, so every byte of B in shared memory serves 256 rows.
// Two accumulators alternate, so the epilogue of a tile runs under the next one's MMAs.
//   warp 0 TMA producer, warp 1 MMA issuer (rank 0), warp 2 tensor memory, warps 4-11 epilogue (one thread per row and half)
template <class P0, class P1>
__global__ void __launch_bounds__(kGemmThreads, 1) head_gemm_kernel(const __grid_constant__ GemmMaps maps0, const GemmParams p0,
                                                                    const __grid_constant__ GemmMaps maps1, const GemmParams p1) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  GemmSmem& sm = *reinterpret_cast<GemmSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int kPair = P0::kPair;
  constexpr bool kTwo = !std::is_same<P1, void>::value;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kPair == 2 ? static_cast<int>(blockIdx.x & 1) : 0;
  const int worker = static_cast<int>(blockIdx.x) / kPair, workers = static_cast<int>(gridDim.x) / kPair;

  if (threadIdx.x == 0) {
    sm.failed = *reinterpret_cast<volatile int*>(&g_head_status) != 0 ? 1 : 0;
    for (int i = 0; i < kMaxStages; ++i) { mbar_init(&sm.full[i], 1); mbar_init(&sm.empty[i], 1); }
    for (int i = 0; i < kMaxAccs; ++i) { mbar_init(&sm.acc_full[i], 1); mbar_init(&sm.acc_free[i], P0::kEpi == kEpiFew16 ? 4 : kEpiWarps * kPair); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    if (kPair == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)), "r"(512u));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)), "r"(512u));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (kPair == 2) pair::cluster_sync();
  tc_fence_after();
  wait_prerequisites();                          // nothing before this reads what an earlier kernel wrote
  launch_dependents();
  const uint32_t tmem = sm.tmem_base;

  PipeState st{0, 0, 0u};
  const GemmParams q0 = in_use<P0>(p0);
  GemmParams q1{};
  if constexpr (kTwo) {
    q1 = in_use<P1>(p1);
    if (p0.rows_used != nullptr) balance(q0, q1);
  }
  // the control warps give registers back, the epilogue warps (128 logits of a row each) take them
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLow));
    if (warp == 0) {
      if (lane == 0) {
        produce<P0>(maps0, q0, sm, rank, worker, workers, st);
        if constexpr (kTwo) produce<P1>(maps1, q1, sm, rank, worker, workers, st);
      }
    } else if (warp == 1 && rank == 0) {
      uint32_t leader;
      asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(leader));
      issue<P0>(q0, sm, tmem, leader, worker, workers, st);
      if constexpr (kTwo) issue<P1>(q1, sm, tmem, leader, worker, workers, st);
    } else if (P0::kEpi == kEpiDz && warp == 3 && p0.counted != nullptr) {
      copy_counted(p0, lane);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsHigh));
    finish<P0>(maps0, q0, sm, tmem, warp - 4, lane, rank, worker, workers, st);
    if constexpr (kTwo) finish<P1>(maps1, q1, sm, tmem, warp - 4, lane, rank, worker, workers, st);
    if (lane == 0) bulk_wait_all();
  }

  __syncthreads();
  if (*reinterpret_cast<volatile int*>(&sm.failed)) {      // a wait gave up: copies and MMAs under way have long landed after 1 ms
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000 * 1000) {}
  }
  if (kPair == 2) pair::cluster_sync();          // neither CTA leaves (or frees tensor memory) while the other may still signal it
  if (warp == 2) {
    tc_fence_after();
    if (kPair == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
  if (threadIdx.x == 0 && sm.failed) atomicExch(&g_head_status, 1);
}

// (maximum, r, lowest index of the maximum) of two disjoint sets of logits, where 1 + r is the sum of exponentials relative to the
// maximum: the 1 is the maximum's own.  Kept apart, it does not round away what the others add up to, and log1p(r) is the loss of a
// row that is sure of its label: with one sum, a loss of 1e-6 was off by up to a quarter.  No logits: (-inf, -1).
__device__ __forceinline__ void join_scores(float& m, float& r, int& arg, float om, float orest, int oa) {
  if (om > m || (om == m && oa < arg)) arg = oa;
  const bool other = om > m;
  const float hi = other ? om : m, lo = other ? m : om, ref = hi == -INFINITY ? 0.f : hi;
  r = (other ? orest : r) + (1.f + (other ? r : orest)) * fast_exp2((lo - ref) * kLog2e);
  m = hi;
}

// Folds the tiles' partials of a row; kWarps warps share a row (8 when there are few rows: 731 partials of one row took
// one warp 14 us).  Every lane reads 4 partials at a time.
template <int kWarps>
__global__ void __launch_bounds__(256) scores_fold_kernel(const float2* part, const int* part_arg, const float* picked, int tiles, int64_t N, int64_t V,
                                                          const int64_t* labels, int64_t ignore, float* nll, float* lse, int64_t* top,
                                                          const int32_t* rows_used, const int32_t* place, int64_t row0) {
  __shared__ float sm[8], sr[8];
  __shared__ int sa[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (8 / kWarps) + warp / kWarps;
  wait_prerequisites();
  launch_dependents();
  float m = -INFINITY, r = -1.f;
  int arg = 0x7fffffff;
  if (rows_used != nullptr && *rows_used - row0 < N) N = *rows_used - row0;
  if (row < N) {
    for (int i0 = (warp % kWarps) * 32 + lane; i0 < tiles; i0 += 4 * 32 * kWarps) {
      float2 p[4];
      int a[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * 32 * kWarps;
        p[j] = i < tiles ? part[row * tiles + i] : make_float2(-INFINITY, -1.f);
        a[j] = i < tiles && part_arg != nullptr ? part_arg[row * tiles + i] : 0x7fffffff;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) join_scores(m, r, arg, p[j].x, p[j].y, a[j]);
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    join_scores(m, r, arg, __shfl_xor_sync(0xffffffffu, m, off), __shfl_xor_sync(0xffffffffu, r, off), __shfl_xor_sync(0xffffffffu, arg, off));
  if (kWarps > 1) {
    if (lane == 0) { sm[warp] = m; sr[warp] = r; sa[warp] = arg; }
    __syncthreads();
    if (warp != 0) return;
    for (int i = 1; i < kWarps; ++i) join_scores(m, r, arg, sm[i], sr[i], sa[i]);
  }
  if (lane != 0 || row >= N) return;
  const float log_s = log1pf(r), l = m + log_s;
  const int64_t at = place != nullptr ? place[row0 + row] : row;
  if (lse != nullptr) lse[at] = l;
  if (top != nullptr) top[row] = arg == 0x7fffffff ? 0 : arg;
  if (nll != nullptr) {
    const int64_t y = labels[row];
    // (m - z_y) + log s, not lse - z_y: a small loss keeps its digits
    nll[at] = y == ignore ? 0.f : (y >= 0 && y < V ? (m - picked[row]) + log_s : __int_as_float(0x7fc00000));
  }
}

// sum of nll, number of counted rows and their quotient, in a fixed order (one block)
__global__ void __launch_bounds__(1024) loss_sum_kernel(const float* nll, const int64_t* labels, int64_t ignore, int64_t N, float* sum, float* count,
                                                        float* mean) {
  __shared__ float ss[32], sc[32];
  float s = 0.f, c = 0.f;
  for (int64_t i = threadIdx.x; i < N; i += 1024) c += labels[i] != ignore ? 1.f : 0.f;
  wait_prerequisites();
  for (int64_t i = threadIdx.x; i < N; i += 1024) s += nll[i];
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
  if (mean != nullptr) *mean = s / c;
}

// d_hidden = scale * (sum of the K splits' fp32 results), rounded once; 4 values a thread.  place: where a row's results are (NULL:
// at the row itself), -1: it has none.
__global__ void __launch_bounds__(256) grad_round_kernel(const float* x, int splits, int64_t n, __nv_bfloat16* out, GradScale g, const int32_t* place,
                                                         int row_len) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  wait_prerequisites();
  launch_dependents();
  if (i >= n) return;
  int64_t from = i;
  if (place != nullptr) {
    const int64_t row = i / row_len;
    const int32_t at = place[row];
    if (at < 0) {
      *reinterpret_cast<uint2*>(out + i) = make_uint2(0u, 0u);
      return;
    }
    from += (at - row) * row_len;
  }
  float4 a = *reinterpret_cast<const float4*>(x + from);
#pragma unroll 8
  for (int s = 1; s < splits; ++s) {
    const float4 b = *reinterpret_cast<const float4*>(x + s * n + from);
    a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
  }
  const float c = g.get();
  *reinterpret_cast<uint2*>(out + i) = make_uint2(pack_bf16x2(a.x * c, a.y * c), pack_bf16x2(a.z * c, a.w * c));
}

// Rows that count: row_of[r] is the r-th row whose label is not `ignore`, place[i] the r of row i or -1, *used their number.
// What does not count gets nll = lse = 0 (where asked for).  One block; 8192 rows a round.
__global__ void __launch_bounds__(1024) rows_used_kernel(const int64_t* labels, int64_t ignore, int64_t N, int32_t* row_of, int32_t* place, int32_t* used,
                                                         float* nll, float* lse) {
  __shared__ int before[8 * 32];                   // counts of (chunk of 1024 rows, warp), then their prefix sums
  __shared__ int base;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) base = 0;
  wait_prerequisites();
  launch_dependents();
  for (int64_t i0 = 0; i0 < N; i0 += 8192) {
    uint32_t votes[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t i = i0 + j * 1024 + threadIdx.x;
      votes[j] = __ballot_sync(0xffffffffu, i < N && labels[i] != ignore);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (lane == 0) before[j * 32 + warp] = __popc(votes[j]);
    __syncthreads();
    if (warp == 0) {
      int c[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) { c[j] = before[lane * 8 + j]; sum += c[j]; }
      int incl = sum;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += o;
      }
      int at = base + incl - sum;
#pragma unroll
      for (int j = 0; j < 8; ++j) { before[lane * 8 + j] = at; at += c[j]; }
      __syncwarp();
      if (lane == 31) base = at;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t i = i0 + j * 1024 + threadIdx.x;
      const bool in = (votes[j] >> lane) & 1u;
      const int r = before[j * 32 + warp] + __popc(votes[j] & ((1u << lane) - 1u));
      if (i < N) {
        place[i] = in ? r : -1;
        if (in) {
          row_of[r] = static_cast<int32_t>(i);
        } else {
          if (nll != nullptr) nll[i] = 0.f;
          if (lse != nullptr) lse[i] = 0.f;
        }
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) *used = base;
}

// Rows row0 .. row0 + gridDim.x of those in use, packed: hidden states, labels and, where given, lse with nll and row gradients.  Up to the
// next multiple of 64 (a K block of the weight's gradient) the rows after the last are zero; every label after it is `ignore`.
__global__ void __launch_bounds__(128) rows_gather_kernel(const __nv_bfloat16* hidden, int64_t stride, int row_len, const int64_t* labels, int64_t ignore,
                                                          const float* lse, const float* nll, const float* row_grad, const int32_t* row_of, const int32_t* used,
                                                          int64_t row0, __nv_bfloat16* hidden_out, int64_t* labels_out, float* lse_out, float* nll_out,
                                                          float* row_grad_out) {
  wait_prerequisites();
  launch_dependents();
  const int64_t r = row0 + blockIdx.x, n = *used;
  const bool in = r < n;
  const int64_t from = in ? row_of[r] : 0;
  if (threadIdx.x == 0) {
    labels_out[blockIdx.x] = in ? labels[from] : ignore;
    if (lse != nullptr) {
      lse_out[blockIdx.x] = in ? lse[from] : 0.f;
      nll_out[blockIdx.x] = in ? nll[from] : 0.f;
    }
    if (row_grad != nullptr) row_grad_out[blockIdx.x] = in ? row_grad[from] : 0.f;
  }
  if (r >= (n + kBK - 1) / kBK * kBK && r >= kBK) return;
  const uint4* src = reinterpret_cast<const uint4*>(hidden + from * stride);
  uint4* dst = reinterpret_cast<uint4*>(hidden_out + static_cast<int64_t>(blockIdx.x) * row_len);
  for (int c = threadIdx.x; c < row_len / 8; c += 128) dst[c] = in ? src[c] : make_uint4(0u, 0u, 0u, 0u);
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------

int64_t cdiv(int64_t x, int64_t y) { return (x + y - 1) / y; }
size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

// (rows, cols) row-major operand or result as a 2-D (loads) or 3-D (results) map; a box is box_x elements by box_y rows
int make_map2(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_x, int box_y, bool f32, int64_t planes, bool three) {
  EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return fail(JL_ERR_LAUNCH, "jl_head: cuTensorMapEncodeTiled is not available from the driver");
  const int es_bytes = f32 ? 4 : 2;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(planes)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld) * es_bytes, static_cast<cuuint64_t>(ld) * es_bytes * static_cast<cuuint64_t>(rows)};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(box_x), static_cast<cuuint32_t>(box_y), 1};
  const cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = enc(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, three ? 3 : 2, const_cast<void*>(base), dims, strides,
                         box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(JL_ERR_BAD_ARG, "jl_head: tensor map encoding failed (CUresult %d)", static_cast<int>(r));
  return JL_OK;
}

struct Matrix {               // bf16, row-major with rows `ld` apart, or (ld 0) in blocks of 64 columns, each block row-major
  const void* p;
  int64_t rows, cols, ld;
};

// Result of the product: base (NULL: none), row length (0: blocks of 64 columns) and type
struct Result {
  void* p;
  int64_t ld;
  bool f32;
  int64_t planes;
};

// Tiles of a launch over an M x N result: rows per tile follow from `pair`, the width is the one whose rounds over the GPU's
// workers cost least (a tile costs its width, plus some columns' worth of hand-over).
// `step`: what the width has to be a multiple of (16 columns of each CTA's B; 64 where boxes of 64 columns are loaded or stored).
struct Plan { int pair, bn, m_tiles, n_tiles; };
Plan plan_tiles(int64_t M, int64_t N, int pair, int step) {
  Plan best{pair, 0, static_cast<int>(cdiv(M, 128 * pair)), 0};
  double cost = 1e30;
  for (int bn = kMaxBN; bn >= step && bn >= 64; bn -= step) {
    const int64_t tiles = best.m_tiles * cdiv(N, bn);
    const double rounds = static_cast<double>(cdiv(tiles, kSms / pair)) * (bn + 24);
    if (rounds < cost * 0.995) { cost = rounds; best.bn = bn; }
  }
  best.n_tiles = static_cast<int>(cdiv(N, best.bn));
  return best;
}

// The dh product has few tiles and a long K: width and K splits together, least bytes of operands per worker.
Plan plan_split(int64_t M, int64_t N, int pair, int64_t k_blocks, int& splits) {
  Plan best{pair, 0, static_cast<int>(cdiv(M, 128 * pair)), 0};
  double cost = 1e30;
  const int workers = kSms / pair;
  splits = 1;
  for (int bn = kMaxBN; bn >= 64 * pair; bn -= 64 * pair) {
    const int64_t tiles = best.m_tiles * cdiv(N, bn);
    int64_t s = workers / tiles;
    if (s > k_blocks / 8) s = k_blocks / 8;
    if (s < 1) s = 1;
    const int64_t depth = cdiv(k_blocks, s);
    const double c = static_cast<double>(cdiv(tiles * s, workers)) * depth * (128 * pair + bn);
    if (c < cost * 0.995) { cost = c; best.bn = bn; splits = static_cast<int>(cdiv(k_blocks, depth)); }
  }
  best.n_tiles = static_cast<int>(cdiv(N, best.bn));
  return best;
}

struct Gemm { GemmMaps maps; GemmParams p; };

template <class P>
int prepare(Gemm& g, const Matrix& A, const Matrix& B, const Result& out, const Plan& plan, int64_t K, int splits) {
  GemmParams& p = g.p;
  p.M = P::kAMn ? A.cols : A.rows;
  p.N = P::kBMn ? B.cols : B.rows;
  p.m_tiles = plan.m_tiles;
  p.n_tiles = plan.n_tiles;
  p.bn = plan.bn;
  p.k_blocks = static_cast<int>(cdiv(K, kBK));
  p.kb_per_split = static_cast<int>(cdiv(p.k_blocks, splits));
  p.splits = static_cast<int>(cdiv(p.k_blocks, p.kb_per_split));
  p.behind = p.alone_rounds = 0;
  int rc = bind_context();
  // a single CTA's one row tile may be short: only its rows are loaded (what the others hold reaches no result)
  const int a_rows = P::kAMn ? kBK : P::kPair == 1 && p.M < 128 ? static_cast<int>(cdiv(p.M, 8)) * 8 : 128;
  p.m_step = 128;
  p.a_bytes = P::kAMn ? kABytes : a_rows * kBK * 2;
  p.tx_bytes = p.a_bytes + plan.bn / P::kPair * kBK * 2;
  // pairs have one geometry, so that two products can share a launch; a single CTA's ring is as deep as its tiles allow (reads of
  // A rows past a short tile stay inside the ring and the staging behind it)
  p.stage_bytes = P::kPair == 2 ? kABytes + kMaxBN / 2 * kBK * 2 : p.a_bytes + plan.bn * kBK * 2;
  p.stages = kRingBytes / p.stage_bytes < 8 ? kRingBytes / p.stage_bytes : 8;
  if (rc == JL_OK) rc = A.ld == 0 ? make_map2(&g.maps.a, A.p, A.rows, 64, 64, 64, a_rows, false, cdiv(A.cols, 64), true)
                                  : make_map2(&g.maps.a, A.p, A.rows, A.cols, A.ld, kBK, a_rows, false, 1, false);
  if (rc == JL_OK) rc = make_map2(&g.maps.b, B.p, B.rows, B.cols, B.ld, kBK, P::kBMn ? kBK : plan.bn / P::kPair, false, 1, false);
  if (rc == JL_OK && out.p != nullptr)
    rc = out.ld == 0 ? make_map2(&g.maps.out, out.p, p.M, 64, 64, 64, 32, false, cdiv(p.N, 64), true)
                     : make_map2(&g.maps.out, out.p, p.M, p.N, out.ld, out.f32 ? 32 : 64, 32, out.f32, out.planes, true);
  return rc;
}

// Scores of up to 32 rows: the weight's rows are the rows of the product and the hidden states its columns, so that a tile
// multiplies 16 columns for one row instead of 128 rows, in equal shares for all SMs.  At the power cap the saved work is time:
// 151936 x 4096, 1 row 240 us -> 200 in a loop and 202 -> 189 (6.6 TB/s) after a pause, 16 rows 243 -> 203 and 207 -> 193, 32 rows
// 246 -> 218 and 208 -> 198.  With more rows the hidden states, loaded once for 115 weight rows instead of 208, cost what the MMAs
// save: 48 rows 247 -> 236 and 210 -> 216.
struct FewPlan { int step, tiles, bn; };
FewPlan plan_few(int64_t rows, int64_t vocab) {
  const int64_t rounds = cdiv(vocab, int64_t(128) * kSms);
  int64_t step = cdiv(vocab, rounds * kSms);
  if (step < 8) step = 8;
  return FewPlan{static_cast<int>(step), static_cast<int>(cdiv(vocab, step)), static_cast<int>(cdiv(rows, 16)) * 16};
}
int prepare_few(Gemm& g, const Matrix& w, const Matrix& h, const FewPlan& f) {
  GemmParams& p = g.p;
  p.M = w.rows;
  p.N = h.rows;
  p.m_tiles = f.tiles;
  p.n_tiles = p.splits = 1;
  p.bn = f.bn;
  p.m_step = f.step;
  p.k_blocks = p.kb_per_split = static_cast<int>(cdiv(w.cols, kBK));
  p.group_m = p.behind = p.alone_rounds = 0;
  // Stages are packed: an MMA reads 128 rows of A and bn of B whatever is loaded, at the end of the ring into the staging behind it;
  // what the rows past the loaded ones hold reaches no result.
  p.a_bytes = static_cast<int>(cdiv(f.step * kBK * 2, 1024)) * 1024;
  p.stage_bytes = p.a_bytes + static_cast<int>(cdiv(h.rows * kBK * 2, 1024)) * 1024;
  p.tx_bytes = (f.step + static_cast<int>(h.rows)) * kBK * 2;
  const int stages = (kRingBytes + kStagingBytes - static_cast<int>(h.rows) * 512) / p.stage_bytes;
  p.stages = stages < kMaxStages ? stages : kMaxStages;
  int rc = bind_context();
  if (rc == JL_OK) rc = make_map2(&g.maps.a, w.p, w.rows, w.cols, w.ld, kBK, f.step, false, 1, false);
  if (rc == JL_OK) rc = make_map2(&g.maps.b, h.p, h.rows, h.cols, h.ld, kBK, static_cast<int>(h.rows), false, 1, false);
  return rc;
}

template <class P0, class P1>
int launch(const Gemm& g0, const Gemm& g1, cudaStream_t stream) {
  constexpr int kPair = P0::kPair;
  auto kernel = head_gemm_kernel<P0, P1>;
  static bool attr_set[64] = {false};
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(JL_ERR_LAUNCH, "jl_head: no current CUDA device");
  if (!attr_set[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemmSmemBytes) != cudaSuccess)
      return check_launch("jl_head (shared memory opt-in)");
    attr_set[dev] = true;
  }
  const int64_t tiles = std::is_same<P1, void>::value ? tiles_of(g0.p) : kSms;
  const int workers = static_cast<int>(tiles < kSms / kPair ? tiles : kSms / kPair);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(workers * kPair);
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = kGemmSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = kPair;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kernel, g0.maps, g0.p, g1.maps, g1.p) != cudaSuccess) return check_launch("jl_head");
  return JL_OK;
}

template <class P>
int launch_one(const Gemm& g, cudaStream_t stream) { return launch<P, void>(g, g, stream); }

using ScoresFew16 = Product<1, false, false, kEpiFew16>;
using ScoresFew32 = Product<1, false, false, kEpiFew32>;
using Scores1 = Product<1, false, false, kEpiScores>;
using Scores2 = Product<2, false, false, kEpiScores>;
using Dz1 = Product<1, false, false, kEpiDz>;
using Dz2 = Product<2, false, false, kEpiDz>;
using Dh1 = Product<1, false, true, kEpiF32>;
using Dh2 = Product<2, false, true, kEpiF32>;
using Dw2 = Product<2, true, true, kEpiBf16>;

int pair_of(int64_t rows) { return rows > 128 ? 2 : 1; }

// Rows of m tiles whose A panel stays in L2 beside the streamed B: 40 MB of hidden states.
int group_of(int64_t K, int pair) {
  const int64_t g = (int64_t(40) << 20) / (K * 2 * 128 * pair);
  return static_cast<int>(g < 1 ? 1 : g);
}

// The tiles' partials take 24 bytes per row and tile; rows beyond 16384 go through the same workspace in further launches
// (each reads the weight once more, 0.2 ms beside 14 ms of products at a hidden size of 4096).
constexpr int64_t kScoreRows = 16384;
// Rows whose label is ignored are left out of the products where there are more row tiles than one: the others are packed first
// (1000 rows x 4096 x 151936, two in five ignored: loss and gradients 3.58 -> 2.69 ms after a pause, 4.10 -> 3.10 in a loop).
constexpr int64_t kPackRows = 257;
struct Packed { size_t hidden, labels, lse, nll, row_grad, row_of, place, used; };      // offsets in the workspace
Packed packed_layout(size_t& total, int64_t rows, int64_t chunk, int32_t hd) {
  Packed k{};
  auto take = [&](int64_t bytes) { const size_t at = total; total += up256(static_cast<size_t>(bytes)); return at; };
  k.hidden = take(chunk * hd * 2);
  k.labels = take(chunk * 8);
  k.lse = take(chunk * 4);
  k.nll = take(chunk * 4);
  k.row_grad = take(chunk * 4);
  k.row_of = take(rows * 4);
  k.place = take(rows * 4);
  k.used = take(4);
  return k;
}
struct ScoresLayout { Plan plan; FewPlan few; int tiles; size_t part, arg, picked, nll, total; bool pack; Packed packed; };      // tiles: partials of a row
ScoresLayout scores_layout(int64_t rows, int32_t hd, int32_t vocab, bool skip_ignored) {
  ScoresLayout l{};
  const int64_t n = rows < 1 ? 1 : rows < kScoreRows ? rows : kScoreRows;
  l.plan = plan_tiles(n, vocab, pair_of(n), 16 * pair_of(n));
  l.few = plan_few(n <= kFewRows ? n : 1, vocab);
  l.tiles = n <= kFewRows ? l.few.tiles : l.plan.n_tiles * 2;
  const size_t parts = static_cast<size_t>(n) * l.tiles;
  l.part = 0;
  l.arg = up256(parts * sizeof(float2));
  l.picked = l.arg + up256(parts * sizeof(int));
  l.nll = l.picked + up256(n * sizeof(float));
  l.total = l.nll + up256(static_cast<size_t>(rows) * sizeof(float));
  l.pack = skip_ignored && rows >= kPackRows;
  if (l.pack) l.packed = packed_layout(l.total, rows, n, hd);
  return l;
}

// Pieces of the vocabulary in the gradient pass: as large as 256 MB of dz allow (fewer, longer launches), balanced, a
// multiple of 256.
struct GradsLayout { int64_t piece; Plan dz, dh, dw; int splits; size_t dh32, counted, total; bool pack; Packed packed; };
GradsLayout grads_layout(int64_t rows, int32_t hd, int32_t vocab) {
  GradsLayout l{};
  const int64_t n = rows > 0 ? rows : 1;
  int64_t most = (int64_t(256) << 20) / (n * 2) / 256 * 256;
  if (most < 2048) most = 2048;
  const int64_t pieces = cdiv(vocab, most);
  l.piece = cdiv(cdiv(vocab, pieces), 256) * 256;
  l.dz = plan_tiles(n, l.piece < vocab ? l.piece : vocab, pair_of(n), 64);
  l.dw = plan_tiles(l.piece < vocab ? l.piece : vocab, hd, 2, 128);
  l.dh = plan_split(n, hd, pair_of(n), cdiv(l.piece, kBK), l.splits);
  l.dh32 = up256(static_cast<size_t>(n) * l.piece * 2);
  l.total = l.dh32 + up256(static_cast<size_t>(n) * hd * 4 * l.splits);
  l.pack = rows >= kPackRows;
  l.counted = l.total;
  if (l.pack) l.packed = packed_layout(l.total, rows, rows, hd);
  else l.total += up256(static_cast<size_t>(n) * hd * 2);
  return l;
}

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

int launch_scores(const jl_head_scores_args* a, cudaStream_t stream) {
  int rc = validate("jl_head_scores", a->hidden, a->weight, a->hidden_stride, a->weight_stride, a->rows, a->hidden_size, a->vocab);
  if (rc != JL_OK) return rc;
  const bool want_loss = a->loss_sum != nullptr || a->loss_count != nullptr || a->loss_mean != nullptr;
  if (a->labels == nullptr && (a->nll != nullptr || want_loss))
    return fail(JL_ERR_BAD_ARG, "jl_head_scores: nll and the loss need labels");
  if (a->skip_ignored && (a->labels == nullptr || a->top != nullptr))
    return fail(JL_ERR_BAD_ARG, "jl_head_scores: skip_ignored needs labels and leaves no top");
  if (misaligned(8, a->labels, a->top) || misaligned(4, a->nll, a->lse, a->loss_sum, a->loss_count, a->loss_mean))
    return fail(JL_ERR_BAD_ARG, "jl_head_scores: labels and top must be 8-byte aligned, the fp32 results 4-byte");
  const ScoresLayout l = scores_layout(a->rows, a->hidden_size, a->vocab, a->skip_ignored != 0);
  if (a->workspace == nullptr || a->workspace_bytes < l.total)
    return fail(JL_ERR_WORKSPACE, "jl_head_scores: workspace of %zu bytes needed, %zu given", l.total, a->workspace_bytes);
  if (reinterpret_cast<uintptr_t>(a->workspace) & 15) return fail(JL_ERR_BAD_ARG, "jl_head_scores: workspace not 16-byte aligned");
  rc = check_device_arch();
  if (rc != JL_OK) return rc;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  float* nll = a->nll != nullptr || !want_loss ? a->nll : reinterpret_cast<float*>(ws + l.nll);
  int32_t *const row_of = reinterpret_cast<int32_t*>(ws + l.packed.row_of), *const place = reinterpret_cast<int32_t*>(ws + l.packed.place),
          *const used = reinterpret_cast<int32_t*>(ws + l.packed.used);
  int64_t* const labels_packed = reinterpret_cast<int64_t*>(ws + l.packed.labels);
  __nv_bfloat16* const hidden_packed = reinterpret_cast<__nv_bfloat16*>(ws + l.packed.hidden);
  if (l.pack && launch_dependent(rows_used_kernel, dim3(1), dim3(1024), 0, stream, a->labels, a->ignore_index, a->rows, row_of, place, used, nll, a->lse) !=
                    cudaSuccess)
    return check_launch("jl_head_scores (rows in use)");
  for (int64_t r0 = 0; r0 < a->rows; r0 += kScoreRows) {
    const int64_t n = a->rows - r0 < kScoreRows ? a->rows - r0 : kScoreRows;
    Plan plan = l.plan;
    plan.m_tiles = static_cast<int>(cdiv(n, 128 * plan.pair));
    Gemm g{};
    GemmParams& p = g.p;
    p.part = reinterpret_cast<float2*>(ws + l.part);
    p.part_arg = a->top != nullptr ? reinterpret_cast<int*>(ws + l.arg) : nullptr;
    p.picked = reinterpret_cast<float*>(ws + l.picked);
    p.labels = l.pack ? labels_packed : a->labels != nullptr ? a->labels + r0 : nullptr;
    p.ignore = a->ignore_index; p.vocab = a->vocab;
    p.group_m = group_of(a->hidden_size, plan.pair);
    p.rows_used = l.pack ? used : nullptr;
    p.row0 = r0;
    if (l.pack && launch_dependent(rows_gather_kernel, dim3(static_cast<unsigned>(n)), dim3(128), 0, stream, static_cast<const __nv_bfloat16*>(a->hidden),
                                   a->hidden_stride, a->hidden_size, a->labels, a->ignore_index, static_cast<const float*>(nullptr),
                                   static_cast<const float*>(nullptr), static_cast<const float*>(nullptr), static_cast<const int32_t*>(row_of),
                                   static_cast<const int32_t*>(used), r0, hidden_packed, labels_packed, static_cast<float*>(nullptr), static_cast<float*>(nullptr),
                                   static_cast<float*>(nullptr)) != cudaSuccess)
      return check_launch("jl_head_scores (packing)");
    const Matrix h = l.pack ? Matrix{hidden_packed, n, a->hidden_size, a->hidden_size}
                            : Matrix{static_cast<const __nv_bfloat16*>(a->hidden) + r0 * a->hidden_stride, n, a->hidden_size, a->hidden_stride};
    const Matrix w{a->weight, a->vocab, a->hidden_size, a->weight_stride};
    if (a->rows <= kFewRows) {
      rc = prepare_few(g, w, h, l.few);
      if (rc == JL_OK) rc = a->rows <= 16 ? launch_one<ScoresFew16>(g, stream) : launch_one<ScoresFew32>(g, stream);
    } else if (plan.pair == 2) {
      rc = prepare<Scores2>(g, h, w, Result{}, plan, a->hidden_size, 1);
      if (rc == JL_OK) rc = launch_one<Scores2>(g, stream);
    } else {
      rc = prepare<Scores1>(g, h, w, Result{}, plan, a->hidden_size, 1);
      if (rc == JL_OK) rc = launch_one<Scores1>(g, stream);
    }
    if (rc != JL_OK) return rc;
    const bool few = n < 16 * kSms;          // (1000 rows of 1188 partials: 25 us with a warp each, 12 with eight)
    if (launch_dependent(few ? scores_fold_kernel<8> : scores_fold_kernel<1>, dim3(static_cast<unsigned>(few ? n : cdiv(n, 8))), dim3(256), 0, stream,
                         static_cast<const float2*>(p.part), static_cast<const int*>(p.part_arg), static_cast<const float*>(p.picked), l.tiles, n,
                         static_cast<int64_t>(a->vocab), p.labels, a->ignore_index, nll != nullptr ? nll + (l.pack ? 0 : r0) : nullptr,
                         a->lse != nullptr ? a->lse + (l.pack ? 0 : r0) : nullptr, a->top != nullptr ? a->top + r0 : nullptr, p.rows_used,
                         l.pack ? static_cast<const int32_t*>(row_of) : nullptr, r0) != cudaSuccess)
      return check_launch("jl_head_scores (fold)");
  }
  if (want_loss && launch_dependent(loss_sum_kernel, dim3(1), dim3(1024), 0, stream, static_cast<const float*>(nll), a->labels, a->ignore_index, a->rows,
                                    a->loss_sum, a->loss_count, a->loss_mean) != cudaSuccess)
    return check_launch("jl_head_scores (loss)");
  return JL_OK;
}

int launch_grads(const jl_head_grads_args* a, cudaStream_t stream) {
  int rc = validate("jl_head_grads", a->hidden, a->weight, a->hidden_stride, a->weight_stride, a->rows, a->hidden_size, a->vocab);
  if (rc != JL_OK) return rc;
  if (a->labels == nullptr || a->lse == nullptr || a->grad == nullptr) return fail(JL_ERR_BAD_ARG, "jl_head_grads: NULL pointer");
  if (a->grad_stride != 0 && a->grad_stride != 1) return fail(JL_ERR_BAD_ARG, "jl_head_grads: grad_stride must be 0 or 1");
  if ((reinterpret_cast<uintptr_t>(a->d_hidden) | reinterpret_cast<uintptr_t>(a->d_weight)) & 15)
    return fail(JL_ERR_BAD_ARG, "jl_head_grads: d_hidden and d_weight must be 16-byte aligned");
  const GradsLayout l = grads_layout(a->rows, a->hidden_size, a->vocab);
  if (a->workspace == nullptr || a->workspace_bytes < l.total)
    return fail(JL_ERR_WORKSPACE, "jl_head_grads: workspace of %zu bytes needed, %zu given", l.total, a->workspace_bytes);
  if (reinterpret_cast<uintptr_t>(a->workspace) & 15) return fail(JL_ERR_BAD_ARG, "jl_head_grads: workspace not 16-byte aligned");
  if (a->nll == nullptr) return fail(JL_ERR_BAD_ARG, "jl_head_grads: nll is NULL");
  if (misaligned(8, a->labels) || misaligned(4, a->lse, a->nll, a->grad, a->grad_count))
    return fail(JL_ERR_BAD_ARG, "jl_head_grads: labels must be 8-byte aligned, the fp32 operands 4-byte");
  rc = check_device_arch();
  if (rc != JL_OK) return rc;
  const int64_t N = a->rows, H = a->hidden_size, V = a->vocab;
  if (N == 0) {
    if (a->d_weight != nullptr && cudaMemsetAsync(a->d_weight, 0, V * H * 2, stream) != cudaSuccess) return check_launch("jl_head_grads");
    return JL_OK;
  }
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  float* dh32 = reinterpret_cast<float*>(ws + l.dh32);
  GemmParams base{};
  base.labels = a->labels; base.ignore = a->ignore_index; base.vocab = V;
  base.lse = a->lse;
  base.nll = a->nll;
  base.row_grad = a->grad_stride != 0 ? a->grad : nullptr;
  base.scale = GradScale{a->grad, a->grad_count, a->grad_stride != 0};
  Matrix h{a->hidden, N, H, a->hidden_stride};
  const int32_t* place = nullptr;
  if (l.pack) {
    int32_t *const row_of = reinterpret_cast<int32_t*>(ws + l.packed.row_of), *const used = reinterpret_cast<int32_t*>(ws + l.packed.used);
    int64_t* const labels = reinterpret_cast<int64_t*>(ws + l.packed.labels);
    float *const lse = reinterpret_cast<float*>(ws + l.packed.lse), *const nll = reinterpret_cast<float*>(ws + l.packed.nll),
          *const row_grad = reinterpret_cast<float*>(ws + l.packed.row_grad);
    __nv_bfloat16* const hidden = reinterpret_cast<__nv_bfloat16*>(ws + l.packed.hidden);
    place = reinterpret_cast<int32_t*>(ws + l.packed.place);
    if (launch_dependent(rows_used_kernel, dim3(1), dim3(1024), 0, stream, a->labels, a->ignore_index, N, row_of, const_cast<int32_t*>(place), used,
                         static_cast<float*>(nullptr), static_cast<float*>(nullptr)) != cudaSuccess)
      return check_launch("jl_head_grads (rows in use)");
    if (launch_dependent(rows_gather_kernel, dim3(static_cast<unsigned>(N)), dim3(128), 0, stream, static_cast<const __nv_bfloat16*>(a->hidden),
                         a->hidden_stride, a->hidden_size, a->labels, a->ignore_index, a->lse, a->nll, base.row_grad, static_cast<const int32_t*>(row_of),
                         static_cast<const int32_t*>(used), int64_t(0), hidden, labels, lse, nll, row_grad) != cudaSuccess)
      return check_launch("jl_head_grads (packing)");
    base.labels = labels;
    base.lse = lse;
    base.nll = nll;
    if (base.row_grad != nullptr) base.row_grad = row_grad;
    base.rows_used = used;
    h = Matrix{hidden, N, H, H};
  }
  // the weight's gradient multiplies every row, if by zero: it takes rows that do not count as zero (packed rows are that already)
  __nv_bfloat16* const counted = l.pack || a->d_weight == nullptr ? nullptr : reinterpret_cast<__nv_bfloat16*>(ws + l.counted);
  const Matrix hw = counted != nullptr ? Matrix{counted, N, H, H} : h;
  int splits = 1;
  bool rounded = false;
  auto round_rows = [&]() -> int {
    if (launch_dependent(grad_round_kernel, dim3(static_cast<unsigned>(cdiv(N * H, 1024))), dim3(256), 0, stream, static_cast<const float*>(dh32), splits, N * H,
                         static_cast<__nv_bfloat16*>(a->d_hidden), base.scale, place, a->hidden_size) != cudaSuccess)
      return check_launch("jl_head_grads (rounding)");
    return JL_OK;
  };
  for (int64_t v0 = 0; v0 < V; v0 += l.piece) {
    const int64_t piece = V - v0 < l.piece ? V - v0 : l.piece;
    const Matrix w{static_cast<const __nv_bfloat16*>(a->weight) + v0 * a->weight_stride, piece, H, a->weight_stride};
    const Matrix dz{ws, N, piece, 0};
    Gemm z{GemmMaps{}, base}, dh{GemmMaps{}, base}, dw{GemmMaps{}, base};
    z.p.v0 = v0;
    if (v0 == 0) {
      z.p.hidden = static_cast<const __nv_bfloat16*>(a->hidden);
      z.p.counted = counted;
      z.p.hidden_stride = a->hidden_stride;
      z.p.row_len = a->hidden_size;
    }
    z.p.group_m = group_of(H, l.dz.pair);
    Plan plan = l.dz;
    plan.n_tiles = static_cast<int>(cdiv(piece, plan.bn));
    const Result z_out{ws, 0, false, 1};
    if (plan.pair == 2) {
      rc = prepare<Dz2>(z, h, w, z_out, plan, H, 1);
      if (rc == JL_OK) rc = launch_one<Dz2>(z, stream);
    } else {
      rc = prepare<Dz1>(z, h, w, z_out, plan, H, 1);
      if (rc == JL_OK) rc = launch_one<Dz1>(z, stream);
    }
    if (rc == JL_OK && a->d_hidden != nullptr) {
      dh.p.reduce = v0 > 0;
      dh.p.group_m = 1 << 20;
      const int64_t kb = cdiv(piece, kBK);
      // a short last piece has fewer K splits than the others: the planes it does not reach keep their sums
      const int s = static_cast<int>(kb < l.splits ? kb : l.splits);
      const Result out{dh32, H, true, l.splits};
      rc = l.dh.pair == 2 ? prepare<Dh2>(dh, dz, w, out, l.dh, piece, s) : prepare<Dh1>(dh, dz, w, out, l.dh, piece, s);
      if (v0 == 0) splits = dh.p.splits;
    }
    if (rc == JL_OK && a->d_weight != nullptr) {
      plan = l.dw;
      plan.m_tiles = static_cast<int>(cdiv(piece, 256));
      dw.p.group_m = 0;
      rc = prepare<Dw2>(dw, dz, hw, Result{static_cast<__nv_bfloat16*>(a->d_weight) + v0 * H, H, false, 1}, plan, N, 1);
    }
    if (rc == JL_OK && a->d_hidden != nullptr && a->d_weight != nullptr && l.dh.pair == 2) {
      // dh has few, long tiles (160 on 74 pairs for 4096 rows x 2560: 72 % of three rounds); dW's many short ones fill in
      balance(dh.p, dw.p);
      rc = launch<Dh2, Dw2>(dh, dw, stream);
    } else {
      if (rc == JL_OK && a->d_hidden != nullptr) rc = l.dh.pair == 2 ? launch_one<Dh2>(dh, stream) : launch_one<Dh1>(dh, stream);
      // the row gradients are rounded while they are in L2, ahead of the weight's (127 x 2048 x 50257: 191 -> 184 us)
      if (rc == JL_OK && a->d_hidden != nullptr && v0 + piece == V) rc = round_rows();
      if (rc == JL_OK && a->d_weight != nullptr) rc = launch_one<Dw2>(dw, stream);
      rounded = true;
    }
    if (rc != JL_OK) return rc;
  }
  return a->d_hidden != nullptr && !rounded ? round_rows() : JL_OK;
}

}  // namespace

}  // namespace jl

extern "C" {

size_t jl_head_scores_workspace_bytes(int64_t rows, int32_t hidden_size, int32_t vocab, int32_t skip_ignored) {
  return rows < 0 || hidden_size < 1 || vocab < 1 ? 0 : jl::scores_layout(rows, hidden_size, vocab, skip_ignored != 0).total + 256;
}

int jl_head_scores(const jl_head_scores_args* args, void* cuda_stream) {
  if (args == nullptr) return jl::fail(JL_ERR_BAD_ARG, "jl_head_scores: args is NULL");
  return jl::launch_scores(args, static_cast<cudaStream_t>(cuda_stream));
}

size_t jl_head_grads_workspace_bytes(int64_t rows, int32_t hidden_size, int32_t vocab) {
  return rows < 0 || hidden_size < 1 || vocab < 1 ? 0 : jl::grads_layout(rows, hidden_size, vocab).total + 256;
}

int jl_head_grads(const jl_head_grads_args* args, void* cuda_stream) {
  if (args == nullptr) return jl::fail(JL_ERR_BAD_ARG, "jl_head_grads: args is NULL");
  return jl::launch_grads(args, static_cast<cudaStream_t>(cuda_stream));
}

int jl_head_status(void) {
  int v = 0;
  if (cudaDeviceSynchronize() != cudaSuccess) return -1;      // the copy alone waits for the legacy stream and what blocks on it
  if (cudaMemcpyFromSymbol(&v, jl::g_head_status, sizeof(int)) != cudaSuccess) return -1;
  const int zero = 0;
  if (v != 0) cudaMemcpyToSymbol(jl::g_head_status, &zero, sizeof(int));
  return v;
}

}  // extern "C"
