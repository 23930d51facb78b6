// Attention of a tree of drafted tokens over the bifocal cache, on the Blackwell tensor path.
//
// The rows of one product are the (node, query head) pairs that share a key head: row r of a 128-row tile is node
// r / rep, head r % rep of the key head's group (rep = heads / kv_heads), so one pass over the cache serves every drafted
// token.  A tree of up to 128 rows per key head takes ONE row tile, whose two softmax warpgroups work on alternate key
// tiles of the same rows (two running states, joined at the end of a segment); a larger tree takes TWO row tiles per CTA, and further
// CTAs that walk the same keys at the same time for its further rows; the last tile of an odd number has CTAs of its own.
//
// Work is a line of VISITS: for every (sample, key head) the key tiles of the far class, then those of the near class (a
// tile crossed by the boundary is visited in both with complementary masks).  The line is cut into equal parts, one per
// SM, wherever that falls, so a batch of any lengths fills the GPU evenly; a part is made of SEGMENTS of one (sample, key
// head) each.  A segment that is all of its (sample, key head) writes the result, every other one leaves one normalised fp32
// partial (O, LSE) per row that tree_combine_kernel joins.
// Nothing on the host depends on the lengths, which are read on the device.
//
//   warp 0      TMA producer of K and V tiles (one ring of 5, in the order of their use), running ahead over all borders; it
//               also leaves one word per visit that tells the issuers what is particular about it
//   warp 1      issues S_t = Q K^T;  warp 2 issues O_t += P V (and owns tensor memory).  Two issuers, because the issue of an MMA
//               blocks while two or three are queued: with one, the waits for one tile's operands stood between the products of
//               the other (2000 clocks per 128 x 128 x 256 product pair instead of 1450)
//   warp 3      TMA producer of the query tiles of the current class
//   warps 4-11  softmax: one thread per row, P back to tensor memory over S
//
// The softmax is one pass over the keys: with the running maximum m (raised lazily, only when a score exceeds it by 2^8), O and l hold
// sum e^(s - m) v and sum e^(s - m) in fp32; P is rounded to bf16 for the product, as the values are.  Times of a replayed graph of the
// call, the join included, after a pause and (in brackets) in a loop at the power cap.  16 nodes x 4 heads over 131056 keys: 96 us
// [107] for 537 MB of keys and values, bound by their stream (6.0 TB/s of 6.56 inside the kernel).  64 nodes x 4 heads: 143 us [170],
// bound by the chain of a row tile's products and softmax (tensor pipe 58 %).
#include "tc_common.cuh"
#include "../../include/jetlong_b200_tree.h"

namespace jl {

namespace {

using namespace tc;

__device__ int g_tree_status = 0;            // raised when a bounded wait gave up

constexpr int kTileN = 128;                  // keys per visit
// Tiles in the ring: K of visit g is its tile 2 g, V is tile 2 g + 1.  The number is odd, so a slot holds K and V in turn, and each
// issuer waits for every second use of it only; the use between has landed by then: before Q K of visit g its issuer has waited for
// P V of visit g - 3 (whose V was there), and before P V of visit g for scores of visit g - 1.
constexpr int kStages = 5;
constexpr int kTileBytes = 128 * 256;        // 128 rows x 128 bf16
constexpr int kHalfBytes = 128 * 128;        // one 64-column half (a TMA box)
constexpr int kThreads = 384;
constexpr int kRegsLow = 72, kRegsHigh = 216;     // 128 x 72 + 256 x 216 = the launch total 384 x 168
constexpr int kSms = 148;

struct TreeParams {
  int batch, nodes, words, rep, kv_heads, rows;
  int npt;                     // nodes per row tile
  int rpt;                     // rows per row tile that can be in use
  int pairs, workers;          // CTAs of two row tiles per part of the line, parts
  int workers_one;             // the last row tile of an odd number has CTAs of its own (two states of the one tile): parts, 0: none
  int unrolled;                // enough visits per part to pay for the unrolled softmax's instruction fetches
  int two_classes, nodes_far;  // nodes_far: w_0 is so small that drafted keys can be in the far class
  int64_t w_0;
  float scale_log2;
  const int32_t *lens, *depth;
  const uint64_t* mask;
  float *part_o, *part_lse;    // [place] (two row tiles: [place][tile]) of [32 column groups][rpt rows][4] and [rpt rows]
  __nv_bfloat16* out;
  float* lse;
  int64_t os_b, os_s, os_h;
};

struct TreeMaps { CUtensorMap q[2], k[2], v; };       // [0] near (base), [1] far (regrouped)

// What is particular about a visit.
enum : int { kQFirst = 1, kQLast = 2, kOFirst = 4, kTail = 8 };
constexpr int kVisitRing = 8;                // the producer is at most 3 visits ahead of the last consumer

struct TreeSmem {
  alignas(1024) uint8_t q[2][kTileBytes];    // two row tiles, or two class operands of one
  alignas(1024) uint8_t kv[kStages][kTileBytes];
  uint64_t q_full[2], q_free[2], full[kStages], empty[kStages];
  uint64_t s_full[2], p_half[2][2], pv_done[2];
  alignas(16) int4 visit[kVisitRing];        // flags, sample, node index of the key tile's first row
  float2 stats[2][128];                      // two states of one tile meet: reference maximum and sum of each row
  int64_t lo, hi;                            // this CTA's part of the line
  int start_b, start_kvh, start_v;
  uint32_t tmem_base;
  int failed;
};

// The visits of one (sample, key head): far key tiles [0, far), then near key tiles near0 ..
// `nodes`: the places of the tree that the cache has rows for.  A node behind them is an absent one, as tree_append stored no key of it.
// A length that is none of this cache counts as the nearest one that leaves a row to every place.
struct Visits { int len, nodes, far, near0, n; };
__device__ __forceinline__ Visits visits_of(const TreeParams& p, int b) {
  Visits v;
  v.len = max(p.lens[b], 0);
  if (v.len > p.rows) v.len = p.rows - p.nodes;
  v.nodes = min(p.nodes, p.rows - v.len);
  const int64_t end = static_cast<int64_t>(v.len) + v.nodes;
  v.far = v.near0 = 0;
  if (p.two_classes) {
    int64_t hi = p.nodes_far ? end : static_cast<int64_t>(v.len) + p.nodes - 1 - p.w_0;      // keys below this can be far for some node
    hi = hi < 0 ? 0 : (hi > end ? end : hi);
    v.far = static_cast<int>((hi + kTileN - 1) / kTileN);
    const int64_t lo = v.len - p.w_0;                                          // keys from this on can be near
    v.near0 = static_cast<int>((lo < 0 ? 0 : lo) / kTileN);
  }
  v.n = v.far + static_cast<int>((end + kTileN - 1) / kTileN) - v.near0;
  return v;
}

// Row tiles 2 mb and 2 mb + 1 are worked on together, or tile 2 mb alone.
__device__ __forceinline__ bool has_two(const TreeParams& p, int mb) { return mb < p.pairs; }

// Parts that the line is cut into for these row tiles: one per worker, but none empty.
__device__ __forceinline__ int64_t parts_of(const TreeParams& p, int mb, int64_t total) {
  return min(static_cast<int64_t>(has_two(p, mb) ? p.workers : p.workers_one), total);
}

// Place of a partial of row tile 2 mb + t.  Only a part's first and last segment can be less than their (sample, key head): `i` is
// twice the part for the first, one more for the last.
__device__ __forceinline__ int64_t place_of(const TreeParams& p, int mb, int t, int64_t i) {
  const int64_t per = 2 * static_cast<int64_t>(p.workers);
  return has_two(p, mb) ? (mb * per + i) * 2 + t : p.pairs * per * 2 + i;
}

struct Segment {
  int b, kvh, v0, v1;          // visits [v0, v1)
  Visits vis;
  __device__ __forceinline__ int key_tile(int v) const { return v < vis.far ? v : vis.near0 + v - vis.far; }
  __device__ __forceinline__ bool tail(int v) const { return (key_tile(v) + 1) * kTileN > vis.len; }     // holds rows that are not committed
};

struct Walk {
  int b, kvh, v;
  int64_t left;
  __device__ __forceinline__ explicit Walk(const TreeSmem& sm) : b(sm.start_b), kvh(sm.start_kvh), v(sm.start_v), left(sm.hi - sm.lo) {}
  __device__ __forceinline__ bool next(const TreeParams& p, Segment& s) {
    if (left <= 0) return false;
    s.b = b;
    s.kvh = kvh;
    s.vis = visits_of(p, b);
    s.v0 = v;
    s.v1 = static_cast<int>(min(static_cast<int64_t>(s.vis.n), v + left));
    left -= s.v1 - s.v0;
    v = 0;
    if (++kvh == p.kv_heads) { kvh = 0; ++b; }
    return true;
  }
};

// Ring slot of the next K or V tile and the parity of its use
struct RingPos {
  int slot;
  uint32_t parity;
  __device__ __forceinline__ explicit RingPos(int first) : slot(first), parity(0) {}
  __device__ __forceinline__ void next() {       // two tiles per visit
    slot += 2;
    if (slot >= kStages) { slot -= kStages; parity ^= 1; }
  }
};

__global__ void __launch_bounds__(kThreads, 1) tree_attention_kernel(const __grid_constant__ TreeMaps maps, const TreeParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  TreeSmem& sm = *reinterpret_cast<TreeSmem*>(smem_raw);
  if (smem_u32(smem_raw) & 1023) {               // not seen: the array's alignment is declared
    if (threadIdx.x == 0) atomicExch(&g_tree_status, 1);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int alone = static_cast<int>(blockIdx.x) - p.pairs * p.workers;      // >= 0: on the one tile that is left
  const bool two_tiles = alone < 0;
  const int mb = two_tiles ? static_cast<int>(blockIdx.x) % p.pairs : p.pairs, worker = two_tiles ? static_cast<int>(blockIdx.x) / p.pairs : alone;
  if (threadIdx.x >= 64 && threadIdx.x < 69) {   // the tensor maps: q[0], q[1], k[0], k[1], v
    const CUtensorMap* m = reinterpret_cast<const CUtensorMap*>(&maps) + (threadIdx.x - 64);
    asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
  }
  const int q_slots = two_tiles ? 1 : 2;

  if (threadIdx.x == 32) {
    sm.failed = *reinterpret_cast<volatile int*>(&g_tree_status) != 0 ? 1 : 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.q_full[i], 1);
      mbar_init(&sm.q_free[i], 1);
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_half[i][0], 128);
      mbar_init(&sm.p_half[i][1], 128);
    }
    for (int i = 0; i < kStages; ++i) { mbar_init(&sm.full[i], 1); mbar_init(&sm.empty[i], 1); }
    for (int i = 0; i < 2; ++i) mbar_init(&sm.pv_done[i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  wait_prerequisites();                          // nothing before this reads what an earlier kernel wrote
  launch_dependents();                           // the combine kernel may take its place and wait there for our end
  if (warp == 0) {
    // ---- this CTA's part of the line of visits: total and start, 32 samples at a time ----
    int64_t total = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) total += b0 + lane < p.batch ? visits_of(p, b0 + lane).n : 0;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
    total *= p.kv_heads;
    const int64_t parts = parts_of(p, mb, total), lo = min(static_cast<int64_t>(worker), parts) * total / parts;
    const int64_t hi = min(static_cast<int64_t>(worker) + 1, parts) * total / parts;
    int64_t base = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      const int64_t mine = b0 + lane < p.batch ? static_cast<int64_t>(visits_of(p, b0 + lane).n) * p.kv_heads : 0;
      int64_t before = mine;                           // inclusive prefix sum over the 32 samples
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int64_t o = __shfl_up_sync(0xffffffffu, before, off);
        if (lane >= off) before += o;
      }
      const int64_t from = base + before - mine;
      if (mine > 0 && lo >= from && lo < from + mine) {
        const int n = static_cast<int>(mine / p.kv_heads);
        sm.start_b = b0 + lane;
        sm.start_kvh = static_cast<int>((lo - from) / n);
        sm.start_v = static_cast<int>((lo - from) % n);
      }
      base += __shfl_sync(0xffffffffu, before, 31);
    }
    if (lane == 0) { sm.lo = lo; sm.hi = hi; }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  volatile int* const failed = &sm.failed;       // a wait gave up: no more copies are issued, every later wait returns at once

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLow));
    if (warp == 0) {
      // ================================ TMA producer of K and V ================================
      if (lane == 0) {
        Walk w(sm);
        Segment seg;
        int g = 0;
        RingPos pos[2] = {RingPos(0), RingPos(1)};
        const int step = two_tiles ? 1 : 2;
        while (w.next(p, seg) && !*failed) {
          for (int v = seg.v0; v < seg.v1; ++v, ++g) {
            const int row = seg.key_tile(v) * kTileN;
            const int flags = (v == seg.v0 || v == seg.vis.far ? kQFirst : 0) | (v + 1 == seg.v1 || v + 1 == seg.vis.far ? kQLast : 0) |
                              (v - seg.v0 < step ? kOFirst : 0) | (seg.tail(v) ? kTail : 0);
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
              const CUtensorMap* map = kv == 1 ? &maps.v : &maps.k[v < seg.vis.far ? 1 : 0];
              const int st = pos[kv].slot;
              mbar_wait(&sm.empty[st], pos[kv].parity ^ 1, sm);
              if (*failed) break;
              if (kv == 0) sm.visit[g % kVisitRing] = make_int4(flags, seg.b, row - seg.vis.len, 0);      // published by the arrivals below
              mbar_expect_tx(&sm.full[st], kTileBytes);
              for (int h = 0; h < 2; ++h) tma_load_4d(sm.kv[st] + h * kHalfBytes, map, &sm.full[st], h * 64, seg.kvh, row, seg.b);
              pos[kv].next();
            }
          }
        }
      }
    } else if (warp == 3) {
      // ================================ TMA producer of the queries ================================
      if (lane == 0) {
        Walk w(sm);
        Segment seg;
        int u = 0;
        const uint32_t half = static_cast<uint32_t>(p.npt) * p.rep * 128;
        while (w.next(p, seg)) {
          for (int cls = 1; cls >= 0; --cls) {
            const bool any = cls == 1 ? seg.v0 < seg.vis.far : seg.v1 > seg.vis.far;
            if (!any) continue;
            const int slot = u % q_slots;
            mbar_wait(&sm.q_free[slot], ((u / q_slots) & 1) ^ 1, sm);
            if (*failed) break;
            mbar_expect_tx(&sm.q_full[slot], (two_tiles ? 4 : 2) * half);
            for (int t = 0; t < (two_tiles ? 2 : 1); ++t)
              for (int h = 0; h < 2; ++h)
                tma_load_4d(sm.q[slot + t] + h * kHalfBytes, &maps.q[cls], &sm.q_full[slot], h * 64, seg.kvh * p.rep, (mb * 2 + t) * p.npt, seg.b);
            ++u;
          }
        }
      }
    } else {
      // ==================================== MMA issuers ====================================
      // The whole warp walks the visits, so that ring indices, parities and descriptors are warp-uniform; one elected lane issues.
      uint32_t leader;
      asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(leader));
      const int n = static_cast<int>(sm.hi - sm.lo), tiles = two_tiles ? 2 : 1;
      RingPos pos(warp - 1);                           // K tiles are the ring's even tiles, V tiles the odd ones
      uint32_t parity = 0u;                            // bit t: parity of state t's next barrier phase
      if (warp == 1) {
        const uint32_t idesc = instr_desc(128, kTileN, 0);
        const uint64_t q_desc = smem_desc(smem_u32(sm.q[0]), 16, 1024), k_desc = smem_desc(smem_u32(sm.kv[0]), 16, 1024);
        int use = -1;                                  // query operands taken so far
        for (int g = 0; g < n; ++g, pos.next()) {
          mbar_wait(&sm.full[pos.slot], pos.parity, sm);
          const int flags = *reinterpret_cast<volatile int*>(&sm.visit[g % kVisitRing].x);
          if (__any_sync(0xffffffffu, flags & kQFirst)) {
            ++use;
            mbar_wait(&sm.q_full[two_tiles ? 0 : use & 1], (two_tiles ? use : use >> 1) & 1, sm);
          }
          if (*failed) break;
          const uint64_t kd = k_desc + static_cast<uint64_t>((pos.slot * kTileBytes) >> 4);
          for (int i = 0; i < tiles; ++i) {
            const int t = two_tiles ? i : g & 1;
            // The second tile starts when the first one's probabilities are out: half a visit apart, one tile's softmax runs under the
            // other's products, and they stay apart (64 nodes over 131072 keys: 142 -> 137 us).
            if (two_tiles && g == 0 && i == 1) mbar_wait(&sm.p_half[0][1], 0u, sm);
            // the scores go where the probabilities of the state's previous item are: P V has to be done with them
            if (g >= (two_tiles ? 1 : 2)) {
              mbar_wait(&sm.pv_done[t], (parity >> t) & 1u, sm);
              parity ^= 1u << t;
            }
            tc_fence_after();
            const uint64_t qd = q_desc + static_cast<uint64_t>(((two_tiles ? i : use & 1) * kTileBytes) >> 4);
            if (leader) {
#pragma unroll
              for (int kk = 0; kk < 8; ++kk) {
                const uint64_t off = static_cast<uint64_t>(((kk >> 2) * kHalfBytes + (kk & 3) * 32) >> 4);
                mma_ss(tmem + t * 128, qd + off, kd + off, idesc, kk > 0);
              }
              mma_commit(&sm.s_full[t]);
            }
            __syncwarp();
          }
          if (leader) {
            mma_commit(&sm.empty[pos.slot]);
            if (flags & kQLast) mma_commit(&sm.q_free[two_tiles ? 0 : use & 1]);
          }
          __syncwarp();
        }
      } else {
        const uint32_t idesc = instr_desc(128, kHeadDim, 1);
        const uint64_t v_desc = smem_desc(smem_u32(sm.kv[0]), kHalfBytes, 1024);
        for (int g = 0; g < n; ++g, pos.next()) {
          mbar_wait(&sm.full[pos.slot], pos.parity, sm);
          if (*failed) break;
          const int4 visit = make_int4(*reinterpret_cast<volatile int*>(&sm.visit[g % kVisitRing].x), *reinterpret_cast<volatile int*>(&sm.visit[g % kVisitRing].y),
                                       *reinterpret_cast<volatile int*>(&sm.visit[g % kVisitRing].z), 0);
          if (__any_sync(0xffffffffu, visit.x & kTail)) {
            // value rows that belong to no node may hold anything, and 0 * NaN is NaN
            int dep[kTileN / 32];                      // together: one latency instead of four
#pragma unroll
            for (int i = 0; i < kTileN / 32; ++i) {
              const int u = visit.z + i * 32 + lane;
              dep[i] = u < 0 ? 0 : u < p.nodes ? p.depth[static_cast<int64_t>(visit.y) * p.nodes + u] : -1;
            }
            uint32_t dead[kTileN / 32], any = 0u;
#pragma unroll
            for (int i = 0; i < kTileN / 32; ++i) any |= dead[i] = __ballot_sync(0xffffffffu, dep[i] < 0);
            if (any != 0u) {
              uint8_t* const base = sm.kv[pos.slot] + ((lane >> 3) & 1) * kHalfBytes + (lane & 7) * 16;      // 16 lanes a row, two rows at a time
#pragma unroll
              for (int i = 0; i < kTileN / 32; ++i)
#pragma unroll 1
                for (int r = lane >> 4; dead[i] >> r != 0u; r += 2) {
                  if ((dead[i] >> r) & 1u) *reinterpret_cast<uint4*>(base + (i * 32 + r) * 128) = make_uint4(0u, 0u, 0u, 0u);
                  if (r >= 30) break;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
          const uint64_t vd = v_desc + static_cast<uint64_t>((pos.slot * kTileBytes) >> 4);
          for (int i = 0; i < tiles; ++i) {
            const int t = two_tiles ? i : g & 1;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              mbar_wait(&sm.p_half[t][h], (parity >> t) & 1u, sm);
              tc_fence_after();
              if (leader) {
#pragma unroll
                for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
                  mma_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, vd + static_cast<uint64_t>((kk * 2048) >> 4), idesc,
                         (!(visit.x & kOFirst) || kk > 0) ? 1u : 0u);
              }
              __syncwarp();
            }
            parity ^= 1u << t;
            if (leader) mma_commit(&sm.pv_done[t]);
            __syncwarp();
          }
          if (leader) mma_commit(&sm.empty[pos.slot]);
          __syncwarp();
        }
      }
    }
  } else {
    // ===================================== softmax =====================================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsHigh));
    const int t = (warp - 4) >> 2, quad = warp & 3;
    const int r = quad * 32 + lane;
    const int node = (mb * 2 + (two_tiles ? t : 0)) * p.npt + r / p.rep;
    const bool row_used = r < p.npt * p.rep && node < p.nodes;
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t t_s = tmem + lane_base + t * 128;        // my row of scores; the bf16 P overlays its first 64 columns
    const uint32_t t_o = tmem + lane_base + 256 + t * 128;  // my row of the output accumulator
    const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2);
    float m_ref = -INFINITY, l_sum = 0.f;

    // The end of a segment.  Two states of one tile are joined, each warpgroup taking half of the columns (tensor memory is shared by
    // the warps of a row quarter).  A segment that is all of its (sample, key head) leaves the result, another one a partial: O / l in
    // fp32 (zero where the row saw nothing) and the LSE in the log2 domain.  A row has seen something when its sum is not 0: scores of
    // NaN leave the maximum at -inf, their sum is NaN, and so is then all that the row leaves.
    auto leave = [&](const Segment& s, bool leads, int d, bool any) {      // leads: the part's first segment
      float m = any && d >= 0 ? m_ref : -INFINITY, l = any && d >= 0 ? l_sum : 0.f, mine = 1.f, other = 0.f;
      if (!two_tiles) {
        sm.stats[t][r] = make_float2(m, l);
        tc_fence_before();
        asm volatile("bar.sync 2, 256;" ::: "memory");
        tc_fence_after();
        const float2 o = sm.stats[t ^ 1][r];
        const float top = fmaxf(m, o.x), ref = top == -INFINITY ? 0.f : top;
        mine = m == -INFINITY ? 0.f : fast_exp2(m - ref);
        other = o.x == -INFINITY ? 0.f : fast_exp2(o.x - ref);
        l = l * mine + o.y * other;
        m = top;
      }
      const bool seen = l != 0.f, whole = s.v0 == 0 && s.v1 == s.vis.n;
      const float inv = seen ? 1.f / l : 0.f;
      mine = seen ? mine * inv : 0.f;
      other *= inv;
      const int64_t prow = place_of(p, mb, t, 2 * worker + (leads ? 0 : 1)) * p.rpt;
      const int ch0 = two_tiles ? 0 : 2 * t, ch1 = two_tiles ? 4 : 2 * t + 2, h = s.kvh * p.rep + r % p.rep;
#pragma unroll 1
      for (int ch = ch0; ch < ch1; ++ch) {
        uint32_t o[32];
        JL_TMEM_LD32(t_o + ch * 32, o, 0);
        JL_TMEM_WAIT_LD32(o, 0);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = mine != 0.f ? __float_as_uint(__uint_as_float(o[i]) * mine) : 0u;      // (nothing: stale, perhaps NaN)
        if (!two_tiles) {
          uint32_t x[32];
          JL_TMEM_LD32(t_o + (1 - 2 * t) * 128 + ch * 32, x, 0);
          JL_TMEM_WAIT_LD32(x, 0);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = other != 0.f ? __float_as_uint(fmaf(__uint_as_float(x[i]), other, __uint_as_float(o[i]))) : o[i];
        }
        if (row_used && whole) {
          uint4* dst = reinterpret_cast<uint4*>(p.out + s.b * p.os_b + node * p.os_s + h * p.os_h + ch * 32);
          auto pk = [&](int i) { return pack_bf16x2(__uint_as_float(o[i]), __uint_as_float(o[i + 1])); };
#pragma unroll
          for (int i = 0; i < 4; ++i) dst[i] = make_uint4(pk(8 * i), pk(8 * i + 2), pk(8 * i + 4), pk(8 * i + 6));
        } else if (row_used) {               // [4 columns][row]: 32 rows of a warp are 512 contiguous bytes (a row at a time cost 7000 clocks)
          float4* dst = reinterpret_cast<float4*>(p.part_o + prow * kHeadDim) + r;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            dst[(ch * 8 + i) * p.rpt] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]),
                                                    __uint_as_float(o[4 * i + 3]));
        }
      }
      if (row_used && (two_tiles || t == 0)) {
        const float lse = seen ? m + log2f(l) : -INFINITY;
        if (!whole) p.part_lse[prow + r] = lse;
        else if (p.lse != nullptr) p.lse[(static_cast<int64_t>(s.b) * p.kv_heads * p.rep + h) * p.nodes + node] = lse * kLn2;
      }
      tc_fence_before();                               // the next segment's P V follows our next P
      if (!two_tiles) asm volatile("bar.sync 2, 256;" ::: "memory");      // and the other state's reading
    };

    Walk w(sm);
    Segment seg;
    int n_done = 0, g = 0;
    while (w.next(p, seg)) {
      const bool leads = g == 0;
      const int step = two_tiles ? 1 : 2, first = seg.v0 + (two_tiles ? 0 : (g ^ t) & 1);
      g += seg.v1 - seg.v0;
      const int64_t nrow = static_cast<int64_t>(seg.b) * p.nodes + (row_used ? node : 0);
      const int d = row_used && node < seg.vis.nodes ? p.depth[nrow] : -1;
      const int len = seg.vis.len;
      m_ref = -INFINITY;
      l_sum = 0.f;
      if (first >= seg.v1) {                           // this state has no visit in the segment
        leave(seg, leads, -1, false);
        continue;
      }
      for (int v = first; v < seg.v1; v += step, ++n_done) {
        const bool far = v < seg.vis.far;
        const int tp0 = seg.key_tile(v) * kTileN;
        // every key of the tile is committed and of this class for nodes of any depth
        bool uniform = tp0 + kTileN <= len;
        if (p.two_classes) uniform &= far ? tp0 + kTileN <= len - p.w_0 : tp0 >= len + p.nodes - 1 - p.w_0;
        // otherwise: committed keys of this class at columns [c_lo, c_hi), drafted keys by the bits of the node's mask and their depth
        int c_lo = 0, c_hi = 0;
        if (!uniform) {
          const int64_t edge = static_cast<int64_t>(len) + d - p.w_0;          // pk < edge: far
          const int64_t lo = (p.two_classes && !far ? edge : 0) - tp0, hi = (p.two_classes && far && edge < len ? edge : len) - tp0;
          c_lo = lo < 0 ? 0 : (lo > 128 ? 128 : static_cast<int>(lo));
          c_hi = d < 0 || hi < 0 ? 0 : (hi > 128 ? 128 : static_cast<int>(hi));
        }
        // the mask's bits of the tile's columns, fetched while the scores are formed: word i holds bits of columns 32 (i - 1) + shift ..
        const int u_tile = tp0 - len;                  // node of the tile's first column (negative: columns before the nodes)
        uint32_t words[kTileN / 32 + 1];
        bool with_nodes = false;
        if (!uniform) {
          with_nodes = d >= 0 && u_tile > -kTileN && u_tile < seg.vis.nodes && (!far || p.nodes_far);
#pragma unroll
          for (int i = 0; i <= kTileN / 32; ++i) {
            const int at = (u_tile >> 5) + i;
            words[i] = with_nodes && at >= 0 && at < 2 * p.words ? __ldg(reinterpret_cast<const uint32_t*>(p.mask + nrow * p.words) + at) : 0u;
          }
        }
        mbar_wait(&sm.s_full[t], n_done & 1, sm);
        tc_fence_after();
        auto raise_reference = [&](float mx) {
          // lazy rescale: only when some row of the warp outgrew its reference maximum by 2^8
          if (__any_sync(0xffffffffu, mx > m_ref + 8.f)) {
            const float m_new = fmaxf(m_ref, mx);
            const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_ref - m_new);
            l_sum *= alpha;
            if (v > first) {                           // O holds something of this segment
              // O is quiescent: these scores ready implies P V of the state's previous item retired, and the next one waits for our P
#pragma unroll 1
              for (int oc = 0; oc < 4; ++oc) {
                uint32_t o[32];
                JL_TMEM_LD32(t_o + oc * 32, o, 0);
                JL_TMEM_WAIT_LD32(o, 0);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                JL_TMEM_ST32(t_o + oc * 32, o, 0);
              }
            }
            m_ref = m_new;
          }
        };
        auto exp_block = [&](const uint32_t* s, uint64_t negm2, uint32_t col, uint64_t (&acc2)[4]) {      // 32 scores -> 16 packed pairs
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint64_t x = fma2(pack2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale2, negm2);
            const uint64_t pp = exp2_pair_sfu(x);      // (a quarter of them on the FMA pipe: 3 % slower here, and 1e-6 off in the LSE)
            acc2[i & 3] = add2(acc2[i & 3], pp);
            float p0, p1;
            unpack2(pp, p0, p1);
            pk[i] = pack_bf16x2(p0, p1);
          }
          JL_TMEM_ST16(t_s + col, pk, 0);
        };
        auto publish = [&](int half) {
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&sm.p_half[t][half]);
        };
        if (!uniform) {
          // what the row does not see in this class becomes -inf, in place
#pragma unroll 1
          for (int ch = 0; ch < 4; ++ch) {
            const int a = max(c_lo - ch * 32, 0), z = min(c_hi - ch * 32, 32);
            uint32_t keep = z > a ? (0xffffffffu >> (32 - (z - a))) << a : 0u;
            if (with_nodes) {
              const int u0 = u_tile + ch * 32;         // first node of these columns
              uint32_t bits = __funnelshift_r(words[0], words[1], u_tile & 31);
#pragma unroll
              for (int i = 0; i < kTileN / 32; ++i) words[i] = words[i + 1];
              const int left = seg.vis.nodes - u0;
              if (left < 32) bits = left > 0 ? bits & (0xffffffffu >> (32 - left)) : 0u;
              if (p.nodes_far) {
                for (uint32_t todo = bits; todo != 0u; todo &= todo - 1) {
                  const int j = __ffs(todo) - 1;
                  if ((d - p.depth[static_cast<int64_t>(seg.b) * p.nodes + u0 + j] > p.w_0) != far) bits &= ~(1u << j);
                }
              }
              keep |= bits;
            }
            uint32_t s[32];
            JL_TMEM_LD32(t_s + ch * 32, s, 0);
            JL_TMEM_WAIT_LD32(s, 0);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((keep >> i) & 1u)) s[i] = 0xff800000u;
            JL_TMEM_ST32(t_s + ch * 32, s, 0);
          }
          tmem_wait_st();
        }
        uint64_t acc2[4] = {0ull, 0ull, 0ull, 0ull};
        if (p.unrolled) {
          // all 128 scores in registers: half the loads, and P published 1300 clocks earlier than by the loop below
          uint32_t s[128];
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          JL_TMEM_LD32(t_s + 0, s, 0);
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) {
            JL_TMEM_WAIT_LD32(s, ch * 32);
            if (ch + 1 < 4) JL_TMEM_LD32(t_s + (ch + 1) * 32, s, (ch + 1) * 32);
#pragma unroll
            for (int i = 0; i < 16; ++i) m4[i & 3] = max3(m4[i & 3], __uint_as_float(s[ch * 32 + 2 * i]), __uint_as_float(s[ch * 32 + 2 * i + 1]));
          }
          raise_reference(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * p.scale_log2);
          const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
          const uint64_t negm2 = pack2(-m_use, -m_use);
          exp_block(s, negm2, 0, acc2);
          exp_block(s + 32, negm2, 16, acc2);
          publish(0);
          exp_block(s + 64, negm2, 32, acc2);
          exp_block(s + 96, negm2, 48, acc2);
          publish(1);
          float a0, a1;
          unpack2(add2(add2(acc2[0], acc2[1]), add2(acc2[2], acc2[3])), a0, a1);
          l_sum += a0 + a1;
          continue;
        }
        // Two passes over the row's scores, 32 columns at a time: maximum, then probabilities (written over scores that have
        // been read).  The loop is kept rolled on purpose: the stream of keys evicts the kernel's code from L2, so its first
        // pass runs at the rate of instruction fetches from HBM; unrolled over 128 columns that took 9 us of a 100 us launch.
        float mx = -INFINITY;
        uint64_t negm2 = 0ull;
#pragma unroll 1
        for (int step32 = 0; step32 < 8; ++step32) {
          const int ch = step32 & 3;
          uint32_t s[32];
          JL_TMEM_LD32(t_s + ch * 32, s, 0);
          JL_TMEM_WAIT_LD32(s, 0);
          if (step32 < 4) {
            float m2[2] = {mx, -INFINITY};
#pragma unroll
            for (int i = 0; i < 16; ++i) m2[i & 1] = max3(m2[i & 1], __uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
            mx = fmaxf(m2[0], m2[1]);
            if (step32 < 3) continue;
            mx *= p.scale_log2;
            raise_reference(mx);
            const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
            negm2 = pack2(-m_use, -m_use);
            continue;
          }
          exp_block(s, negm2, ch * 16, acc2);
          if (ch & 1) publish(ch >> 1);                // keys 0..63 are published with their own barrier, then keys 64..127
        }
        float a0, a1;
        unpack2(add2(add2(acc2[0], acc2[1]), add2(acc2[2], acc2[3])), a0, a1);
        l_sum += a0 + a1;
      }
      mbar_wait(&sm.pv_done[t], (n_done - 1) & 1, sm);
      tc_fence_after();
      leave(seg, leads, d, true);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*failed) {                                 // copies and MMAs that were under way have long landed after 1 ms
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000 * 1000) {}
  }
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
  if (threadIdx.x == 0 && sm.failed) atomicExch(&g_tree_status, 1);
}

// Joins the partials of the segments that cover a (sample, key head), where one segment did not have it all.  One thread per
// (row, 4 columns), rows fastest, so that partials are read as they were written.  grid x: blocks of 128 threads over a tile's
// 32 * rpt such items, y: row tile of the (sample, key head), z: (sample, key head).
__global__ void __launch_bounds__(128) tree_combine_kernel(const TreeParams p) {
  const int lane = threadIdx.x & 31;
  const int heads = p.kv_heads * p.rep, b = static_cast<int>(blockIdx.z) / p.kv_heads, kvh = static_cast<int>(blockIdx.z) % p.kv_heads;
  int64_t total = 0, before = 0;
  for (int i = lane; i < p.batch; i += 32) {
    const int n = visits_of(p, i).n;
    total += n;
    before += i < b ? n : 0;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, off);
    before += __shfl_xor_sync(0xffffffffu, before, off);
  }
  total *= p.kv_heads;
  const int n_b = visits_of(p, b).n;
  const int64_t lo = before * p.kv_heads + static_cast<int64_t>(kvh) * n_b, hi = lo + n_b - 1;     // first and last visit
  const int tile = blockIdx.y, mb = tile >> 1;
  const int64_t parts = parts_of(p, mb, total);
  // the part that holds visit x of the line: the largest i with i * total / parts <= x
  const int i0 = static_cast<int>(((lo + 1) * parts + total - 1) / total) - 1, i1 = static_cast<int>(((hi + 1) * parts + total - 1) / total) - 1;
  if (i0 == i1) {                                          // one segment had it all: the result is there
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) wait_prerequisites();      // this kernel ends after the one before it
    return;
  }
  const int n_parts = i1 - i0 + 1, stride = has_two(p, mb) ? 2 : 1;
  // in part i0 it is the first segment if it starts there, else the last; in every later part the first
  const int64_t first = place_of(p, mb, tile & 1, 2 * static_cast<int64_t>(i0));
  const int64_t skip = static_cast<int64_t>(i0) * total / parts < lo ? stride * p.rpt : 0;
  const int64_t lse_step = 2 * static_cast<int64_t>(stride) * p.rpt, o_step = lse_step * 32;
  wait_prerequisites();
  for (int item = blockIdx.x * 128 + threadIdx.x; item < 32 * p.rpt; item += gridDim.x * 128) {
    const int c = item / p.rpt, r = item - c * p.rpt;
    const int nd = tile * p.npt + r / p.rep, h = kvh * p.rep + r % p.rep;
    if (nd >= p.nodes) continue;
    const float* lse = p.part_lse + first * p.rpt + r;
    const float4* o = reinterpret_cast<const float4*>(p.part_o) + first * p.rpt * 32 + item;
    float m = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = 0; k0 < n_parts; k0 += 8) {              // 8 partials in flight; the running maximum moves once a round
      float l[8];
      float4 x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool in = k0 + j < n_parts;
        const int64_t late = k0 + j == 0 ? skip : 0;
        l[j] = in ? lse[(k0 + j) * lse_step + late] : -INFINITY;
        x[j] = in ? o[(k0 + j) * o_step + late * 32] : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float mn = m;
#pragma unroll
      for (int j = 0; j < 8; ++j) mn = fmaxf(mn, l[j]);
      const float ref = mn == -INFINITY ? 0.f : mn, f = fast_exp2(m - ref);
      m = mn;
      sum *= f; acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float w = fast_exp2(l[j] - ref);
        sum += w;
        acc.x = fmaf(w, x[j].x, acc.x); acc.y = fmaf(w, x[j].y, acc.y); acc.z = fmaf(w, x[j].z, acc.z); acc.w = fmaf(w, x[j].w, acc.w);
      }
    }
    const float inv = sum != 0.f ? 1.f / sum : 0.f;            // NaN where a partial is
    *reinterpret_cast<uint2*>(p.out + b * p.os_b + nd * p.os_s + h * p.os_h + 4 * c) =
        make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
    if (p.lse != nullptr && c == 0) p.lse[(static_cast<int64_t>(b) * heads + h) * p.nodes + nd] = sum != 0.f ? (m + log2f(sum)) * kLn2 : -INFINITY;
  }
}

struct Layout { int npt, rpt, pairs, workers, workers_one; size_t lse, total; };
Layout layout_of(int32_t nodes, int32_t heads, int32_t kv_heads) {
  Layout l{};
  const int rep = heads / kv_heads;
  l.npt = 128 / rep;
  const int tiles = (nodes + l.npt - 1) / l.npt;
  l.pairs = tiles / 2;
  l.rpt = (tiles > 1 ? l.npt : nodes) * rep;
  // SMs for pairs of row tiles and for the one that is left, by what a visit costs them, 36 : 17 (80 nodes over 131056 keys, three
  // tiles: 217 us, with 36 : 13 250, 36 : 22 228; 259 with the last tile paired with an empty one).  The ratio was varied at that size
  // alone; with it, 40 nodes x 8 heads over 74631 keys took 129 us instead of 160, 8 samples of 78 nodes 158 instead of 184.
  const bool odd = tiles % 2 != 0;
  l.workers = l.pairs == 0 ? 0 : odd ? kSms * 36 / (36 * l.pairs + 17) : kSms / l.pairs;
  if (l.pairs > 0 && l.workers < 1) l.workers = 1;
  l.workers_one = !odd ? 0 : kSms - l.pairs * l.workers < 1 ? 1 : kSms - l.pairs * l.workers;
  const size_t rows = static_cast<size_t>(l.pairs * l.workers * 2 + l.workers_one) * 2 * l.rpt;      // two places a part
  l.lse = rows * kHeadDim * sizeof(float);
  l.total = l.lse + rows * sizeof(float);
  return l;
}

// (B, S, Hx, 128) bf16 view -> 4-D map (d, h, s, b), box 64 x box_h x box_s x 1, 128-byte swizzle, zero fill past the end
int make_map4(CUtensorMap* m, const void* base, int batch, int seq, int heads, int64_t sb, int64_t ss, int64_t sh, int box_h, int box_s) {
  EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return fail(JL_ERR_LAUNCH, "jl_tree_attention: cuTensorMapEncodeTiled is not available from the driver");
  const int64_t dflt = 128;                      // size-1 dimensions may arrive with stride 0; the encoder wants positive multiples of 16 bytes
  const cuuint64_t dims[4] = {128, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(seq), static_cast<cuuint64_t>(batch)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>((heads > 1 && sh > 0 ? sh : dflt) * 2), static_cast<cuuint64_t>((seq > 1 && ss > 0 ? ss : dflt) * 2),
                                 static_cast<cuuint64_t>((batch > 1 && sb > 0 ? sb : dflt) * 2)};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_h), static_cast<cuuint32_t>(box_s), 1};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(JL_ERR_BAD_ARG, "jl_tree_attention: tensor map encoding failed (CUresult %d)", static_cast<int>(r));
  return JL_OK;
}

}  // namespace

size_t tree_attention_workspace_bytes(int32_t batch, int32_t nodes, int32_t heads, int32_t kv_heads, int32_t) {
  if (batch < 1 || nodes < 1 || kv_heads < 1 || heads < kv_heads || heads / kv_heads > 128) return 0;
  return layout_of(nodes, heads, kv_heads).total;
}

int launch_tree_attention(const jl_tree_attention_args* a, cudaStream_t stream) {
  const Layout l = layout_of(a->nodes, a->heads, a->kv_heads);
  if (a->workspace == nullptr || a->workspace_bytes < l.total)
    return fail(JL_ERR_WORKSPACE, "jl_tree_attention: workspace of %zu bytes needed, %zu given", l.total, a->workspace_bytes);
  if (reinterpret_cast<uintptr_t>(a->workspace) & 15) return fail(JL_ERR_BAD_ARG, "jl_tree_attention: workspace not 16-byte aligned");
  TreeParams p{};
  p.batch = a->batch; p.nodes = a->nodes; p.words = (a->nodes + 63) / 64; p.kv_heads = a->kv_heads; p.rep = a->heads / a->kv_heads; p.rows = a->rows;
  p.npt = l.npt; p.rpt = l.rpt; p.pairs = l.pairs; p.workers = l.workers; p.workers_one = l.workers_one;
  p.two_classes = a->q_group != nullptr;
  p.w_0 = a->w_0 < (int64_t(1) << 32) ? a->w_0 : (int64_t(1) << 32);           // no cache reaches further
  p.nodes_far = p.two_classes && p.w_0 < a->nodes - 1;
  // The unrolled softmax saves 1300 clocks a visit, and its instructions, cold, cost 8 us once: 16 nodes over 131072 keys 106.5 us
  // rolled and 102.8 unrolled, 64 nodes 171 and 142; the two are equal at 8 visits a part.  The choice goes by the rows that the
  // cache has, since its lengths are on the device: 4 nodes over 1037 keys in a cache of 131072 rows take 18.4 us, in one of 1044 16.4.
  p.unrolled = static_cast<int64_t>(a->batch) * a->kv_heads * (a->rows / kTileN) >= 16ll * (l.pairs > 0 ? l.workers : l.workers_one);
  p.scale_log2 = a->softmax_scale * kLog2e;
  p.lens = a->lens; p.depth = a->depth; p.mask = a->mask;
  p.part_o = static_cast<float*>(a->workspace);
  p.part_lse = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + l.lse);
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.lse = a->lse;
  p.os_b = a->o_stride_b; p.os_s = a->o_stride_s; p.os_h = a->o_stride_h;
  TreeMaps maps;
  int rc = bind_context();
  for (int c = 0; c < 2 && rc == JL_OK; ++c) {
    const bool far = c == 1 && p.two_classes;
    rc = make_map4(&maps.q[c], far ? a->q_group : a->q_base, a->batch, a->nodes, a->heads, a->q_stride_b, a->q_stride_s, a->q_stride_h, p.rep, p.npt);
    if (rc == JL_OK)
      rc = make_map4(&maps.k[c], far ? a->k_group : a->k_base, a->batch, a->rows, a->kv_heads, a->k_stride_b, a->k_stride_s, a->k_stride_h, 1, kTileN);
  }
  if (rc == JL_OK) rc = make_map4(&maps.v, a->v, a->batch, a->rows, a->kv_heads, a->v_stride_b, a->v_stride_s, a->v_stride_h, 1, kTileN);
  if (rc != JL_OK) return rc;
  constexpr int kSmemBytes = sizeof(TreeSmem);
  static_assert(kSmemBytes <= 227 * 1024, "shared memory");
  static bool attr_set[64] = {false};
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(JL_ERR_LAUNCH, "jl_tree_attention: no current CUDA device");
  if (!attr_set[dev]) {
    if (cudaFuncSetAttribute(tree_attention_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) != cudaSuccess)
      return check_launch("jl_tree_attention (shared memory opt-in)");
    attr_set[dev] = true;
  }
  const int row_tiles = (a->nodes + l.npt - 1) / l.npt;
  if (static_cast<int64_t>(a->batch) * a->kv_heads > 65535)
    return fail(JL_ERR_UNSUPPORTED, "jl_tree_attention: batch * kv_heads must be at most 65535");
  if (launch_dependent(tree_attention_kernel, dim3(p.pairs * p.workers + p.workers_one), dim3(kThreads), kSmemBytes, stream, maps, p) != cudaSuccess)
    return check_launch("jl_tree_attention");
  // enough blocks to fill the GPU, but no more: what most of them do for many samples is to see that nothing is left to do
  const int64_t pairs = static_cast<int64_t>(a->batch) * a->kv_heads * row_tiles;
  int64_t blocks = (int64_t(8) * kSms + pairs - 1) / pairs;
  if (blocks > (32 * l.rpt + 127) / 128) blocks = (32 * l.rpt + 127) / 128;
  if (launch_dependent(tree_combine_kernel, dim3(static_cast<unsigned>(blocks), row_tiles, a->batch * a->kv_heads), dim3(128), 0, stream, p) != cudaSuccess)
    return check_launch("jl_tree_attention (combine)");
  return JL_OK;
}

int tree_status() {
  int v = 0;
  if (cudaDeviceSynchronize() != cudaSuccess) return -1;      // the copy alone waits for the legacy stream and what blocks on it
  if (cudaMemcpyFromSymbol(&v, g_tree_status, sizeof(int)) != cudaSuccess) return -1;
  const int zero = 0;
  if (v != 0) cudaMemcpyToSymbol(g_tree_status, &zero, sizeof(int));
  return v;
}

}  // namespace jl
