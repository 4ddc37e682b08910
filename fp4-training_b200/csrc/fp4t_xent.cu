// Softmax cross entropy of a projection onto a large vocabulary, without keeping the logits:
//
//   x = h W^T (+ b)                      h [T, D], W [V, D] bf16, fp32 accumulation
//   lse_t = log sum_v exp(x_tv)          loss_t = lse_t - x_t,y(t)   (0 for ignored tokens)
//   dl = (exp(x - lse) - onehot) g_t     dh = dl W,  dW = dl^T h,  db = sum_t dl
//
// All products run on the 5th-generation tensor cores (tcgen05, bf16 operands, accumulators in tensor
// memory), one persistent kernel with four epilogues:
//   forward   the tile of logits never leaves tensor memory: each epilogue thread owns a row of it and
//             keeps a running maximum and sum of exponentials (fp32), two numbers per row and half tile
//             that a small kernel joins along the vocabulary;
//   backward  in pieces of the vocabulary: the logits of a piece are computed again, turned into dl in
//             the epilogue and written once, in bf16 (the operand type of the two products that read
//             it; a rounding of 2^-9 on average per term, as large as the one that dh and dW get at the end);
//             dh accumulates over the pieces in fp32, dW's rows of the piece are final.
// Recomputing costs 2 T V D operations on top of the 6 T V D that cannot be avoided, and saves the
// T x V logits (4 GB of fp32 at 8192 x 131072).
//
// The tile is 256 x 256 (or 256 x 128) on a pair of CTAs (cta_group::2): each CTA loads its 128 rows of
// the first operand and half of the second one, 64 elements of K per stage, with plain tiled TMA
// loads into 128-byte-swizzled shared memory.  Operands that run along the other dimension (W for dh, both
// for dW) are loaded as 64 x 64 boxes and read by the tensor core in their MN-major form, so nothing is
// transposed in memory.  Two accumulators fill tensor memory (2 x 256 columns): the epilogue of a tile
// (eight warps, two per lane quadrant) runs under the products of the next.
//
// Outputs of few tiles over a long K (dh of few tokens, dW of few classes) split K over the idle
// clusters into fp32 slices that a small kernel adds in a fixed order.  No atomics on results: every
// output is reproducible.  Every wait is bounded as in the block-scaled GEMM.
#include <algorithm>

#include "fp4t_common.cuh"
#include "fp4t_tcgen05.cuh"

namespace fp4t {
namespace {

enum { kStats = 0, kGrad = 1, kProduct = 2, kProductT = 3 };   // epilogue / operand forms

constexpr int kXM = 256, kXK = 64;               // rows and K elements of a tile
constexpr int kXEpiWarps = 8;
constexpr int kXThreads = 128 + 32 * kXEpiWarps; // producer, MMA issuer, tensor-memory owner, an idle warp, epilogue
constexpr int kXTmemCols = 512;
constexpr float kLog2e = 1.4426950408889634f;
// Logits are scaled by log2(e) in the multiply-add that subtracts the maximum.  A maximum (or lse) beyond
// this would overflow there -- a row masked with the type's lowest value, or infinite -- and is
// subtracted first instead.
constexpr float kFar = 2e38f;
constexpr int kXBadTarget = 41;                  // status: a target outside the vocabulary

constexpr int64_t kTokenBlock = 16384;           // tokens whose partial statistics are held at once
constexpr int64_t kPieceBytes = 512ll << 20;     // dl of one piece of the vocabulary, unless that makes
constexpr int64_t kMinPiece = 4096;              // the piece narrower than this

struct XParams {
  int rows, cols;                                // of the output
  int m_tiles, n_tiles, group_m, k_stages, splits, ks_per_split, slice_rows;
  // kStats, kGrad
  const void* bias;
  int bias_f32;
  const int64_t* target;
  int64_t ignore;
  int64_t col0;                                  // first vocabulary entry of the piece
  float2* part;                                  // kStats: [2 * n_tiles][rows] (maximum, sum)
  float* picked;                                 // kStats: the target's logit
  unsigned int* counter;                         // kStats: put to zero for the joining kernel
  const float* lse;
  const float* grad;
  int grad_per_row;
  const float* count;                            // kGrad, mean: number of counted tokens
  // kProduct, kProductT
  int out_f32;
  const float* acc;                              // added to the result (fp32, pitch ldacc)
  int64_t ldacc;
  int32_t* status;
};

template <int kBN>
struct XCfg {
  static constexpr int kBRows = kBN / 2;                         // rows of the second operand per CTA
  static constexpr int kABytes = 128 * kXK * 2, kBBytes = kBRows * kXK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kEpiBytes = kXEpiWarps * 4096;
  static constexpr int kBarBytes = 512;
  static constexpr int kBudget = 227 * 1024 - kEpiBytes - kBarBytes;
  static constexpr int kStages = kBudget / kStageBytes > 8 ? 8 : kBudget / kStageBytes;
  static constexpr int kEpi0 = kStages * kStageBytes, kBar0 = kEpi0 + kEpiBytes;
  static constexpr int kSmemBytes = kBar0 + kBarBytes;
  static constexpr int kHalf = kBN / 2;                          // columns of an epilogue warp
  static_assert(kSmemBytes <= 227 * 1024 && 2 * kBN <= kXTmemCols, "shared or tensor memory budget");
  static_assert((2 * kStages + 4) * 8 + 8 <= kBarBytes, "barrier block");
};

// Instruction descriptor of kind::f16: [4,6) D format (1 = f32), [7,10) / [10,13) A / B format (1 = bf16),
// 15 / 16 A / B major (1 = MN), [17,23) N >> 3, [24,29) M >> 4.
template <int kBN, bool kAMn, bool kBMn>
__device__ __forceinline__ constexpr uint32_t xent_idesc() {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((kAMn ? 1u : 0u) << 15) | ((kBMn ? 1u : 0u) << 16) |
         ((uint32_t)(kBN >> 3) << 17) | ((uint32_t)(kXM >> 4) << 24);
}
__device__ __forceinline__ void tc_mma_bf16_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Operand descriptors.  K-major: rows of 128 bytes (64 elements of K), 8-row groups 1024 bytes apart; a
// step of 16 in K is 32 bytes.  MN-major: rows of K, each 128 bytes (64 elements of M or N); 8-row
// groups 1024 bytes apart, the next 64 elements of M or N 64 rows (8192 bytes, the leading offset) further; a
// step of 16 in K is two 8-row groups.
constexpr uint32_t kMnLead = (8192u >> 4) << 16;
template <bool kMn>
__device__ __forceinline__ uint64_t xent_desc(uint32_t lo, int k16) {
  return kMn ? make_desc((lo + (uint32_t)k16 * (2048u >> 4)) | kMnLead, kDescHiOperand)
             : make_desc(lo + (uint32_t)k16 * (32u >> 4), kDescHiOperand);
}

struct TilePos {
  int m, n, split;
};
// Tiles go down a group of group_m tile rows before the next column: the first operand's rows of the
// group stay in L2 while the second operand streams past once per group.
__device__ __forceinline__ TilePos tile_at(const XParams& g, int unit) {
  TilePos t;
  const int tile = unit / g.splits;
  t.split = unit - tile * g.splits;
  const int span = g.group_m * g.n_tiles;
  const int grp = tile / span, rem = tile - grp * span;
  const int rows = min(g.group_m, g.m_tiles - grp * g.group_m);
  t.n = rem / rows;
  t.m = grp * g.group_m + rem - t.n * rows;
  return t;
}

// bias of the 32 columns from c on (columns behind the last read as zero)
__device__ __forceinline__ void add_bias(const XParams& g, int c, float (&v)[32]) {
  if (g.bias == nullptr) return;
  if (c + 32 <= g.cols) {
    if (g.bias_f32) {
      const float4* b = reinterpret_cast<const float4*>(static_cast<const float*>(g.bias) + c);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 f = __ldg(b + j);
        v[4 * j] += f.x; v[4 * j + 1] += f.y; v[4 * j + 2] += f.z; v[4 * j + 3] += f.w;
      }
    } else {
      const uint4* b = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(g.bias) + c);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 u = __ldg(b + j);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[8 * j + 2 * i] += __uint_as_float(w[i] << 16);
          v[8 * j + 2 * i + 1] += __uint_as_float(w[i] & 0xFFFF0000u);
        }
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (c + j < g.cols) v[j] += g.bias_f32 ? __ldg(static_cast<const float*>(g.bias) + c + j) : __bfloat162float(static_cast<const __nv_bfloat16*>(g.bias)[c + j]);
  }
}

// One 32 x 32 chunk (a row per lane) to a swizzled staging tile and from there with one tiled TMA
// store, clipped at the matrix edges.  bf16: two 2-KB tiles that alternate; fp32: one of 4 KB.
__device__ __forceinline__ void store_chunk_bf16(const CUtensorMap* map, uint8_t* buf, uint32_t& n_emit, int lane, int row, int col,
                                                 const float (&v)[32]) {
  uint8_t* tile = buf + (n_emit & 1u) * 2048;
  if (lane == 0) bulk_wait_read<1>();
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t w[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[8 * j + 2 * t], v[8 * j + 2 * t + 1]);
      w[t] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(tile + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  fence_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(map, smem_u32(tile), col, row);
    bulk_commit();
  }
  ++n_emit;
}
__device__ __forceinline__ void store_chunk_f32(const CUtensorMap* map, uint8_t* buf, int lane, int row, int col, const float (&v)[32]) {
  if (lane == 0) bulk_wait_read<0>();
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *reinterpret_cast<float4*>(buf + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  fence_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(map, smem_u32(buf), col, row);
    bulk_commit();
  }
}

template <int kMode, int kBN>
__global__ void __launch_bounds__(kXThreads, 1)
xent_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const __grid_constant__ CUtensorMap map_d, const XParams g) {
  using C = XCfg<kBN>;
  constexpr bool kAMn = kMode == kProductT, kBMn = kMode == kProduct || kMode == kProductT;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t smem_base = smem_u32(smem);
  pdl_launch_dependents();
  if (smem_base & 1023u) {   // the swizzled tiles need the alignment the declaration asks for
    pdl_wait();
    if (threadIdx.x == 0 && g.status) atomicCAS(g.status, 0, 29);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBar0);
  const uint32_t bar_full = smem_u32(bars);                   // [kStages] both CTAs' tiles landed (the leader's copy is used)
  const uint32_t bar_empty = bar_full + 8 * C::kStages;       // [kStages] the products that read the stage are done (own copy)
  const uint32_t bar_tmem_full = bar_empty + 8 * C::kStages;  // [2] accumulator complete (own copy)
  const uint32_t bar_tmem_empty = bar_tmem_full + 16;         // [2] accumulator drained (the leader's copy)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * C::kStages + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int cluster_id = blockIdx.x >> 1, num_clusters = gridDim.x >> 1;

  if (threadIdx.x == 32) {
    tma_prefetch_map(&map_a);
    tma_prefetch_map(&map_b);
    if (kMode != kStats) tma_prefetch_map(&map_d);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(bar_tmem_full + 8 * a, 1);
      mbar_init(bar_tmem_empty + 8 * a, 2 * kXEpiWarps);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)kXTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();          // barriers of both CTAs are initialised before any remote arrive
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();                  // from here on memory that the predecessor wrote is touched

  const int units = g.m_tiles * g.n_tiles * g.splits;
  const uint32_t leader_full = mapa_u32(bar_full, 0);
  const uint32_t leader_tmem_empty = mapa_u32(bar_tmem_empty, 0);

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------ producer (each CTA) ------------------------------
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int unit = cluster_id; ok && unit < units; unit += num_clusters) {
        const TilePos t = tile_at(g, unit);
        const int ks0 = t.split * g.ks_per_split, ks1 = min(ks0 + g.ks_per_split, g.k_stages);
        const int row_a = t.m * kXM + (int)rank * 128, row_b = t.n * kBN + (int)rank * C::kBRows;
        for (int ks = ks0; ks < ks1; ++ks) {
          if (!mbar_wait(bar_empty + 8 * stage, phase ^ 1u, abort_flag, g.status, 21)) { ok = false; break; }
          const uint32_t a_s = smem_base + stage * C::kStageBytes, b_s = a_s + C::kABytes;
          const uint32_t bar = leader_full + 8 * stage;
          if (leader) mbar_expect_tx(bar_full + 8 * stage, 2u * C::kStageBytes);
          if (kAMn) {
            tma_load_2d_pair(a_s, &map_a, bar, row_a, ks * kXK);
            tma_load_2d_pair(a_s + 8192, &map_a, bar, row_a + 64, ks * kXK);
          } else {
            tma_load_2d_pair(a_s, &map_a, bar, ks * kXK, row_a);
          }
          if (kBMn) {
#pragma unroll
            for (int o = 0; o < C::kBRows / 64; ++o) tma_load_2d_pair(b_s + o * 8192, &map_b, bar, row_b + o * 64, ks * kXK);
          } else {
            tma_load_2d_pair(b_s, &map_b, bar, ks * kXK, row_b);
          }
          if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
        }
      }
      if (*abort_flag) {   // let copies in flight land before shared memory is given back
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) {}
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (leader) {
      // ------------------------------ MMA issuer (leader CTA, whole warp) ------------------------------
      const uint32_t elected = elect_one();
      constexpr uint32_t idesc = xent_idesc<kBN, kAMn, kBMn>();
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      int it = 0;
      for (int unit = cluster_id; ok && unit < units; unit += num_clusters, ++it) {
        const int split = unit % g.splits;
        const int ks0 = split * g.ks_per_split, ks1 = min(ks0 + g.ks_per_split, g.k_stages);
        const int a = it & 1;
        ok = mbar_wait(bar_tmem_empty + 8 * a, ((it >> 1) & 1) ^ 1u, abort_flag, g.status, 22);
        if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
        tc_fence_after();
        const uint32_t acc = tmem_base + (uint32_t)(a * kBN);
        for (int ks = ks0; ks < ks1; ++ks) {
          ok = mbar_wait(bar_full + 8 * stage, phase, abort_flag, g.status, 23);
          if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
          tc_fence_after();
          if (elected) {
            const uint32_t a_lo = ((smem_base + stage * C::kStageBytes) & 0x3FFFFu) >> 4;
            const uint32_t b_lo = a_lo + (C::kABytes >> 4);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              tc_mma_bf16_pair(acc, xent_desc<kAMn>(a_lo, j), xent_desc<kBMn>(b_lo, j), idesc, (ks > ks0 || j > 0) ? 1u : 0u);
            tc_commit_all<2>(bar_empty + 8 * stage);   // frees the stage in both CTAs
          }
          __syncwarp();
          if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
        }
        if (ok) {
          if (elected) tc_commit_all<2>(bar_tmem_full + 8 * a);
          __syncwarp();
        }
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------ epilogue (each CTA) ------------------------------
    const int quad = warp & 3, half = (warp - 4) >> 2;
    uint8_t* buf = smem + C::kEpi0 + (warp - 4) * 4096;
    uint32_t n_emit = 0;
    float scale = 0.f;
    if (kMode == kStats && blockIdx.x == 0 && threadIdx.x == 128) *g.counter = 0u;
    if (kMode == kGrad && !g.grad_per_row) scale = g.count != nullptr ? __ldg(g.grad) / __ldg(g.count) : __ldg(g.grad);
    int it = 0;
    for (int unit = cluster_id; unit < units; unit += num_clusters, ++it) {
      const TilePos t = tile_at(g, unit);
      const int a = it & 1;
      int ok = 1;
      if (lane == 0) ok = mbar_wait(bar_tmem_full + 8 * a, (uint32_t)((it >> 1) & 1), abort_flag, g.status, 24) ? 1 : 0;
      ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(a * kBN + half * C::kHalf);
      const int row0 = t.m * kXM + (int)rank * 128 + quad * 32, row = row0 + lane;
      const bool row_ok = row < g.rows;
      const int colbase = t.n * kBN + half * C::kHalf;
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(leader_tmem_empty + 8 * a);
      };
      if (kMode == kStats || kMode == kGrad) {
        const int64_t y = row_ok ? __ldg(reinterpret_cast<const long long*>(g.target) + row) : g.ignore;
        const bool counted = y != g.ignore;
        // the target's column in this warp's part of the tile; anything outside [0, cols) never matches
        const int64_t yc = y - g.col0;
        const int mine = counted && yc >= colbase && yc < colbase + C::kHalf && yc < g.cols ? (int)yc - colbase : -1;
        float m = -INFINITY, s = 0.f, x_y = 0.f;
        float lse = 0.f, gr = 0.f;
        if (kMode == kGrad) {
          lse = row_ok ? __ldg(g.lse + row) : 0.f;
          gr = g.grad_per_row ? (row_ok ? __ldg(g.grad + row) : 0.f) : scale;
        }
#pragma unroll 1
        for (int c = 0; c < C::kHalf / 32; ++c) {
          uint32_t r[32];
          tc_ld32(acc + (uint32_t)(c * 32), r);
          tc_wait_ld();
          if (c == C::kHalf / 32 - 1) release();
          const int col = colbase + c * 32;
          if (col >= g.cols || row0 >= g.rows) continue;      // warp-uniform
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
          add_bias(g, col, v);
          if (kMode == kStats) {
            if (col + 32 > g.cols) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (col + j >= g.cols) v[j] = -INFINITY;
            }
            if (__any_sync(0xFFFFFFFFu, (mine >> 5) == c)) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (mine == c * 32 + j) x_y = v[j];
            }
            float top = v[0];
#pragma unroll
            for (int j = 1; j < 32; ++j) top = fmaxf(top, v[j]);
            const float mn = fmaxf(m, top);
            if (fabsf(mn) < kFar) {              // by row: its result does not depend on its neighbours
              const float ref = mn * kLog2e;
              float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                s0 += exp2_fast(fmaf(v[j], kLog2e, -ref));
                s1 += exp2_fast(fmaf(v[j + 1], kLog2e, -ref));
                s2 += exp2_fast(fmaf(v[j + 2], kLog2e, -ref));
                s3 += exp2_fast(fmaf(v[j + 3], kLog2e, -ref));
              }
              s = fmaf(s, exp2_fast(fmaf(m, kLog2e, -ref)), (s0 + s1) + (s2 + s3));
            } else {
              const float ref = mn == -INFINITY ? 0.f : mn;           // a row of -inf so far: all terms are 0
              float s0 = 0.f;
#pragma unroll
              for (int j = 0; j < 32; ++j) s0 += exp2_fast((v[j] - ref) * kLog2e);
              s = fmaf(s, exp2_fast((m - ref) * kLog2e), s0);
            }
            m = mn;
          } else {
            if (fabsf(lse) < kFar) {
              const float lse2 = lse * kLog2e;
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = exp2_fast(fmaf(v[j], kLog2e, -lse2));
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = exp2_fast((v[j] - lse) * kLog2e);
            }
            if (__any_sync(0xFFFFFFFFu, (mine >> 5) == c)) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (mine == c * 32 + j) v[j] -= 1.f;
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = counted ? v[j] * gr : 0.f;
            store_chunk_bf16(&map_d, buf, n_emit, lane, row0, col, v);
          }
        }
        if (kMode == kStats && row_ok) {
          g.part[(int64_t)(2 * t.n + half) * g.rows + row] = make_float2(m, s);
          if (mine >= 0) g.picked[row] = x_y;
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < C::kHalf / 32; ++c) {
          uint32_t r[32];
          tc_ld32(acc + (uint32_t)(c * 32), r);
          tc_wait_ld();
          if (c == C::kHalf / 32 - 1) release();
          const int col = colbase + c * 32;
          if (col >= g.cols || row0 >= g.rows) continue;
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
          if (g.acc != nullptr && row_ok) {                    // columns are a multiple of 8: whole vectors
            const float4* p = reinterpret_cast<const float4*>(g.acc + (int64_t)row * g.ldacc + col);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (col + 4 * j < g.cols) {
                const float4 f = p[j];
                v[4 * j] += f.x; v[4 * j + 1] += f.y; v[4 * j + 2] += f.z; v[4 * j + 3] += f.w;
              }
            }
          }
          const int srow = row0 + t.split * g.slice_rows;
          if (g.out_f32) store_chunk_f32(&map_d, buf, lane, srow, col, v);
          else store_chunk_bf16(&map_d, buf, n_emit, lane, srow, col, v);
        }
      }
    }
    if (lane == 0) bulk_wait_all<0>();
    __syncwarp();
  }

  // ------------------------------ teardown ------------------------------
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();          // the other CTA no longer signals into this one's shared memory
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)kXTmemCols) : "memory");
  }
}

// Joins the partial statistics of a row along the vocabulary: `lanes` rows a block (a power of two, at
// most 8), 256 / lanes threads a row, so that a single token's partials are read by a whole block.  The last
// block to finish adds the blocks' sums in block order (fp64) and writes the mean or sum.
constexpr int kJoinThreads = 256;
struct JoinParams {
  const float2* part;
  int parts;
  const float* picked;
  const int64_t* target;
  int64_t ignore, vocab;
  int rows, lanes;                 // rows of this token block
  float* lse;
  float* row_loss;                 // losses token by token, or null
  float* out;                      // their mean or sum, or null
  int mean;
  float* count;                    // number of counted tokens
  double* block_loss;              // [blocks of all token blocks]
  int* block_count;
  int first_block, all_blocks;
  unsigned int* counter;
  int32_t* status;
};
__global__ void __launch_bounds__(kJoinThreads) xent_join_kernel(const JoinParams p) {
  __shared__ float2 red[kJoinThreads];
  __shared__ double sum_s[kJoinThreads];
  __shared__ int cnt_s[kJoinThreads];
  __shared__ bool last;
  pdl_launch_dependents();
  pdl_wait();
  const int slices = kJoinThreads / p.lanes;
  const int r = threadIdx.x & (p.lanes - 1), slice = threadIdx.x / p.lanes;
  const int64_t row = (int64_t)blockIdx.x * p.lanes + r;
  float m = -INFINITY, s = 0.f;
  if (row < p.rows) {
#pragma unroll 4
    for (int i = slice; i < p.parts; i += slices) {
      const float2 q = p.part[(int64_t)i * p.rows + row];
      const float mn = fmaxf(m, q.x), ref = mn == -INFINITY ? 0.f : mn;
      s = s * exp2_fast((m - ref) * kLog2e) + q.y * exp2_fast((q.x - ref) * kLog2e);
      m = mn;
    }
  }
  red[threadIdx.x] = make_float2(m, s);
  __syncthreads();
  for (int o = slices >> 1; o > 0; o >>= 1) {
    if (slice < o) {
      const float2 a = red[threadIdx.x], b = red[threadIdx.x + o * p.lanes];
      const float mn = fmaxf(a.x, b.x), ref = mn == -INFINITY ? 0.f : mn;
      red[threadIdx.x] = make_float2(mn, a.y * exp2_fast((a.x - ref) * kLog2e) + b.y * exp2_fast((b.x - ref) * kLog2e));
    }
    __syncthreads();
  }
  double sum = 0.0;
  int cnt = 0;
  if (slice == 0 && row < p.rows) {
    const float2 q = red[threadIdx.x];
    const float lse = q.x + logf(q.y);
    p.lse[row] = lse;
    const int64_t y = p.target[row];
    float loss = 0.f;
    if (y != p.ignore) {
      cnt = 1;
      if (y >= 0 && y < p.vocab) {
        loss = lse - p.picked[row];
      } else {
        loss = NAN;
        if (p.status) atomicCAS(p.status, 0, kXBadTarget);
      }
    }
    if (p.row_loss) p.row_loss[row] = loss;
    sum = loss;
  }
  if (threadIdx.x < p.lanes) {
    sum_s[threadIdx.x] = sum;
    cnt_s[threadIdx.x] = cnt;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    cnt = 0;
    for (int i = 0; i < p.lanes; ++i) {
      sum += sum_s[i];
      cnt += cnt_s[i];
    }
    p.block_loss[p.first_block + blockIdx.x] = sum;
    p.block_count[p.first_block + blockIdx.x] = cnt;
    __threadfence();
    last = atomicAdd(p.counter, 1u) == (unsigned int)p.all_blocks - 1u;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  sum = 0.0;
  cnt = 0;
  for (int i = threadIdx.x; i < p.all_blocks; i += kJoinThreads) {
    sum += __ldcg(p.block_loss + i);
    cnt += __ldcg(p.block_count + i);
  }
  sum_s[threadIdx.x] = sum;
  cnt_s[threadIdx.x] = cnt;
  __syncthreads();
  for (int o = kJoinThreads >> 1; o > 0; o >>= 1) {
    if (threadIdx.x < o) {
      sum_s[threadIdx.x] += sum_s[threadIdx.x + o];
      cnt_s[threadIdx.x] += cnt_s[threadIdx.x + o];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    *p.count = (float)cnt_s[0];
    if (p.out) *p.out = (float)(p.mean ? sum_s[0] / (double)cnt_s[0] : sum_s[0]);   // no token counted: 0 / 0
  }
}

// out[r, c] = sum over the slices (+ acc[r, c]), four columns a thread, slices in order.
__global__ void __launch_bounds__(256) xent_slices_kernel(const float* __restrict__ slices, int n, int64_t slice_elems, const float* acc,
                                                          void* out, int out_f32, int64_t total4) {
  pdl_launch_dependents();
  pdl_wait();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total4; i += (int64_t)gridDim.x * 256) {
    float4 v = acc ? reinterpret_cast<const float4*>(acc)[i] : make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < n; ++s) {
      const float4 f = reinterpret_cast<const float4*>(slices + s * slice_elems)[i];
      v.x += f.x; v.y += f.y; v.z += f.z; v.w += f.w;
    }
    if (out_f32) {
      static_cast<float4*>(out)[i] = v;
    } else {
      const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
      static_cast<uint2*>(out)[i] = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
  }
}

// Column sums of dl: a block per 64 columns, 32 warps over the rows, their sums added in warp order.
__global__ void __launch_bounds__(1024) xent_bias_grad_kernel(const __nv_bfloat16* __restrict__ dl, int64_t ld, int rows, int cols, void* db,
                                                              int db_f32) {
  __shared__ float red[32][64];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 64 + 2 * lane;
  float a = 0.f, b = 0.f;
  if (c < cols) {                      // the pitch is even: the second element of the last pair may be padding, and is not used
#pragma unroll 8
    for (int r = warp; r < rows; r += 32) {
      const uint32_t u = __ldg(reinterpret_cast<const uint32_t*>(dl + (int64_t)r * ld + c));
      a += __uint_as_float(u << 16);
      b += __uint_as_float(u & 0xFFFF0000u);
    }
  }
  red[warp][2 * lane] = a;
  red[warp][2 * lane + 1] = b;
  __syncthreads();
  if (threadIdx.x < 64 && blockIdx.x * 64 + threadIdx.x < cols) {
    float s = 0.f;
    for (int w = 0; w < 32; ++w) s += red[w][threadIdx.x];
    const int at = blockIdx.x * 64 + threadIdx.x;
    if (db_f32) static_cast<float*>(db)[at] = s;
    else static_cast<__nv_bfloat16*>(db)[at] = __float2bfloat16_rn(s);
  }
}

// ------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------
template <int kMode, int kBN>
int xent_clusters() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (cached[dev] == 0) {
    auto kern = xent_gemm_kernel<kMode, kBN>;
    int n = -1;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, XCfg<kBN>::kSmemBytes) == cudaSuccess) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(2 * 148, 1, 1);
      cfg.blockDim = dim3(kXThreads, 1, 1);
      cfg.dynamicSmemBytes = XCfg<kBN>::kSmemBytes;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = 2;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) n = -1;
    }
    cudaGetLastError();
    cached[dev] = n;
  }
  return cached[dev];
}

// Clusters that the persistent kernel may fill: one CTA pair per two SMs, less under an SM limit.
int cluster_budget() {
  const int sms = sm_count();
  return sms > 0 ? std::max(1, sms / 2) : -1;
}

// How a product [m, n] over k is cut: tile width, and K splits when its tiles leave most clusters idle.
struct Cut {
  int bn = 256, splits = 1, ks_per_split = 0;
  int64_t slice_rows = 0;
  int64_t slice_bytes(int64_t n) const { return splits > 1 ? splits * slice_rows * n * 4 : 0; }
};
Cut cut_product(int64_t m, int64_t n, int64_t k, bool may_split, int clusters) {
  Cut c;
  const int64_t mt = ceil_div(m, kXM), stages = ceil_div(k, kXK);
  c.bn = n <= 128 ? 128 : 256;
  const int64_t tiles = mt * ceil_div(n, c.bn);
  c.ks_per_split = (int)stages;
  if (may_split && tiles * 2 <= clusters && stages >= 4) {
    int64_t s = std::min<int64_t>(clusters / tiles, stages / 2);
    if (s >= 2) {
      c.ks_per_split = (int)ceil_div(stages, s);
      c.splits = (int)ceil_div(stages, c.ks_per_split);
    }
  }
  c.slice_rows = mt * kXM;
  return c;
}

struct Operand {
  const void* p;
  int64_t outer, inner, ld;          // rows, contiguous elements, pitch in elements
};
int bf16_map(CUtensorMap* map, const Operand& o, int box_inner, int box_outer, CUtensorMapSwizzle sw) {
  return encode_tensor_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, o.p, (uint64_t)o.inner, (uint64_t)o.outer, (uint64_t)o.ld * 2,
                              (uint32_t)box_inner, (uint32_t)box_outer, sw);
}

template <int kMode, int kBN>
int launch_width(const Operand& a, const Operand& b, void* out, int64_t ldo, XParams g, int64_t k, cudaStream_t stream) {
  using C = XCfg<kBN>;
  constexpr bool kAMn = kMode == kProductT, kBMn = kMode == kProduct || kMode == kProductT;
  const int resident = xent_clusters<kMode, kBN>();
  int clusters = cluster_budget();
  if (resident <= 0 || clusters <= 0) {
    set_error("linear cross entropy: the kernel cannot be resident on this device");
    return FP4T_ERR_DEVICE;
  }
  clusters = std::min(clusters, resident);
  g.m_tiles = (int)ceil_div(g.rows, kXM);
  g.n_tiles = (int)ceil_div(g.cols, kBN);
  g.k_stages = (int)ceil_div(k, kXK);
  if (g.splits <= 1) {
    g.splits = 1;
    g.ks_per_split = g.k_stages;
  }
  // the first operand's rows of a group: 32 MB, a quarter of L2
  g.group_m = (int)std::min<int64_t>(g.m_tiles, std::max<int64_t>(1, (32ll << 20) / ((int64_t)kXM * 2 * std::max<int64_t>(k, 1))));
  CUtensorMap map_a, map_b, map_d = {};
  int rc = kAMn ? bf16_map(&map_a, a, 64, kXK, CU_TENSOR_MAP_SWIZZLE_128B) : bf16_map(&map_a, a, kXK, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == FP4T_OK)
    rc = kBMn ? bf16_map(&map_b, b, 64, kXK, CU_TENSOR_MAP_SWIZZLE_128B) : bf16_map(&map_b, b, kXK, C::kBRows, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == FP4T_OK && kMode != kStats) {
    const uint64_t rows = g.splits > 1 ? (uint64_t)g.splits * g.slice_rows : (uint64_t)g.rows;
    rc = encode_tensor_map_2d(&map_d, g.out_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, out, (uint64_t)g.cols, rows,
                              (uint64_t)ldo * (g.out_f32 ? 4 : 2), 32u, 32u, g.out_f32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
  }
  if (rc != FP4T_OK) return rc;
  const int64_t units = (int64_t)g.m_tiles * g.n_tiles * g.splits;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(units, clusters)), 1, 1);
  cfg.blockDim = dim3(kXThreads, 1, 1);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  pdl_attribute(&attr[1]);
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  FP4T_CUDA(cudaLaunchKernelEx(&cfg, xent_gemm_kernel<kMode, kBN>, map_a, map_b, map_d, g));
  return FP4T_OK;
}
template <int kMode>
int launch_xent(int bn, const Operand& a, const Operand& b, void* out, int64_t ldo, const XParams& g, int64_t k, cudaStream_t stream) {
  return bn == 128 ? launch_width<kMode, 128>(a, b, out, ldo, g, k, stream) : launch_width<kMode, 256>(a, b, out, ldo, g, k, stream);
}

template <typename... Args, typename... Actual>
int launch_small(void (*kern)(Args...), int grid, int threads, cudaStream_t stream, Actual... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  pdl_attribute(&attr);
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  FP4T_CUDA(cudaLaunchKernelEx(&cfg, kern, args...));
  return FP4T_OK;
}

// One product into `out` (contiguous rows of `cols`), through slices when it is split.
template <int kMode>
int run_product(const Cut& cut, const Operand& a, const Operand& b, int64_t k, int64_t rows, int64_t cols, void* out, int out_f32,
                const float* acc, float* slices, int32_t* status, cudaStream_t stream) {
  XParams g = {};
  g.rows = (int)rows;
  g.cols = (int)cols;
  g.status = status;
  g.out_f32 = out_f32;
  g.splits = cut.splits;
  g.ks_per_split = cut.ks_per_split;
  if (cut.splits == 1) {
    g.acc = acc;
    g.ldacc = cols;
    return launch_xent<kMode>(cut.bn, a, b, out, cols, g, k, stream);
  }
  g.slice_rows = (int)cut.slice_rows;
  g.out_f32 = 1;
  int rc = launch_xent<kMode>(cut.bn, a, b, slices, cols, g, k, stream);
  if (rc != FP4T_OK) return rc;
  const int64_t total4 = rows * cols / 4;
  const int grid = (int)std::min<int64_t>(ceil_div(total4, 256), 148 * 8);
  return launch_small(xent_slices_kernel, grid, 256, stream, (const float*)slices, cut.splits, cut.slice_rows * cols, acc, out, out_f32, total4);
}

int64_t round_up(int64_t v, int64_t to) { return ceil_div(v, to) * to; }

int width_for(int64_t vocab) { return vocab <= 128 ? 128 : 256; }   // of a tile of logits

// Forward workspace: counter, block sums and counts, the targets' logits, partial statistics.
struct ForwardPlan {
  int64_t block, parts, join_blocks;      // tokens per block, partials per token, joining blocks of all token blocks
  int lanes;
  int64_t o_loss, o_count, o_picked, o_part, bytes;
};
ForwardPlan plan_forward(int64_t tokens, int64_t vocab) {
  ForwardPlan p;
  p.block = std::min(tokens, kTokenBlock);
  p.parts = 2 * ceil_div(vocab, width_for(vocab));
  p.lanes = 1;
  while (p.lanes < 8 && p.lanes < tokens) p.lanes <<= 1;
  p.join_blocks = (tokens / p.block) * ceil_div(p.block, p.lanes) + ceil_div(tokens % p.block, p.lanes);
  p.o_loss = 128;
  p.o_count = p.o_loss + round_up(p.join_blocks * 8, 128);
  p.o_picked = p.o_count + round_up(p.join_blocks * 4, 128);
  p.o_part = p.o_picked + round_up(p.block * 4, 128);
  p.bytes = p.o_part + p.parts * p.block * 8;
  return p;
}

// Backward workspace: dl of a piece, dh in fp32 when there are several pieces, K slices.
struct BackwardPlan {
  int64_t piece, pieces, ld;
  Cut dh, dw;
  int64_t o_acc, o_slices, bytes;
};
BackwardPlan plan_backward(int64_t tokens, int64_t dim, int64_t vocab, bool want_dh, bool want_dw, int clusters) {
  BackwardPlan p;
  p.piece = std::min(round_up(vocab, 256), std::max(kMinPiece, kPieceBytes / (2 * tokens) / 256 * 256));
  p.pieces = ceil_div(vocab, p.piece);
  p.piece = round_up(ceil_div(vocab, p.pieces), 256);       // even pieces
  p.pieces = ceil_div(vocab, p.piece);
  p.ld = std::min(p.piece, round_up(vocab, 8));
  p.dh = cut_product(tokens, dim, std::min(p.piece, vocab), true, clusters);
  p.dw = cut_product(std::min(p.piece, vocab), dim, tokens, true, clusters);
  p.o_acc = round_up(tokens * p.ld * 2, 1024);
  p.o_slices = p.o_acc + (want_dh && p.pieces > 1 ? round_up(tokens * dim * 4, 1024) : 0);
  p.bytes = p.o_slices + std::max(want_dh ? p.dh.slice_bytes(dim) : 0, want_dw ? p.dw.slice_bytes(dim) : 0);
  return p;
}

int check_sizes(const char* name, int64_t tokens, int64_t dim, int64_t vocab) {
  FP4T_REQUIRE(tokens >= 0 && tokens <= (1 << 26) && vocab >= 1 && vocab <= (1 << 26) && dim >= 8 && dim <= (1 << 20),
               "%s: bad shape tokens=%lld dim=%lld vocab=%lld", name, (long long)tokens, (long long)dim, (long long)vocab);
  FP4T_REQUIRE(dim % 8 == 0, "%s: dim (%lld) must be a multiple of 8", name, (long long)dim);
  FP4T_REQUIRE(ceil_div(tokens, kXM) * ceil_div(vocab, 128) < (1ll << 30), "%s: too many tiles", name);
  return FP4T_OK;
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check_inputs(const char* name, const void* h, int64_t ldh, const void* w, int64_t ldw, const void* bias, int bias_dtype, const void* target,
                 int64_t dim, int reduction, const void* workspace) {
  FP4T_REQUIRE(h && w && target && workspace, "%s: null pointer", name);
  FP4T_REQUIRE(ldh >= dim && ldw >= dim && ldh % 8 == 0 && ldw % 8 == 0, "%s: row pitches must be multiples of 8, at least dim", name);
  FP4T_REQUIRE(aligned16(h) && aligned16(w) && aligned16(bias) && aligned16(workspace), "%s: pointers must be 16-byte aligned", name);
  FP4T_REQUIRE(reinterpret_cast<uintptr_t>(target) % 8 == 0, "%s: misaligned target", name);
  FP4T_REQUIRE(!bias || bias_dtype == FP4T_DT_F32 || bias_dtype == FP4T_DT_BF16, "%s: the bias must be f32 or bf16", name);
  FP4T_REQUIRE(reduction == FP4T_XENT_NONE || reduction == FP4T_XENT_MEAN || reduction == FP4T_XENT_SUM, "%s: bad reduction", name);
  return FP4T_OK;
}

}  // namespace

FP4T_DEFINE_WAIT_TIMEOUT_SETTER(set_wait_timeout_xent)

}  // namespace fp4t

using namespace fp4t;

extern "C" int64_t fp4t_linear_xent_forward_workspace_bytes(int64_t tokens, int64_t vocab) {
  if (check_sizes("fp4t_linear_xent_forward_workspace_bytes", tokens, 8, vocab) != FP4T_OK) return -1;
  return tokens == 0 ? 128 : plan_forward(tokens, vocab).bytes;
}

extern "C" int fp4t_linear_xent_forward(const void* h, int64_t ldh, const void* w, int64_t ldw, const void* bias, int bias_dtype,
                                        const int64_t* target, int64_t tokens, int64_t dim, int64_t vocab, int64_t ignore_index,
                                        int reduction, float* loss, float* lse, float* count, void* workspace, int64_t workspace_bytes,
                                        int32_t* status, fp4t_stream_t stream) {
  const char* name = "fp4t_linear_xent_forward";
  int rc = check_sizes(name, tokens, dim, vocab);
  if (rc != FP4T_OK) return rc;
  FP4T_REQUIRE(tokens > 0, "%s: no tokens", name);
  rc = check_inputs(name, h, ldh, w, ldw, bias, bias_dtype, target, dim, reduction, workspace);
  if (rc != FP4T_OK) return rc;
  FP4T_REQUIRE(loss && lse && count, "%s: null pointer", name);
  const ForwardPlan p = plan_forward(tokens, vocab);
  FP4T_REQUIRE(workspace_bytes >= p.bytes, "%s: the workspace holds %lld bytes of %lld", name, (long long)workspace_bytes, (long long)p.bytes);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (!status) status = current_status_word();
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  int64_t first_block = 0;
  for (int64_t t0 = 0; t0 < tokens; t0 += p.block) {
    const int64_t rows = std::min(p.block, tokens - t0);
    XParams g = {};
    g.rows = (int)rows;
    g.cols = (int)vocab;
    g.bias = bias;
    g.bias_f32 = bias_dtype == FP4T_DT_F32;
    g.target = target + t0;
    g.ignore = ignore_index;
    g.part = reinterpret_cast<float2*>(ws + p.o_part);
    g.picked = reinterpret_cast<float*>(ws + p.o_picked);
    g.counter = reinterpret_cast<unsigned int*>(ws + (t0 == 0 ? 0 : 64));      // counts over all token blocks: zeroed by the first
    g.status = status;
    rc = launch_xent<kStats>(width_for(vocab), Operand{static_cast<const __nv_bfloat16*>(h) + t0 * ldh, rows, dim, ldh}, Operand{w, vocab, dim, ldw},
                             nullptr, 0, g, dim, s);
    if (rc != FP4T_OK) return rc;
    JoinParams j = {};
    j.part = g.part;
    j.parts = (int)p.parts;
    j.picked = g.picked;
    j.target = g.target;
    j.ignore = ignore_index;
    j.vocab = vocab;
    j.rows = (int)rows;
    j.lanes = p.lanes;
    j.lse = lse + t0;
    j.row_loss = reduction == FP4T_XENT_NONE ? loss + t0 : nullptr;
    j.out = reduction == FP4T_XENT_NONE ? nullptr : loss;
    j.mean = reduction == FP4T_XENT_MEAN;
    j.count = count;
    j.block_loss = reinterpret_cast<double*>(ws + p.o_loss);
    j.block_count = reinterpret_cast<int*>(ws + p.o_count);
    j.first_block = (int)first_block;
    j.all_blocks = (int)p.join_blocks;
    j.counter = reinterpret_cast<unsigned int*>(ws);
    j.status = status;
    const int blocks = (int)ceil_div(rows, p.lanes);
    first_block += blocks;
    rc = launch_small(xent_join_kernel, blocks, kJoinThreads, s, j);
    if (rc != FP4T_OK) return rc;
  }
  return FP4T_OK;
}

extern "C" int64_t fp4t_linear_xent_backward_workspace_bytes(int64_t tokens, int64_t dim, int64_t vocab, int want_dh, int want_dw) {
  if (check_sizes("fp4t_linear_xent_backward_workspace_bytes", tokens, dim, vocab) != FP4T_OK) return -1;
  const int clusters = cluster_budget();
  if (tokens == 0 || clusters <= 0) return tokens == 0 ? 128 : -1;
  return plan_backward(tokens, dim, vocab, want_dh != 0, want_dw != 0, clusters).bytes;
}

extern "C" int fp4t_linear_xent_backward(const float* grad_loss, const void* h, int64_t ldh, const void* w, int64_t ldw, const void* bias,
                                         int bias_dtype, const int64_t* target, const float* lse, const float* count, int64_t tokens,
                                         int64_t dim, int64_t vocab, int64_t ignore_index, int reduction, void* dh, int dh_dtype, void* dw,
                                         int dw_dtype, void* db, int db_dtype, void* workspace, int64_t workspace_bytes, int32_t* status,
                                         fp4t_stream_t stream) {
  const char* name = "fp4t_linear_xent_backward";
  int rc = check_sizes(name, tokens, dim, vocab);
  if (rc != FP4T_OK) return rc;
  FP4T_REQUIRE(tokens > 0, "%s: no tokens", name);
  rc = check_inputs(name, h, ldh, w, ldw, bias, bias_dtype, target, dim, reduction, workspace);
  if (rc != FP4T_OK) return rc;
  FP4T_REQUIRE(grad_loss && lse && count, "%s: null pointer", name);
  FP4T_REQUIRE((!dh || dh_dtype == FP4T_DT_F32 || dh_dtype == FP4T_DT_BF16) && (!dw || dw_dtype == FP4T_DT_F32 || dw_dtype == FP4T_DT_BF16) &&
                   (!db || db_dtype == FP4T_DT_F32 || db_dtype == FP4T_DT_BF16),
               "%s: gradients must be f32 or bf16", name);
  FP4T_REQUIRE(aligned16(dh) && aligned16(dw) && aligned16(db), "%s: pointers must be 16-byte aligned", name);
  if (!dh && !dw && !db) return FP4T_OK;
  const int clusters = cluster_budget();
  if (clusters <= 0) {
    set_error("%s: the current device is not an sm_100 part", name);
    return FP4T_ERR_DEVICE;
  }
  const BackwardPlan p = plan_backward(tokens, dim, vocab, dh != nullptr, dw != nullptr, clusters);
  FP4T_REQUIRE(workspace_bytes >= p.bytes, "%s: the workspace holds %lld bytes of %lld", name, (long long)workspace_bytes, (long long)p.bytes);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (!status) status = current_status_word();
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  __nv_bfloat16* dl = reinterpret_cast<__nv_bfloat16*>(ws);
  float* acc = reinterpret_cast<float*>(ws + p.o_acc);
  float* slices = reinterpret_cast<float*>(ws + p.o_slices);
  for (int64_t i = 0; i < p.pieces; ++i) {
    const int64_t v0 = i * p.piece, vc = std::min(p.piece, vocab - v0);
    const Operand hop{h, tokens, dim, ldh}, wop{static_cast<const __nv_bfloat16*>(w) + v0 * ldw, vc, dim, ldw}, dop{dl, tokens, vc, p.ld};
    XParams g = {};
    g.rows = (int)tokens;
    g.cols = (int)vc;
    g.bias = bias ? static_cast<const uint8_t*>(bias) + v0 * (bias_dtype == FP4T_DT_F32 ? 4 : 2) : nullptr;
    g.bias_f32 = bias_dtype == FP4T_DT_F32;
    g.target = target;
    g.ignore = ignore_index;
    g.col0 = v0;
    g.lse = lse;
    g.grad = grad_loss;
    g.grad_per_row = reduction == FP4T_XENT_NONE;
    g.count = reduction == FP4T_XENT_MEAN ? count : nullptr;
    g.status = status;
    rc = launch_xent<kGrad>(width_for(vc), hop, wop, dl, p.ld, g, dim, s);
    if (rc != FP4T_OK) return rc;
    if (dh) {
      const bool last = i == p.pieces - 1;
      Cut cut = p.dh;
      if (vc != std::min(p.piece, vocab)) {            // a shorter last piece: the same slices, fewer of them
        const int64_t stages = ceil_div(vc, kXK);
        cut.ks_per_split = (int)std::min<int64_t>(cut.ks_per_split, stages);
        cut.splits = (int)std::min<int64_t>(cut.splits, ceil_div(stages, cut.ks_per_split));
      }
      rc = run_product<kProduct>(cut, dop, wop, vc, tokens, dim, last ? dh : static_cast<void*>(acc), last ? dh_dtype == FP4T_DT_F32 : 1,
                                 i > 0 ? acc : nullptr, slices, status, s);
      if (rc != FP4T_OK) return rc;
    }
    if (dw) {
      void* out = static_cast<uint8_t*>(dw) + v0 * dim * (dw_dtype == FP4T_DT_F32 ? 4 : 2);
      rc = run_product<kProductT>(p.dw, dop, hop, tokens, vc, dim, out, dw_dtype == FP4T_DT_F32, nullptr, slices, status, s);
      if (rc != FP4T_OK) return rc;
    }
    if (db) {
      void* out = static_cast<uint8_t*>(db) + v0 * (db_dtype == FP4T_DT_F32 ? 4 : 2);
      rc = launch_small(xent_bias_grad_kernel, (int)ceil_div(vc, 64), 1024, s, (const __nv_bfloat16*)dl, p.ld, (int)tokens, (int)vc, out,
                        (int)(db_dtype == FP4T_DT_F32));
      if (rc != FP4T_OK) return rc;
    }
  }
  return FP4T_OK;
}
