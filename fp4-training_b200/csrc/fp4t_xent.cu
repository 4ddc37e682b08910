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
//             it); dh accumulates over the pieces in fp32, dW's rows of the piece are final.
//             That rounding is off by half a step, 2^-8, per term at most, as the one that dh and dW get at the
//             end, and at many tokens as independent.  A scalar g_t is kept out of it (it scales the products'
//             epilogues): rounded into every term it would be one error in all of them.  Up to 64 tokens, where a
//             few roundings do not average out, dl is kept as a sum of two bf16, rows 64 to 127 holding
//             what rows 0 to 63 lost; the tiles are 256 rows high and wait for W, so this costs no time.
// Recomputing costs 2 T V D operations on top of the 6 T V D that cannot be avoided, and saves the
// T x V logits (4 GB of fp32 at 8192 x 131072).
//
// The tile is 256 x 256 (or 256 x 128) on a pair of CTAs (cta_group::2): each CTA loads its 128 rows of
// the first operand and half of the second one, 64 elements of K per stage, with plain tiled TMA
// loads into 128-byte-swizzled shared memory.  Operands that run along the other dimension (W for dh, both
// for dW) are loaded as 64 x 64 boxes and read by the tensor core in their MN-major form, so nothing is
// transposed in memory.  Two accumulators fill tensor memory (2 x 256 columns): the epilogue of a tile
// (eight warps, two per lane quadrant) runs under the products of the next.  Measured (B200, nominal 2.25
// PFLOP/s, cuBLAS 1.38 sustained): 8192 x 4096 x 131072 forward 6.5 ms, 1.36 PFLOP/s, backward 20.1 ms (26.4 TFLOP, 1.31);
// bound by the power limit.  An epilogue takes 5000 cycles a tile forward and 8000 backward (the exponentials and
// the chain of a chunk's steps), so widths below about 600 and 1000 are bound by it instead of the products.
//
// Outputs of few tiles over a long K (dh of few tokens, dW of few classes) split K over the idle
// clusters into fp32 slices that a small kernel adds in a fixed order.  No atomics on results: every
// output is reproducible.  Every wait is bounded as in the block-scaled GEMM.
#include <algorithm>

#include "fp4t_common.cuh"
#include "fp4t_pack.cuh"
#include "fp4t_tcgen05.cuh"

namespace fp4t {
namespace {

enum { kStats = 0, kGrad = 1, kProduct = 2, kProductT = 3 };   // epilogue / operand forms

constexpr int kXM = 256, kXK = 64;               // rows and K elements of a tile
constexpr int kXEpiWarps = 8;
constexpr int kXThreads = 128 + 32 * kXEpiWarps; // producer, MMA issuer, tensor-memory owner, an idle warp, epilogue
constexpr int kXTmemCols = 512;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Logits are scaled by log2(e) in the multiply-add that subtracts the maximum.  A maximum (or lse) beyond
// this would overflow there -- a row masked with the type's lowest value, or infinite -- and is
// subtracted first instead.
constexpr float kFar = 2e38f;
constexpr int kXBadTarget = 60;                  // status: a target outside the vocabulary

constexpr int kFew = 64;                         // tokens up to which dl is kept in two bf16 (one K stage)
constexpr int64_t kTokenBlock = 16384;           // tokens whose partial statistics are held at once
constexpr int64_t kPieceBytes = 512ll << 20;     // dl of one piece of the vocabulary, unless that makes
constexpr int64_t kMinPiece = 4096;              // the piece narrower than this

// Counted tokens are numbered in order ("slots"); everything between the operands and the gradients has
// slots for rows.  Their number is known on the device only.
struct XParams {
  int rows, cols;                                // of the output; rows: the most there can be
  int m_tiles, n_tiles, group_m, k_stages, splits, ks_per_split, slice_rows;
  const int* slots;                              // number of counted tokens
  int tokens;                                    // all tokens: slots == tokens means that h can be read as it is
  int slot0;                                     // kStats: first slot of the block
  int few;                                       // backward, at most kFew tokens: dl has 2 kFew rows, h is packed twice
  int split_clusters;                            // kProduct: clusters that K may be split over (0: it may not)
  // kStats, kGrad
  const void* bias;
  int bias_f32;
  const int* target;                             // of the slots; -1: outside the vocabulary
  int col0;                                      // first vocabulary entry of the piece
  float2* part;                                  // kStats: [2 * n_tiles][rows] (maximum, sum)
  float* picked;                                 // kStats: the target's logit
  const float* lse;
  const float* grad;
  int grad_per_row;
  int mean;                                      // divide by the number of counted tokens
  const int* token;                              // slot -> token (grad_per_row, and kProduct's rows)
  float* col_part;                               // kGrad: column sums of dl over 32 slots, [slots / 32][col_ld], or null
  int64_t col_ld;
  // where the tile goes: kGrad dl, else the result or (splits) fp32 slices
  void* dst;
  int64_t ldd;                                   // pitch in elements
  int out_f32;
  int to_tokens;                                 // kProduct: the result's rows are tokens, not slots
  float* slices;                                 // kProduct: in place of dst when it splits K itself (pitch: cols)
  const float* acc;                              // added to the result (fp32, pitch ldacc)
  int64_t ldacc;
  int32_t* status;
};

// kStats stores nothing through shared memory and gets a seventh stage instead.
template <int kMode, int kBN>
struct XCfg {
  static constexpr int kBRows = kBN / 2;                         // rows of the second operand per CTA
  static constexpr int kABytes = 128 * kXK * 2, kBBytes = kBRows * kXK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kEpiWarpBytes = kMode == kStats ? 0 : 4096;   // one 32 x 32 chunk
  static constexpr int kEpiBytes = kXEpiWarps * kEpiWarpBytes;
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

// kProduct's K splits follow the number of slots too: over the clusters that its tiles leave idle, if those
// are at least half, into pieces of kMinSplitStages or more (fewer stages take less than the kernel that
// adds the slices).  splits * m_tiles * n_tiles <= clusters, which bounds the slices.
constexpr int kMinSplitStages = 8;
struct SlotSplit {
  int splits, ks_per_split;
};
__host__ __device__ __forceinline__ SlotSplit split_slots(int m_tiles, int n_tiles, int k_stages, int clusters) {
  const int tiles = m_tiles * n_tiles;
  SlotSplit r{1, k_stages};
  if (tiles > 0 && (int64_t)m_tiles * n_tiles * 2 <= clusters) {
    const int s = min(clusters / tiles, k_stages / kMinSplitStages);
    if (s >= 2) {
      r.ks_per_split = (k_stages + s - 1) / s;
      r.splits = (k_stages + r.ks_per_split - 1) / r.ks_per_split;
    }
  }
  return r;
}

// A cluster's tiles.  They go down a group of group_m tile rows before the next column: the first operand's rows
// of the group stay in L2 while the second operand streams past once per group.  The next tile is found by
// adding (the divisions of finding it afresh took 400 cycles of every epilogue warp and tile); a
// product that is split has about one unit per cluster, and divides.
struct TileWalk {
  int m, n, split;
  int unit, step;
  int grp, in_grp, rows;           // group, tile row in it, tile rows of it
  int dn, dm;                      // a step in columns and rows of a whole group

  __device__ __forceinline__ void start(const XParams& g, int first, int stride) {
    unit = first;
    step = stride;
    const int tile = unit / g.splits;
    split = unit - tile * g.splits;
    const int span = g.group_m * g.n_tiles;
    grp = tile / span;
    locate(g, tile - grp * span);
  }
  __device__ __forceinline__ void locate(const XParams& g, int rem) {
    rows = max(1, min(g.group_m, g.m_tiles - grp * g.group_m));
    n = rem / rows;
    in_grp = rem - n * rows;
    m = grp * g.group_m + in_grp;
    dn = step / rows;
    dm = step - dn * rows;
  }
  __device__ __forceinline__ void advance(const XParams& g) {
    if (g.splits > 1) {
      start(g, unit + step, step);
      return;
    }
    unit += step;
    in_grp += dm;
    n += dn;
    if (in_grp >= rows) {
      in_grp -= rows;
      ++n;
    }
    if (n >= g.n_tiles) {          // into a later group
      int rem = n * rows + in_grp;
      do {
        rem -= rows * g.n_tiles;
        ++grp;
        rows = max(1, min(g.group_m, g.m_tiles - grp * g.group_m));
      } while (rem >= rows * g.n_tiles && grp * g.group_m < g.m_tiles);
      locate(g, rem);
    } else {
      m = grp * g.group_m + in_grp;
    }
  }
};

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

// Sums over the warp's 32 rows of 32 columns, column j's in lane j: in each step a lane hands half of its
// columns to the lane across and adds what it gets for the other half, 31 shuffles in all.
__device__ __forceinline__ float column_sums(const float (&v)[32], int lane) {
  float w[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) w[j] = v[j];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool upper = (lane & o) != 0;
#pragma unroll
    for (int j = 0; j < o; ++j) {
      const float give = upper ? w[j] : w[j + o], keep = upper ? w[j + o] : w[j];
      w[j] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, o);
    }
  }
  return w[0];
}

// One 32 x 32 chunk (a row per lane) through the warp's staging tile to whole 64- or 128-byte pieces of
// rows.  Plain stores: handing the tile to the copy engine (proxy fence, TMA store, wait for the tile) was no
// faster on many tokens and 6 % slower on few (16 tokens, 131072 x 4096: backward 926 against 870 us).  Columns end at a multiple of 8 (of dl at its pitch).  `token`: rows of the result by slot, or null.
struct Dest {
  uint8_t* p;
  int64_t pitch;                   // bytes
  int row_end, col_end;
  const int* token;
};
template <bool kF32>
__device__ __forceinline__ void store_chunk(const Dest& d, uint8_t* tile, int lane, int row0, int col, const float (&v)[32]) {
  constexpr int kPiece = kF32 ? 8 : 4;            // 16-byte pieces of a row of the chunk
  __syncwarp();                                   // the chunk before has been read
#pragma unroll
  for (int j = 0; j < kPiece; ++j) {
    uint4 q;
    if (kF32) {
      q = make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[8 * j + 2 * t], v[8 * j + 2 * t + 1]);
        w[t] = *reinterpret_cast<const uint32_t*>(&h);
      }
      q = make_uint4(w[0], w[1], w[2], w[3]);
    }
    const int at = kF32 ? j ^ (lane & 7) : j ^ ((lane >> 1) & 3);        // conflict-free both ways
    *reinterpret_cast<uint4*>(tile + lane * (kPiece * 16) + (at << 4)) = q;
  }
  __syncwarp();
  const int piece = lane & (kPiece - 1);
  const int c = col + piece * (kF32 ? 4 : 8);
  uint8_t* base = d.p + (int64_t)c * (kF32 ? 4 : 2);
#pragma unroll
  for (int i = 0; i < kPiece; ++i) {
    const int r = i * (32 / kPiece) + lane / kPiece, row = row0 + r;
    const int at = kF32 ? piece ^ (r & 7) : piece ^ ((r >> 1) & 3);
    const uint4 q = *reinterpret_cast<const uint4*>(tile + r * (kPiece * 16) + (at << 4));
    if (row < d.row_end && c < d.col_end) {
      const int to = d.token != nullptr ? __ldcg(d.token + row) : row;
      *reinterpret_cast<uint4*>(base + (int64_t)to * d.pitch) = q;
    }
  }
}

// The wait for a tcgen05.ld that was issued before other work: its registers pass through, so that nothing
// reads them earlier.
__device__ __forceinline__ void tc_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                 "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                 "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// v <- v log2(e) - ref, two at a time
__device__ __forceinline__ void scale_to_log2(float (&v)[32], float ref) {
  const Pack<2> l = Pack<2>::all(kLog2e), m = Pack<2>::all(-ref);
#pragma unroll
  for (int j = 0; j < 32; j += 2) fma(Pack<2>::of(v + j), l, m).to(v + j);
}

template <int kMode, int kBN>
__global__ void __launch_bounds__(kXThreads, 1)
xent_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const __grid_constant__ CUtensorMap map_packed, const XParams gp) {
  using C = XCfg<kMode, kBN>;
  XParams g = gp;
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
    if (kMode != kProduct) tma_prefetch_map(&map_packed);
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

  // The work follows the number of counted tokens: rows of the output, or the length of K.
  const int slots = *static_cast<const volatile int*>(g.slots);
  const bool dense = slots == g.tokens && !g.few;
  const int dl_rows = g.few ? 2 * kFew : slots;
  if (kMode == kProductT) {
    g.k_stages = (dl_rows + kXK - 1) / kXK;
    g.ks_per_split = (g.k_stages + g.splits - 1) / g.splits;
  } else {
    g.rows = max(0, min(g.rows, dl_rows - g.slot0));
    g.m_tiles = (g.rows + kXM - 1) / kXM;
    if (kMode == kProduct && g.split_clusters > 0) {
      const SlotSplit sp = split_slots(g.m_tiles, g.n_tiles, g.k_stages, g.split_clusters);
      g.splits = sp.splits;
      g.ks_per_split = sp.ks_per_split;
      g.slice_rows = g.m_tiles * kXM;
    }
  }
  const bool sliced = kMode == kProduct && (g.splits > 1 || g.few);   // fp32 slices, summed by another kernel
  const CUtensorMap* tma_a = (kMode == kStats || kMode == kGrad) && !dense ? &map_packed : &map_a;
  const CUtensorMap* tma_b = kMode == kProductT && !dense ? &map_packed : &map_b;
  const int units = g.m_tiles * g.n_tiles * g.splits;
  const uint32_t leader_full = mapa_u32(bar_full, 0);
  const uint32_t leader_tmem_empty = mapa_u32(bar_tmem_empty, 0);

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------ producer (each CTA) ------------------------------
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      TileWalk t;
      for (t.start(g, cluster_id, num_clusters); ok && t.unit < units; t.advance(g)) {
        const int ks0 = t.split * g.ks_per_split, ks1 = min(ks0 + g.ks_per_split, g.k_stages);
        const int row_a = t.m * kXM + (int)rank * 128, row_b = t.n * kBN + (int)rank * C::kBRows;
        for (int ks = ks0; ks < ks1; ++ks) {
          if (!mbar_wait(bar_empty + 8 * stage, phase ^ 1u, abort_flag, g.status, 21)) { ok = false; break; }
          const uint32_t a_s = smem_base + stage * C::kStageBytes, b_s = a_s + C::kABytes;
          const uint32_t bar = leader_full + 8 * stage;
          if (leader) mbar_expect_tx(bar_full + 8 * stage, 2u * C::kStageBytes);
          if (kAMn) {
            tma_load_2d_pair(a_s, tma_a, bar, row_a, ks * kXK);
            tma_load_2d_pair(a_s + 8192, tma_a, bar, row_a + 64, ks * kXK);
          } else {
            tma_load_2d_pair(a_s, tma_a, bar, ks * kXK, row_a);
          }
          if (kBMn) {
#pragma unroll
            for (int o = 0; o < C::kBRows / 64; ++o) tma_load_2d_pair(b_s + o * 8192, tma_b, bar, row_b + o * 64, ks * kXK);
          } else {
            tma_load_2d_pair(b_s, tma_b, bar, ks * kXK, row_b);
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
        const int split = g.splits > 1 ? unit % g.splits : 0;
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
    uint8_t* buf = smem + C::kEpi0 + (warp - 4) * C::kEpiWarpBytes;
    // a scalar gradient of the loss scales the products (and db), one per token is part of dl
    float scale = 1.f;
    if (kMode != kStats && !g.grad_per_row) scale = g.mean ? (slots > 0 ? __ldcg(g.grad) / (float)slots : 0.f) : __ldcg(g.grad);
    int it = 0;
    TileWalk t;
    t.start(g, cluster_id, num_clusters);
    // What a row brings to its tile (target, lse, gradient) is loaded a tile ahead.  Through L2: the kernel may
    // have been resident before its predecessor wrote them, which the read-only path must not see.
    int row0 = 0, slot = 0, y = -1;
    bool row_ok = false;
    float lse = 0.f, gr = 1.f;
    const auto look = [&]() {
      row0 = t.m * kXM + (int)rank * 128 + quad * 32;
      const int row = row0 + lane;
      slot = kMode == kGrad && g.few ? row & (kFew - 1) : row;
      row_ok = t.unit < units && row < g.rows && (kMode != kGrad || slot < slots);
      if (kMode == kStats || kMode == kGrad) {
        y = row_ok ? __ldcg(g.target + slot) : -1;
        if (kMode == kGrad) {
          lse = row_ok ? __ldcg(g.lse + slot) : 0.f;
          if (g.grad_per_row) gr = row_ok ? __ldcg(g.grad + __ldcg(g.token + slot)) : 0.f;
        }
      }
    };
    look();
    for (; t.unit < units; ++it) {
      const int a = it & 1;
      const int my_row0 = row0, row = row0 + lane, n_tile = t.n, split = t.split, my_y = y;
      const bool my_ok = row_ok;
      const float my_lse = lse, my_gr = gr;
      t.advance(g);
      look();
      const bool ok = mbar_wait(bar_tmem_full + 8 * a, (uint32_t)((it >> 1) & 1), abort_flag, g.status, 24);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      tc_fence_after();
      const uint32_t acc = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(a * kBN + half * C::kHalf);
      const int colbase = n_tile * kBN + half * C::kHalf;
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(leader_tmem_empty + 8 * a);
      };
      if (kMode == kStats || kMode == kGrad) {
        // the target's column in this warp's part of the tile; anything outside [0, cols) never matches
        const int yc = my_ok ? my_y - g.col0 : -1;
        const int mine = yc >= colbase && yc < colbase + C::kHalf && yc < g.cols ? yc - colbase : -1;
        // dl's rows up to the end of the last K stage that reads them are written (as zeros)
        const int row_end = kMode == kGrad ? (g.rows + kXK - 1) / kXK * kXK : g.rows;
        float m = -INFINITY, s = 0.f, x_y = 0.f;
        const bool all_ok = __all_sync(0xFFFFFFFFu, my_ok);
        const Dest dest{static_cast<uint8_t*>(g.dst), g.ldd * 2, min(row_end, gp.rows), (g.cols + 7) / 8 * 8, nullptr};
        constexpr int kN = C::kHalf / 32;
        uint32_t r[2][32];
        tc_ld32(acc, r[0]);
#pragma unroll
        for (int c = 0; c < kN; ++c) {
          tc_wait_ld(r[c & 1]);
          if (c + 1 < kN) tc_ld32(acc + (uint32_t)((c + 1) * 32), r[(c + 1) & 1]);    // under this chunk's work
          else release();
          const int col = colbase + c * 32;
          if (col >= g.cols || my_row0 >= row_end) continue;     // warp-uniform
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[c & 1][j]);
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
            float top[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) top[j] = fmaxf(fmaxf(v[j], v[j + 8]), fmaxf(v[j + 16], v[j + 24]));
            const float mn = fmaxf(fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]))),
                                   fmaxf(fmaxf(top[4], top[5]), fmaxf(top[6], top[7])));
            if (fabsf(mn) < kFar) {              // by row: its result does not depend on its neighbours
              const float ref = mn * kLog2e;
              scale_to_log2(v, ref);
              Pack<2> sum[4];
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                const float e[2] = {exp2_fast(v[j]), exp2_fast(v[j + 1])};
                sum[(j >> 1) & 3] = j < 8 ? Pack<2>::of(e) : add(sum[(j >> 1) & 3], Pack<2>::of(e));
              }
              // ref is mn log2(e) rounded, the same error in all terms: the residual takes it out of their sum
              s = fmaf(s, exp2_fast((m - mn) * kLog2e),
                       add(add(sum[0], sum[1]), add(sum[2], sum[3])).sum() * fmaf(fmaf(mn, kLog2e, -ref), -kLn2, 1.f));
            } else {
              const float ref = mn == -INFINITY ? 0.f : mn;           // a row of -inf so far: all terms are 0
              float s0 = 0.f;
#pragma unroll
              for (int j = 0; j < 32; ++j) s0 += exp2_fast((v[j] - ref) * kLog2e);
              s = fmaf(s, exp2_fast((m - ref) * kLog2e), s0);
            }
            m = mn;
          } else {
            if (fabsf(my_lse) < kFar) {
              scale_to_log2(v, my_lse * kLog2e);
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = exp2_fast(v[j]);
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = exp2_fast((v[j] - my_lse) * kLog2e);
            }
            if (__any_sync(0xFFFFFFFFu, (mine >> 5) == c)) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (mine == c * 32 + j) v[j] -= 1.f;
            }
            if (g.grad_per_row) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] *= my_gr;
            }
            if (!all_ok) {                                    // rows without a token: zeros, whatever the tile holds there
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = my_ok ? v[j] : 0.f;
            }
            if (g.col_part != nullptr && (!g.few || my_row0 < kFew)) {
              const float sum = column_sums(v, lane) * scale;
              if (col + lane < g.cols) g.col_part[(int64_t)(my_row0 >> 5) * g.col_ld + col + lane] = sum;
            }
            if (g.few && my_row0 >= kFew) {                      // what the rows' first bf16 lose
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] -= __bfloat162float(__float2bfloat16_rn(v[j]));
            }
            store_chunk<false>(dest, buf, lane, my_row0, col, v);
          }
        }
        if (kMode == kStats && my_ok) {
          g.part[(int64_t)(2 * n_tile + half) * gp.rows + row] = make_float2(m, s);
          if (mine >= 0) g.picked[row] = x_y;
        }
      } else {
        const bool nothing = split * g.ks_per_split >= g.k_stages;      // no stage of K: no product was issued
        const bool f32 = sliced || g.out_f32;
        const int64_t first = sliced ? (int64_t)split * g.slice_rows * g.cols : kMode == kProductT ? (int64_t)split * g.slice_rows * g.ldd : 0;
        const int64_t pitch = sliced ? g.cols : g.ldd;
        const Dest dest{static_cast<uint8_t*>(sliced ? static_cast<void*>(g.slices) : g.dst) + first * (f32 ? 4 : 2), pitch * (f32 ? 4 : 2), g.rows,
                        g.cols, !sliced && g.to_tokens && !dense ? g.token : nullptr};
        constexpr int kN = C::kHalf / 32;
        uint32_t r[2][32];
        tc_ld32(acc, r[0]);
#pragma unroll
        for (int c = 0; c < kN; ++c) {
          tc_wait_ld(r[c & 1]);
          if (c + 1 < kN) tc_ld32(acc + (uint32_t)((c + 1) * 32), r[(c + 1) & 1]);
          else release();
          const int col = colbase + c * 32;
          if (col >= g.cols || my_row0 >= g.rows) continue;
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = nothing ? 0.f : __uint_as_float(r[c & 1][j]) * scale;
          if (g.acc != nullptr && my_ok && !sliced) {         // columns are a multiple of 8: whole vectors
            const float4* p = reinterpret_cast<const float4*>(g.acc + (int64_t)row * g.ldacc + col);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (col + 4 * j < g.cols) {
                const float4 f = p[j];
                v[4 * j] += f.x; v[4 * j + 1] += f.y; v[4 * j + 2] += f.z; v[4 * j + 3] += f.w;
              }
            }
          }
          if (f32) store_chunk<true>(dest, buf, lane, my_row0, col, v);
          else store_chunk<false>(dest, buf, lane, my_row0, col, v);
        }
      }
    }
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

// Numbers the counted tokens in order and, unless all are counted, copies their rows of h together, so
// that padded and masked-out tokens (a third to nine tenths of a fine-tuning batch) cost no products and their
// contents reach nothing.  Each block takes a run of tokens; the counted ones before it are counted by
// the block itself (64 KB of targets at 8192 tokens), for long inputs from per-run counts.
constexpr int kPackThreads = 256;
constexpr int64_t kPackSelf = 32768;             // tokens up to which every block counts for itself
struct PackParams {
  const int64_t* target;
  int64_t ignore;
  int vocab, tokens, run;                        // run: tokens per block
  const int* run_counts;                         // counted tokens of every run, or null
  const __nv_bfloat16* h;
  int64_t ldh;
  int dim;
  __nv_bfloat16* packed;                         // [tokens][dim]; few: [2 kFew][dim], the rows twice
  int few;
  int* slots;
  int* token;                                    // slot -> token
  int* slot_target;
  float* row_loss;                               // forward, losses token by token: 0 for the others
  void* dh;                                      // backward: rows of the others are zero
  int dh_f32;
  unsigned int* counter;                         // forward: put to zero for the joining kernel
  float* count;                                  // forward: number of counted tokens for the caller
};
__device__ __forceinline__ int pack_block_sum(int v, int* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = __reduce_add_sync(0xFFFFFFFFu, v);
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  int s = 0;
#pragma unroll
  for (int w = 0; w < kPackThreads / 32; ++w) s += red[w];
  return s;
}
__global__ void __launch_bounds__(kPackThreads) xent_run_count_kernel(const int64_t* target, int64_t ignore, int tokens, int run, int* run_counts) {
  __shared__ int red[kPackThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t0 = (int64_t)blockIdx.x * run, t1 = min((int64_t)tokens, t0 + run);
  int n = 0;
  for (int64_t t = t0 + threadIdx.x; t < t1; t += kPackThreads) n += target[t] != ignore;
  n = pack_block_sum(n, red);
  if (threadIdx.x == 0) run_counts[blockIdx.x] = n;
}
__global__ void __launch_bounds__(kPackThreads) xent_pack_kernel(const PackParams p) {
  __shared__ int red[kPackThreads / 32];
  __shared__ int source[kPackThreads];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = blockIdx.x * p.run, t1 = min(p.tokens, t0 + p.run);      // gridDim * run < 2^31
  int before = 0, all = 0;
  if (p.run_counts != nullptr) {
    for (int i = threadIdx.x; i < (int)gridDim.x; i += kPackThreads) {
      const int c = p.run_counts[i];
      all += c;
      if (i < (int)blockIdx.x) before += c;
    }
  } else {
#pragma unroll 8
    for (int t = threadIdx.x; t < p.tokens; t += kPackThreads) {
      const int c = __ldcg(reinterpret_cast<const long long*>(p.target) + t) != p.ignore;
      all += c;
      if (t < t0) before += c;
    }
  }
  all = pack_block_sum(all, red);
  before = pack_block_sum(before, red);
  const bool dense = all == p.tokens && !p.few;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *p.slots = all;
    if (p.counter) *p.counter = 0u;
    if (p.count) *p.count = (float)all;
  }
  for (int base = t0; base < t1; base += kPackThreads) {
    const int t = base + (int)threadIdx.x;
    const int64_t y = t < t1 ? __ldcg(reinterpret_cast<const long long*>(p.target) + t) : p.ignore;
    const bool counted = t < t1 && y != p.ignore;
    const uint32_t votes = __ballot_sync(0xFFFFFFFFu, counted);
    __syncthreads();                              // red and source of the round before are read
    if (lane == 0) red[warp] = __popc(votes);
    __syncthreads();
    int at = __popc(votes & ((1u << lane) - 1u)), total = 0;
#pragma unroll
    for (int w = 0; w < kPackThreads / 32; ++w) {
      if (w < warp) at += red[w];
      total += red[w];
    }
    if (counted) {
      p.token[before + at] = t;
      p.slot_target[before + at] = y >= 0 && y < p.vocab ? (int)y : -1;
      source[at] = t;
    } else if (t < t1 && p.row_loss != nullptr) {
      p.row_loss[t] = 0.f;
    }
    __syncthreads();
    if (!dense) {
      const int vecs = p.dim / 8;
      for (int64_t c0 = threadIdx.x; c0 < (int64_t)total * vecs; c0 += 4 * kPackThreads) {
        uint4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int64_t c = c0 + k * kPackThreads;
          const int i = (int)(c / vecs);
          if (i < total) v[k] = __ldcg(reinterpret_cast<const uint4*>(p.h + (int64_t)source[i] * p.ldh) + (c - (int64_t)i * vecs));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int64_t c = c0 + k * kPackThreads;
          if (c < (int64_t)total * vecs) {
            uint4* to = reinterpret_cast<uint4*>(p.packed) + (int64_t)before * vecs + c;
            to[0] = v[k];
            if (p.few) to[(int64_t)kFew * vecs] = v[k];
          }
        }
      }
      if (p.dh != nullptr) {
        const int dvecs = p.dim / (p.dh_f32 ? 4 : 8);
        for (int i = 0; i < 32; ++i) {            // a warp its own 32 tokens
          const int tt = base + warp * 32 + i;
          if (tt < t1 && !((votes >> i) & 1u)) {
            uint4* to = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.dh) + (int64_t)tt * dvecs * 16);
            for (int c = lane; c < dvecs; c += 32) to[c] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
      }
    }
    before += total;
  }
  // the rows behind the last slot that the last K stage of dW reads are zero
  if (!dense) {
    const int end = p.few ? kFew : min(p.tokens, (all + kXK - 1) / kXK * kXK);
    for (int64_t c = (int64_t)all * (p.dim / 8) + blockIdx.x * kPackThreads + threadIdx.x; c < (int64_t)end * (p.dim / 8);
         c += (int64_t)gridDim.x * kPackThreads) {
      reinterpret_cast<uint4*>(p.packed)[c] = make_uint4(0u, 0u, 0u, 0u);
      if (p.few) reinterpret_cast<uint4*>(p.packed)[c + (int64_t)kFew * (p.dim / 8)] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
}

// The forward statistics of one to four tokens: reading W is all there is to it, and whole rows in a row
// read better than the tensor core's 128-byte columns of 256 rows (131072 x 4096, one token: 184 against 245 us; the
// bytes' floor is 163).  A warp
// takes four neighbouring rows of W at a time, the tokens' states wait in shared memory as bf16; products
// and sums in fp32.  One partial (maximum, sum) per block and token.
constexpr int kRowsThreads = 256, kRowsPerWarp = 4, kRowsTokens = 4;
constexpr int64_t kRowsElems = 24000;            // tokens * dim: 47 KB of shared memory
struct RowsParams {
  const __nv_bfloat16* h;
  const __nv_bfloat16* w;
  int64_t ldh, ldw;
  const void* bias;
  int bias_f32;
  int dim, vocab, tokens;
  const int* slots;
  const int* token;
  const int* target;
  float2* part;                                  // [gridDim.x][tokens]
  float* picked;
};
__device__ __forceinline__ float dot8(const uint4& a, const uint4& b, float acc) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    acc = fmaf(__uint_as_float(x[i] << 16), __uint_as_float(y[i] << 16), acc);
    acc = fmaf(__uint_as_float(x[i] & 0xFFFF0000u), __uint_as_float(y[i] & 0xFFFF0000u), acc);
  }
  return acc;
}
// adds one logit to a running (maximum, sum of exponentials)
__device__ __forceinline__ void running_add(float x, float& m, float& s) {
  const float mn = fmaxf(m, x), ref = mn == -INFINITY ? 0.f : mn;
  s = s * exp2_fast((m - ref) * kLog2e) + exp2_fast((x - ref) * kLog2e);
  m = mn;
}
template <int kT>
__global__ void __launch_bounds__(kRowsThreads) xent_rows_kernel(const RowsParams p) {
  extern __shared__ __align__(16) uint4 state[];             // [kT][dim / 8]
  __shared__ float2 red[kRowsThreads / 32][kT];
  pdl_launch_dependents();
  pdl_wait();
  const int slots = *static_cast<const volatile int*>(p.slots);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int vecs = p.dim / 8;
  int target[kT];
#pragma unroll
  for (int t = 0; t < kT; ++t) target[t] = t < slots ? p.target[t] : -1;
#pragma unroll
  for (int t = 0; t < kT; ++t) {
    const uint4* from = t < slots ? reinterpret_cast<const uint4*>(p.h + (int64_t)p.token[t] * p.ldh) : nullptr;
    for (int c = threadIdx.x; c < vecs; c += kRowsThreads) state[t * vecs + c] = from ? from[c] : make_uint4(0u, 0u, 0u, 0u);
  }
  __syncthreads();
  float m[kT], s[kT];
#pragma unroll
  for (int t = 0; t < kT; ++t) {
    m[t] = -INFINITY;
    s[t] = 0.f;
  }
  const int stride = gridDim.x * (kRowsThreads / 32) * kRowsPerWarp;
  for (int v0 = (blockIdx.x * (kRowsThreads / 32) + warp) * kRowsPerWarp; v0 < p.vocab && slots > 0; v0 += stride) {
    const uint4* row[kRowsPerWarp];
#pragma unroll
    for (int r = 0; r < kRowsPerWarp; ++r) row[r] = reinterpret_cast<const uint4*>(p.w + (int64_t)min(v0 + r, p.vocab - 1) * p.ldw);
    float acc[kRowsPerWarp][kT];
#pragma unroll
    for (int r = 0; r < kRowsPerWarp; ++r)
#pragma unroll
      for (int t = 0; t < kT; ++t) acc[r][t] = 0.f;
    int c = lane;
    for (; c + 96 < vecs; c += 128) {                        // sixteen 16-byte loads in flight per lane
      uint4 q[4][kRowsPerWarp];
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int r = 0; r < kRowsPerWarp; ++r) q[k][r] = __ldcs(row[r] + c + 32 * k);
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int t = 0; t < kT; ++t) {
          const uint4 hv = state[t * vecs + c + 32 * k];
#pragma unroll
          for (int r = 0; r < kRowsPerWarp; ++r) acc[r][t] = dot8(q[k][r], hv, acc[r][t]);
        }
    }
    for (; c < vecs; c += 32) {
      uint4 q[kRowsPerWarp];
#pragma unroll
      for (int r = 0; r < kRowsPerWarp; ++r) q[r] = __ldcs(row[r] + c);
#pragma unroll
      for (int t = 0; t < kT; ++t) {
        const uint4 hv = state[t * vecs + c];
#pragma unroll
        for (int r = 0; r < kRowsPerWarp; ++r) acc[r][t] = dot8(q[r], hv, acc[r][t]);
      }
    }
#pragma unroll
    for (int r = 0; r < kRowsPerWarp; ++r) {
      const int v = v0 + r;
      float b = 0.f;
      if (p.bias != nullptr && v < p.vocab)
        b = p.bias_f32 ? __ldg(static_cast<const float*>(p.bias) + v) : __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[v]);
#pragma unroll
      for (int t = 0; t < kT; ++t) {
        float x = acc[r][t];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
        x += b;
        if (v < p.vocab) {
          running_add(x, m[t], s[t]);
          if (lane == 0 && v == target[t]) p.picked[t] = x;
        }
      }
    }
  }
  if (lane == 0) {
#pragma unroll
    for (int t = 0; t < kT; ++t) red[warp][t] = make_float2(m[t], s[t]);
  }
  __syncthreads();
  if (threadIdx.x < kT && (int)threadIdx.x < p.tokens) {
    float mm = -INFINITY, ss = 0.f;
    for (int w = 0; w < kRowsThreads / 32; ++w) {
      const float2 q = red[w][threadIdx.x];
      const float mn = fmaxf(mm, q.x), ref = mn == -INFINITY ? 0.f : mn;
      ss = ss * exp2_fast((mm - ref) * kLog2e) + q.y * exp2_fast((q.x - ref) * kLog2e);
      mm = mn;
    }
    p.part[(int64_t)blockIdx.x * p.tokens + threadIdx.x] = make_float2(mm, ss);
  }
}

// Joins the partial statistics of a slot along the vocabulary: `lanes` rows a block (a power of two, at
// most 8), 256 / lanes threads a row, so that a single token's partials are read by a whole block.  The last
// block to finish adds the blocks' sums in block order (fp64) and writes the mean or sum.
constexpr int kJoinThreads = 256;
struct JoinParams {
  const float2* part;
  int parts;
  const float* picked;
  const int* target;
  const int* token;
  const int* slots;
  int slot0, rows, lanes;          // of this block of slots; rows: the most it can hold
  float* lse;
  float* row_loss;                 // losses token by token, or null
  float* out;                      // their mean or sum, or null
  int mean;
  double* block_loss;              // [joining blocks of all blocks of slots]
  int first_block, all_blocks;
  unsigned int* counter;
  int32_t* status;
};
__global__ void __launch_bounds__(kJoinThreads) xent_join_kernel(const JoinParams p) {
  __shared__ float2 red[kJoinThreads];
  __shared__ double sum_s[kJoinThreads];
  __shared__ bool last;
  pdl_launch_dependents();
  pdl_wait();
  const int slots = *static_cast<const volatile int*>(p.slots);
  const int rows = max(0, min(p.rows, slots - p.slot0));
  const int slices = kJoinThreads / p.lanes;
  const int r = threadIdx.x & (p.lanes - 1), slice = threadIdx.x / p.lanes;
  const int64_t row = (int64_t)blockIdx.x * p.lanes + r;
  float m = -INFINITY, s = 0.f;
  if (row < rows) {
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
  if (slice == 0 && row < rows) {
    const float2 q = red[threadIdx.x];
    const double lse = (double)q.x + (double)logf(q.y);      // the loss is a small difference of large numbers
    p.lse[row] = (float)lse;
    float loss = NAN;
    if (p.target[row] >= 0) loss = (float)(lse - (double)p.picked[row]);
    else if (p.status) atomicCAS(p.status, 0, kXBadTarget);
    if (p.row_loss) p.row_loss[p.token[row]] = loss;
    sum = loss;
  }
  if (p.out == nullptr) return;
  if (threadIdx.x < p.lanes) sum_s[threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    for (int i = 0; i < p.lanes; ++i) sum += sum_s[i];
    p.block_loss[p.first_block + blockIdx.x] = sum;
    __threadfence();
    last = atomicAdd(p.counter, 1u) == (unsigned int)p.all_blocks - 1u;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  sum = 0.0;
  for (int i = threadIdx.x; i < p.all_blocks; i += kJoinThreads) sum += __ldcg(p.block_loss + i);
  sum_s[threadIdx.x] = sum;
  __syncthreads();
  for (int o = kJoinThreads >> 1; o > 0; o >>= 1) {
    if (threadIdx.x < o) sum_s[threadIdx.x] += sum_s[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) *p.out = (float)(p.mean ? sum_s[0] / (double)slots : sum_s[0]);   // no token counted: 0 / 0
}

// out[r, c] = sum over the slices (+ acc[r, c]), four columns a thread, slices in order.  `slots` (dh): the
// rows are slots and go to their tokens' places if `token` is given.
struct SliceParams {
  const float* slices;
  int n;
  int64_t slice_elems;
  const float* acc;
  void* out;
  int out_f32, rows, cols4, tokens;
  const int* slots;                      // dh: the splits are kProduct's own
  const int* token;
  int n_tiles, k_stages, split_clusters;
  int few;                               // dh: rows kFew further on are added
};
__global__ void __launch_bounds__(256) xent_slices_kernel(const SliceParams p) {
  pdl_launch_dependents();
  pdl_wait();
  int rows = p.rows, n = p.n;
  int64_t slice_elems = p.slice_elems;
  bool scatter = false;
  if (p.slots != nullptr) {
    rows = min(rows, *static_cast<const volatile int*>(p.slots));
    scatter = p.token != nullptr && rows < p.tokens;
    const int m_tiles = p.few ? 1 : (rows + kXM - 1) / kXM;
    n = split_slots(m_tiles, p.n_tiles, p.k_stages, p.split_clusters).splits;
    if (n == 1 && !p.few) return;        // written by kProduct itself
    slice_elems = (int64_t)m_tiles * kXM * p.cols4 * 4;
  }
  const int64_t total4 = (int64_t)rows * p.cols4;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total4; i += (int64_t)gridDim.x * 256) {
    float4 v = p.acc ? reinterpret_cast<const float4*>(p.acc)[i] : make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < n; ++s) {
      const float4 f = reinterpret_cast<const float4*>(p.slices + s * slice_elems)[i];
      v.x += f.x; v.y += f.y; v.z += f.z; v.w += f.w;
      if (p.few) {
        const float4 l = reinterpret_cast<const float4*>(p.slices + s * slice_elems)[i + (int64_t)kFew * p.cols4];
        v.x += l.x; v.y += l.y; v.z += l.z; v.w += l.w;
      }
    }
    int64_t to = i;
    if (scatter) {
      const int64_t r = i / p.cols4;
      to += ((int64_t)p.token[r] - r) * p.cols4;
    }
    if (p.out_f32) {
      static_cast<float4*>(p.out)[to] = v;
    } else {
      const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
      static_cast<uint2*>(p.out)[to] = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
  }
}

// db: the column sums of dl that the gradient epilogue left per 32 slots (taken in fp32, before dl is
// rounded).  A block per 32 columns; its 8 warps take the rows in turn and are added in warp order.
__global__ void __launch_bounds__(256) xent_bias_grad_kernel(const float* __restrict__ part, int64_t ld, const int* slots, int cols, void* db,
                                                              int db_f32) {
  __shared__ float red[8][32];
  pdl_launch_dependents();
  pdl_wait();
  const int rows = (*static_cast<const volatile int*>(slots) + 31) / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float a = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int r = warp; r < rows; r += 8) a += part[(int64_t)r * ld + c];
  }
  red[warp][lane] = a;
  __syncthreads();
  if (warp == 0 && c < cols) {
    float s = 0.f;
    for (int w = 0; w < 8; ++w) s += red[w][lane];
    if (db_f32) static_cast<float*>(db)[c] = s;
    else static_cast<__nv_bfloat16*>(db)[c] = __float2bfloat16_rn(s);
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
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, XCfg<kMode, kBN>::kSmemBytes) == cudaSuccess) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(2 * 148, 1, 1);
      cfg.blockDim = dim3(kXThreads, 1, 1);
      cfg.dynamicSmemBytes = XCfg<kMode, kBN>::kSmemBytes;
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

int64_t round_up(int64_t v, int64_t to) { return ceil_div(v, to) * to; }

int width_for(int64_t cols) { return cols <= 128 ? 128 : 256; }     // of a tile

// How a product [m, n] over k is cut: tile width, and K splits when its tiles leave most clusters idle.
struct Cut {
  int bn = 256, splits = 1, ks_per_split = 0;
  int64_t slice_rows = 0;
  int64_t slice_bytes(int64_t n) const { return splits > 1 ? splits * slice_rows * n * 4 : 0; }
};
Cut cut_product(int64_t m, int64_t n, int64_t k, int clusters) {
  Cut c;
  const int64_t mt = ceil_div(m, kXM), stages = ceil_div(k, kXK);
  c.bn = width_for(n);
  const int64_t tiles = mt * ceil_div(n, c.bn);
  c.ks_per_split = (int)stages;
  if (tiles * 2 <= clusters) {
    const int64_t s = std::min<int64_t>(clusters / tiles, stages / kMinSplitStages);
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

// `packed`: the counted tokens' rows of h, read in place of operand a (kStats, kGrad) or b (kProductT).
template <int kMode, int kBN>
int launch_width(const Operand& a, const Operand& b, const Operand& packed, XParams g, int64_t k, cudaStream_t stream) {
  using C = XCfg<kMode, kBN>;
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
  CUtensorMap map_a, map_b, map_packed = {};
  int rc = kAMn ? bf16_map(&map_a, a, 64, kXK, CU_TENSOR_MAP_SWIZZLE_128B) : bf16_map(&map_a, a, kXK, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == FP4T_OK)
    rc = kBMn ? bf16_map(&map_b, b, 64, kXK, CU_TENSOR_MAP_SWIZZLE_128B) : bf16_map(&map_b, b, kXK, C::kBRows, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == FP4T_OK && kMode != kProduct)
    rc = kBMn ? bf16_map(&map_packed, packed, 64, kXK, CU_TENSOR_MAP_SWIZZLE_128B) : bf16_map(&map_packed, packed, kXK, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != FP4T_OK) return rc;
  const int64_t units = kMode == kProduct && g.split_clusters > 0 ? clusters : (int64_t)g.m_tiles * g.n_tiles * g.splits;
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
  FP4T_CUDA(cudaLaunchKernelEx(&cfg, xent_gemm_kernel<kMode, kBN>, map_a, map_b, map_packed, g));
  return FP4T_OK;
}
template <int kMode>
int launch_xent(int bn, const Operand& a, const Operand& b, const Operand& packed, const XParams& g, int64_t k, cudaStream_t stream) {
  return bn == 128 ? launch_width<kMode, 128>(a, b, packed, g, k, stream) : launch_width<kMode, 256>(a, b, packed, g, k, stream);
}

template <typename... Args, typename... Actual>
int launch_small_shared(void (*kern)(Args...), int grid, int threads, int64_t shared, cudaStream_t stream, Actual... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = (size_t)shared;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  pdl_attribute(&attr);
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  FP4T_CUDA(cudaLaunchKernelEx(&cfg, kern, args...));
  return FP4T_OK;
}
template <typename... Args, typename... Actual>
int launch_small(void (*kern)(Args...), int grid, int threads, cudaStream_t stream, Actual... args) {
  return launch_small_shared(kern, grid, threads, 0, stream, args...);
}

// What both passes know about the counted tokens (device memory in the workspace).
struct Slots {
  int* slots;
  int* token;
  int* target;
  int* run_counts;
  __nv_bfloat16* packed;
};

// The loss's gradient as the kernels take it.
struct Scale {
  const float* grad;
  int reduction;
  void to(XParams& g) const {
    g.grad = grad;
    g.grad_per_row = reduction == FP4T_XENT_NONE;
    g.mean = reduction == FP4T_XENT_MEAN;
  }
};

// dh (or its sum over the pieces so far) into `out`, rows of `dim`: slots, or tokens' places if to_tokens.
int run_dh(const Operand& dl, const Operand& w, int64_t tokens, int64_t dim, int64_t vc, void* out, int out_f32, bool to_tokens, const float* acc,
           float* slices, int64_t slice_rows, int split_clusters, const Scale& scale, const Slots& sl, int32_t* status, cudaStream_t stream) {
  XParams g = {};
  g.few = tokens <= kFew;
  g.tokens = (int)tokens;
  g.rows = g.few ? 2 * kFew : (int)tokens;
  scale.to(g);
  g.cols = (int)dim;
  g.slots = sl.slots;
  g.token = sl.token;
  g.status = status;
  g.out_f32 = out_f32;
  g.acc = acc;
  g.ldacc = dim;
  g.dst = out;
  g.ldd = dim;
  g.to_tokens = to_tokens;
  g.slices = slices;
  const int bn = width_for(dim);
  split_clusters = std::min(split_clusters, bn == 128 ? xent_clusters<kProduct, 128>() : xent_clusters<kProduct, 256>());
  g.split_clusters = slice_rows > 0 ? split_clusters : 0;      // (the kernel's launch refuses when none can be resident)
  int rc = launch_xent<kProduct>(bn, dl, w, Operand{}, g, vc, stream);
  if (rc != FP4T_OK || g.split_clusters <= 0) return rc;
  SliceParams p = {};
  p.slices = slices;
  p.acc = acc;
  p.out = out;
  p.out_f32 = out_f32;
  p.rows = p.tokens = (int)tokens;
  p.cols4 = (int)(dim / 4);
  p.slots = sl.slots;
  p.token = to_tokens ? sl.token : nullptr;
  p.few = g.few;
  p.n_tiles = (int)ceil_div(dim, bn);
  p.k_stages = (int)ceil_div(vc, kXK);
  p.split_clusters = split_clusters;
  const int grid = (int)std::min<int64_t>(ceil_div(std::min(tokens, slice_rows) * dim / 4, 256), 148 * 8);
  return launch_small(xent_slices_kernel, grid, 256, stream, p);
}

// dW's rows of a piece, through slices when it is split (few entries, many tokens).
int run_dw(const Cut& cut, const Operand& dl, const Operand& h, const Operand& packed, int64_t tokens, int64_t dim, int64_t vc, void* out, int out_f32,
           float* slices, const Scale& scale, const Slots& sl, int32_t* status, cudaStream_t stream) {
  XParams g = {};
  g.few = tokens <= kFew;
  g.rows = (int)vc;
  g.cols = (int)dim;
  g.tokens = (int)tokens;
  scale.to(g);
  g.slots = sl.slots;
  g.status = status;
  g.splits = cut.splits;
  g.ks_per_split = cut.ks_per_split;
  g.out_f32 = cut.splits > 1 ? 1 : out_f32;
  g.slice_rows = (int)cut.slice_rows;
  g.dst = cut.splits > 1 ? slices : out;
  g.ldd = dim;
  int rc = launch_xent<kProductT>(cut.bn, dl, h, packed, g, dl.outer, stream);
  if (rc != FP4T_OK || cut.splits == 1) return rc;
  SliceParams p = {};
  p.slices = slices;
  p.n = cut.splits;
  p.slice_elems = cut.slice_rows * dim;
  p.out = out;
  p.out_f32 = out_f32;
  p.rows = (int)vc;
  p.cols4 = (int)(dim / 4);
  const int grid = (int)std::min<int64_t>(ceil_div(vc * dim / 4, 256), 148 * 8);
  return launch_small(xent_slices_kernel, grid, 256, stream, p);
}

// Slots in the workspace: their number, the token and target of each, counts per run, the packed rows of h.
struct SlotPlan {
  int64_t run, runs, o_token, o_target, o_runs, o_packed, packed_rows, bytes;
};
SlotPlan plan_slots(int64_t tokens, int64_t dim, bool backward) {
  SlotPlan p;
  p.run = tokens <= 148 * 8 ? ceil_div(tokens, 148) : round_up(ceil_div(tokens, 148 * 4), 8);
  p.runs = ceil_div(tokens, p.run);
  p.o_token = 256;                       // slot count at 0, joining kernel's counter at 128
  p.o_target = p.o_token + round_up(tokens * 4, 128);
  p.o_runs = p.o_target + round_up(tokens * 4, 128);
  p.o_packed = round_up(p.o_runs + p.runs * 4, 1024);
  p.packed_rows = backward && tokens <= kFew ? 2 * kFew : tokens;
  p.bytes = p.o_packed + round_up(p.packed_rows * dim * 2, 1024);
  return p;
}
Slots slots_at(uint8_t* ws, const SlotPlan& p) {
  return Slots{reinterpret_cast<int*>(ws), reinterpret_cast<int*>(ws + p.o_token), reinterpret_cast<int*>(ws + p.o_target),
               reinterpret_cast<int*>(ws + p.o_runs), reinterpret_cast<__nv_bfloat16*>(ws + p.o_packed)};
}
int launch_pack(const SlotPlan& plan, const Slots& sl, const void* h, int64_t ldh, const int64_t* target, int64_t tokens, int64_t dim, int64_t vocab,
                int64_t ignore, float* row_loss, void* dh, int dh_f32, unsigned int* counter, float* count, cudaStream_t stream) {
  PackParams p = {};
  p.target = target;
  p.ignore = ignore;
  p.vocab = (int)vocab;
  p.tokens = (int)tokens;
  p.run = (int)plan.run;
  p.h = static_cast<const __nv_bfloat16*>(h);
  p.ldh = ldh;
  p.dim = (int)dim;
  p.packed = sl.packed;
  p.few = plan.packed_rows > tokens;
  p.slots = sl.slots;
  p.token = sl.token;
  p.slot_target = sl.target;
  p.row_loss = row_loss;
  p.dh = dh;
  p.dh_f32 = dh_f32;
  p.counter = counter;
  p.count = count;
  if (tokens > kPackSelf) {
    p.run_counts = sl.run_counts;
    const int rc = launch_small(xent_run_count_kernel, (int)plan.runs, kPackThreads, stream, target, ignore, (int)tokens, (int)plan.run, sl.run_counts);
    if (rc != FP4T_OK) return rc;
  }
  return launch_small(xent_pack_kernel, (int)plan.runs, kPackThreads, stream, p);
}

// Forward workspace: slots, the joining blocks' sums, the targets' logits, partial statistics of a block of slots.
struct ForwardPlan {
  SlotPlan slots;
  int64_t rows_blocks;                    // blocks of the few-tokens kernel, 0: the tensor-core one
  int64_t block, parts, join_blocks;      // slots per block, partials per slot, joining blocks of all blocks of slots
  int lanes;
  int64_t o_loss, o_picked, o_part, bytes;
};
ForwardPlan plan_forward(int64_t tokens, int64_t dim, int64_t vocab) {
  ForwardPlan p;
  p.slots = plan_slots(tokens, dim, false);
  p.block = std::min(tokens, kTokenBlock);
  p.rows_blocks = tokens <= kRowsTokens && (tokens == 1 ? 1 : 4) * dim <= kRowsElems ? std::min<int64_t>(ceil_div(vocab, kRowsThreads / 32 * kRowsPerWarp), 148 * 2) : 0;
  p.parts = p.rows_blocks > 0 ? p.rows_blocks : 2 * ceil_div(vocab, width_for(vocab));
  p.lanes = 1;                            // rows of a joining block: up to 8 (64 bytes of a partial's row) while there are blocks for all SMs
  while (p.lanes < 8 && p.lanes * 148 < tokens) p.lanes <<= 1;
  p.join_blocks = (tokens / p.block) * ceil_div(p.block, p.lanes) + ceil_div(tokens % p.block, p.lanes);
  p.o_loss = p.slots.bytes;
  p.o_picked = p.o_loss + round_up(p.join_blocks * 8, 128);
  p.o_part = p.o_picked + round_up(p.block * 4, 128);
  p.bytes = p.o_part + p.parts * p.block * 8;
  return p;
}

// Backward workspace: slots, dl of a piece, dh in fp32 when there are several pieces, column sums, K slices.
struct BackwardPlan {
  SlotPlan slots;
  int64_t piece, pieces, ld;
  Cut dw;
  int64_t dh_slice_rows;                    // of dh's slices, all splits together; 0: never split
  int64_t o_dl, o_acc, o_cols, o_slices, bytes;
};
BackwardPlan plan_backward(int64_t tokens, int64_t dim, int64_t vocab, bool want_dh, bool want_dw, bool want_db, int clusters) {
  BackwardPlan p;
  p.slots = plan_slots(tokens, dim, true);
  p.piece = std::min(round_up(vocab, 256), std::max(kMinPiece, kPieceBytes / (2 * tokens) / 256 * 256));
  p.pieces = ceil_div(vocab, p.piece);
  p.piece = round_up(ceil_div(vocab, p.pieces), 256);       // even pieces
  p.pieces = ceil_div(vocab, p.piece);
  p.ld = std::min(p.piece, round_up(vocab, 8));
  p.dw = cut_product(std::min(p.piece, vocab), dim, p.slots.packed_rows, clusters);
  const int64_t dh_tiles = ceil_div(dim, width_for(dim));
  p.dh_slice_rows = want_dh && dh_tiles * 2 <= clusters && ceil_div(std::min(p.piece, vocab), kXK) >= 2 * kMinSplitStages ? clusters / dh_tiles * kXM : 0;
  if (want_dh && tokens <= kFew) p.dh_slice_rows = std::max<int64_t>(p.dh_slice_rows, kXM);
  const int64_t dl_rows = p.slots.packed_rows;
  p.o_dl = p.slots.bytes;
  p.o_acc = p.o_dl + round_up(dl_rows * p.ld * 2, 1024);
  p.o_cols = p.o_acc + (want_dh && p.pieces > 1 ? round_up(tokens * dim * 4, 1024) : 0);
  p.o_slices = p.o_cols + (want_db ? round_up(round_up(tokens, kXK) / 32 * p.ld * 4, 1024) : 0);
  p.bytes = p.o_slices + std::max(p.dh_slice_rows * dim * 4, want_dw ? p.dw.slice_bytes(dim) : 0);
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

extern "C" int64_t fp4t_linear_xent_forward_workspace_bytes(int64_t tokens, int64_t dim, int64_t vocab) {
  if (check_sizes("fp4t_linear_xent_forward_workspace_bytes", tokens, dim, vocab) != FP4T_OK) return -1;
  return tokens == 0 ? 128 : plan_forward(tokens, dim, vocab).bytes;
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
  const ForwardPlan p = plan_forward(tokens, dim, vocab);
  FP4T_REQUIRE(workspace_bytes >= p.bytes, "%s: the workspace holds %lld bytes of %lld", name, (long long)workspace_bytes, (long long)p.bytes);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (!status) status = current_status_word();
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const Slots sl = slots_at(ws, p.slots);
  unsigned int* counter = reinterpret_cast<unsigned int*>(ws + 128);
  rc = launch_pack(p.slots, sl, h, ldh, target, tokens, dim, vocab, ignore_index, reduction == FP4T_XENT_NONE ? loss : nullptr, nullptr, 0, counter,
                   count, s);
  if (rc != FP4T_OK) return rc;
  int64_t first_block = 0;
  for (int64_t t0 = 0; t0 < tokens; t0 += p.block) {
    const int64_t rows = std::min(p.block, tokens - t0);
    XParams g = {};
    g.rows = (int)rows;
    g.cols = (int)vocab;
    g.tokens = (int)tokens;
    g.slots = sl.slots;
    g.slot0 = (int)t0;
    g.bias = bias;
    g.bias_f32 = bias_dtype == FP4T_DT_F32;
    g.target = sl.target + t0;
    g.part = reinterpret_cast<float2*>(ws + p.o_part);
    g.picked = reinterpret_cast<float*>(ws + p.o_picked);
    g.status = status;
    if (p.rows_blocks > 0) {
      RowsParams r = {};
      r.h = static_cast<const __nv_bfloat16*>(h);
      r.w = static_cast<const __nv_bfloat16*>(w);
      r.ldh = ldh;
      r.ldw = ldw;
      r.bias = bias;
      r.bias_f32 = g.bias_f32;
      r.dim = (int)dim;
      r.vocab = (int)vocab;
      r.tokens = (int)tokens;
      r.slots = sl.slots;
      r.token = sl.token;
      r.target = sl.target;
      r.part = g.part;
      r.picked = g.picked;
      auto kern = tokens == 1 ? xent_rows_kernel<1> : xent_rows_kernel<4>;
      rc = launch_small_shared(kern, (int)p.rows_blocks, kRowsThreads, (tokens == 1 ? 1 : 4) * dim * 2, s, r);
    } else
      rc = launch_xent<kStats>(width_for(vocab), Operand{static_cast<const __nv_bfloat16*>(h) + t0 * ldh, rows, dim, ldh}, Operand{w, vocab, dim, ldw},
                             Operand{sl.packed + t0 * dim, rows, dim, dim}, g, dim, s);
    if (rc != FP4T_OK) return rc;
    JoinParams j = {};
    j.part = g.part;
    j.parts = (int)p.parts;
    j.picked = g.picked;
    j.target = g.target;
    j.token = sl.token + t0;
    j.slots = sl.slots;
    j.slot0 = (int)t0;
    j.rows = (int)rows;
    j.lanes = p.lanes;
    j.lse = lse + t0;
    j.row_loss = reduction == FP4T_XENT_NONE ? loss : nullptr;
    j.out = reduction == FP4T_XENT_NONE ? nullptr : loss;
    j.mean = reduction == FP4T_XENT_MEAN;
    j.block_loss = reinterpret_cast<double*>(ws + p.o_loss);
    j.first_block = (int)first_block;
    j.all_blocks = (int)p.join_blocks;
    j.counter = counter;
    j.status = status;
    const int blocks = (int)ceil_div(rows, p.lanes);
    first_block += blocks;
    rc = launch_small(xent_join_kernel, blocks, kJoinThreads, s, j);
    if (rc != FP4T_OK) return rc;
  }
  return FP4T_OK;
}

extern "C" int64_t fp4t_linear_xent_backward_workspace_bytes(int64_t tokens, int64_t dim, int64_t vocab, int want_dh, int want_dw,
                                                              int want_db) {
  if (check_sizes("fp4t_linear_xent_backward_workspace_bytes", tokens, dim, vocab) != FP4T_OK) return -1;
  const int clusters = cluster_budget();
  if (tokens == 0 || clusters <= 0) return tokens == 0 ? 128 : -1;
  return plan_backward(tokens, dim, vocab, want_dh != 0, want_dw != 0, want_db != 0, clusters).bytes;
}

extern "C" int fp4t_linear_xent_backward(const float* grad_loss, const void* h, int64_t ldh, const void* w, int64_t ldw, const void* bias,
                                         int bias_dtype, const int64_t* target, const float* lse, int64_t tokens, int64_t dim, int64_t vocab,
                                         int64_t ignore_index, int reduction, void* dh, int dh_dtype, void* dw, int dw_dtype, void* db,
                                         int db_dtype, void* workspace, int64_t workspace_bytes, int32_t* status, fp4t_stream_t stream) {
  const char* name = "fp4t_linear_xent_backward";
  int rc = check_sizes(name, tokens, dim, vocab);
  if (rc != FP4T_OK) return rc;
  FP4T_REQUIRE(tokens > 0, "%s: no tokens", name);
  rc = check_inputs(name, h, ldh, w, ldw, bias, bias_dtype, target, dim, reduction, workspace);
  if (rc != FP4T_OK) return rc;
  FP4T_REQUIRE(grad_loss && lse, "%s: null pointer", name);
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
  const BackwardPlan p = plan_backward(tokens, dim, vocab, dh != nullptr, dw != nullptr, db != nullptr, clusters);
  FP4T_REQUIRE(workspace_bytes >= p.bytes, "%s: the workspace holds %lld bytes of %lld", name, (long long)workspace_bytes, (long long)p.bytes);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (!status) status = current_status_word();
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const Slots sl = slots_at(ws, p.slots);
  rc = launch_pack(p.slots, sl, h, ldh, target, tokens, dim, vocab, ignore_index, nullptr, dh, dh_dtype == FP4T_DT_F32, nullptr, nullptr, s);
  if (rc != FP4T_OK) return rc;
  __nv_bfloat16* dl = reinterpret_cast<__nv_bfloat16*>(ws + p.o_dl);
  float* acc = reinterpret_cast<float*>(ws + p.o_acc);
  float* slices = reinterpret_cast<float*>(ws + p.o_slices);
  const Operand hop{h, tokens, dim, ldh}, packed{sl.packed, p.slots.packed_rows, dim, dim};
  const Scale scale{grad_loss, reduction};
  for (int64_t i = 0; i < p.pieces; ++i) {
    const int64_t v0 = i * p.piece, vc = std::min(p.piece, vocab - v0);
    const Operand wop{static_cast<const __nv_bfloat16*>(w) + v0 * ldw, vc, dim, ldw}, dop{dl, p.slots.packed_rows, vc, p.ld};
    XParams g = {};
    g.rows = (int)p.slots.packed_rows;
    g.few = tokens <= kFew;
    g.cols = (int)vc;
    g.tokens = (int)tokens;
    g.slots = sl.slots;
    g.token = sl.token;
    g.bias = bias ? static_cast<const uint8_t*>(bias) + v0 * (bias_dtype == FP4T_DT_F32 ? 4 : 2) : nullptr;
    g.bias_f32 = bias_dtype == FP4T_DT_F32;
    g.target = sl.target;
    g.col0 = (int)v0;
    g.lse = lse;
    scale.to(g);
    g.col_part = db ? reinterpret_cast<float*>(ws + p.o_cols) : nullptr;
    g.col_ld = p.ld;
    g.status = status;
    g.dst = dl;
    g.ldd = p.ld;
    rc = launch_xent<kGrad>(width_for(vc), hop, wop, packed, g, dim, s);
    if (rc != FP4T_OK) return rc;
    if (dh) {
      const bool last = i == p.pieces - 1;
      rc = run_dh(dop, wop, tokens, dim, vc, last ? dh : static_cast<void*>(acc), last ? dh_dtype == FP4T_DT_F32 : 1, last, i > 0 ? acc : nullptr,
                  slices, p.dh_slice_rows, clusters, scale, sl, status, s);
      if (rc != FP4T_OK) return rc;
    }
    if (dw) {
      void* out = static_cast<uint8_t*>(dw) + v0 * dim * (dw_dtype == FP4T_DT_F32 ? 4 : 2);
      rc = run_dw(p.dw, dop, hop, packed, tokens, dim, vc, out, dw_dtype == FP4T_DT_F32, slices, scale, sl, status, s);
      if (rc != FP4T_OK) return rc;
    }
    if (db) {
      void* out = static_cast<uint8_t*>(db) + v0 * (db_dtype == FP4T_DT_F32 ? 4 : 2);
      rc = launch_small(xent_bias_grad_kernel, (int)ceil_div(vc, 32), 256, s, (const float*)g.col_part, p.ld, (const int*)sl.slots, (int)vc, out,
                        (int)(db_dtype == FP4T_DT_F32));
      if (rc != FP4T_OK) return rc;
    }
  }
  return FP4T_OK;
}
