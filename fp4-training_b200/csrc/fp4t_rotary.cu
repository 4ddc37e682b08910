// Between the stacked q / k / v projection and the attention core: rotary positions with several
// axes, and the RMS norm of every query / key head with that rotation in the same pass.
//
//   rotary      (a, b) -> (a cos t - b sin t, a sin t + b cos t) for every turning pair p of a head,
//               t = position[axis(p)] * frequency(p); elements behind the turning ones are copied
//   norm        xh = x / sqrt(mean(x^2) + eps), y = R(t) (w * xh)
//   backward    g = R(-t) dy, dw = sum g xh, u = g w, dx = r (u - xh mean(u xh)), r recomputed from x
//
// The angle is kept in turns as a 64-bit fixed-point fraction: position * (frequency / 2 pi * 2^64)
// wraps modulo one turn by itself, so a position of a million is as exact as one of ten (an fp32
// product is off by 0.06 radians there) and costs one integer multiply, no fp64.
//
// The arithmetic is packed, two floats an instruction: element by element the norm kernels took 211
// instructions per lane and head and were bound by their issue.
//
// A head is held by a group of 1 to 32 lanes, up to eight pairs (two 16-byte vectors of bf16) a lane, so the
// norm is a shuffle reduction inside the group and every element is read and written once:
// HBM-bound (forward 4 bytes per bf16 element, norm backward 6).  Measured (B200, copy bandwidth 6.57 TB/s):
// 65536 tokens x 40 heads x 128 bf16 rotation 204 us, 6.58 TB/s; 32768 tokens with norms forward 107 us, 6.3 TB/s,
// backward 183 us, 5.5 TB/s (bound by the chain of two reductions per head at 16 warps per SM).
//
// A group walks heads of ONE token, queries and keys, with the cosines and sines of its pairs in registers: no
// table, no barrier, and the trigonometry is paid once per token, not per head.  Several heads' vectors are under way
// before the first is worked on, the first ones before the angles are computed.
#include <algorithm>

#include "fp4t_common.cuh"
#include "fp4t_pack.cuh"

namespace fp4t {
namespace {

constexpr int kRotThreads = 128;
constexpr int kRotWarps = kRotThreads / 32;
constexpr int kRotMaxDim = 512;           // 256 pairs: 32 lanes x 8
constexpr int kRotBlocksPerSm = 4;        // of the norm backward: resident at once, and rows of its workspace

struct HeadsIn {
  const void* p;
  int64_t sb, st, sh;
};
struct HeadsOut {
  void* p;
  int64_t sb, st, sh;
};
struct RotParams {
  HeadsIn x[2], dy[2];
  HeadsOut y[2];
  int heads[2];
  const float* w[2];
  float eps, inv_dim;
  int64_t n;                              // batch * tokens
  int64_t tokens;
  int dim, pairs, turned, group, log_group;
  int chunk, chunks;                      // heads of a token per group, groups per token
  int blocks0;                            // norm backward: blocks that work on the first tensor
  const void* pos;
  int pos_i64, axes;
  int64_t pos_sb, pos_st, pos_sa;
  const uint64_t* turns;
  const int32_t* axis;
  float sign;                             // -1: rotate back
  float* partial;                         // norm backward: [gridDim.x][dim]
};

// One vector of V elements as it lies in memory (bf16 stays packed until its head's turn comes: several
// heads in flight fit the registers).
template <typename T, int V>
struct Raw {
  static constexpr int kWords = sizeof(T) == 4 ? V : (V + 1) / 2;
  uint32_t u[kWords];

  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kWords >= 4) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 q = reinterpret_cast<const uint4*>(p)[i / 4];
        u[i] = q.x; u[i + 1] = q.y; u[i + 2] = q.z; u[i + 3] = q.w;
      }
    } else if constexpr (kWords == 2) {
      const uint2 q = *reinterpret_cast<const uint2*>(p);
      u[0] = q.x; u[1] = q.y;
    } else if constexpr (sizeof(T) == 4 || V == 2) {
      u[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      u[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) u[i] = 0u;
  }
  __device__ __forceinline__ void expand(float* v) const {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(u[i]);
      else v[i] = __uint_as_float((i & 1) ? u[i / 2] & 0xFFFF0000u : u[i / 2] << 16);
    }
  }
};

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (V >= 4) {
#pragma unroll
      for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else if constexpr (V == 2) {
      *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    } else {
      *p = v[0];
    }
  } else if constexpr (V == 1) {
    *p = __float2bfloat16_rn(v[0]);
  } else {
    uint32_t u[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    if constexpr (V == 8) *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    else if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
    else *reinterpret_cast<uint32_t*>(p) = u[0];
  }
}

// Cosine and sine of a fraction of a turn held in 64 bits (the integer part has wrapped away).  The
// nearest quarter turn is taken off as an integer, so the float that is left is at most an eighth of
// a turn and its rounding stays below 2^-25 of a quarter; the quarter swaps and negates.  For bf16 tensors the
// hardware's approximations serve: off by 2^-20 at most, 2^-11 of a bf16 step.
template <bool kPrecise>
__device__ __forceinline__ float2 turn_cos_sin(uint64_t fraction) {
  const uint32_t hi = (uint32_t)(fraction >> 32);
  const uint32_t quarter = (hi + 0x20000000u) >> 30;
  const int32_t rest = (int32_t)(hi - (quarter << 30));          // 2^-32 turns, |rest| <= 2^29
  float s, c;
  if constexpr (kPrecise) {
    sincospif((float)rest * 0x1p-31f, &s, &c);                   // half turns
  } else {
    const float x = (float)rest * 1.4629180792671596e-9f;        // 2 pi / 2^32
    s = __sinf(x);
    c = __cosf(x);
  }
  const float a = (quarter & 1u) ? s : c, b = (quarter & 1u) ? c : s;
  return make_float2((quarter + 1u) & 2u ? -a : a, quarter & 2u ? -b : b);
}

__device__ __forceinline__ float group_sum(float v, int group) {
  for (int o = group >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Element offsets of the two V-vectors of the chunk that starts at pair p0.  Adjacent pairs and the
// elements behind the turning ones are 2V consecutive elements; in the half layout the members of a
// pair are `turned` apart.
template <int V, bool kHalf>
__device__ __forceinline__ void chunk_offsets(int p0, int turned, int& ea, int& eb) {
  if (kHalf && p0 < turned) {
    ea = p0;
    eb = turned + p0;
  } else {
    ea = 2 * p0;
    eb = ea + V;
  }
}

enum { kRotate = 0, kNormRotate = 1, kNormRotateBackward = 2 };

// What a lane holds of a head: kSlots chunks of V pairs each (V * kSlots = 8 pairs), chunk s of lane j
// starting at pair (j + s * group) * V.
template <typename T, int V, bool kHalf>
struct LaneView {
  static constexpr int kSlots = 8 / V;
  int ea[kSlots], eb[kSlots];      // element offsets of the chunk's two vectors
  bool has[kSlots], turns[kSlots];

  __device__ __forceinline__ void init(const RotParams& p, int lane) {
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      const int p0 = (lane + s * p.group) * V;
      has[s] = p0 < p.pairs;
      turns[s] = p0 < p.turned;
      // a lane without a chunk loads the head's first one and is left out of sums and stores
      chunk_offsets<V, kHalf>(has[s] ? p0 : 0, p.turned, ea[s], eb[s]);
    }
  }
  struct Head {
    Raw<T, V> a[kSlots], b[kSlots];
  };
  __device__ __forceinline__ void load(const T* x, Head& r) const {
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      r.a[s].load(x + ea[s]);
      r.b[s].load(x + eb[s]);
    }
  }
  // the same from two 16-byte vectors (V = 8, bf16)
  static __device__ __forceinline__ void from_shared(const uint4& a, const uint4& b, Head& r) {
    uint32_t* w = r.a[0].u;
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w = r.b[0].u;
    w[0] = b.x; w[1] = b.y; w[2] = b.z; w[3] = b.w;
  }
  // A lane's pairs as packs: first members in a, second ones in b; pack j belongs to chunk slot(j).
  static constexpr int W = V == 1 ? 1 : 2, kPacks = 8 / W;
  static __device__ __forceinline__ constexpr int slot(int j) { return j * W / V; }
  using P = Pack<W>;
  static __device__ __forceinline__ void pairs(const float (&e)[16], P (&a)[kPacks], P (&b)[kPacks]) {
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
      const int at = 2 * V * slot(j), i = j * W % V;           // chunk, and pair in it
      float t[2], u[2];
#pragma unroll
      for (int k = 0; k < W; ++k) {
        t[k] = e[at + (kHalf ? i + k : 2 * (i + k))];
        u[k] = e[at + (kHalf ? V + i + k : 2 * (i + k) + 1)];
      }
      a[j] = P::of(t);
      b[j] = P::of(u);
    }
  }
  __device__ __forceinline__ void expand(const Head& r, P (&a)[kPacks], P (&b)[kPacks]) const {
    float e[16];
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      r.a[s].expand(e + 2 * V * s);
      r.b[s].expand(e + 2 * V * s + V);
    }
    pairs(e, a, b);
  }
  __device__ __forceinline__ void load_weight(const float* w, P (&wa)[kPacks], P (&wb)[kPacks]) const {
    float e[16];
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      Raw<float, V> a, b;
      a.load(w + ea[s]);
      b.load(w + eb[s]);
      a.expand(e + 2 * V * s);
      b.expand(e + 2 * V * s + V);
    }
    pairs(e, wa, wb);
  }
  // sum of a b + c d over what the lane holds
  __device__ __forceinline__ float sum_of_products(const P (&a)[kPacks], const P (&b)[kPacks], const P (&c)[kPacks], const P (&d)[kPacks]) const {
    float total = 0.f;
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      constexpr int kPer = V / W;                              // packs of a chunk
      P x = mul(a[s * kPer], b[s * kPer]), y = mul(c[s * kPer], d[s * kPer]);
#pragma unroll
      for (int j = 1; j < kPer; ++j) {
        x = fma(a[s * kPer + j], b[s * kPer + j], x);
        y = fma(c[s * kPer + j], d[s * kPer + j], y);
      }
      total += has[s] ? x.sum() + y.sum() : 0.f;
    }
    return total;
  }
  // pairs back to the order of the elements
  static __device__ __forceinline__ void elements(const P (&a)[kPacks], const P (&b)[kPacks], float (&e)[16]) {
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
      const int at = 2 * V * slot(j), i = j * W % V;
      float t[2], u[2];
      a[j].to(t);
      b[j].to(u);
#pragma unroll
      for (int k = 0; k < W; ++k) {
        e[at + (kHalf ? i + k : 2 * (i + k))] = t[k];
        e[at + (kHalf ? V + i + k : 2 * (i + k) + 1)] = u[k];
      }
    }
  }
  __device__ __forceinline__ void store(T* y, const P (&a)[kPacks], const P (&b)[kPacks]) const {
    float e[16];
    elements(a, b, e);
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      if (has[s]) {
        store_vec<T, V>(y + ea[s], e + 2 * V * s);
        store_vec<T, V>(y + eb[s], e + 2 * V * s + V);
      }
    }
  }
  // cosines and sines (times sign) of the lane's pairs for the token at (b, l); 1 and 0 for those that stay
  __device__ __forceinline__ void angles(const RotParams& p, int lane, int64_t b, int64_t l, float sign, float (&c)[8], float (&sn)[8]) const {
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      const int p0 = (lane + s * p.group) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        c[V * s + i] = 1.f;
        sn[V * s + i] = 0.f;
      }
      if (turns[s]) {
        const int64_t at = b * p.pos_sb + l * p.pos_st;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const uint32_t a = min((uint32_t)__ldg(p.axis + p0 + i), (uint32_t)(p.axes - 1));   // never outside the positions
          const int64_t j = at + (int64_t)a * p.pos_sa;
          const int64_t pos = p.pos_i64 ? __ldg(static_cast<const long long*>(p.pos) + j) : (int64_t)__ldg(static_cast<const int*>(p.pos) + j);
          const float2 cs = turn_cos_sin<sizeof(T) == 4>((uint64_t)pos * __ldg(reinterpret_cast<const unsigned long long*>(p.turns) + p0 + i));
          c[V * s + i] = cs.x;
          sn[V * s + i] = cs.y * sign;
        }
      }
    }
  }
};
// Asynchronous 16-byte copies to shared memory, waited for by the thread that started them.
__device__ __forceinline__ void copy_ahead(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_ahead_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void copy_ahead_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// Forward (and the plain rotation's backward).  A warp works on 32 / group tokens and one chunk of
// their heads; kBatch heads are in flight per lane, or (norm, bf16 in whole 16-byte vectors) kDepth heads through
// shared memory, each lane's own copies, which leaves registers for the factors: 121 -> 113 us, without the norm it
// made no difference.  Blocks in the order of the tokens, not persistent: what runs at one time then touches one
// stretch of memory (an even share of far-apart stretches for each resident warp took 271 instead of 204 us on
// 65536 tokens).  With the norm the weights are multiplied into the
// cosines and sines once per token and tensor, y = r (x_a (w_a c) - x_b (w_b s), x_a (w_a s) + x_b (w_b c)), six packed
// instructions for two pairs.
template <typename T, int V, bool kHalf, bool kNorm>
__global__ void __launch_bounds__(kRotThreads, 4) qk_rotary_kernel(const RotParams p) {
  constexpr bool kAhead = kNorm && sizeof(T) == 2 && V == 8;
  constexpr int kBatch = sizeof(T) == 4 ? 2 : V == 1 ? 2 : 4, kDepth = 4;      // 32 registers of raw vectors
  __shared__ uint4 ring[kAhead ? kDepth : 1][2][kAhead ? kRotThreads : 1];
  using View = LaneView<T, V, kHalf>;
  using P = typename View::P;
  constexpr int N = View::kPacks;
  const int lane = threadIdx.x & (p.group - 1);
  const int per_warp = 32 >> p.log_group;
  const int64_t unit = (int64_t)blockIdx.x * kRotWarps + (threadIdx.x >> 5);
  const int64_t tb = unit / p.chunks;
  const int chunk = (int)(unit - tb * p.chunks);
  const int64_t n = tb * per_warp + ((threadIdx.x & 31) >> p.log_group);
  if (tb * per_warp >= p.n) return;                       // the whole warp
  const bool token_live = n < p.n;
  const int64_t nn = token_live ? n : p.n - 1, b = nn / p.tokens, l = nn - b * p.tokens;
  View view;
  view.init(p, lane);
  float cf[8], sf[8];
  bool have_angles = false;
  const int h0 = chunk * p.chunk, h1 = h0 + p.chunk;      // heads of the chunk, keys behind the queries
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const int shift = which == 0 ? 0 : p.heads[0];
    const int first = max(h0 - shift, 0), last = min(h1 - shift, p.heads[which]);
    if (first >= last) continue;                          // warp-uniform
    const int64_t xs = p.x[which].sh, ys = p.y[which].sh;
    const T* x = static_cast<const T*>(p.x[which].p) + b * p.x[which].sb + l * p.x[which].st + first * xs;
    T* y = static_cast<T*>(p.y[which].p) + b * p.y[which].sb + l * p.y[which].st + first * ys;
    typename View::Head raw[kBatch];
    if constexpr (kAhead) {
#pragma unroll
      for (int u = 0; u < kDepth; ++u) {
        if (first + u < last) {
          copy_ahead(&ring[u][0][threadIdx.x], x + u * xs + view.ea[0]);
          copy_ahead(&ring[u][1][threadIdx.x], x + u * xs + view.eb[0]);
        }
        copy_ahead_commit();
      }
    } else {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) view.load(x + min(u, last - 1 - first) * xs, raw[u]);
    }
    if (!have_angles) {
      view.angles(p, lane, b, l, p.sign, cf, sf);
      have_angles = true;
    }
    // the four factors of a pair: y_a = x_a ka - x_b kb, y_b = x_a la + x_b lb
    P ka[N], kb[N], la[N], lb[N];
    if constexpr (kNorm) view.load_weight(p.w[which], ka, kb);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const P c = P::of(cf + j * View::W), sn = P::of(sf + j * View::W), minus = P::all(-1.f);
      if constexpr (kNorm) {
        const P wa = ka[j], wb = kb[j];
        ka[j] = mul(wa, c);
        la[j] = mul(wa, sn);
        kb[j] = mul(mul(wb, sn), minus);
        lb[j] = mul(wb, c);
      } else {
        ka[j] = lb[j] = c;
        la[j] = sn;
        kb[j] = mul(sn, minus);
      }
    }
    const auto work = [&](const typename View::Head& head, T* out) {
      P a[N], d[N];
      view.expand(head, a, d);
      P r = P::all(1.f);
      if constexpr (kNorm) r = P::all(rsqrtf(group_sum(view.sum_of_products(a, a, d, d), p.group) * p.inv_dim + p.eps));
#pragma unroll
      for (int j = 0; j < N; ++j) {
        P ya = a[j], yb = d[j];
        if (view.turns[View::slot(j)]) {
          ya = fma(d[j], kb[j], mul(a[j], ka[j]));
          yb = fma(d[j], lb[j], mul(a[j], la[j]));
        } else if constexpr (kNorm) {                     // c = 1: the factors are the weights
          ya = mul(a[j], ka[j]);
          yb = mul(d[j], lb[j]);
        }
        a[j] = kNorm ? mul(ya, r) : ya;
        d[j] = kNorm ? mul(yb, r) : yb;
      }
      if (token_live) view.store(out, a, d);
    };
    if constexpr (kAhead) {
      for (int h = first; h < last; ++h) {
        const int slot = (h - first) & (kDepth - 1);
        copy_ahead_wait<kDepth - 1>();
        view.from_shared(ring[slot][0][threadIdx.x], ring[slot][1][threadIdx.x], raw[0]);
        work(raw[0], y);
        if (h + kDepth < last) {
          copy_ahead(&ring[slot][0][threadIdx.x], x + kDepth * xs + view.ea[0]);
          copy_ahead(&ring[slot][1][threadIdx.x], x + kDepth * xs + view.eb[0]);
        }
        copy_ahead_commit();
        x += xs;
        y += ys;
      }
    } else {
      for (int h = first; h < last; h += kBatch) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
          if (h + u < last) work(raw[u], y + u * ys);     // warp-uniform
        x += kBatch * xs;
        y += kBatch * ys;
        if (h + kBatch < last) {
#pragma unroll
          for (int u = 0; u < kBatch; ++u) view.load(x + min(u, last - 1 - h - kBatch) * xs, raw[u]);
        }
      }
    }
  }
}

// Norm backward.  A block works on one of the tensors, so that a lane's weight gradients are 16 registers;
// persistent: they are kept over all its tokens and reduced once.
template <typename T, int V, bool kHalf>
__global__ void __launch_bounds__(kRotThreads, 4) qk_norm_rotary_bwd_kernel(const RotParams p) {
  // bf16 in whole 16-byte vectors is copied to shared memory kDepth heads ahead, each lane its own (nothing to wait for
  // but its own copies): 218 -> 190 us at 32768 tokens x 40 heads x 128.  Everything else is loaded into registers,
  // kBatch heads at a time (fp32 through shared memory took 179 instead of 138 us at 16384 tokens x 32 heads x 80).
  constexpr bool kAhead = sizeof(T) == 2 && V == 8;
  constexpr int kBatch = sizeof(T) == 4 || V == 1 ? 1 : 2, kDepth = 4;
  __shared__ uint4 ring[kAhead ? kDepth : 1][2][2][kAhead ? kRotThreads : 1];   // x, dy; the lane's two vectors
  __shared__ float red[kRotMaxDim];
  const int which = (int)blockIdx.x < p.blocks0 ? 0 : 1;
  const int block = which == 0 ? blockIdx.x : blockIdx.x - p.blocks0;
  const int blocks = which == 0 ? p.blocks0 : gridDim.x - p.blocks0;
  const HeadsIn px = p.x[which], pg = p.dy[which];
  const HeadsOut py = p.y[which];
  const int heads = p.heads[which];
  const int lane = threadIdx.x & (p.group - 1), warp = threadIdx.x >> 5;
  const int per_warp = 32 >> p.log_group;
  using View = LaneView<T, V, kHalf>;
  using P = typename View::P;
  constexpr int N = View::kPacks;
  View view;
  view.init(p, lane);
  // the weights wait in shared memory: their registers hold a second head's vectors instead
  __shared__ __align__(16) float ws[kRotMaxDim];
  for (int i = threadIdx.x; i < p.dim; i += kRotThreads) ws[i] = p.w[which][i];
  __syncthreads();
  P dwa[N], dwb[N];
#pragma unroll
  for (int j = 0; j < N; ++j) dwa[j] = dwb[j] = P::all(0.f);
  const int chunks = (heads + p.chunk - 1) / p.chunk;
  const int64_t units = (p.n + per_warp - 1) / per_warp * chunks;
  for (int64_t unit = (int64_t)block * kRotWarps + warp; unit < units; unit += (int64_t)blocks * kRotWarps) {
    const int64_t tb = unit / chunks;
    const int first = (int)(unit - tb * chunks) * p.chunk, last = min(first + p.chunk, heads);
    const int64_t n = tb * per_warp + ((threadIdx.x & 31) >> p.log_group);
    const bool live = n < p.n;
    const int64_t nn = live ? n : p.n - 1, b = nn / p.tokens, l = nn - b * p.tokens;
    const T* x = static_cast<const T*>(px.p) + b * px.sb + l * px.st + first * px.sh;
    const T* g = static_cast<const T*>(pg.p) + b * pg.sb + l * pg.st + first * pg.sh;
    T* y = static_cast<T*>(py.p) + b * py.sb + l * py.st + first * py.sh;
    typename View::Head raw_x[kBatch], raw_g[kBatch];
    const auto ahead = [&](int slot, int k) {              // starts the copies of the k-th head from `first` on
      if constexpr (kAhead) {
        copy_ahead(&ring[slot][0][0][threadIdx.x], x + k * px.sh + view.ea[0]);
        copy_ahead(&ring[slot][0][1][threadIdx.x], x + k * px.sh + view.eb[0]);
        copy_ahead(&ring[slot][1][0][threadIdx.x], g + k * pg.sh + view.ea[0]);
        copy_ahead(&ring[slot][1][1][threadIdx.x], g + k * pg.sh + view.eb[0]);
      }
    };
    if constexpr (kAhead) {
#pragma unroll
      for (int k = 0; k < kDepth; ++k) {
        if (first + k < last) ahead(k, k);
        copy_ahead_commit();
      }
    } else {
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        view.load(x + min(k, last - 1 - first) * px.sh, raw_x[k]);
        view.load(g + min(k, last - 1 - first) * pg.sh, raw_g[k]);
      }
    }
    P c[N], sn[N];
    {
      float cf[8], sf[8];
      view.angles(p, lane, b, l, -1.f, cf, sf);           // back
#pragma unroll
      for (int j = 0; j < N; ++j) {
        c[j] = P::of(cf + j * View::W);
        sn[j] = P::of(sf + j * View::W);
      }
    }
    // one head, its vectors in registers
    const auto work = [&](const typename View::Head& hx, const typename View::Head& hg, T* out) {
      P xa[N], xb[N], ga[N], gb[N];
      view.expand(hx, xa, xb);
      view.expand(hg, ga, gb);
      const float r = rsqrtf(group_sum(view.sum_of_products(xa, xa, xb, xb), p.group) * p.inv_dim + p.eps);
      // t = r R(-angle) dy;  dw += t x;  u = t w;  dx = u - x r^2 mean(u x)
      const P rr = P::all(r), minus = P::all(-1.f);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (view.turns[View::slot(j)]) {
          const P ta = fma(mul(gb[j], minus), sn[j], mul(ga[j], c[j]));
          gb[j] = fma(gb[j], c[j], mul(ga[j], sn[j]));
          ga[j] = ta;
        }
        ga[j] = mul(ga[j], rr);
        gb[j] = mul(gb[j], rr);
        if (live) {                                   // a group behind the last token repeats it and adds nothing
          dwa[j] = fma(ga[j], xa[j], dwa[j]);
          dwb[j] = fma(gb[j], xb[j], dwb[j]);
        }
      }
      {
        P wa[N], wb[N];
        view.load_weight(ws, wa, wb);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          ga[j] = mul(ga[j], wa[j]);
          gb[j] = mul(gb[j], wb[j]);
        }
      }
      const float dot = group_sum(view.sum_of_products(ga, xa, gb, xb), p.group) * p.inv_dim;
      const P f = P::all(-r * r * dot);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        ga[j] = fma(xa[j], f, ga[j]);
        gb[j] = fma(xb[j], f, gb[j]);
      }
      if (live) view.store(out, ga, gb);
    };
    if constexpr (kAhead) {
      for (int h = first; h < last; ++h) {
        const int slot = (h - first) & (kDepth - 1);
        copy_ahead_wait<kDepth - 1>();
        view.from_shared(ring[slot][0][0][threadIdx.x], ring[slot][0][1][threadIdx.x], raw_x[0]);
        view.from_shared(ring[slot][1][0][threadIdx.x], ring[slot][1][1][threadIdx.x], raw_g[0]);
        work(raw_x[0], raw_g[0], y + (h - first) * py.sh);
        if (h + kDepth < last) ahead(slot, h - first + kDepth);
        copy_ahead_commit();
      }
    } else {
      for (int h = first; h < last; h += kBatch) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
          if (h + k < last) work(raw_x[k], raw_g[k], y + k * py.sh);      // warp-uniform
        x += kBatch * px.sh;
        g += kBatch * pg.sh;
        y += kBatch * py.sh;
        if (h + kBatch < last) {
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            view.load(x + min(k, last - 1 - h - kBatch) * px.sh, raw_x[k]);
            view.load(g + min(k, last - 1 - h - kBatch) * pg.sh, raw_g[k]);
          }
        }
      }
    }
  }
  float dw[16];
  View::elements(dwa, dwb, dw);
  // The block's weight gradients: the groups of a warp by shuffles, the warps in warp order, then one
  // row of the workspace -- a fixed association, whatever the scheduling.
#pragma unroll
  for (int i = 0; i < 16; ++i)
    for (int o = p.group; o < 32; o <<= 1) dw[i] += __shfl_xor_sync(0xFFFFFFFFu, dw[i], o);
  for (int wi = 0; wi < kRotWarps; ++wi) {
    if (warp == wi && (threadIdx.x & 31) < p.group) {
#pragma unroll
      for (int s = 0; s < view.kSlots; ++s) {
        if (view.has[s]) {
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) {
            float* at = red + (i < V ? view.ea[s] + i : view.eb[s] + i - V);
            *at = wi == 0 ? dw[2 * V * s + i] : *at + dw[2 * V * s + i];
          }
        }
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < p.dim; i += kRotThreads) p.partial[(size_t)blockIdx.x * p.dim + i] = red[i];
}

// dweight[c] = sum over a tensor's blocks' partial rows, in a fixed order: one block per 32 columns of a
// tensor, warp w adds rows w, w + 32, ..., then the warps' sums are added in warp order.
__global__ void __launch_bounds__(1024) qk_weight_grad_kernel(const float* __restrict__ partial, int blocks0, int blocks, int dim,
                                                              float* __restrict__ dq, float* __restrict__ dk) {
  __shared__ float red[32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + lane;
  const int from = blockIdx.y == 0 ? 0 : blocks0, to = blockIdx.y == 0 ? blocks0 : blocks;
  float s = 0.f;
  if (i < dim) {
#pragma unroll 8
    for (int k = from + warp; k < to; k += 32) s += partial[(size_t)k * dim + i];
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && i < dim) {
    float v = 0.f;
    for (int w = 0; w < 32; ++w) v += red[w][lane];
    (blockIdx.y == 0 ? dq : dk)[i] = v;
  }
}

using RotKernel = void (*)(const RotParams);

template <typename T, int V, bool kHalf>
RotKernel pick_mode(int mode) {
  return mode == kRotate ? qk_rotary_kernel<T, V, kHalf, false>
         : mode == kNormRotate ? qk_rotary_kernel<T, V, kHalf, true> : qk_norm_rotary_bwd_kernel<T, V, kHalf>;
}
template <typename T, int V>
RotKernel pick_layout(bool half, int mode) {
  return half ? pick_mode<T, V, true>(mode) : pick_mode<T, V, false>(mode);
}
template <typename T>
RotKernel pick_width(int v, bool half, int mode) {
  return v == 8 ? pick_layout<T, 8>(half, mode) : v == 4 ? pick_layout<T, 4>(half, mode)
         : v == 2 ? pick_layout<T, 2>(half, mode) : pick_layout<T, 1>(half, mode);
}

int check_heads(const char* name, const char* what, const fp4t_heads_t* t, int count, const fp4t_heads_t* like) {
  FP4T_REQUIRE(t, "%s: %s is null", name, what);
  for (int i = 0; i < count; ++i) {
    FP4T_REQUIRE(t[i].heads > 0 && t[i].heads <= 65535, "%s: %s[%d] has %lld heads", name, what, i, (long long)t[i].heads);
    FP4T_REQUIRE(t[i].heads == like[i].heads, "%s: %s[%d] has another number of heads than x", name, what, i);
  }
  return FP4T_OK;
}

bool aligned_to(const fp4t_heads_t* t, int count, int elem, int64_t vec_bytes) {
  for (int i = 0; i < count; ++i)
    if (reinterpret_cast<uintptr_t>(t[i].data) % vec_bytes || (t[i].stride_batch * elem) % vec_bytes ||
        (t[i].stride_token * elem) % vec_bytes || (t[i].stride_head * elem) % vec_bytes)
      return false;
  return true;
}

int run(const char* name, int mode, const fp4t_heads_t* x, const fp4t_heads_t* dy, const fp4t_heads_t* y, int count, int dtype,
        int64_t batch, int64_t tokens, int64_t dim, const fp4t_rotary_t* rot, int inverse, const float* const* w, float eps,
        float* const* dw, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  FP4T_REQUIRE(count == 1 || count == 2, "%s: count must be 1 or 2", name);
  FP4T_REQUIRE(dtype == FP4T_DT_F32 || dtype == FP4T_DT_BF16, "%s: dtype must be f32 or bf16", name);
  FP4T_REQUIRE(batch >= 0 && tokens >= 0 && (tokens == 0 || batch <= INT64_MAX / 65536 / (tokens + 1)), "%s: bad shape batch=%lld tokens=%lld", name,
               (long long)batch, (long long)tokens);
  FP4T_REQUIRE(dim >= 2 && dim % 2 == 0 && dim <= kRotMaxDim, "%s: head_dim (%lld) must be even, at most %d", name, (long long)dim, kRotMaxDim);
  FP4T_REQUIRE(x, "%s: x is null", name);
  int rc = check_heads(name, "x", x, count, x);
  if (rc == FP4T_OK) rc = check_heads(name, "y", y, count, x);
  if (rc == FP4T_OK && mode == kNormRotateBackward) rc = check_heads(name, "dy", dy, count, x);
  if (rc != FP4T_OK) return rc;
  FP4T_REQUIRE(rot, "%s: the rotary description is null", name);
  FP4T_REQUIRE(rot->turned >= 0 && 2 * (int64_t)rot->turned <= dim, "%s: %d turning pairs do not fit head_dim %lld", name, rot->turned, (long long)dim);
  const bool empty = batch == 0 || tokens == 0;
  if (rot->turned > 0) {
    FP4T_REQUIRE(rot->axes >= 1 && rot->turns && rot->axis && (empty || rot->positions), "%s: null positions or frequency table", name);
    FP4T_REQUIRE(reinterpret_cast<uintptr_t>(rot->turns) % 8 == 0 && reinterpret_cast<uintptr_t>(rot->axis) % 4 == 0 &&
                     reinterpret_cast<uintptr_t>(rot->positions) % (rot->positions_i64 ? 8 : 4) == 0,
                 "%s: misaligned positions or frequency table", name);
  }
  const int elem = dtype == FP4T_DT_F32 ? 4 : 2;
  const bool norm = mode != kRotate;
  for (int i = 0; i < count; ++i) {
    FP4T_REQUIRE(empty || (x[i].data && y[i].data && (mode != kNormRotateBackward || dy[i].data)), "%s: null pointer", name);
    FP4T_REQUIRE(!norm || (w && w[i] && reinterpret_cast<uintptr_t>(w[i]) % 16 == 0), "%s: weights must be 16-byte aligned", name);
    if (mode == kNormRotateBackward) FP4T_REQUIRE(dw && dw[i], "%s: null weight gradient", name);
  }
  FP4T_REQUIRE(aligned_to(x, count, elem, elem) && aligned_to(y, count, elem, elem) &&
                   (mode != kNormRotateBackward || aligned_to(dy, count, elem, elem)),
               "%s: a tensor is not aligned to its elements", name);
  if (norm) FP4T_REQUIRE(eps >= 0.0f, "%s: eps must not be negative", name);
  if (mode == kNormRotateBackward) FP4T_REQUIRE(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: the workspace must be 16-byte aligned", name);
  const int64_t row_bytes = dim * (int64_t)sizeof(float);        // of the workspace: one row per block
  if (mode == kNormRotateBackward) FP4T_REQUIRE(workspace_bytes >= count * row_bytes, "%s: the workspace holds %lld bytes, %lld are the least", name,
                                                (long long)workspace_bytes, (long long)(count * row_bytes));
  if (empty) {
    if (mode == kNormRotateBackward)
      for (int i = 0; i < count; ++i) FP4T_CUDA(cudaMemsetAsync(dw[i], 0, (size_t)dim * sizeof(float), stream));
    return FP4T_OK;
  }
  const int sms = sm_count();
  if (sms <= 0) {
    set_error("%s: the current device is not an sm_100 part", name);
    return FP4T_ERR_DEVICE;
  }
  RotParams p = {};
  for (int i = 0; i < count; ++i) {
    p.x[i] = HeadsIn{x[i].data, x[i].stride_batch, x[i].stride_token, x[i].stride_head};
    p.y[i] = HeadsOut{y[i].data, y[i].stride_batch, y[i].stride_token, y[i].stride_head};
    if (mode == kNormRotateBackward) p.dy[i] = HeadsIn{dy[i].data, dy[i].stride_batch, dy[i].stride_token, dy[i].stride_head};
    p.heads[i] = (int)x[i].heads;
    if (norm) p.w[i] = w[i];
  }
  p.eps = eps;
  p.inv_dim = 1.0f / (float)dim;
  p.n = batch * tokens;
  p.tokens = tokens;
  p.dim = (int)dim;
  p.pairs = (int)dim / 2;
  p.turned = rot->turned;
  p.pos = rot->positions;
  p.pos_i64 = rot->positions_i64;
  p.axes = rot->axes;
  p.pos_sb = rot->stride_batch;
  p.pos_st = rot->stride_token;
  p.pos_sa = rot->stride_axis;
  p.turns = rot->turns;
  p.axis = rot->axis;
  p.sign = inverse ? -1.f : 1.f;
  p.partial = static_cast<float*>(workspace);
  const bool half = !rot->interleaved;
  // The widest vector that every pointer, stride and chunk boundary allows.
  int v = 8;
  for (; v > 1; v >>= 1) {
    const int64_t vec = std::min<int64_t>(16, (int64_t)v * elem);
    if (p.pairs % v == 0 && p.turned % v == 0 && aligned_to(x, count, elem, vec) && aligned_to(y, count, elem, vec) &&
        (mode != kNormRotateBackward || aligned_to(dy, count, elem, vec)))
      break;
  }
  const int lanes = (p.pairs + 7) / 8;
  p.group = 1;
  while (p.group < lanes) {
    p.group <<= 1;
    ++p.log_group;
  }
  // A token's heads go to one group unless that leaves warps short of eight per SM (about the number that
  // hides the loads' latency); then they are dealt out, down to one head per group.
  const int per_warp = 32 >> p.log_group;
  const int64_t token_warps = ceil_div(p.n, per_warp);
  const auto chunk_for = [&](int heads) { return (int)ceil_div(heads, std::min<int64_t>(heads, ceil_div(8ll * sms, token_warps))); };
  RotKernel kern = dtype == FP4T_DT_F32 ? pick_width<float>(v, half, mode) : pick_width<__nv_bfloat16>(v, half, mode);
  if (mode != kNormRotateBackward) {
    const int heads = p.heads[0] + p.heads[1];
    p.chunk = chunk_for(heads);
    p.chunks = (int)ceil_div(heads, p.chunk);
    const int64_t blocks = ceil_div(token_warps * p.chunks, kRotWarps);
    FP4T_REQUIRE(blocks <= INT32_MAX, "%s: too many tokens", name);
    kern<<<(unsigned)blocks, kRotThreads, 0, stream>>>(p);
    FP4T_CUDA(cudaGetLastError());
    return FP4T_OK;
  }
  // Persistent blocks, kRotBlocksPerSm per SM, dealt out to the tensors by their heads; no more than there is work or
  // workspace for.  A token's heads are split into up to eight parts where the blocks' rounds then come out more even; a
  // part costs the angles again, about a head's work (16384 tokens x 32 heads x 80 fp32: 138 -> 130 us, bf16 heads of
  // 128, bound by memory, the same either way).
  const int most = std::max(p.heads[0], p.heads[1]);
  const int64_t room = std::min<int64_t>((int64_t)kRotBlocksPerSm * sms, workspace_bytes / row_bytes);
  const int64_t share = count == 1 ? room : std::max<int64_t>(1, std::min<int64_t>(room - 1, room * p.heads[0] / (p.heads[0] + p.heads[1])));
  int64_t b0 = 0, b1 = 0, best = INT64_MAX;
  const int whole = chunk_for(most);
  for (int parts = 1; parts <= 8; ++parts) {
    const int chunk = (int)ceil_div(whole, parts);
    const auto units = [&](int i) { return token_warps * ceil_div(p.heads[i], chunk); };
    const auto blocks_for = [&](int i) { return std::max<int64_t>(1, ceil_div(units(i), kRotWarps)); };
    int64_t n0 = blocks_for(0), n1 = count == 2 ? blocks_for(1) : 0;
    if (n0 + n1 > room) {
      n0 = std::min(n0, share);
      n1 = std::min(n1, room - share);
    }
    int64_t steps = ceil_div(units(0), n0 * kRotWarps) * (std::min(chunk, p.heads[0]) + 1);
    if (count == 2) steps = std::max(steps, ceil_div(units(1), n1 * kRotWarps) * (std::min(chunk, p.heads[1]) + 1));
    if (steps < best) {
      best = steps;
      b0 = n0;
      b1 = n1;
      p.chunk = chunk;
    }
  }
  p.blocks0 = (int)b0;
  kern<<<(unsigned)(b0 + b1), kRotThreads, 0, stream>>>(p);
  FP4T_CUDA(cudaGetLastError());
  qk_weight_grad_kernel<<<dim3((unsigned)ceil_div(dim, 32), (unsigned)count), 1024, 0, stream>>>(p.partial, (int)b0, (int)(b0 + b1), (int)dim,
                                                                                                dw[0], count == 2 ? dw[1] : nullptr);
  FP4T_CUDA(cudaGetLastError());
  return FP4T_OK;
}

}  // namespace
}  // namespace fp4t

using namespace fp4t;

extern "C" int fp4t_rotary(const fp4t_heads_t* x, const fp4t_heads_t* y, int count, int dtype, int64_t batch, int64_t tokens,
                           int64_t head_dim, const fp4t_rotary_t* rotary, int inverse, fp4t_stream_t stream) {
  return run("fp4t_rotary", kRotate, x, nullptr, y, count, dtype, batch, tokens, head_dim, rotary, inverse, nullptr, 0.f, nullptr,
             nullptr, 0, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int fp4t_qk_norm_rotary_forward(const fp4t_heads_t* x, const float* const* weights, float eps, const fp4t_heads_t* y,
                                           int count, int dtype, int64_t batch, int64_t tokens, int64_t head_dim,
                                           const fp4t_rotary_t* rotary, fp4t_stream_t stream) {
  return run("fp4t_qk_norm_rotary_forward", kNormRotate, x, nullptr, y, count, dtype, batch, tokens, head_dim, rotary, 0, weights, eps,
             nullptr, nullptr, 0, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int64_t fp4t_qk_norm_rotary_backward_workspace_bytes(int64_t head_dim) {
  const int sms = sm_count();
  if (head_dim < 2 || head_dim > kRotMaxDim || sms <= 0) return -1;
  return (int64_t)sms * kRotBlocksPerSm * head_dim * (int64_t)sizeof(float);
}

extern "C" int fp4t_qk_norm_rotary_backward(const fp4t_heads_t* dy, const fp4t_heads_t* x, const float* const* weights, float eps,
                                            const fp4t_heads_t* dx, float* const* dweights, int count, int dtype, int64_t batch,
                                            int64_t tokens, int64_t head_dim, const fp4t_rotary_t* rotary, void* workspace,
                                            int64_t workspace_bytes, fp4t_stream_t stream) {
  return run("fp4t_qk_norm_rotary_backward", kNormRotateBackward, x, dy, dx, count, dtype, batch, tokens, head_dim, rotary, 0, weights,
             eps, dweights, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}
