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
// product is off by 0.06 radians there) and costs one integer multiply, no fp64.  Cosine and sine of a
// (token, pair) are computed once per tile of tokens into shared memory and used by all heads of
// queries AND keys of the token; with 3 + 3 heads the trigonometry is a third of the instructions,
// with 32 + 8 it disappears.
//
// A head is held by a group of 1 to 32 lanes, up to eight pairs (two 16-byte vectors of bf16) a lane, so the
// norm is a shuffle reduction inside the group and every element is read and written once:
// HBM-bound (forward 4 bytes per bf16 element, norm backward 6).
#include <algorithm>

#include "fp4t_common.cuh"

namespace fp4t {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotWarps = kRotThreads / 32;
constexpr int kRotMaxTile = 32;           // tokens per tile
constexpr int kRotMaxDim = 512;           // 256 pairs: 32 lanes x 8
constexpr int kRotTableBytes = 32768;     // cosines and sines of one tile
constexpr int kRotBlocksPerSm = 4;        // upper bound of the backward grid per SM (workspace size)

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
  int tile;                               // tokens per tile
  const void* pos;
  int pos_i64, axes;
  int64_t pos_sb, pos_st, pos_sa;
  const uint64_t* turns;
  const int32_t* axis;
  float sign;                             // -1: rotate back
  float* partial;                         // norm backward: [gridDim.x][2][dim]
};

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (V >= 4) {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 f = *reinterpret_cast<const float4*>(p + i);
        v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
      }
    } else if constexpr (V == 2) {
      const float2 f = *reinterpret_cast<const float2*>(p);
      v[0] = f.x; v[1] = f.y;
    } else {
      v[0] = *p;
    }
  } else if constexpr (V == 1) {
    v[0] = __bfloat162float(*p);
  } else {
    uint32_t u[V / 2];
    if constexpr (V == 8) {
      const uint4 q = *reinterpret_cast<const uint4*>(p);
      u[0] = q.x; u[1] = q.y; u[2] = q.z; u[3] = q.w;
    } else if constexpr (V == 4) {
      const uint2 q = *reinterpret_cast<const uint2*>(p);
      u[0] = q.x; u[1] = q.y;
    } else {
      u[0] = *reinterpret_cast<const uint32_t*>(p);
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  }
}

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
// a turn and its rounding stays below 2^-25 of a quarter; the quarter swaps and negates.
__device__ __forceinline__ float2 turn_cos_sin(uint64_t fraction) {
  const uint32_t hi = (uint32_t)(fraction >> 32);
  const uint32_t quarter = (hi + 0x20000000u) >> 30;
  const int32_t rest = (int32_t)(hi - (quarter << 30));          // 2^-32 turns, |rest| <= 2^29
  float s, c;
  sincospif((float)rest * 0x1p-31f, &s, &c);                     // half turns
  const float a = (quarter & 1u) ? s : c, b = (quarter & 1u) ? c : s;
  return make_float2((quarter + 1u) & 2u ? -a : a, quarter & 2u ? -b : b);
}

// Index of pair p's cosine in a tile row: for eight-pair lanes the row is two halves, so that the
// 16-byte reads of neighbouring lanes touch different banks.
template <int V>
__device__ __forceinline__ int table_index(int p, int turned) {
  if constexpr (V == 8) return ((p >> 2) & 1) * (turned >> 1) + (p >> 3) * 4 + (p & 3);
  else return p;
}
template <int V>
__device__ __forceinline__ void load_table(const float* row, int p0, int turned, float* v) {
  if constexpr (V == 8) {
    const float4 a = *reinterpret_cast<const float4*>(row + (p0 >> 1));
    const float4 b = *reinterpret_cast<const float4*>(row + (turned >> 1) + (p0 >> 1));
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else if constexpr (V == 4) {
    const float4 a = *reinterpret_cast<const float4*>(row + p0);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else if constexpr (V == 2) {
    const float2 a = *reinterpret_cast<const float2*>(row + p0);
    v[0] = a.x; v[1] = a.y;
  } else {
    v[0] = row[p0];
  }
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

// Rotates the chunk in place by (cos, sin): e[0..V) and e[V..2V) are the two vectors.
template <int V, bool kHalf>
__device__ __forceinline__ void turn_chunk(float* e, const float* c, const float* s, float sign) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int ia = kHalf ? i : 2 * i, ib = kHalf ? V + i : 2 * i + 1;
    const float a = e[ia], b = e[ib], sn = s[i] * sign;
    e[ia] = a * c[i] - b * sn;
    e[ib] = a * sn + b * c[i];
  }
}

enum { kRotate = 0, kNormRotate = 1, kNormRotateBackward = 2 };

// V pairs per vector, kSlots vectors pairs per lane (V * kSlots = 8 pairs).
template <typename T, int V, bool kHalf, int kMode>
__global__ void __launch_bounds__(kRotThreads) qk_rotary_kernel(const RotParams p) {
  constexpr int kSlots = 8 / V;
  constexpr bool kNorm = kMode != kRotate, kBack = kMode == kNormRotateBackward;
  extern __shared__ __align__(16) float table[];        // [tile][2][turned]; reused for the weight gradients
  __shared__ int64_t off_x[2][kRotMaxTile], off_y[2][kRotMaxTile], off_g[2][kRotMaxTile];
  const int lane_in_group = threadIdx.x & (p.group - 1);
  const int first = threadIdx.x >> p.log_group, stride = kRotThreads >> p.log_group;
  float dw[2][16];
  if (kBack) {
#pragma unroll
    for (int i = 0; i < 16; ++i) dw[0][i] = dw[1][i] = 0.f;
  }
  const int64_t tiles = (p.n + p.tile - 1) / p.tile;
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t n0 = t * p.tile;
    const int count = (int)min((int64_t)p.tile, p.n - n0);
    __syncthreads();                                     // the previous tile's table is no longer read
    if (threadIdx.x < count) {
      const int64_t n = n0 + threadIdx.x, b = n / p.tokens, l = n - b * p.tokens;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        off_x[i][threadIdx.x] = b * p.x[i].sb + l * p.x[i].st;
        off_y[i][threadIdx.x] = b * p.y[i].sb + l * p.y[i].st;
        if (kBack) off_g[i][threadIdx.x] = b * p.dy[i].sb + l * p.dy[i].st;
      }
    }
    for (int i = threadIdx.x; i < count * p.turned; i += kRotThreads) {
      const int tok = i / p.turned, pr = i - tok * p.turned;
      const int64_t n = n0 + tok, b = n / p.tokens, l = n - b * p.tokens;
      const uint32_t a = min((uint32_t)__ldg(p.axis + pr), (uint32_t)(p.axes - 1));   // never outside the positions
      const int64_t at = b * p.pos_sb + l * p.pos_st + (int64_t)a * p.pos_sa;
      const int64_t pos = p.pos_i64 ? __ldg(static_cast<const long long*>(p.pos) + at) : (int64_t)__ldg(static_cast<const int*>(p.pos) + at);
      const float2 cs = turn_cos_sin((uint64_t)pos * __ldg(reinterpret_cast<const unsigned long long*>(p.turns) + pr));
      const int j = table_index<V>(pr, p.turned);
      table[(2 * tok) * p.turned + j] = cs.x;
      table[(2 * tok + 1) * p.turned + j] = cs.y;
    }
    __syncthreads();
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int heads = p.heads[which];
      const int items = count * heads;
      const T* x0 = static_cast<const T*>(p.x[which].p);
      T* y0 = static_cast<T*>(p.y[which].p);
      // all lanes of a warp take the same number of turns (shuffles); groups behind the last item idle
      const int rounds = (items + stride - 1) / stride;
      for (int it = 0; it < rounds; ++it) {
        const int item = first + it * stride;
        const bool live = item < items;
        const int tok = live ? item / heads : 0, head = live ? item - tok * heads : 0;
        const T* x = x0 + off_x[which][tok] + head * p.x[which].sh;
        T* y = y0 + off_y[which][tok] + head * p.y[which].sh;
        const float* crow = table + 2 * tok * p.turned;
        const float* srow = crow + p.turned;
        float e[kSlots][2 * V];
        float sq = 0.f;
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
          const int p0 = (lane_in_group + s * p.group) * V;
          if (live && p0 < p.pairs) {
            int ea, eb;
            chunk_offsets<V, kHalf>(p0, p.turned, ea, eb);
            load_vec<T, V>(x + ea, e[s]);
            load_vec<T, V>(x + eb, e[s] + V);
          } else {
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) e[s][i] = 0.f;
          }
          if (kNorm) {
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) sq = fmaf(e[s][i], e[s][i], sq);
          }
        }
        float r = 1.f;
        if (kNorm) r = rsqrtf(group_sum(sq, p.group) * p.inv_dim + p.eps);
        if (!kBack) {
          if (!live) continue;                           // no shuffles below
#pragma unroll
          for (int s = 0; s < kSlots; ++s) {
            const int p0 = (lane_in_group + s * p.group) * V;
            if (p0 >= p.pairs) continue;
            int ea, eb;
            chunk_offsets<V, kHalf>(p0, p.turned, ea, eb);
            if (kNorm) {
              float w[2 * V];
              load_vec<float, V>(p.w[which] + ea, w);
              load_vec<float, V>(p.w[which] + eb, w + V);
#pragma unroll
              for (int i = 0; i < 2 * V; ++i) e[s][i] = (e[s][i] * r) * w[i];
            }
            if (p0 < p.turned) {
              float c[V], sn[V];
              load_table<V>(crow, p0, p.turned, c);
              load_table<V>(srow, p0, p.turned, sn);
              turn_chunk<V, kHalf>(e[s], c, sn, p.sign);
            }
            store_vec<T, V>(y + ea, e[s]);
            store_vec<T, V>(y + eb, e[s] + V);
          }
        } else {
          const T* dy = static_cast<const T*>(p.dy[which].p) + off_g[which][tok] + head * p.dy[which].sh;
          float u[kSlots][2 * V];
          float dot = 0.f;
#pragma unroll
          for (int s = 0; s < kSlots; ++s) {
            const int p0 = (lane_in_group + s * p.group) * V;
            if (live && p0 < p.pairs) {
              int ea, eb;
              chunk_offsets<V, kHalf>(p0, p.turned, ea, eb);
              load_vec<T, V>(dy + ea, u[s]);
              load_vec<T, V>(dy + eb, u[s] + V);
              if (p0 < p.turned) {
                float c[V], sn[V];
                load_table<V>(crow, p0, p.turned, c);
                load_table<V>(srow, p0, p.turned, sn);
                turn_chunk<V, kHalf>(u[s], c, sn, -1.f);
              }
              float w[2 * V];
              load_vec<float, V>(p.w[which] + ea, w);
              load_vec<float, V>(p.w[which] + eb, w + V);
#pragma unroll
              for (int i = 0; i < 2 * V; ++i) {
                e[s][i] *= r;                                               // xh
                dw[which][s * 2 * V + i] = fmaf(u[s][i], e[s][i], dw[which][s * 2 * V + i]);
                u[s][i] *= w[i];
                dot = fmaf(u[s][i], e[s][i], dot);
              }
            }
          }
          dot = group_sum(dot, p.group) * p.inv_dim;
          if (!live) continue;
#pragma unroll
          for (int s = 0; s < kSlots; ++s) {
            const int p0 = (lane_in_group + s * p.group) * V;
            if (p0 >= p.pairs) continue;
            int ea, eb;
            chunk_offsets<V, kHalf>(p0, p.turned, ea, eb);
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) u[s][i] = r * (u[s][i] - e[s][i] * dot);
            store_vec<T, V>(y + ea, u[s]);
            store_vec<T, V>(y + eb, u[s] + V);
          }
        }
      }
    }
  }
  if (kBack) {
    // The block's weight gradients: the groups of a warp by shuffles, the warps in warp order, then one
    // row of the workspace -- a fixed association, whatever the scheduling.
    float* red = table;                                  // [2][dim]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        for (int o = p.group; o < 32; o <<= 1) dw[which][i] += __shfl_xor_sync(0xFFFFFFFFu, dw[which][i], o);
    }
    for (int wi = 0; wi < kRotWarps; ++wi) {
      __syncthreads();
      if (warp == wi && lane < p.group) {
#pragma unroll
        for (int which = 0; which < 2; ++which) {
#pragma unroll
          for (int s = 0; s < kSlots; ++s) {
            const int p0 = (lane + s * p.group) * V;
            if (p0 >= p.pairs) continue;
            int ea, eb;
            chunk_offsets<V, kHalf>(p0, p.turned, ea, eb);
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) {
              float* at = red + which * p.dim + (i < V ? ea + i : eb + i - V);
              *at = wi == 0 ? dw[which][s * 2 * V + i] : *at + dw[which][s * 2 * V + i];
            }
          }
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.dim; i += kRotThreads) p.partial[(size_t)blockIdx.x * 2 * p.dim + i] = red[i];
  }
}

// dweight[c] = sum over the blocks' partial rows, in a fixed order: one block per 32 columns, warp w adds
// rows w, w + 32, ..., then the warps' sums are added in warp order.
__global__ void __launch_bounds__(1024) qk_weight_grad_kernel(const float* __restrict__ partial, int parts, int dim,
                                                              float* __restrict__ dq, float* __restrict__ dk) {
  __shared__ float red[32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (i < 2 * dim)
    for (int k = warp; k < parts; k += 32) s += partial[(size_t)k * 2 * dim + i];
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && i < 2 * dim) {
    float v = 0.f;
    for (int w = 0; w < 32; ++w) v += red[w][lane];
    if (i < dim) dq[i] = v;
    else if (dk != nullptr) dk[i - dim] = v;
  }
}

using RotKernel = void (*)(const RotParams);

template <typename T, int V, bool kHalf>
RotKernel pick_mode(int mode) {
  return mode == kRotate ? qk_rotary_kernel<T, V, kHalf, kRotate>
         : mode == kNormRotate ? qk_rotary_kernel<T, V, kHalf, kNormRotate> : qk_rotary_kernel<T, V, kHalf, kNormRotateBackward>;
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
  const int64_t row_bytes = 2 * dim * (int64_t)sizeof(float);    // of the workspace: one row per block
  if (mode == kNormRotateBackward) FP4T_REQUIRE(workspace_bytes >= row_bytes, "%s: the workspace holds %lld bytes, %lld are the least", name,
                                                (long long)workspace_bytes, (long long)row_bytes);
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
  // Tokens per tile: enough items for two rounds of all groups, a table of at most 32 KB, and no
  // fewer tiles than SMs while there are tokens to spread.
  const int per_round = kRotThreads >> p.log_group, heads = p.heads[0] + p.heads[1];
  int64_t tile = std::max<int64_t>(1, (2 * per_round + heads - 1) / heads);
  tile = std::max<int64_t>(tile, 4);
  tile = std::min<int64_t>(tile, kRotMaxTile);
  if (p.turned > 0) tile = std::min<int64_t>(tile, kRotTableBytes / (8 * p.turned));
  tile = std::min<int64_t>(tile, std::max<int64_t>(1, p.n / (2 * sms)));
  p.tile = (int)tile;
  RotKernel kern = dtype == FP4T_DT_F32 ? pick_width<float>(v, half, mode) : pick_width<__nv_bfloat16>(v, half, mode);
  const size_t smem = std::max((size_t)tile * 2 * p.turned * 4, mode == kNormRotateBackward ? (size_t)2 * dim * 4 : (size_t)0);
  int occ = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, kRotThreads, smem) != cudaSuccess || occ <= 0) {
    cudaGetLastError();
    occ = 1;
  }
  if (mode == kNormRotateBackward) occ = std::min(occ, kRotBlocksPerSm);
  const int64_t tiles = ceil_div(p.n, tile);
  int grid = (int)std::min<int64_t>(tiles, (int64_t)sms * occ);
  if (mode == kNormRotateBackward) grid = (int)std::min<int64_t>(grid, workspace_bytes / row_bytes);
  kern<<<grid, kRotThreads, smem, stream>>>(p);
  FP4T_CUDA(cudaGetLastError());
  if (mode == kNormRotateBackward) {
    qk_weight_grad_kernel<<<(int)ceil_div(2 * dim, 32), 1024, 0, stream>>>(p.partial, grid, (int)dim, dw[0], count == 2 ? dw[1] : nullptr);
    FP4T_CUDA(cudaGetLastError());
  }
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
  return (int64_t)sms * kRotBlocksPerSm * 2 * head_dim * (int64_t)sizeof(float);
}

extern "C" int fp4t_qk_norm_rotary_backward(const fp4t_heads_t* dy, const fp4t_heads_t* x, const float* const* weights, float eps,
                                            const fp4t_heads_t* dx, float* const* dweights, int count, int dtype, int64_t batch,
                                            int64_t tokens, int64_t head_dim, const fp4t_rotary_t* rotary, void* workspace,
                                            int64_t workspace_bytes, fp4t_stream_t stream) {
  return run("fp4t_qk_norm_rotary_backward", kNormRotateBackward, x, dy, dx, count, dtype, batch, tokens, head_dim, rotary, 0, weights,
             eps, dweights, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}
