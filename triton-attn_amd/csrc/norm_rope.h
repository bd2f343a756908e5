// Norms of query and key heads and the position rotation: device code shared by the kernels for one axis
// (norm_rope.hip, whose comment has the mathematics and the layout) and for several (rope_axes.hip).
#pragma once

#include <algorithm>

#include "common.h"
#include "ops.h"

namespace tattn {
namespace {

constexpr int kHeads = 4;      // heads per lane group and turn
constexpr int kBwdThreads = 512;

template <typename T, int D>
struct RowCfg {
  static constexpr int EPC = 16 / (int)sizeof(T);  // elements of a 16-byte chunk
  static constexpr int LPR = D / (2 * EPC);        // lanes per row
  static constexpr int E = 2 * EPC;                // elements per lane
};

template <typename T, int N>
__device__ __forceinline__ void load_floats(const void* p, float* x) {
  static_assert(N * sizeof(T) % 16 == 0 || N * sizeof(T) == 8, "whole vectors");
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f32x4 v = *reinterpret_cast<const f32x4*>((const char*)p + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i + j] = v[j];
    }
  } else {
    typedef T V8 __attribute__((ext_vector_type(8)));
    const V8 v = *reinterpret_cast<const V8*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)v[j];
  }
}

template <typename T>
__device__ __forceinline__ void store_chunk(T* p, const float* x) {
  constexpr int EPC = 16 / (int)sizeof(T);
  typedef T V __attribute__((ext_vector_type(EPC)));
  V v;
#pragma unroll
  for (int i = 0; i < EPC; ++i) v[i] = (T)x[i];
  *reinterpret_cast<V*>(p) = v;
}

// The lane's E elements of a row: its chunk c of the lower half, then of the upper half.
template <typename T, int D>
__device__ __forceinline__ void load_row(const T* row, int c, float* x) {
  using C = RowCfg<T, D>;
  load_floats<T, C::EPC>(row + C::EPC * c, x);
  load_floats<T, C::EPC>(row + D / 2 + C::EPC * c, x + C::EPC);
}
template <typename T, int D>
__device__ __forceinline__ void store_row(T* row, int c, const float* x) {
  using C = RowCfg<T, D>;
  store_chunk<T>(row + C::EPC * c, x);
  store_chunk<T>(row + D / 2 + C::EPC * c, x + C::EPC);
}
template <typename T, int D>
__device__ __forceinline__ void load_weight(const void* w, bool wide, int c, float* x) {
  using C = RowCfg<T, D>;
  if (wide) {
    load_floats<float, C::EPC>((const float*)w + C::EPC * c, x);
    load_floats<float, C::EPC>((const float*)w + D / 2 + C::EPC * c, x + C::EPC);
  } else {
    load_row<T, D>((const T*)w, c, x);
  }
}

// Cosines (or sines) of the lane's EPC pairs: of pairs EPC c .. in order, or interleaved EPC / 2 in each half.
template <typename T, int D, bool IL>
__device__ __forceinline__ void load_angles(const float* row, int c, float* x) {
  using C = RowCfg<T, D>;
  if constexpr (!IL) {
    load_floats<float, C::EPC>(row + C::EPC * c, x);
  } else {
    constexpr int P = C::EPC / 2;
#pragma unroll
    for (int i = 0; i < P; i += 2) {
      const f32x2 a = *reinterpret_cast<const f32x2*>(row + P * c + i);
      const f32x2 b = *reinterpret_cast<const f32x2*>(row + D / 4 + P * c + i);
      x[i] = a[0], x[i + 1] = a[1], x[P + i] = b[0], x[P + i + 1] = b[1];
    }
  }
}

// Turns the lane's pairs by their angles (sign = 1) or back (-1), but for those whose bits in `still` are set: a turn by cosine 1 and
// sine 0 would carry an infinity or a NaN of one of a pair into the other.
template <int E, bool IL>
__device__ __forceinline__ void rotate(float* x, const float* cs, const float* sn, float sign, uint32_t still) {
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    float& a = IL ? x[2 * i] : x[i];
    float& b = IL ? x[2 * i + 1] : x[i + E / 2];
    const float s = sign * sn[i], a0 = a, b0 = b;
    a = still >> i & 1 ? a0 : a0 * cs[i] - b0 * s;
    b = still >> i & 1 ? b0 : b0 * cs[i] + a0 * s;
  }
}

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int d = 1; d < LPR; d <<= 1) x += __shfl_xor(x, d);
  return x;
}

// What a lane group works on: up to four heads of one token of q or of k.
struct Unit {
  int z, n, head, heads;  // heads >= 1
};
__device__ __forceinline__ Unit unit_of(uint32_t u, uint32_t per, int N, int H) {
  const uint32_t token = u / per, part = u % per;
  const int head = (int)part * kHeads;
  return {(int)(token / (uint32_t)N), (int)(token % (uint32_t)N), head, min(kHeads, H - head)};
}

// Angles of the unit's position; a position outside the table makes them NaN. Returns the pairs that are not turned: none.
template <typename T, int D, bool IL>
__device__ __forceinline__ uint32_t unit_angles(const NormRopeParams& p, const Unit& u, int c, float* cs, float* sn) {
  constexpr int EPC = RowCfg<T, D>::EPC;
  const int pos = p.positions ? p.positions[u.z * p.pos_stride + u.n] : u.n;
  const bool ok = pos >= 0 && pos < p.P;
  const int64_t at = (int64_t)(ok ? pos : 0) * (D / 2);
  load_angles<T, D, IL>(p.cos + at, c, cs);
  load_angles<T, D, IL>(p.sin + at, c, sn);
  if (!ok) {
#pragma unroll
    for (int i = 0; i < EPC; ++i) cs[i] = sn[i] = __builtin_nanf("");
  }
  return 0;
}

// Angles of the unit's positions where each pair has an axis of its own. Quads: four pairs in a row share one, and are loaded
// together. A position outside the table makes its axis's pairs NaN. Returns a bit for each pair without an axis, which is not turned.
template <typename T, int D, bool IL>
__device__ __forceinline__ uint32_t unit_angles(const RopeAxesParams& p, const Unit& u, int c, float* cs, float* sn) {
  constexpr int EPC = RowCfg<T, D>::EPC, RUN = IL ? EPC / 2 : EPC, W = RUN < 4 ? RUN : 4;  // pairs in a row, and in a load
  const int64_t at = u.z * p.pos_stride + u.n;
  uint32_t still = 0;
#pragma unroll
  for (int i0 = 0; i0 < EPC; i0 += W) {
    const int first = IL ? i0 / RUN * (D / 4) + RUN * c + i0 % RUN : RUN * c + i0;  // of the pairs
    uint32_t axes;
    if constexpr (W == 4) axes = reinterpret_cast<const uint16_t*>(p.axes)[first / 4];
    else axes = reinterpret_cast<const uint8_t*>(p.axes)[first / 2];
    auto row = [&](uint32_t axis, bool& ok) __attribute__((always_inline)) {
      const int pos = axis < kNoAxis ? p.positions[axis * p.axis_stride + at] : 0;
      ok = pos >= 0 && pos < p.P;
      return (int64_t)(ok ? pos : 0) * (D / 2) + first;
    };
    auto put = [&](int i, uint32_t axis, bool ok, float x, float y) __attribute__((always_inline)) {
      cs[i0 + i] = ok ? x : __builtin_nanf("");
      sn[i0 + i] = ok ? y : __builtin_nanf("");
      still |= axis == kNoAxis ? 1u << (i0 + i) : 0;
    };
    if (W == 4 && p.quads) {
      bool ok;
      const uint32_t axis = axes & 15;
      const int64_t r = row(axis, ok);
      const f32x4 x = *reinterpret_cast<const f32x4*>(p.cos + r), y = *reinterpret_cast<const f32x4*>(p.sin + r);
#pragma unroll
      for (int i = 0; i < W; ++i) put(i, axis, ok, x[i], y[i]);
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        bool ok;
        const uint32_t axis = axes >> (4 * i) & 15;
        const int64_t r = row(axis, ok) + i;
        put(i, axis, ok, p.cos[r], p.sin[r]);
      }
    }
  }
  return still;
}

// NORM: the rows are divided by their root mean square and weighted before the rotation; otherwise they are turned by p.sign times
// the angles, which is the gradient's way too.
template <typename T, int D, bool IL, typename P, bool NORM>
__global__ __launch_bounds__(256) void norm_rope_fwd_kernel(const P p) {
  using C = RowCfg<T, D>;
  const int c = threadIdx.x % C::LPR;
  uint32_t id = blockIdx.x * (256 / C::LPR) + threadIdx.x / C::LPR;
  if (id >= p.units_q + p.units_k) return;
  const bool is_k = id >= p.units_q;
  if (is_k) id -= p.units_q;
  const Unit u = is_k ? unit_of(id, p.per_k, p.N, p.Hk) : unit_of(id, p.per_q, p.N, p.H);
  const int64_t* st = is_k ? p.sk : p.sq;
  const int64_t* so = is_k ? p.sko : p.sqo;
  const T* src = (const T*)(is_k ? p.k : p.q) + u.z * st[0] + u.head * st[1] + u.n * st[2];
  T* dst = (T*)(is_k ? p.ko : p.qo) + u.z * so[0] + u.head * so[1] + u.n * so[2];
  float x[kHeads][C::E], w[C::E], cs[C::EPC], sn[C::EPC];
#pragma unroll
  for (int j = 0; j < kHeads; ++j) load_row<T, D>(src + (j < u.heads ? j : 0) * st[1], c, x[j]);
  const uint32_t still = unit_angles<T, D, IL>(p, u, c, cs, sn);
  if constexpr (NORM) load_weight<T, D>(is_k ? p.kw : p.qw, p.wide_w, c, w);
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    if (j >= u.heads) break;
    if constexpr (NORM) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < C::E; ++i) s = __builtin_fmaf(x[j][i], x[j][i], s);
      const float r = rsqrtf(row_sum<C::LPR>(s) * (1.0f / D) + p.eps);
#pragma unroll
      for (int i = 0; i < C::E; ++i) x[j][i] = x[j][i] * r * w[i];
      rotate<C::E, IL>(x[j], cs, sn, 1.0f, still);
    } else {
      rotate<C::E, IL>(x[j], cs, sn, p.sign, still);
    }
    store_row<T, D>(dst + j * so[1], c, x[j]);
  }
}

// dx of every row, and per workgroup the sum of its rows' weight gradients. Workgroups below p.blocks_q
// take q's units, the others k's, each a fixed set of them, so that the sums do not depend on
// timing; norm_rope_dw_kernel adds the workgroups' sums in order.
template <typename T, int D, bool IL, typename P>
__global__ __launch_bounds__(kBwdThreads) void norm_rope_bwd_kernel(const P p) {
  using C = RowCfg<T, D>;
  constexpr int GROUPS = kBwdThreads / C::LPR, HB = 2;  // rows in flight: x and dy of two
  __shared__ float part[kBwdThreads / 64][D];
  const int c = threadIdx.x % C::LPR;
  const bool is_k = (int)blockIdx.x >= p.blocks_q;
  const uint32_t block = is_k ? blockIdx.x - p.blocks_q : blockIdx.x;
  const uint32_t blocks = is_k ? p.blocks_k : p.blocks_q;
  const uint32_t units = is_k ? p.units_k : p.units_q;
  const int64_t* st = is_k ? p.sk : p.sq;
  const int64_t* so = is_k ? p.sko : p.sqo;
  const int64_t* sg = is_k ? p.sgk : p.sgq;
  float w[C::E], dw[C::E];
  load_weight<T, D>(is_k ? p.kw : p.qw, p.wide_w, c, w);
#pragma unroll
  for (int i = 0; i < C::E; ++i) dw[i] = 0.0f;

  for (uint32_t id = block * GROUPS + threadIdx.x / C::LPR; id < units; id += blocks * GROUPS) {
    const Unit u = is_k ? unit_of(id, p.per_k, p.N, p.Hk) : unit_of(id, p.per_q, p.N, p.H);
    const T* src = (const T*)(is_k ? p.k : p.q) + u.z * st[0] + u.head * st[1] + u.n * st[2];
    const T* grad = (const T*)(is_k ? p.gk : p.gq) + u.z * sg[0] + u.head * sg[1] + u.n * sg[2];
    T* dst = (T*)(is_k ? p.ko : p.qo) + u.z * so[0] + u.head * so[1] + u.n * so[2];
    float cs[C::EPC], sn[C::EPC];
    const uint32_t still = unit_angles<T, D, IL>(p, u, c, cs, sn);
#pragma unroll
    for (int j0 = 0; j0 < kHeads; j0 += HB) {
      if (j0 >= u.heads) break;
      float x[HB][C::E], t[HB][C::E];
#pragma unroll
      for (int j = 0; j < HB; ++j) {
        const int at = j0 + j < u.heads ? j0 + j : j0;
        load_row<T, D>(src + at * st[1], c, x[j]);
        load_row<T, D>(grad + at * sg[1], c, t[j]);
      }
#pragma unroll
      for (int j = 0; j < HB; ++j) {
        if (j0 + j >= u.heads) break;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < C::E; ++i) s = __builtin_fmaf(x[j][i], x[j][i], s);
        const float r = rsqrtf(row_sum<C::LPR>(s) * (1.0f / D) + p.eps);
        rotate<C::E, IL>(t[j], cs, sn, -1.0f, still);
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < C::E; ++i) {
          x[j][i] *= r;
          dw[i] = __builtin_fmaf(t[j][i], x[j][i], dw[i]);
          t[j][i] *= w[i];
          m = __builtin_fmaf(t[j][i], x[j][i], m);
        }
        m = row_sum<C::LPR>(m) * (1.0f / D);
#pragma unroll
        for (int i = 0; i < C::E; ++i) t[j][i] = r * (t[j][i] - x[j][i] * m);
        store_row<T, D>(dst + (j0 + j) * so[1], c, t[j]);
      }
    }
  }
  if (!p.partial) return;
  // The wave's row groups, then the waves.
#pragma unroll
  for (int i = 0; i < C::E; ++i)
#pragma unroll
    for (int d = C::LPR; d < 64; d <<= 1) dw[i] += __shfl_xor(dw[i], d);
  const int lane = threadIdx.x & 63;
  if (lane < C::LPR) {
#pragma unroll
    for (int i = 0; i < C::E; ++i)
      part[threadIdx.x >> 6][(i < C::EPC ? 0 : D / 2 - C::EPC) + C::EPC * lane + i] = dw[i];
  }
  __syncthreads();
  if (threadIdx.x < D) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kBwdThreads / 64; ++i) s += part[i][threadIdx.x];
    p.partial[(int64_t)blockIdx.x * D + threadIdx.x] = s;
  }
}

// Workgroups of q and of k in the backward: as many as their units fill, at most two per CU of an MI355X in all, shared out by
// units.
template <typename T, int D>
void norm_rope_bwd_blocks(NormRopeParams& p) {
  constexpr int64_t GROUPS = kBwdThreads / RowCfg<T, D>::LPR, MOST = kNormRopeRows;
  const int64_t uq = p.units_q, uk = p.units_k;
  const int64_t nq = (uq + GROUPS - 1) / GROUPS, nk = (uk + GROUPS - 1) / GROUPS;
  const int64_t share = std::min<int64_t>(MOST - 1, std::max<int64_t>(1, MOST * uq / (uq + uk)));
  p.blocks_q = (int)std::min(nq, share);
  p.blocks_k = (int)std::min(nk, MOST - share);
}

}  // namespace
}  // namespace tattn
