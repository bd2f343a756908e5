// Attention over few keys: device code shared by the kernels of cross_short.hip and cross_short_pipe.hip.
#pragma once

#include "cross_bwd.h"

namespace tattn {
namespace {

constexpr int kShortWaves = 4;
constexpr int short_part(int D) { return (D + 31) / 32 * 16 * 64 * 4; }  // bytes of a wave's sums for 32 keys

// K and V of the slice into `tiles` (K's, then V's), rows at or past len as zeros; waits for them.
template <typename T, int D, int NT>
__device__ __forceinline__ void stage_keys(const CrossParams& p, const CrossSlice& sl, char* tiles, int wu, int lane) {
  using Tile = CrossTile<D>;
  const __amdgpu_buffer_rsrc_t krs = rows_rsrc<T, D>(p.k, sl.zs * p.sk[0] + sl.hk * p.sk[1], sl.len, p.sk[2]);
  const __amdgpu_buffer_rsrc_t vrs = rows_rsrc<T, D>(p.v, sl.zs * p.sv[0] + sl.hk * p.sv[1], sl.len, p.sv[2]);
  for (int i = wu; i < NT * Tile::PIECES; i += kShortWaves) {
    const int t = i / Tile::PIECES, piece = i % Tile::PIECES;
    dma16(krs, tiles + 1024 * i, Tile::source(piece, lane, p.sk[2]) + (uint32_t)(64 * t * p.sk[2]));
    dma16(vrs, tiles + NT * Tile::BYTES + 1024 * i, Tile::source(piece, lane, p.sv[2]) + (uint32_t)(64 * t * p.sv[2]));
  }
  all_landed_barrier();
}

// Row tiles of the workgroup's part.
struct ShortRows {
  int slice, part, rows, t0, t1;
  bool ok;
  __device__ __forceinline__ ShortRows(const CrossParams& p, int parts) {
    ok = cross_coord(p, parts, slice, part);
    rows = p.B * p.G * p.N;
    const int tiles = (rows + 31) >> 5;
    t0 = (int)((int64_t)tiles * part / parts);
    t1 = (int)((int64_t)tiles * (part + 1) / parts);
  }
};

// What the scores of a tile's keys start from: 0, or -inf for those at or past len, whose K is zeros. One float a key.
template <int NT>
__device__ __forceinline__ void stage_mask(const CrossSlice& sl, float* mask) {
  if (threadIdx.x < 32 * NT) mask[threadIdx.x] = (int)threadIdx.x < sl.len ? 0.0f : -__builtin_inff();
}
__device__ __forceinline__ f32x16 masked_start(const float* mask, int k, int h2) {
  f32x16 s;
  int at = 8 * h2;
  asm volatile("" : "+v"(at));  // read where it is used: held over the rows it would take 16 registers a tile
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const f32x4 x = *reinterpret_cast<const TATTN_LDS f32x4*>((const TATTN_LDS float*)mask + 32 * k + 16 * (a >> 1) + at + 4 * (a & 1));
#pragma unroll
    for (int e = 0; e < 4; ++e) s[4 * a + e] = x[e];
  }
  return s;
}
// Where the scale is negative the signs of q and of the scale change: scores rise with their exponents.
template <typename V8>
__device__ __forceinline__ V8 signed_rows(u32x4 x, uint32_t sign) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] ^= sign;
  return __builtin_bit_cast(V8, x);
}

// The lane's row of a tile as operand chunks (row l32, 16 bytes of every 32).
template <typename T, int D>
__device__ __forceinline__ void load_rows(const T* base, int64_t off, int h2, u32x4 (&x)[D / 16]) {
#pragma unroll
  for (int s = 0; s < D / 16; ++s) x[s] = ld16(base + off + 16 * s + 8 * h2);
}

// The waves' sums of dK and dV, tile by tile of keys, added through `smem` and stored: C register r of a lane is key 8 (r / 4) + 4 h2 +
// r % 4, column 32 u + l32. Keys at or past len get zeros: their P and dS are 0, but not their products with what is not finite.
template <typename T, int D, int NT, int DT>
__device__ __forceinline__ void short_sums(const CrossParams& p, const CrossSlice& sl, const ShortRows& b, char* smem,
                                           const f32x16 (&dk)[NT][DT], const f32x16 (&dv)[NT][DT], float unlift) {
  using V8 = typename H16<T>::V8;
  constexpr int CPR = D / 8, KEYS = 32 * NT, PART = short_part(D);
  const int tid = threadIdx.x, lane = tid & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(tid >> 6));
  TATTN_LDS float* sums = (TATTN_LDS float*)smem;
  float* part = p.kpart + ((int64_t)b.slice * p.parts + b.part) * (2 * KEYS * D);
#pragma unroll
  for (int k = 0; k < NT; ++k)
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int u = 0; u < DT; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int in = 8 * (r >> 2) + 4 * h2 + (r & 3), d = 32 * u + l32;
          if (d < D) sums[wu * (PART / 4) + in * D + d] = which ? dv[k][u][r] : dk[k][u][r] * unlift;
        }
      __syncthreads();
      for (int i = tid; i < 32 * CPR; i += kShortWaves * 64) {
        const int in = i / CPR, cc = i % CPR, key = 32 * k + in;
        if (key >= p.S) continue;
        f32x4 lo = f32x4{}, hi = f32x4{};
#pragma unroll
        for (int w = 0; w < kShortWaves; ++w) {
          lo += *reinterpret_cast<const TATTN_LDS f32x4*>(sums + w * (PART / 4) + in * D + 8 * cc);
          hi += *reinterpret_cast<const TATTN_LDS f32x4*>(sums + w * (PART / 4) + in * D + 8 * cc + 4);
        }
        if (key >= sl.len) lo = hi = f32x4{};
        if (p.parts > 1) {
          float* dst = part + (which ? KEYS * D : 0) + key * D + 8 * cc;
          *reinterpret_cast<f32x4*>(dst) = lo;
          *reinterpret_cast<f32x4*>(dst + 4) = hi;
        } else {
          const float mul = which ? 1.0f : p.scale;
          V8 y;
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = (T)((e < 4 ? lo[e & 3] : hi[e & 3]) * mul);
          T* dst = which ? (T*)p.dv + sl.zs * p.sdv[0] + sl.hk * p.sdv[1] + (int64_t)key * p.sdv[2]
                         : (T*)p.dk + sl.zs * p.sdk[0] + sl.hk * p.sdk[1] + (int64_t)key * p.sdk[2];
          *reinterpret_cast<V8*>(dst + 8 * cc) = y;
        }
      }
    }
}

}  // namespace
}  // namespace tattn
