// Tiles of 32 rows in float32 for v_mfma_f32_32x32x2f32: A lane holds A[m = lane % 32][k = lane / 32], B lane
// B[k = lane / 32][n = lane % 32]. Workgroups of 256 threads.
#pragma once

#include "common.h"

namespace tattn {

__device__ __forceinline__ f32x16 mfma2(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }

template <int D>
struct F32 {
  static constexpr int H = D / 2;               // d per lane half, and matrix instructions over d
  static constexpr int DT = (D + 31) / 32;
  static constexpr int LD = D + 4;              // floats per row in LDS
  static constexpr int CPR = D / 4;             // 16-byte chunks per row
  static constexpr int CPT = (32 * CPR + 255) / 256;
};

// A 32-row tile on its way from memory to LDS.
template <int D>
struct Tile32 {
  using C = F32<D>;
  f32x4 x[C::CPT];
  // Row i of the tile where ok(i), else zeros.
  template <typename Ok>
  __device__ __forceinline__ void load(const float* base, int64_t stride, int first, Ok ok) {
#pragma unroll
    for (int i = 0; i < C::CPT; ++i) {
      const int ch = threadIdx.x + 256 * i, row = ch / C::CPR;
      x[i] = f32x4{};
      if (row < 32 && ok(first + row)) x[i] = *reinterpret_cast<const f32x4*>(base + (int64_t)(first + row) * stride + 4 * (ch % C::CPR));
    }
  }
  __device__ __forceinline__ void store(float* lds) const {
#pragma unroll
    for (int i = 0; i < C::CPT; ++i) {
      const int ch = threadIdx.x + 256 * i, row = ch / C::CPR;
      if (row < 32) *reinterpret_cast<TATTN_LDS f32x4*>((TATTN_LDS float*)lds + row * C::LD + 4 * (ch % C::CPR)) = x[i];
    }
  }
};

// A product over d: rows of the LDS tile in perm32 order against the lane's own row.
template <int D>
__device__ __forceinline__ f32x16 rows_dot(const float* lds, const float (&own)[D / 2], f32x16 s, int l32, int h2) {
  using C = F32<D>;
  const TATTN_LDS float* row = (const TATTN_LDS float*)lds + perm32(l32) * C::LD + h2 * C::H;
#pragma unroll
  for (int j = 0; j < C::H; j += 4) {
    const f32x4 a = *reinterpret_cast<const TATTN_LDS f32x4*>(row + j);
#pragma unroll
    for (int e = 0; e < 4; ++e) s = mfma2(a[e], own[j + e], s);
  }
  return s;
}

// Element d of tile row kappa(r, h2): an operand of the second products.
template <int D>
__device__ __forceinline__ float cell(const float* lds, int r, int d, int h2) {
  return D >= 32 || d < D ? ((const TATTN_LDS float*)lds)[kappa(r, h2) * F32<D>::LD + d] : 0.0f;
}

template <int D>
__device__ __forceinline__ void own_row(const float* row, bool live, int h2, float (&x)[D / 2]) {
#pragma unroll
  for (int j = 0; j < D / 2; j += 4) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(row + h2 * (D / 2) + j);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[j + e] = live ? a[e] : 0.0f;
  }
}

}  // namespace tattn
