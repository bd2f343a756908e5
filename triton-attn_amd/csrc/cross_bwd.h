// Attention over keys of another length, backward: device code shared by its kernels.
#pragma once

#include "cross.h"

namespace tattn {

// A step's rows on their way from memory to LDS: two tiles of 32 rows, NT threads.
template <int D, int NT>
struct StepRows {
  using B = BwdPipe<D>;
  static constexpr int CPT = (B::CHUNKS + NT - 1) / NT;
  uint32_t goff[2][CPT];
  int ldst[CPT];
  u32x4 x[2][CPT];
  __device__ __forceinline__ void init(int tid, int64_t sa, int64_t sb) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int ch = min(tid + i * NT, B::CHUNKS - 1), row = ch / B::CPR, cb = (ch % B::CPR) * 16;
      goff[0][i] = (uint32_t)(row * sa * 2 + cb);
      goff[1][i] = (uint32_t)(row * sb * 2 + cb);
      ldst[i] = Swz<D>::addr(perm32(row), cb);
    }
  }
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t a, __amdgpu_buffer_rsrc_t b, uint32_t oa, uint32_t ob) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      x[0][i] = rsrc_load(a, goff[0][i] + oa);
      x[1][i] = rsrc_load(b, goff[1][i] + ob);
    }
  }
  __device__ __forceinline__ void store(char* stage, int tid) const {
#pragma unroll
    for (int i = 0; i < CPT; ++i)
      if (B::CHUNKS % NT == 0 || tid + i * NT < B::CHUNKS) {
        st16(stage + ldst[i], x[0][i]);
        st16(stage + B::TILE + ldst[i], x[1][i]);
      }
  }
  __device__ __forceinline__ void clear(char* stage, int tid) const {
#pragma unroll
    for (int i = 0; i < CPT; ++i)
      if (B::CHUNKS % NT == 0 || tid + i * NT < B::CHUNKS) {
        st16(stage + ldst[i], u32x4{});
        st16(stage + B::TILE + ldst[i], u32x4{});
      }
  }
};

}  // namespace tattn
