// Attention over keys of another length: parameters, and device code shared by its kernels.
//
// No mask but the keys' number: every row of sequence z sees the first len_z keys. The rows that share the keys of a slice (a
// sequence, or a group of them behind one prefix, and a key head) are numbered one after the other, row R = (b G + g) N + n for
// sequence b of B, query head g of G and query n of N, whatever their addresses: tiles of 32 rows hold any of them, so a
// single token's heads share a tile, and so do the sequences behind a prefix.
#pragma once

#include "bwd_pipe.h"
#include "common.h"
#include "ops.h"
#include "window.h"

namespace tattn {

// Workgroup -> (slice, block); false past the last. Workgroups go round-robin over the 8 XCDs. Blocks of a slice stay on one, whose
// L2 then holds its keys, and the slices are dealt out one by one, so that sequences of other lengths meet on every XCD
// (cross_dealt); where that would leave XCDs idle each takes a run of all blocks. 8 x 16 x 1,024 rows over 375 to 1,500 keys x 64, us
// forward and backward: runs 53 and 200, dealt out 47 and 185 (long sequences first, or long and short ones side by side: no faster).
__device__ __forceinline__ bool cross_coord(const CrossParams& p, int nblk, int& slice, int& blk) {
  const int slices = p.Zs * p.Hk;
  if (!cross_dealt(slices)) return window_coord(slices, nblk, 0, 0, slice, blk);
  const int l = (int)(blockIdx.x >> 3);
  slice = 8 * (l / nblk) + (int)(blockIdx.x & 7);
  blk = l % nblk;
  return slice < slices;
}

// The sequence group and key head of a slice and the keys that its rows see.
struct CrossSlice {
  int zs, hk, len;
  __device__ __forceinline__ CrossSlice(const CrossParams& p, int slice) {
    zs = slice / p.Hk;
    hk = slice % p.Hk;
    len = p.lens ? min(max(p.lens[zs], 0), p.S) : p.S;
  }
};

// Row R of a slice: its sequence, query head and query.
struct CrossRow {
  int z, h, n;
  __device__ __forceinline__ CrossRow(const CrossParams& p, const CrossSlice& s, int row) {
    const int b = row / (p.G * p.N), rest = row - b * (p.G * p.N), g = rest / p.N;
    z = s.zs * p.B + b;
    h = s.hk * p.G + g;
    n = rest - g * p.N;
  }
  __device__ __forceinline__ int64_t at(const int64_t (&st)[3]) const { return (int64_t)z * st[0] + (int64_t)h * st[1] + (int64_t)n * st[2]; }
  __device__ __forceinline__ int64_t index(const CrossParams& p) const { return ((int64_t)z * p.H + h) * p.N + n; }
};

template <typename T, int D>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* base, int64_t off, int64_t rows, int64_t stride) {
  return slice_rsrc((const T*)base + off, rows > 0 ? slice_bytes(rows, stride, D) : 0);
}

// A 32-row tile in LDS: swizzled rows (Swz) in perm32 order, 1 KB pieces.
template <int D>
struct CrossTile {
  static constexpr int RB = Swz<D>::RB, BYTES = 32 * RB, PIECES = BYTES / 1024;
  // Byte offset, from the tile's first row, of what lane `lane` of piece i fetches.
  static __device__ __forceinline__ uint32_t source(int i, int lane, int64_t stride) {
    constexpr int CPR = RB / 16;
    const int j = 64 * i + lane, row = j / CPR, cc = ((j % CPR) ^ Swz<D>::f(row)) & (D / 8 - 1);
    return (uint32_t)(perm32(row) * stride * 2 + cc * 16);
  }
};

// Operand addresses within a tile: natural rows, and the transposed reads of 16-row slice 0 (the swizzle depends on a row's
// index mod 16, so slice 1 is a constant further).
template <int D>
struct CrossOp {
  static constexpr int NSD = D / 16, DT = (D + 31) / 32;
  int nat[NSD], lo[DT], hi[DT];
  __device__ __forceinline__ void init(int lane) {
    const int l32 = lane & 31, h2 = lane >> 5;
#pragma unroll
    for (int s = 0; s < NSD; ++s) nat[s] = Swz<D>::addr(l32, (16 * s + 8 * h2) * 2);
#pragma unroll
    for (int u = 0; u < DT; ++u) tr_addrs<D>(0, u, lane, lo[u], hi[u]);
  }
  template <typename T>
  __device__ __forceinline__ typename H16<T>::V8 tr(const char* tile, int sl, int u, int lane) const {
    typename H16<T>::V8 x = tr_pair<T>(tile + 16 * sl * Swz<D>::RB, lo[u], hi[u]);
    if (D < 32 && 16 * ((lane >> 4) & 1) >= D) x = typename H16<T>::V8{};
    return x;
  }
};

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, char* lds, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (TATTN_LDS void*)lds, 16, (int)off, 0, 0, 0);
}

// At most OUT of this wave's memory operations are still in flight, and its LDS reads are done.
template <int OUT>
__device__ __forceinline__ void wave_landed() {
  static_assert(OUT < 64, "vmcnt field");
  __builtin_amdgcn_s_waitcnt((OUT & 15) | ((OUT >> 4) << 14) | 0x0070);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// This wave's LDS reads are done: a load into what it read may start.
__device__ __forceinline__ void reads_done() {
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// Hides the keys past a row's last one in a tile of S^T: register r of lane half h2 is key 32 t + 8 h2 + 16 (r / 8) + r % 8.
__device__ __forceinline__ void hide_after(f32x16& s, int last, int t, int h2, float hidden) {
  const int hi = last - 32 * t - 8 * h2;
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = 16 * (r >> 3) + (r & 7) > hi ? hidden : s[r];
}

// Rounded probabilities of a tile against the running max as it stands, as operands; returns the lane's sum of them.
template <typename T>
__device__ __forceinline__ float tile_probs(const f32x16& s, typename H16<T>::V8 (&x)[2], float c, float nm) {
  float ps = 0.0f;
#pragma unroll
  for (int sg = 0; sg < 2; ++sg)
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const int r = 8 * sg + i;
      const auto pr = H16<T>::pack(fast_exp2(__builtin_fmaf(s[r], c, nm)), fast_exp2(__builtin_fmaf(s[r + 1], c, nm)));
      ps = H16<T>::sum2(pr, ps);
      x[sg][i] = pr[0];
      x[sg][i + 1] = pr[1];
    }
  return ps;
}

// The max that a tile's scores ask for: it moves only where they exceed it by more than 2^kRescaleLog2.
__device__ __forceinline__ float moved_max(const f32x16& s, float c, float mrow) {
  float mx = kNoMax;
#pragma unroll
  for (int r = 0; r < 16; ++r) mx = __builtin_fmaxf(mx, s[r] * c);
  const float cand = max_halves(mx);
  return cand > mrow + kRescaleLog2 ? cand : mrow;
}

// A row of O^T in registers (register 4 g + e of tile u: column 32 u + 8 g + 4 h2 + e), times mul, to memory.
template <typename T, int D, int DT>
__device__ __forceinline__ void store_row_t(T* row, const f32x16 (&acc)[DT], float mul, int h2) {
  typedef T V4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int u = 0; u < DT; ++u)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d0 = 32 * u + 8 * g + 4 * h2;
      if (d0 >= D) continue;
      V4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (T)(acc[u][4 * g + e] * mul);
      *reinterpret_cast<V4*>(row + d0) = y;
    }
}

}  // namespace tattn
