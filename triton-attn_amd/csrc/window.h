// Window attention: parameters, and device code shared by its kernels and the one over the 4-bit cache.
//
// Query n of sequence z is at position p = len_z - N + n and sees key j if j <= p and (p - j < window or
// j < sinks). The G query heads of one key head share its keys: their rows are laid one after the other, row
// R = n * G + g, so that a 32-row tile holds whole queries with all their heads where G allows. A tile then spans 32 / G
// positions, which trims the masked ends of its window, and a single token's heads fill one tile.
#pragma once

#include "bwd_pipe.h"
#include "common.h"
#include "ops.h"

namespace tattn {

// Score below every score: the running max before the first visible key. Finite, so that rescaling a
// sum that holds nothing yet multiplies by 0 and never subtracts infinities.
constexpr float kNoMax = -3.0e38f;

// The key tiles (32 keys) that rows at positions [p0, p1] see: the tiles of the first `sinks` keys, then those of
// the window. `last` is the position of the first row of the last wave. Where the tile in which the first keys end lies in the
// window of the first wave's rows and before the last's, it comes twice: of its other keys nothing may be there for waves that
// see none of them (a hidden key's probability is 0, but 0 times a NaN in its value is not), so these waves take an entry
// among the first keys', in which the other keys are zeros, and those whose window holds the tile take it whole.
struct TileList {
  int lo;     // first key of the window
  int sink_tiles, n;
  int jump;   // entry i is tile i, or from sink_tiles on tile i + jump
  int skip;   // the entry of that tile among the first keys', or -1
  __device__ __forceinline__ void init(int p0, int p1, int last, int window, int sinks) {
    lo = max(0, p0 - window + 1);
    int first = lo >> 5;
    const int end = sinks >> 5;
    sink_tiles = min((min(sinks, lo) + 31) >> 5, first);
    skip = -1;
    if ((sinks & 31) != 0 && first <= end && end < (last - window + 1) >> 5) {
      skip = first = end;  // the tiles before it hold first keys alone
      sink_tiles = end + 1;
    }
    jump = first - sink_tiles;
    n = p1 < 0 ? 0 : (p1 >> 5) - jump + 1;
  }
  __device__ __forceinline__ int at(int i) const { return i < sink_tiles ? i : i + jump; }
  // Keys below are zeros in entry i, but for the first keys.
  __device__ __forceinline__ int low(int i) const { return i < sink_tiles ? 0x7fffffff : lo; }
};

// The raw score of a hidden key: its scaled value is -inf, so its probability is 0 whatever the row's max or log-sum-exp
// (the entry points replace a scale of 0, where no such score exists, by a tiny one).
__device__ __forceinline__ float hidden_score(float c) { return c < 0.0f ? __builtin_inff() : -__builtin_inff(); }

// What a lane's row at position p hides in a tile of S^T: register r of lane-half h2 is key 32 t + 8 h2 + 16 (r / 8) + r % 8.
struct RowMask {
  int hi, lb, sk;
  __device__ __forceinline__ RowMask(int p, int t, int h2, int window, int sinks) {
    const int base = 32 * t + 8 * h2;
    hi = p - base;
    lb = hi - window + 1;
    sk = sinks - base;
  }
  __device__ __forceinline__ void hide(f32x16& s, float hidden) const {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int off = 16 * (r >> 3) + (r & 7);
      s[r] = off > hi || (off < lb && off >= sk) ? hidden : s[r];
    }
  }
};

// The same where the lane is a key and register r a query of a tile of S: `gap` from the key to the tile's first
// position, `rows` left from there to the last query.
struct ColMask {
  int gap, window, rows;
  __device__ __forceinline__ ColMask(int gap_, int key, int rows_, int h2, int window_, int sinks) {
    gap = gap_ + 8 * h2;
    rows = rows_ - 8 * h2;
    window = key < sinks ? 0x7fffffff : window_;
  }
  __device__ __forceinline__ void hide(f32x16& s, float hidden) const {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int off = 16 * (r >> 3) + (r & 7);
      s[r] = gap + off < 0 || gap + off >= window || off >= rows ? hidden : s[r];
    }
  }
};

// What a wave whose rows are at positions [p0, p1] sees of the tiles: nothing of a tile (live() is false), or some of it
// (masked()), or all. p1 < 0: no rows.
struct WaveTiles {
  int lo, hi, sinks;                 // live: t <= hi, from lo on or with first keys
  int skip;                          // the entry that is not the wave's of a tile that comes twice
  int full_lo, full_hi, full_sinks;  // seen by all rows
  __device__ __forceinline__ void init(const TileList& list, int p0, int p1, int window, int sinks_) {
    hi = p1 < 0 ? -1 : p1 >> 5;
    lo = max(0, p0 - window + 1) >> 5;
    sinks = (sinks_ + 31) >> 5;
    skip = list.skip >= 0 && list.skip < lo ? list.sink_tiles : list.skip;
    full_hi = ((p0 + 1) >> 5) - 1;
    full_lo = (max(0, p1 - window + 1) + 31) >> 5;
    full_sinks = sinks_ >> 5;
  }
  // Entry i of the list, tile t.
  __device__ __forceinline__ bool live(int i, int t) const { return t <= hi && (t >= lo || t < sinks) && i != skip; }
  __device__ __forceinline__ bool masked(int t) const { return t > full_hi || (t < full_lo && t >= full_sinks); }
};

// In float16 dS is rounded to steps of 2^-24 below 2^-14, where that of small losses lies. It is scaled up by a power of two
// before it is rounded, 2^lift with lift = -floor(log2 |dO|), |dO| the (largest) norm of the rows. |dS| <= |dO| |v| + |delta| must
// stay finite: dK takes its keys' |v| and the rows' |delta| into account, dQ, whose rows see many keys, starts over without a
// factor where a sum is not finite. Of a step's time this is 0.2% at 4 x 16 x 4,096 x 64, window 1,024 (1.7% where dO is small), 1% at
// 16/4 x 32,768 x 64, window 128, and 3% at 4 x 16 x 8,192 x 32, window 512, whose workgroups are short.
__device__ __forceinline__ int norm_exponent(uint32_t norm2) { return ((int)(norm2 >> 23) - 127) >> 1; }  // of a squared norm's bits; NaN: 64
__device__ __forceinline__ int small_gradient_lift(int exponent, int most) { return min(max(-exponent, 0), most); }
__device__ __forceinline__ float unlift_of(int lift) { return __builtin_bit_cast(float, (uint32_t)(127 - lift) << 23); }

// Over the wave, uniform.
__device__ __forceinline__ uint32_t max_wave(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, true));   // quad_perm 1, 0, 3, 2
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, true));   // quad_perm 2, 3, 0, 1
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, true));  // row_half_mirror
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xf, 0xf, true));  // row_mirror
  const uint32_t a = max((uint32_t)__builtin_amdgcn_readlane((int)x, 0), (uint32_t)__builtin_amdgcn_readlane((int)x, 16));
  return max(a, max((uint32_t)__builtin_amdgcn_readlane((int)x, 32), (uint32_t)__builtin_amdgcn_readlane((int)x, 48)));
}

// Everything this wave has in flight has landed, its LDS reads are done, then the barrier.
__device__ __forceinline__ void all_landed_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0)
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// Workgroup -> (slice, block); false past the last. Workgroups go round-robin over the 8 XCDs. The first `head` blocks of the
// slices come before all others and the last `tail`, which are shorter and shorter, after them, the longer ones first; those
// between are equally long: an XCD takes consecutive ones, which read overlapping rows through its L2.
__device__ __forceinline__ bool window_coord(int slices, int nblk, int head, int tail, int& slice, int& blk) {
  const int even = nblk - head - tail;
  const int64_t ahead = (int64_t)slices * head, total = (int64_t)slices * even, chunk = (total + 7) >> 3;
  int64_t i = blockIdx.x;
  blk = 0;
  if (i >= ahead) {
    i -= ahead;
    if (i < 8 * chunk) {
      i = (i & 7) * chunk + (i >> 3);
      if (i >= total) return false;
      slice = (int)(i / even);
      blk = head + (int)(i % even);
      return true;
    }
    i -= 8 * chunk;
    if (i >= (int64_t)slices * tail) return false;
    blk = nblk - tail;
  }
  slice = (int)(i % slices);
  blk += (int)(i / slices);
  return true;
}

}  // namespace tattn
