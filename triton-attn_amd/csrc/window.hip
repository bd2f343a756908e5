// Attention over a sliding window and the first keys, 16-bit, forward and backward, on gfx950.
//
// A workgroup's NW = RW * CS waves own RW 32-row tiles; a step stages CS tiles of the other dimension by LDS DMA
// (buffer_load ... lds, swizzled rows) into one of two stages while the other is worked on. With many rows CS is 1 and each wave
// works on every tile for its own rows; with few, wave (rw, cs) takes every CS-th tile, and the CS partial
// results of a row tile are added through LDS at the end. Only tiles that some row of the workgroup sees are walked
// (TileList), only those at the ends of a row's window pay for masks, and a wave passes over tiles that none of its own rows sees.
//
// Rows that nobody in the workgroup sees (before the window, behind the last key) are fetched from beyond the end of
// the buffer, which reads as zero: whatever a cache holds there cannot reach a sum.
//
// Roundings: the operands of the second products, P and dS, are rounded to the element type, as the matrix instruction takes them
// (what a second operand for the rest would add: as many products again), P's sum is taken from the rounded values, and
// delta from the stored O. Scores, maxima, sums and accumulators are float32. That leaves errors 1.1 to 1.5 times those
// of a float32 computation rounded once (relative to 64 bits, in norm, all outputs: 4 x 16 x 4,096 x 64 in fp16 3.1e-4 for 2.1e-4,
// 11 x 12/4 x 1,500 x 128 in bf16 2.5e-3 for 1.7e-3). dS in fp16 is scaled first (small_gradient_lift).
//
// Bound by the issue of matrix and vector instructions and by the latency of a tile's chain (scores, exponentials, second product),
// which the 8 to 16 waves of a CU overlap only in part: at head dim 64 the forward keeps the matrix cores busy 31% and the vector
// units 49% of the time. us (rate of the products that count); whole calls, and in a profiler's trace, which clocks lower,
// the kernels one by one:
//                                                    call         forward       with gradients  |  traced: forward   dQ   dK / dV
//   4 x 16 x 4,096 x 64 fp16, window 1,024, 4 first keys            89 (680 TF)   380 (556 TF)  |           102    126     204
//   11 x 12/4 x 1,500 x 128 bf16, window 500                        64 (660 TF)   283 (522 TF)  |            79    109     143
//   1 x 32/8 x 16,384 x 128 bf16, window 4,096, 4 first keys       892 (1,080 TF)               |         1,003
//   32 x 32/8 x 128, one token, window 2,048, 4 first keys          51 (5.2 TB/s of the keys and values)  |  49
// Each row was measured in one session; sessions differ by up to 6%.
#include <algorithm>
#include <type_traits>

#include "window.h"

namespace tattn {
namespace {

// A stage: NT tiles of each of two tensors. Each wave fetches PPW 1 KB pieces of a step, TW whole tiles or a part of one,
// the first half of the waves of the first tensor.
template <int D, int NW, int NT>
struct WinRing {
  static constexpr int RB = Swz<D>::RB, TILE = 32 * RB, PIECES = TILE / 1024;
  static constexpr int HALF = NT * TILE;  // bytes of one tensor's tiles
  static constexpr int STAGE = 2 * HALF;
  static constexpr int PPW = 2 * NT * PIECES / NW;
  static constexpr int TW = PPW > PIECES ? PPW / PIECES : 1, PPT = PPW / TW;  // pieces per tile
  static_assert(PPW >= 1 && TW * PPT * NW == 2 * NT * PIECES && PIECES % PPT == 0 && NW % 2 == 0, "whole pieces, one tensor per wave");
};

constexpr uint32_t kBeyond = 0x7fffffffu;  // byte offset past every slice: reads as zero

template <int D, int NW, int NT>
struct WinLoader {
  using R = WinRing<D, NW, NT>;
  uint32_t go[R::PPT];
  uint32_t tile_bytes;
  int first, piece0, base, lane;  // first tile of the wave's TW, first piece of it, and its place in a stage
  bool second;
  __device__ __forceinline__ void init(int64_t sa, int64_t sb, int wu, int lane_) {
    lane = lane_;
    second = wu >= NW / 2;
    const int64_t st = second ? sb : sa;
    tile_bytes = uniform32((uint32_t)(st * 64));
    first = wu % (NW / 2) * R::PPW / R::PIECES;
    piece0 = wu % (NW / 2) * R::PPW % R::PIECES;
    base = (second ? R::HALF : 0) + first * R::TILE + 1024 * piece0;
    constexpr int CPR = R::RB / 16;
#pragma unroll
    for (int i = 0; i < R::PPT; ++i) {
      const int j = 64 * (piece0 + i) + lane;
      const int row = j / CPR, cc = ((j % CPR) ^ Swz<D>::f(row)) & (D / 8 - 1);
      go[i] = (uint32_t)(perm32(row) * st * 2 + cc * 16);
    }
  }
  // Row of a tile that the lane fetches in the wave's piece i.
  __device__ __forceinline__ int row(int i) const { return perm32((64 * (piece0 + i) + lane) / (R::RB / 16)); }
  __device__ __forceinline__ void fetch(__amdgpu_buffer_rsrc_t rs, char* stage, int x, int i, uint32_t off) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (TATTN_LDS void*)(stage + base + x * R::TILE + 1024 * i), 16, (int)off, 0, 0, 0);
  }
};

// Operand addresses within one tile at byte `base`: natural rows, and the transposed reads of 16-row slice 0 (the
// swizzle depends on a row's index mod 16, so slice 1 is a constant further).
template <int D>
struct WinOp {
  static constexpr int NSD = D / 16, DT = (D + 31) / 32;
  int nat[NSD], lo[DT], hi[DT];
  __device__ __forceinline__ void init(int base, int lane) {
    const int l32 = lane & 31, h2 = lane >> 5;
#pragma unroll
    for (int s = 0; s < NSD; ++s) nat[s] = base + Swz<D>::addr(l32, (16 * s + 8 * h2) * 2);
#pragma unroll
    for (int u = 0; u < DT; ++u) {
      tr_addrs<D>(0, u, lane, lo[u], hi[u]);
      lo[u] += base;
      hi[u] += base;
    }
  }
  template <typename T>
  __device__ __forceinline__ typename H16<T>::V8 tr(const char* st, int sl, int u) const {
    return tr_pair<T>(st + 16 * sl * Swz<D>::RB, lo[u], hi[u]);
  }
};

// The rows of a workgroup and of its waves, and the key tiles they see.
struct WinRows {
  int z, hk, slice, len, off;
  int rows;      // N * G
  int tile0;     // first row tile of the workgroup
  int p0, p1;    // positions of the workgroup's rows; p1 is also the last key any of them sees
  int last;      // position of the last row tile's first row
  __device__ __forceinline__ void init(const WindowParams& p, int slice_, int blk, int rw) {
    slice = slice_;
    z = slice / p.Hk;
    hk = slice % p.Hk;
    len = p.lens ? min(max(p.lens[z], 0), p.S) : p.S;
    off = len - p.N;
    rows = p.N * p.G;
    tile0 = blk * rw;
    p0 = off + (32 * tile0) / p.G;
    p1 = off + min(32 * (tile0 + rw) - 1, rows - 1) / p.G;
    last = off + min(32 * (tile0 + rw - 1), rows - 1) / p.G;
  }
};

template <typename T, int D>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t win_rsrc(const void* base, int64_t off, int64_t rows, int64_t stride) {
  return slice_rsrc((const T*)base + off, rows > 0 ? slice_bytes(rows, stride, D) : 0);
}

// K and V tiles of list entries [i0, i0 + NT) into `stage`; entries from i1 on are not fetched.
template <int D, int NW, int NT>
__device__ __forceinline__ void fetch_keys(const WinLoader<D, NW, NT>& ld, __amdgpu_buffer_rsrc_t rs, char* stage,
                                           const TileList& list, int i0, int i1, int top, int sinks) {
  using R = WinRing<D, NW, NT>;
#pragma unroll
  for (int x = 0; x < R::TW; ++x) {
    const int at = i0 + ld.first + x;
    if (at >= i1) break;
    const int t = list.at(at), low = list.low(at);
    const uint32_t o = (uint32_t)t * ld.tile_bytes;
    if (32 * t + 31 > top || (32 * t < low && 32 * t + 31 >= sinks)) {
#pragma unroll
      for (int i = 0; i < R::PPT; ++i) {
        const int key = 32 * t + ld.row(i);
        const bool dead = key > top || (key < low && key >= sinks);
        ld.fetch(rs, stage, x, i, dead ? kBeyond : ld.go[i] + o);
      }
    } else {
#pragma unroll
      for (int i = 0; i < R::PPT; ++i) ld.fetch(rs, stage, x, i, ld.go[i] + o);
    }
  }
}

// ---- forward -----------------------------------------------------------------------------------
template <typename T, int D, int RW, int CS, int OCC, bool SPLIT>
__global__ __launch_bounds__(RW * CS * 64, OCC) void window_fwd_kernel(const WindowParams p) {
  using H = H16<T>;
  using V8 = typename H::V8;
  using V4 = typename H::V4;
  using V2 = typename H::V2;
  constexpr int NW = RW * CS, NSD = D / 16, DT = (D + 31) / 32;
  using R = WinRing<D, NW, CS>;
  // Two arrays: a DMA into one stage does not alias reads of the other.
  __shared__ __attribute__((aligned(1024))) char s0[R::STAGE];
  __shared__ __attribute__((aligned(1024))) char s1[R::STAGE];
  __shared__ float red[2][CS > 1 || SPLIT ? NW : 1][32];

  const int tid = threadIdx.x;
  const int lane = tid & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(tid >> 6));
  const int rw = wu / CS, cs = wu % CS;
  const float c = p.c;
  int slice, blk, split = 0;
  if (!window_coord(p.Z * p.Hk, p.nblk * (SPLIT ? p.splits : 1), p.head, p.tail, slice, blk)) return;
  if (SPLIT) split = blk % p.splits, blk /= p.splits;
  WinRows b;
  b.init(p, slice, p.nblk - 1 - blk, RW);  // longest rows first
  TileList list;
  list.init(b.p0, b.p1, b.last, p.window, p.sinks);
  const int i0 = SPLIT ? (int)((int64_t)list.n * split / p.splits) : 0;
  const int i1 = SPLIT ? (int)((int64_t)list.n * (split + 1) / p.splits) : list.n;
  const int nsteps = (i1 - i0 + CS - 1) / CS;

  WinLoader<D, NW, CS> ld;
  ld.init(p.sk[2], p.sv[2], wu, lane);
  const __amdgpu_buffer_rsrc_t rs =
      ld.second ? win_rsrc<T, D>(p.v, b.z * p.sv[0] + b.hk * p.sv[1], b.len, p.sv[2])
                : win_rsrc<T, D>(p.k, b.z * p.sk[0] + b.hk * p.sk[1], b.len, p.sk[2]);
  auto issue = [&](char* stage, int step) __attribute__((always_inline)) {
    fetch_keys<D, NW, CS>(ld, rs, stage, list, i0 + step * CS, i1, b.p1, p.sinks);
  };
  if (nsteps > 0) issue(s0, 0);

  const int tile0 = 32 * (b.tile0 + rw);
  const int row = tile0 + l32;
  const bool live = row < b.rows;
  const int n = (live ? row : 0) / p.G, g = (live ? row : 0) % p.G;
  const int pos = b.off + n;
  // The wave's positions; a wave without rows sees no tile.
  WaveTiles sees;
  sees.init(list, b.off + tile0 / p.G, tile0 < b.rows ? b.off + min(tile0 + 31, b.rows - 1) / p.G : -1, p.window, p.sinks);
  V8 qop[NSD];
  {
    const T* src = (const T*)p.q + b.z * p.sq[0] + (b.hk * p.G + g) * p.sq[1] + n * p.sq[2] + 8 * h2;
#pragma unroll
    for (int s = 0; s < NSD; ++s) {
      const V8 x = *reinterpret_cast<const V8*>(src + 16 * s);
      qop[s] = live ? x : V8{};
    }
  }
  WinOp<D> at;
  at.init(cs * R::TILE, lane);

  const float hidden = hidden_score(c);
  float mrow = kNoMax, lrow = 0.0f;
  f32x16 acc[DT];
#pragma unroll
  for (int u = 0; u < DT; ++u) acc[u] = f32x16{};

  // Tile t, staged in `st`. Probabilities against the running max as it stands; a lane whose 16 probabilities sum above
  // 2^12 (its first visible tile among them) sends the wave through the row max and a rescale. The branches are
  // one-sided (state updated first, undone inside): two-sided ones make the allocator hold two copies of it and copy the
  // accumulators in every tile.
  auto tile = [&](const char* st, int t) __attribute__((always_inline)) {
    f32x16 s = f32x16{};
#pragma unroll
    for (int sd = 0; sd < NSD; ++sd) s = Elt<T>::mfma(lds8<T>(st + at.nat[sd]), qop[sd], s);
    if (sees.masked(t)) RowMask(pos, t, h2, p.window, p.sinks).hide(s, hidden);
    V8 x[2];
    auto probs = [&]() __attribute__((always_inline)) {
      float ps = 0.0f;
#pragma unroll
      for (int sg = 0; sg < 2; ++sg)
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const int r = 8 * sg + i;
          const V2 pr = H::pack(fast_exp2(__builtin_fmaf(s[r], c, -mrow)), fast_exp2(__builtin_fmaf(s[r + 1], c, -mrow)));
          ps = H::sum2(pr, ps);
          x[sg][i] = pr[0];
          x[sg][i + 1] = pr[1];
        }
      return ps;
    };
    const float lprev = lrow;
    const float ps = probs();
    lrow += ps;
    if (__builtin_amdgcn_ballot_w64(!(ps <= 4096.0f))) {
      float mx = kNoMax;
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = __builtin_fmaxf(mx, s[r] * c);
      const float cand = max_halves(mx);
      const float mnew = cand > mrow + kRescaleLog2 ? cand : mrow;
      const float alpha = fast_exp2(mrow - mnew);
      mrow = mnew;
      const float again = probs();
      lrow = lprev * alpha + again;
#pragma unroll
      for (int u = 0; u < DT; ++u) acc[u] *= alpha;
    }
#pragma unroll
    for (int sg = 0; sg < 2; ++sg)
#pragma unroll
      for (int u = 0; u < DT; ++u) {
        V8 va = at.template tr<T>(st + R::HALF, sg, u);
        if (D < 32 && 16 * ((lane >> 4) & 1) >= D) va = V8{};
        acc[u] = Elt<T>::mfma(va, x[sg], acc[u]);
      }
  };
  auto step = [&](int i, char* cur, char* nxt) __attribute__((always_inline)) {
    if (i + 1 < nsteps) issue(nxt, i + 1);
    const int k = i0 + i * CS + cs;
    if (k < i1) {
      const int t = list.at(k);
      if (sees.live(k, t)) tile(cur, t);
    }
    all_landed_barrier();
  };
  all_landed_barrier();
  int i = 0;
  for (; i + 1 < nsteps; i += 2) {
    step(i, s0, s1);
    step(i + 1, s1, s0);
  }
  if (i < nsteps) step(i, s0, s1);

  // Merge the CS partial rows of each row tile (the stages are free: every wave passed the last barrier and no
  // DMA is in flight). A split keeps the sums as they are; otherwise they are divided by the row's sum, and rows
  // that see no key become 0.
  const float lt = sum_halves(lrow);
  if constexpr (CS == 1 && !SPLIT) {
    const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
    if (!live) return;
    T* orow = (T*)p.out + b.z * p.sout[0] + (b.hk * p.G + g) * p.sout[1] + n * p.sout[2];
#pragma unroll
    for (int u = 0; u < DT; ++u)
#pragma unroll
      for (int gr = 0; gr < 4; ++gr) {
        const int d0 = 32 * u + 8 * gr + 4 * h2;
        if (d0 >= D) continue;
        V4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (T)(acc[u][4 * gr + e] * inv);
        *reinterpret_cast<V4*>(orow + d0) = y;
      }
    if (h2 == 0 && p.m) p.m[((int64_t)b.z * p.H + b.hk * p.G + g) * p.N + n] = mrow + __log2f(lt);
    return;
  }
  if (h2 == 0) {
    red[0][wu][l32] = mrow;
    red[1][wu][l32] = lt;
  }
  __syncthreads();
  float mall = kNoMax;
#pragma unroll
  for (int k = 0; k < CS; ++k) mall = __builtin_fmaxf(mall, red[0][rw * CS + k][l32]);
  float lall = 0.0f;
#pragma unroll
  for (int k = 0; k < CS; ++k) lall += fast_exp2(red[0][rw * CS + k][l32] - mall) * red[1][rw * CS + k][l32];
  float wgt = fast_exp2(mrow - mall);
  if (!SPLIT) wgt = lall == 0.0f ? 0.0f : wgt / lall;
  constexpr int PART = DT * 16 * 64 * 4;  // bytes of one wave's partial O^T
  constexpr int PER = R::STAGE / PART;    // partials per stage array
  static_assert((CS == 1 && !SPLIT) || 2 * PER >= NW, "partials fit the stages");
  auto part = [&](int k) { return (TATTN_LDS float*)(k < PER ? s0 + k * PART : s1 + (k - PER) * PART); };
  {
    TATTN_LDS float* dst = part(wu) + lane;
#pragma unroll
    for (int u = 0; u < DT; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) dst[(16 * u + r) * 64] = acc[u][r] * wgt;
  }
  __syncthreads();
  if (!live) return;
  const int64_t prow = ((int64_t)b.slice * (SPLIT ? p.splits : 1) + split) * b.rows + row;
  T* orow = (T*)p.out + b.z * p.sout[0] + (b.hk * p.G + g) * p.sout[1] + n * p.sout[2];
  float* frow = p.part + prow * D;
  for (int gr = cs; gr < DT * 4; gr += CS) {  // four consecutive columns per register group
    const int d0 = 8 * gr + 4 * h2;
    if (d0 < D) {
      f32x4 x = f32x4{};
#pragma unroll
      for (int k = 0; k < CS; ++k) {
        const TATTN_LDS float* src = part(rw * CS + k) + lane + 4 * gr * 64;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += src[64 * e];
      }
      if (SPLIT) {
        *reinterpret_cast<f32x4*>(frow + d0) = x;
      } else {
        V4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (T)x[e];
        *reinterpret_cast<V4*>(orow + d0) = y;
      }
    }
  }
  if (cs == 0 && h2 == 0) {
    if (SPLIT) {
      float* ml = p.part + (int64_t)p.Z * p.Hk * p.splits * b.rows * D + prow * 2;
      ml[0] = mall;
      ml[1] = lall;
    } else if (p.m) {
      p.m[((int64_t)b.z * p.H + b.hk * p.G + g) * p.N + n] = mall + __log2f(lall);
    }
  }
}

// ---- rows whose keys were split ------------------------------------------------------------------
// O = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s. A workgroup takes one row: D / 4 lanes over the columns, the parts dealt
// to the 1024 / D groups of them, whose sums are added in order through LDS (a group walking all of 125 parts took 60 us).
template <typename T, int D>
__global__ __launch_bounds__(256) void combine_kernel(const float* part, T* out, float* m, int64_t sz, int64_t sh, int64_t sn,
                                                      int Hk, int G, int N, int splits) {
  typedef T V4 __attribute__((ext_vector_type(4)));
  constexpr int LPR = D / 4, GROUPS = 256 / LPR;
  __shared__ float red[4];
  __shared__ __attribute__((aligned(16))) float sums[GROUPS][D];
  __shared__ float ls[GROUPS];
  const int tid = threadIdx.x, rows = N * G;
  const int64_t slice = blockIdx.x / rows, slices = gridDim.x / rows;
  const int row = (int)(blockIdx.x % rows), d0 = tid % LPR * 4, g = tid / LPR;
  const float* ml = part + slices * splits * rows * D;
  const int64_t first = slice * splits * rows + row;
  float mall = kNoMax;
  for (int s = tid; s < splits; s += 256) mall = __builtin_fmaxf(mall, ml[(first + (int64_t)s * rows) * 2]);
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) mall = __builtin_fmaxf(mall, __shfl_xor(mall, i));
  red[tid >> 6] = mall;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) mall = __builtin_fmaxf(mall, red[i]);
  f32x4 x = f32x4{};
  float l = 0.0f;
#pragma unroll 4
  for (int s = g; s < splits; s += GROUPS) {
    const int64_t at = first + (int64_t)s * rows;
    const float w = fast_exp2(ml[at * 2] - mall), part_l = ml[at * 2 + 1];
    if (part_l == 0.0f) continue;  // no visible key: the sums of such a part may not be there
    l = __builtin_fmaf(w, part_l, l);
    const f32x4 y = *reinterpret_cast<const f32x4*>(part + at * D + d0);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(w, y[e], x[e]);
  }
  *reinterpret_cast<f32x4*>(&sums[g][d0]) = x;
  if (d0 == 0) ls[g] = l;
  __syncthreads();
  if (g > 0) return;
  for (int i = 1; i < min(GROUPS, splits); ++i) {
    l += ls[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += sums[i][d0 + e];
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t z = slice / Hk, h = slice % Hk * G + row % G, n = row / G;
  V4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (T)(l == 0.0f ? 0.0f : x[e] * inv);
  *reinterpret_cast<V4*>(out + z * sz + h * sh + n * sn + d0) = y;
  if (m && d0 == 0) m[(z * Hk * G + h) * N + n] = mall + __log2f(l);
}

// ---- dQ ------------------------------------------------------------------------------------------
// Rows and key tiles as in the forward; computes delta = rowsum(dO * O) on the way and stores -delta for dK / dV, in float16 also
// the largest squared norm of the block's rows of dO and its largest |delta|.
template <typename T, int D, int RW, int OCC>
__global__ __launch_bounds__(RW * 64, OCC) void window_dq_kernel(const WindowParams p) {
  using H = H16<T>;
  using V8 = typename H::V8;
  using V4 = typename H::V4;
  using V2 = typename H::V2;
  constexpr int NSD = D / 16, DT = (D + 31) / 32;
  using R = WinRing<D, RW, 1>;
  constexpr bool LIFT = std::is_same_v<T, f16>;
  __shared__ __attribute__((aligned(1024))) char s0[R::STAGE];
  __shared__ __attribute__((aligned(1024))) char s1[R::STAGE];
  __shared__ uint32_t norms[3][LIFT ? RW : 1];  // per wave: largest squared norm, |delta|, whether a row is lifted

  const int tid = threadIdx.x;
  const int lane = tid & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(tid >> 6));
  const float c = p.c;
  int slice, blk;
  if (!window_coord(p.Z * p.Hk, p.nblk, p.head, p.tail, slice, blk)) return;
  blk = p.nblk - 1 - blk;
  WinRows b;
  b.init(p, slice, blk, RW);
  TileList list;
  list.init(b.p0, b.p1, b.last, p.window, p.sinks);

  WinLoader<D, RW, 1> ld;
  ld.init(p.sk[2], p.sv[2], wu, lane);
  const __amdgpu_buffer_rsrc_t rs =
      ld.second ? win_rsrc<T, D>(p.v, b.z * p.sv[0] + b.hk * p.sv[1], b.len, p.sv[2])
                : win_rsrc<T, D>(p.k, b.z * p.sk[0] + b.hk * p.sk[1], b.len, p.sk[2]);
  auto issue = [&](char* stage, int i) __attribute__((always_inline)) {
    fetch_keys<D, RW, 1>(ld, rs, stage, list, i, list.n, b.p1, p.sinks);
  };
  if (list.n > 0) issue(s0, 0);

  const int tile0 = 32 * (b.tile0 + wu);
  const int row = tile0 + l32;
  const bool live = row < b.rows;
  const int n = (live ? row : 0) / p.G, g = (live ? row : 0) % p.G, h = b.hk * p.G + g;
  const int pos = b.off + n;
  WaveTiles sees;
  sees.init(list, b.off + tile0 / p.G, tile0 < b.rows ? b.off + min(tile0 + 31, b.rows - 1) / p.G : -1, p.window, p.sinks);
  const int64_t mrow = ((int64_t)b.z * p.H + h) * p.N + n;
  V8 qop[NSD], dop[NSD];
  float dl;
  int lift = 0;  // dS is scaled by 2^lift
  uint32_t top = 0;
  {
    const T* qs = (const T*)p.q + b.z * p.sq[0] + h * p.sq[1] + n * p.sq[2] + 8 * h2;
    const T* ds = (const T*)p.dout + b.z * p.sd[0] + h * p.sd[1] + n * p.sd[2] + 8 * h2;
    const T* os = (const T*)p.o + b.z * p.so[0] + h * p.so[1] + n * p.so[2] + 8 * h2;
    float sd[NSD], norm = 0.0f;
#pragma unroll
    for (int s = 0; s < NSD; ++s) {
      const V8 x = *reinterpret_cast<const V8*>(qs + 16 * s), y = *reinterpret_cast<const V8*>(ds + 16 * s);
      qop[s] = live ? x : V8{};
      dop[s] = live ? y : V8{};
      sd[s] = chunk_dot(*reinterpret_cast<const V8*>(os + 16 * s), y);
      if (LIFT) norm += chunk_dot(dop[s], dop[s]);
    }
    if constexpr (LIFT) {
      const uint32_t bits = __builtin_bit_cast(uint32_t, sum_halves(norm));
      lift = small_gradient_lift(norm_exponent(bits), 60);
      top = max_wave(bits);  // NaN above all
      norms[0][wu] = top;
      norms[2][wu] = __builtin_amdgcn_ballot_w64(lift > 0) != 0;
    }
    dl = row_delta(sd);
    if (live && h2 == 0) p.delta[mrow] = -dl;
    if (!live) dl = 0.0f;
    if constexpr (LIFT) {  // delta counts where all rows are small
      norms[1][wu] = 0;
      if (norm_exponent(top) < 0) norms[1][wu] = max_wave(__builtin_bit_cast(uint32_t, __builtin_fabsf(dl)));
    }
  }
  const float m = live ? p.m[mrow] : 0.0f;
  float nm = live ? (float)lift - m : 0.0f;
  WinOp<D> at;
  at.init(0, lane);
  f32x16 dq[DT];

  const float hidden = hidden_score(c);
  auto tile = [&](const char* st, int t) __attribute__((always_inline)) {
    f32x16 s = f32x16{}, dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) dp[r] = -dl;  // seeds dP - delta
#pragma unroll
    for (int sd = 0; sd < NSD; ++sd) {
      s = Elt<T>::mfma(lds8<T>(st + at.nat[sd]), qop[sd], s);
      dp = Elt<T>::mfma(lds8<T>(st + R::HALF + at.nat[sd]), dop[sd], dp);
    }
    if (sees.masked(t)) RowMask(pos, t, h2, p.window, p.sinks).hide(s, hidden);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = fast_exp2(__builtin_fmaf(s[r], c, nm)) * dp[r];
    V8 ds[2];
#pragma unroll
    for (int sl = 0; sl < 2; ++sl)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const V2 dh = H::pack(s[8 * sl + i], s[8 * sl + i + 1]);
        ds[sl][i] = dh[0];
        ds[sl][i + 1] = dh[1];
      }
#pragma unroll
    for (int sl = 0; sl < 2; ++sl)
#pragma unroll
      for (int u = 0; u < DT; ++u) {
        V8 a = at.template tr<T>(st, sl, u);
        if (D < 32 && 16 * ((lane >> 4) & 1) >= D) a = V8{};
        dq[u] = Elt<T>::mfma(a, ds[sl], dq[u]);
      }
  };
  auto step = [&](int i, char* cur, char* nxt) __attribute__((always_inline)) {
    if (i + 1 < list.n) issue(nxt, i + 1);
    const int t = list.at(i);
    if (sees.live(i, t)) tile(cur, t);
    all_landed_barrier();
  };
  all_landed_barrier();
  uint32_t lifted = 0;
  if constexpr (LIFT) {
    if (tid < 2) {  // for dK / dV
      top = norms[tid][0];
#pragma unroll
      for (int k = 1; k < RW; ++k) top = max(top, norms[tid][k]);
      p.norms[2 * ((int64_t)b.slice * p.nblk + blk) + tid] = __builtin_bit_cast(float, top);
    }
#pragma unroll
    for (int k = 0; k < RW; ++k) lifted |= norms[2][k];
    lifted = uniform32(lifted);
  }
  for (;;) {
#pragma unroll
    for (int u = 0; u < DT; ++u) dq[u] = f32x16{};
    int i = 0;
    for (; i + 1 < list.n; i += 2) {
      step(i, s0, s1);
      step(i + 1, s1, s0);
    }
    if (i < list.n) step(i, s0, s1);
    if (!LIFT || !lifted) break;
    float zero = 0.0f;  // times every sum: NaN where one is not finite
#pragma unroll
    for (int u = 0; u < DT; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) zero = __builtin_fmaf(dq[u][r], 0.0f, zero);
    if (!__syncthreads_or(lift > 0 && zero != 0.0f)) break;
    lifted = lift = 0;
    nm = -m;
    issue(s0, 0);
    all_landed_barrier();
  }
  const float scale = LIFT ? p.scale * unlift_of(lift) : p.scale;

  if (!live) return;
  T* orow = (T*)p.out + b.z * p.sout[0] + h * p.sout[1] + n * p.sout[2];
#pragma unroll
  for (int u = 0; u < DT; ++u)
#pragma unroll
    for (int gr = 0; gr < 4; ++gr) {
      const int d0 = 32 * u + 8 * gr + 4 * h2;
      if (d0 >= D) continue;
      V4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (T)(dq[u][4 * gr + e] * scale);
      *reinterpret_cast<V4*>(orow + d0) = y;
    }
}

// ---- dK / dV -------------------------------------------------------------------------------------
// A workgroup owns RW tiles of 32 keys and walks the query tiles that see any of them, head after head of
// the group: the sum over shared heads stays in registers. Key blocks that hold first keys are seen by every later query, an
// N / window-fold of the others' work: their list is cut into `splits` parts. Where all blocks of all slices would fill the
// chip only in part, the others' lists are cut into `parts`. Parts write float32 sums that window_parts_kernel adds in order.
struct KeyBlocks {
  int sink_blocks, splits, parts;
  int blocks, items;  // per slice: sink_blocks * splits parts, then the other blocks' parts
  __host__ __device__ explicit KeyBlocks(int rw, const WindowParams& p) : splits(p.splits), parts(p.parts) {
    blocks = (p.S + 32 * rw - 1) / (32 * rw);
    sink_blocks = splits > 1 ? (p.sinks + 32 * rw - 1) / (32 * rw) : 0;
    if (sink_blocks > blocks) sink_blocks = blocks;
    items = sink_blocks * splits + (blocks - sink_blocks) * parts;
  }
  // Key block, part and number of parts of an item.
  __device__ __forceinline__ void block(int item, int& kb, int& part, int& of) const {
    const int rest = item - sink_blocks * splits;
    of = rest < 0 ? splits : parts;
    const int i = rest < 0 ? item : rest;
    kb = i / of + (rest < 0 ? 0 : sink_blocks);
    part = i % of;
  }
  __host__ __device__ int first(int kb) const {  // item of its first part
    return kb < sink_blocks ? kb * splits : sink_blocks * splits + (kb - sink_blocks) * parts;
  }
  __host__ __device__ int parted() const { return parts > 1 ? blocks : sink_blocks; }  // blocks in parts, the first ones
};

// Whether any query sees the key: what lies at another is taken as zero.
__device__ __forceinline__ bool key_seen(const WindowParams& p, int off, int key) {
  return key < p.S && (key < p.sinks || off - key < p.window);
}

// What dS of a block of keys that queries nlo .. nhi see is scaled by (small_gradient_lift), the same for all lanes. Loaded
// first and looked at once the first tiles are on their way.
struct KeysLift {
  const u32x2* norms;
  int i, last;
  u32x2 top;  // squared norm of dO, |delta|
  __device__ __forceinline__ KeysLift(const WindowParams& p, int slice, int nlo, int nhi, int lane) {
    norms = reinterpret_cast<const u32x2*>(p.norms) + (int64_t)slice * window_norm_blocks(p.N, p.G);
    i = (nlo * p.G >> 7) + lane;
    last = (nhi * p.G + p.G - 1) >> 7;
    top = i <= last ? norms[i] : u32x2{};
  }
  template <typename V8, int N>
  __device__ __forceinline__ int lift(const V8 (&v)[N]) {  // v: the lane's half of its key's value
    for (i += 64; i <= last; i += 256) {  // four loads at a time
      const u32x2 a = norms[i], b = norms[min(i + 64, last)], c = norms[min(i + 128, last)], d = norms[min(i + 192, last)];
#pragma unroll
      for (int k = 0; k < 2; ++k) top[k] = max(top[k], max(max(a[k], b[k]), max(c[k], d[k])));
    }
    const int row = norm_exponent(max_wave(top[0]));
    if (row >= 0) return 0;
    float norm = 0.0f;
#pragma unroll
    for (int s = 0; s < N; ++s) norm += chunk_dot(v[s], v[s]);
    const int key = norm_exponent(max_wave(__builtin_bit_cast(uint32_t, sum_halves(norm))));
    const int delta = (int)(max_wave(top[1]) >> 23) - 127;
    // |dS| < 2^(row + key + 2) + 2^(delta + 1)
    return min(small_gradient_lift(row, 15), max(min(12 - row - key, 13 - delta), 0));
  }
};

template <typename T, int D, int RW, int CS, int OCC>
__global__ __launch_bounds__(RW * CS * 64, OCC) void window_dkdv_kernel(const WindowParams p) {
  using H = H16<T>;
  using V8 = typename H::V8;
  using V2 = typename H::V2;
  constexpr int NW = RW * CS, NSD = D / 16, DT = (D + 31) / 32;
  using R = WinRing<D, NW, CS>;
  __shared__ __attribute__((aligned(1024))) char s0[R::STAGE];
  __shared__ __attribute__((aligned(1024))) char s1[R::STAGE];
  __shared__ __attribute__((aligned(16))) float md[NW][2][64];  // per wave and parity: M[32], -delta[32]

  const int tid = threadIdx.x;
  const int lane = tid & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(tid >> 6));
  const int rw = wu / CS, cs = wu % CS;
  const float c = p.c;
  const KeyBlocks kbs(RW, p);
  int slice, item, kb, split, splits;
  if (!window_coord(p.Z * p.Hk, kbs.items, p.head, p.tail, slice, item)) return;
  kbs.block(item, kb, split, splits);
  const bool parted = splits > 1;
  const int z = slice / p.Hk, hk = slice % p.Hk, off = p.S - p.N;
  const int k0 = 32 * RW * kb, k1 = k0 + 32 * RW - 1;
  // Queries that see a key of the block, as tiles of 32 of each head in turn.
  const int nlo = max(0, k0 - off);
  const int nhi = k0 < p.sinks ? p.N - 1 : min(p.N - 1, k1 + p.window - 1 - off);
  const int qt0 = nlo >> 5, nq = nhi < nlo ? 0 : (nhi >> 5) - qt0 + 1;
  const int total = nq * p.G;
  const int i0 = (int)((int64_t)total * split / splits), i1 = (int)((int64_t)total * (split + 1) / splits);
  const int nsteps = (i1 - i0 + CS - 1) / CS;

  WinLoader<D, NW, CS> ld;
  ld.init(p.sq[2], p.sd[2], wu, lane);
  const char* qbase = ld.second ? (const char*)((const T*)p.dout + z * p.sd[0] + (int64_t)hk * p.G * p.sd[1])
                                : (const char*)((const T*)p.q + z * p.sq[0] + (int64_t)hk * p.G * p.sq[1]);
  const int64_t head_bytes = (ld.second ? p.sd[1] : p.sq[1]) * 2;
  const uint32_t qbytes = (uint32_t)slice_bytes(p.N, ld.second ? p.sd[2] : p.sq[2], D);
  auto issue = [&](char* stage, int step) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < R::TW; ++x) {
      const int k = i0 + step * CS + ld.first + x;
      if (k >= i1) break;
      const int g = k / nq, qt = qt0 + k % nq;
      // Rows past the head's last query lie past the end of its slice and read as zero.
      const __amdgpu_buffer_rsrc_t rs = slice_rsrc(qbase + g * head_bytes, qbytes);
#pragma unroll
      for (int i = 0; i < R::PPT; ++i) ld.fetch(rs, stage, x, i, ld.go[i] + (uint32_t)qt * ld.tile_bytes);
    }
  };
  constexpr bool LIFT = std::is_same_v<T, f16>;
  KeysLift kl(p, slice, nlo, LIFT ? nhi : -1, lane);
  if (nsteps > 0) issue(s0, 0);
  // Lanes 0-31 fetch M and lanes 32-63 -delta of the wave's tile; zero past the end.
  const float* mdsrc = (h2 ? p.delta : p.m) + ((int64_t)z * p.H + hk * p.G) * p.N;
  auto md_load = [&](int step) __attribute__((always_inline)) {
    const int k = i0 + step * CS + cs;
    const int q = k < i1 ? 32 * (qt0 + k % nq) + l32 : p.N;
    return q < p.N ? mdsrc[(int64_t)(k / nq) * p.N + q] : 0.0f;
  };
  const float md0 = nsteps > 0 ? md_load(0) : 0.0f;
  const int kt = kb * RW + rw, key = 32 * kt + l32;
  const bool seen = key_seen(p, off, key);
  V8 kop[NSD], vop[NSD];
  {
    const T* ks = (const T*)p.k + z * p.sk[0] + hk * p.sk[1] + (int64_t)(key < p.S ? key : 0) * p.sk[2] + 8 * h2;
    const T* vs = (const T*)p.v + z * p.sv[0] + hk * p.sv[1] + (int64_t)(key < p.S ? key : 0) * p.sv[2] + 8 * h2;
#pragma unroll
    for (int s = 0; s < NSD; ++s) {
      const V8 a = *reinterpret_cast<const V8*>(ks + 16 * s);
      const V8 b = *reinterpret_cast<const V8*>(vs + 16 * s);
      kop[s] = seen ? a : V8{};
      vop[s] = seen ? b : V8{};
    }
  }
  // P, and with it dS, is scaled by 2^lift through M.
  const int by = LIFT ? kl.lift(vop) : 0;
  const float unlift = unlift_of(by), lift = LIFT && h2 == 0 ? (float)by : 0.0f;
  md[wu][0][lane] = md0 - lift;
  WinOp<D> at;
  at.init(cs * R::TILE, lane);
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int u = 0; u < DT; ++u) dk[u] = dv[u] = f32x16{};

  const float hidden = hidden_score(c);
  auto tile = [&](const char* st, const float* mdw, int qt, bool masked) __attribute__((always_inline)) {
    f32x16 s = f32x16{}, dp;
    float mv[16];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int o = 16 * (a >> 1) + 8 * h2 + 4 * (a & 1);
      const f32x4 x = *reinterpret_cast<const TATTN_LDS f32x4*>((const TATTN_LDS float*)mdw + o);
      const f32x4 y = *reinterpret_cast<const TATTN_LDS f32x4*>((const TATTN_LDS float*)mdw + 32 + o);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mv[4 * a + i] = x[i];
        dp[4 * a + i] = y[i];
      }
    }
#pragma unroll
    for (int sd = 0; sd < NSD; ++sd) {
      s = Elt<T>::mfma(lds8<T>(st + at.nat[sd]), kop[sd], s);
      dp = Elt<T>::mfma(lds8<T>(st + R::HALF + at.nat[sd]), vop[sd], dp);
    }
    if (masked) ColMask(off + 32 * qt - key, key, p.N - 32 * qt, h2, p.window, p.sinks).hide(s, hidden);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = fast_exp2(__builtin_fmaf(s[r], c, -mv[r]));
    V8 pp[2], ds[2];
#pragma unroll
    for (int sl = 0; sl < 2; ++sl)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const int r = 8 * sl + i;
        const V2 ph = H::pack(s[r], s[r + 1]), dh = H::pack(s[r] * dp[r], s[r + 1] * dp[r + 1]);
        pp[sl][i] = ph[0];
        pp[sl][i + 1] = ph[1];
        ds[sl][i] = dh[0];
        ds[sl][i + 1] = dh[1];
      }
#pragma unroll
    for (int sl = 0; sl < 2; ++sl)
#pragma unroll
      for (int u = 0; u < DT; ++u) {
        V8 dob = at.template tr<T>(st + R::HALF, sl, u);
        V8 qb = at.template tr<T>(st, sl, u);
        if (D < 32 && 16 * ((lane >> 4) & 1) >= D) dob = qb = V8{};
        dv[u] = Elt<T>::mfma(pp[sl], dob, dv[u]);
        dk[u] = Elt<T>::mfma(ds[sl], qb, dk[u]);
      }
  };
  const int wk0 = 32 * kt, wk1 = wk0 + 31;
  auto step = [&](int i, char* cur, char* nxt, int par) __attribute__((always_inline)) {
    float mdn = 0.0f;
    if (i + 1 < nsteps) {
      issue(nxt, i + 1);
      mdn = md_load(i + 1);
    }
    const int k = i0 + i * CS + cs;
    if (k < i1 && wk0 < p.S) {
      const int qt = qt0 + k % nq, q0 = off + 32 * qt, q1 = q0 + 31;
      if (q1 >= wk0 && (q0 - wk1 < p.window || wk0 < p.sinks))
        tile(cur, md[wu][par], qt, q0 < wk1 || (q1 - wk0 >= p.window && wk1 >= p.sinks) || 32 * qt + 32 > p.N);
    }
    md[wu][par ^ 1][lane] = mdn - lift;  // the wave's own rows: no barrier needed
    all_landed_barrier();
  };
  all_landed_barrier();
  int i = 0;
  for (; i + 1 < nsteps; i += 2) {
    step(i, s0, s1, 0);
    step(i + 1, s1, s0, 1);
  }
  if (i < nsteps) step(i, s0, s1, 0);

  // Sum the CS partials of each key tile, dK then dV: wave 0 of a tile keeps its own in registers. C register r of
  // a lane: key 8 (r / 4) + 4 h2 + r % 4 of the tile, column 32 u + l32.
  constexpr int PART = DT * 16 * 64 * 4;
  constexpr int PER = R::STAGE / PART;
  static_assert(2 * PER >= RW * (CS - 1), "partials fit the stages");
  auto part = [&](int k) { return (TATTN_LDS float*)(k < PER ? s0 + k * PART : s1 + (k - PER) * PART); };
  // A part's sums: [slice][item][dK, dV][32 RW keys][D] float32.
  float* fdst = p.part + ((int64_t)slice * kbs.first(kbs.parted()) + item) * (2 * 32 * RW * D);
  auto reduce = [&](const f32x16 (&a)[DT], float mul, T* dst, int64_t stride, float* fpart) __attribute__((always_inline)) {
    if (cs > 0) {
      TATTN_LDS float* mine = part(rw * (CS - 1) + cs - 1) + lane;
#pragma unroll
      for (int u = 0; u < DT; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) mine[(16 * u + r) * 64] = a[u][r];
    }
    __syncthreads();
    if (cs == 0) {
#pragma unroll
      for (int u = 0; u < DT; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float x = a[u][r];
#pragma unroll
          for (int k = 0; k < CS - 1; ++k) x += (part(rw * (CS - 1) + k) + lane)[(16 * u + r) * 64];
          const int in = 8 * (r >> 2) + 4 * h2 + (r & 3), d = 32 * u + l32;
          if (d >= D) continue;
          if (parted) fpart[(32 * rw + in) * D + d] = x * unlift;
          else if (wk0 + in < p.S) dst[(int64_t)(wk0 + in) * stride + d] = (T)(x * mul);
        }
    }
  };
  reduce(dk, p.scale * unlift, (T*)p.dk + z * p.sdk[0] + hk * p.sdk[1], p.sdk[2], fdst);
  __syncthreads();
  reduce(dv, unlift, (T*)p.dv + z * p.sdv[0] + hk * p.sdv[1], p.sdv[2], fdst + 32 * RW * D);
}

// dK / dV at head dims 64 and 128: two waves per 32-key tile. Over each 32-query tile wave j (role A) computes S = Q K^T,
// P = 2^(S c - M), dV += P^T dO, and wave j + RW (role B) dP - delta = dO V^T - delta, dS = P (dP - delta), dK += dS^T Q,
// taking P from A through LDS in float32. Each keeps one of K / V and one accumulator set: half the registers of a wave that
// does both, so that two waves (head dim 128) or four (64) share a SIMD, with as many matrix instructions in either role.
// Step i, one barrier each: A takes tile i, B tile i - 1, and tile i + 1 (with four stages i + 2 too) is on its way. Nothing is
// pipelined inside a wave: the waves of a SIMD overlap each other's matrix and vector work.
template <typename T, int D, int RW, int NST, int OCC>
__global__ __launch_bounds__(RW * 128, OCC) void window_dkdv_pair_kernel(const WindowParams p) {
  using H = H16<T>;
  using V8 = typename H::V8;
  using V2 = typename H::V2;
  constexpr int NW = 2 * RW, NSD = D / 16, DT = D / 32, RB = Swz<D>::RB, TILE = 32 * RB;
  constexpr int PW = 2 * TILE / 1024 / NW;          // 1 KB pieces per wave and step
  constexpr int STAGE = 2 * TILE + 256;             // Q, dO, M[32], -delta[32]
  constexpr int XB = 32 * 32 * 4;                   // P of a pair
  // Arrays of their own: a DMA into one does not alias reads of the others.
  __shared__ __attribute__((aligned(256))) char st0[STAGE], st1[STAGE], st2[STAGE], st3[NST == 4 ? STAGE : 16];
  __shared__ __attribute__((aligned(256))) char xbuf[2 * RW * XB];
  auto stage = [&](auto tag) __attribute__((always_inline)) -> char* {
    constexpr int I = decltype(tag)::value % NST;
    return I == 0 ? st0 : I == 1 ? st1 : I == 2 ? st2 : st3;
  };

  const int tid = threadIdx.x;
  const int lane = tid & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(tid >> 6));
  const int pr = wu % RW;
  const bool role_b = wu >= RW;
  const float c = p.c;
  const KeyBlocks kbs(RW, p);
  int slice, item, kb, split, splits;
  if (!window_coord(p.Z * p.Hk, kbs.items, p.head, p.tail, slice, item)) return;
  kbs.block(item, kb, split, splits);
  const bool parted = splits > 1;
  const int z = slice / p.Hk, hk = slice % p.Hk, off = p.S - p.N;
  const int k0 = 32 * RW * kb, k1 = k0 + 32 * RW - 1;
  // Queries that see a key of the block, as tiles of 32 of each head in turn.
  const int nlo = max(0, k0 - off);
  const int nhi = k0 < p.sinks ? p.N - 1 : min(p.N - 1, k1 + p.window - 1 - off);
  const int qt0 = nlo >> 5, nq = nhi < nlo ? 0 : (nhi >> 5) - qt0 + 1;
  const int total = nq * p.G;
  const int i0 = (int)((int64_t)total * split / splits), i1 = (int)((int64_t)total * (split + 1) / splits);
  const int n = i1 - i0;
  const int wk0 = 32 * (kb * RW + pr), wk1 = wk0 + 31, key = wk0 + l32;
  constexpr bool LIFT = std::is_same_v<T, f16>;
  KeysLift kl(p, slice, nlo, LIFT && role_b ? nhi : -1, lane);
  int lift = 0;  // dS is scaled by 2^lift

  // The wave's operand: K rows (A) or V rows (B).
  const bool seen = key_seen(p, off, key);
  V8 kv[NSD];
  {
    const T* src = role_b ? (const T*)p.v + z * p.sv[0] + hk * p.sv[1] + (int64_t)(key < p.S ? key : 0) * p.sv[2]
                          : (const T*)p.k + z * p.sk[0] + hk * p.sk[1] + (int64_t)(key < p.S ? key : 0) * p.sk[2];
#pragma unroll
    for (int s = 0; s < NSD; ++s) {
      const V8 a = *reinterpret_cast<const V8*>(src + 16 * s + 8 * h2);
      kv[s] = seen ? a : V8{};
    }
  }

  // Fetching: pieces wu * PW .. of the step's Q tile (waves 0-3) and dO tile (4-7), and by wave 0 M and -delta.
  const int64_t head = (role_b ? p.sd[1] : p.sq[1]) * 2, rowst = role_b ? p.sd[2] : p.sq[2];
  const char* base = role_b ? (const char*)((const T*)p.dout + z * p.sd[0] + (int64_t)hk * p.G * p.sd[1])
                            : (const char*)((const T*)p.q + z * p.sq[0] + (int64_t)hk * p.G * p.sq[1]);
  const uint32_t bytes = (uint32_t)slice_bytes(p.N, rowst, D), tile_bytes = uniform32((uint32_t)(rowst * 64));
  const float* md = (h2 ? p.delta : p.m) + ((int64_t)z * p.H + hk * p.G) * p.N;
  uint32_t go[PW];
#pragma unroll
  for (int i = 0; i < PW; ++i) {
    constexpr int CPR = RB / 16;
    const int j = 64 * (pr * PW + i) + lane, row = j / CPR;
    go[i] = (uint32_t)(perm32(row) * rowst * 2 + (((j % CPR) ^ Swz<D>::f(row)) & (D / 8 - 1)) * 16);
  }
  // Next tile to fetch. Past the last one its rows come again, into a stage that nobody reads: every step has as many
  // loads in flight.
  const int fg0 = nq > 0 ? i0 / nq : 0, fq0 = qt0 + (nq > 0 ? i0 % nq : 0), q_end = qt0 + nq;
  const char* fbase = base + fg0 * head;  // of the head being fetched
  const float* fmd = md + (int64_t)fg0 * p.N;
  int fq = fq0, fi = 1;
  auto fetch = [&](char* st) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t rs = slice_rsrc(fbase, bytes);  // rows past the last query read as zero
    const uint32_t o = (uint32_t)fq * tile_bytes;
#pragma unroll
    for (int i = 0; i < PW; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (TATTN_LDS void*)(st + (wu * PW + i) * 1024), 16, (int)(go[i] + o), 0, 0, 0);
    if (wu == 0)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(fmd + min(32 * fq + l32, p.N - 1)),
                                       (TATTN_LDS void*)(st + 2 * TILE), 4, 0, 0);
    if (fi < n) {
      ++fi;
      if (++fq == q_end) fq = qt0, fbase += head, fmd += p.N;
    }
  };
  // End of a step: with four stages the loads of the step before have landed and this step's may stay in flight, with
  // three all have landed; LDS accesses are done.
  auto step_end = [&]() __attribute__((always_inline)) {
    if (NST == 3) __builtin_amdgcn_s_waitcnt(0x0070);
    else if (wu == 0) __builtin_amdgcn_s_waitcnt(0x0070 | (PW + 1));
    else __builtin_amdgcn_s_waitcnt(0x0070 | PW);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
  };

  int nat[NSD], lo[DT], hi[DT];
#pragma unroll
  for (int s = 0; s < NSD; ++s) nat[s] = Swz<D>::addr(l32, (16 * s + 8 * h2) * 2);
#pragma unroll
  for (int u = 0; u < DT; ++u) tr_addrs<D>(0, u, lane, lo[u], hi[u]);
  const float hidden = hidden_score(c);
  f32x16 acc[DT];  // dV (A) or dK (B)
#pragma unroll
  for (int u = 0; u < DT; ++u) acc[u] = f32x16{};

  // Query tiles of which the pair's keys see something, and those that see all of them (or are seen by all).
  const int far = 0x3fffffff;
  const int live_lo = wk0 < p.S ? (wk0 - off) >> 5 : far, live_hi = wk0 < p.sinks ? far : (p.window + wk1 - off - 1) >> 5;
  const int full_lo = (wk1 - off + 31) >> 5;
  const int full_hi = min((p.N >> 5) - 1, wk1 < p.sinks ? far : (p.window + wk0 - off - 32) >> 5);

  auto run = [&](auto role_tag) __attribute__((always_inline)) {
    constexpr int ROLE = decltype(role_tag)::value;  // 0: A, 1: B, 2: B with dS scaled up
    constexpr bool RB_ = ROLE > 0;
    // S (A) of a stage's tile, or dP - delta (B).
    auto first = [&](f32x16& s, const char* st) __attribute__((always_inline)) {
      if constexpr (RB_) {
        const TATTN_LDS char* nd = (const TATTN_LDS char*)st + 2 * TILE + 128 + 32 * h2;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const f32x4 v = *reinterpret_cast<const TATTN_LDS f32x4*>(nd + 64 * (a >> 1) + 16 * (a & 1));
#pragma unroll
          for (int e = 0; e < 4; ++e) s[4 * a + e] = v[e];
        }
      } else {
        s = f32x16{};
      }
#pragma unroll
      for (int sd = 0; sd < NSD; ++sd) s = Elt<T>::mfma(lds8<T>(st + (RB_ ? TILE : 0) + nat[sd]), kv[sd], s);
    };
    // dV += P^T dO (A), dK += dS^T Q (B).
    auto grad = [&](const V8 (&op)[2], const char* st) __attribute__((always_inline)) {
#pragma unroll
      for (int sl = 0; sl < 2; ++sl)
#pragma unroll
        for (int u = 0; u < DT; ++u)
          acc[u] = Elt<T>::mfma(op[sl], tr_pair<T>(st + (RB_ ? 0 : TILE) + 16 * sl * RB, lo[u], hi[u]), acc[u]);
    };
    auto probs = [&](const f32x16& s, V8 (&pp)[2], const char* st, char* x) __attribute__((always_inline)) {
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const f32x4 m = *reinterpret_cast<const TATTN_LDS f32x4*>((const TATTN_LDS char*)st + 2 * TILE + 32 * h2 + 64 * (a >> 1) + 16 * (a & 1));
        f32x4 pv;
#pragma unroll
        for (int e = 0; e < 4; ++e) pv[e] = fast_exp2(__builtin_fmaf(s[4 * a + e], c, -m[e]));
        *reinterpret_cast<TATTN_LDS f32x4*>((TATTN_LDS char*)x + pr * XB + 1024 * a + 16 * lane) = pv;
        const V2 a0 = H::pack(pv[0], pv[1]), a1 = H::pack(pv[2], pv[3]);
        V8& o8 = pp[a >> 1];
        o8[4 * (a & 1)] = a0[0], o8[4 * (a & 1) + 1] = a0[1], o8[4 * (a & 1) + 2] = a1[0], o8[4 * (a & 1) + 3] = a1[1];
      }
    };
    auto dsv = [&](const f32x16& dp, V8 (&ds)[2], const char* x) __attribute__((always_inline)) {
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const f32x4 pv = *reinterpret_cast<const TATTN_LDS f32x4*>((const TATTN_LDS char*)x + pr * XB + 1024 * a + 16 * lane);
        float d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = pv[e] * dp[4 * a + e];
        const V2 a0 = H::pack(d[0], d[1]), a1 = H::pack(d[2], d[3]);
        V8& o8 = ds[a >> 1];
        o8[4 * (a & 1)] = a0[0], o8[4 * (a & 1) + 1] = a0[1], o8[4 * (a & 1) + 2] = a1[0], o8[4 * (a & 1) + 3] = a1[1];
      }
    };
    int q = fq0;
    bool prev = false;
    auto step = [&](int i, auto tag) __attribute__((always_inline)) {
      constexpr int I = decltype(tag)::value;
      if (i > n) return;
      fetch(stage(IC<I + NST - 2>{}));
      const int odd = (NST == 4 ? I : i) & 1;
      char* xc = xbuf + odd * (RW * XB);
      const char* xp = xbuf + (odd ^ 1) * (RW * XB);
      const bool live = i < n && q >= live_lo && q <= live_hi;
      if constexpr (!RB_) {
        if (live) {
          f32x16 s;
          V8 pp[2];
          first(s, stage(IC<I>{}));
          if (q < full_lo || q > full_hi) ColMask(off + 32 * q - key, key, p.N - 32 * q, h2, p.window, p.sinks).hide(s, hidden);
          probs(s, pp, stage(IC<I>{}), xc);
          grad(pp, stage(IC<I>{}));
        }
      } else if (prev) {
        f32x16 dp;
        V8 ds[2];
        first(dp, stage(IC<I + NST - 1>{}));
        if constexpr (ROLE == 2) {
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[r] *= unlift_of(-lift);
        }
        dsv(dp, ds, xp);
        grad(ds, stage(IC<I + NST - 1>{}));
      }
      prev = live;
      if (++q == q_end) q = qt0;
      step_end();
    };
    for (int i = 0; i <= n; i += NST) {  // in step n B finishes the last tile; none follows
      step(i, IC<0>{});
      step(i + 1, IC<1>{});
      step(i + 2, IC<2>{});
      if constexpr (NST == 4) step(i + 3, IC<3>{});
    }
  };
  if (n > 0) {
    fetch(st0);
    if (NST == 4) fetch(st1);
    if (LIFT && role_b) lift = kl.lift(kv);
    all_landed_barrier();
    if (!role_b) run(IC<0>{});
    else if (!LIFT || lift == 0) run(IC<1>{});
    else run(IC<2>{});
    all_landed_barrier();
  }

  // Every wave has passed the last barrier and nothing is in flight. C register r of a lane: key 8 (r / 4) + 4 h2 + r % 4 of
  // the tile, column 32 u + l32. A part's sums go out in float32; otherwise the tile is turned into rows through LDS.
  const float unlift = role_b ? unlift_of(lift) : 1.0f, mul = role_b ? p.scale * unlift : 1.0f;
  if (parted) {
    float* dst = p.part + ((int64_t)slice * kbs.first(kbs.parted()) + item) * (2 * 32 * RW * D) +
                 (role_b ? 0 : 32 * RW * D) + (int64_t)32 * pr * D;
#pragma unroll
    for (int u = 0; u < DT; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) dst[(8 * (r >> 2) + 4 * h2 + (r & 3)) * D + 32 * u + l32] = acc[u][r] * unlift;
    return;
  }
  T* dst = role_b ? (T*)p.dk + z * p.sdk[0] + hk * p.sdk[1] : (T*)p.dv + z * p.sdv[0] + hk * p.sdv[1];
  const int64_t dst_row = role_b ? p.sdk[2] : p.sdv[2];
  static_assert(2 * NST >= NW, "a block of rows per wave, two in a stage");
  char* mine = (wu >> 1) == 0 ? st0 : (wu >> 1) == 1 ? st1 : (wu >> 1) == 2 ? st2 : st3;
  mine += (wu & 1) * TILE;
#pragma unroll
  for (int u = 0; u < DT; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = 8 * (r >> 2) + 4 * h2 + (r & 3);
      *reinterpret_cast<TATTN_LDS T*>((TATTN_LDS char*)mine + Swz<D>::addr(row, (32 * u + l32) * 2)) = (T)(acc[u][r] * mul);
    }
  constexpr int CPR = D / 8;
#pragma unroll
  for (int i = 0; i < 32 * CPR / 64; ++i) {
    const int j = 64 * i + lane, row = j / CPR, cc = j % CPR;
    const u32x4 v = *reinterpret_cast<const TATTN_LDS u32x4*>((const TATTN_LDS char*)mine + Swz<D>::addr(row, 16 * cc));
    if (wk0 + row < p.S) st16(dst + (int64_t)(wk0 + row) * dst_row + 8 * cc, v);
  }
}

// dK and dV of the key blocks whose queries were cut into parts: four consecutive columns a thread.
template <typename T, int D, int RW>
__global__ __launch_bounds__(256) void window_parts_kernel(const WindowParams p) {
  typedef T V4 __attribute__((ext_vector_type(4)));
  const KeyBlocks kbs(RW, p);
  const int blocks = kbs.parted();
  constexpr int BLOCK = 32 * RW * D;
  const int64_t per = 2ll * BLOCK, i = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
  if (i >= (int64_t)p.Z * p.Hk * blocks * per) return;
  const int64_t block = i / per;
  const int e = (int)(i % per), which = e / BLOCK, in = e % BLOCK / D, d = e % D;
  const int slice = (int)(block / blocks), kb = (int)(block % blocks);
  const int key = 32 * RW * kb + in;
  if (key >= p.S) return;
  const int first = kbs.first(kb), n = kbs.first(kb + 1) - first;
  const float* src = p.part + ((int64_t)slice * kbs.first(blocks) + first) * per + e;
  f32x4 x = f32x4{};
#pragma unroll 4
  for (int s = 0; s < n; ++s) x += *reinterpret_cast<const f32x4*>(src + s * per);
  const int z = slice / p.Hk, hk = slice % p.Hk;
  T* dst = which ? (T*)p.dv + z * p.sdv[0] + hk * p.sdv[1] + (int64_t)key * p.sdv[2] + d
                 : (T*)p.dk + z * p.sdk[0] + hk * p.sdk[1] + (int64_t)key * p.sdk[2] + d;
  V4 y;
#pragma unroll
  for (int k = 0; k < 4; ++k) y[k] = (T)(x[k] * (which ? 1.0f : p.scale));
  *reinterpret_cast<V4*>(dst) = y;
}

// ---- launch ----------------------------------------------------------------------------------------
// Row tiles per workgroup, and waves per SIMD of the forward. One key tile per step: its 32 KB of stages at head dim 128 let three
// workgroups share a CU (two tiles and two workgroups: 1,129 us against 1,048 at 16,384 x 32/8 x 128, window 4,096).
template <int D> struct WinShape { static constexpr int RW = 4, OCC = D == 128 ? 3 : 4; };
// Key tiles per workgroup of dK / dV. At head dim 128 two pairs and three stages let two workgroups share a CU, whose barriers do
// not wait for each other, and a last round of few workgroups is shorter (four pairs, four stages, one workgroup: 149 us
// against 125 at 11 x 12/4 x 1,500, window 500); at 64 four pairs have the CU full (two pairs: 269 against 205 us at
// 4 x 16 x 4,096, window 1,024).
constexpr int key_tiles(int D) { return D == 64 ? 4 : 2; }

// Key tiles that a block of 32 rows walks at most.
int64_t most_tiles(const WindowParams& p) {
  const int64_t seen = std::min<int64_t>(p.S, (int64_t)p.window + 32 / p.G + std::min(p.sinks, p.S));
  return (seen + 31) / 32 + 1;
}

template <typename T, int D>
int fwd_d(WindowParams p, hipStream_t st) {
  const int64_t slices = (int64_t)p.Z * p.Hk, rows = (int64_t)p.N * p.G;
  unsigned blocks;
  int rc;
  if (p.splits > 0) {
    p.nblk = (int)((rows + 31) / 32);
    p.tail = 0;
    if ((rc = window_grid(slices, (int64_t)p.nblk * p.splits, 0, &blocks))) return rc;
    if (p.splits == 1) {
      window_fwd_kernel<T, D, 1, 4, D == 128 ? 1 : 2, false><<<dim3(blocks), dim3(256), 0, st>>>(p);
      return check_launch("tattn_window_fwd");
    }
    window_fwd_kernel<T, D, 1, 4, D == 128 ? 1 : 2, true><<<dim3(blocks), dim3(256), 0, st>>>(p);
    if ((rc = check_launch("tattn_window_fwd"))) return rc;
    return launch_combine(p.part, p.out, p.m, p.sout, slices, p.Hk, p.G, p.N, p.splits, D, std::is_same_v<T, bf16> ? 2 : 0, st);
  }
  using S = WinShape<D>;
  p.nblk = (int)((rows + 32 * S::RW - 1) / (32 * S::RW));
  p.tail = window_row_tail(p, 32 * S::RW, p.nblk);
  if ((rc = window_grid(slices, p.nblk, p.tail, &blocks))) return rc;
  window_fwd_kernel<T, D, S::RW, 1, S::OCC, false><<<dim3(blocks), dim3(S::RW * 64), 0, st>>>(p);
  return check_launch("tattn_window_fwd");
}

template <typename T, int D>
int bwd_d(WindowParams p, hipStream_t st) {
  using S = WinShape<D>;
  constexpr int RW = key_tiles(D);
  const int64_t slices = (int64_t)p.Z * p.Hk, rows = (int64_t)p.N * p.G;
  unsigned blocks;
  int rc;
  p.nblk = (int)((rows + 32 * S::RW - 1) / (32 * S::RW));
  p.tail = window_row_tail(p, 32 * S::RW, p.nblk);
  if ((rc = window_grid(slices, p.nblk, p.tail, &blocks))) return rc;
  window_dq_kernel<T, D, S::RW, D >= 64 ? 2 : 4><<<dim3(blocks), dim3(S::RW * 64), 0, st>>>(p);
  if ((rc = check_launch("tattn_window_bwd"))) return rc;
  const KeyBlocks kbs(RW, p);
  p.head = kbs.sink_blocks * p.splits;  // the longest: 84 -> 73 us for the whole backward at 4/4 x 16,384 x 64, window 512
  p.tail = window_key_tail(p, 32 * RW, kbs.blocks - kbs.sink_blocks) * p.parts;
  if ((rc = window_grid(slices, kbs.items, p.head + p.tail, &blocks))) return rc;
  if constexpr (D >= 64)
    window_dkdv_pair_kernel<T, D, RW, D == 128 ? 3 : 4, D == 128 ? 2 : 4><<<dim3(blocks), dim3(RW * 128), 0, st>>>(p);
  else
    window_dkdv_kernel<T, D, RW, 4, D == 32 ? 3 : 4><<<dim3(blocks), dim3(RW * 256), 0, st>>>(p);
  if ((rc = check_launch("tattn_window_bwd")) || !kbs.parted()) return rc;
  const int64_t n = slices * kbs.parted() * 2 * 32 * RW * D / 4;
  window_parts_kernel<T, D, RW><<<dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st>>>(p);
  return check_launch("tattn_window_bwd");
}

#define TATTN_WIN_SWITCH(FN)                                                     \
  switch (D) {                                                                   \
    case 16: return dtype == 0 ? FN<f16, 16>(p, st) : FN<bf16, 16>(p, st);       \
    case 32: return dtype == 0 ? FN<f16, 32>(p, st) : FN<bf16, 32>(p, st);       \
    case 64: return dtype == 0 ? FN<f16, 64>(p, st) : FN<bf16, 64>(p, st);       \
    case 128: return dtype == 0 ? FN<f16, 128>(p, st) : FN<bf16, 128>(p, st);    \
  }                                                                              \
  return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %d", D);

template <typename T, int D>
int combine_d(const float* part, void* out, float* m, const int64_t so[3], int64_t slices, int Hk, int G, int N, int splits,
              hipStream_t st) {
  const int64_t rows = slices * N * G;
  if (rows > 0x7fffffff) return set_error(TATTN_E_ARG, "grid too large: %lld rows", (long long)rows);
  combine_kernel<T, D><<<dim3((unsigned)rows), dim3(256), 0, st>>>(part, (T*)out, m, so[0], so[1], so[2], Hk, G, N, splits);
  return check_launch("combine");
}

}  // namespace

// Few rows (a single row tile per slice, or few blocks of four tiles): one row tile per workgroup, whose waves share its keys.
// Against blocks of four, us by head dim and number of such blocks, at windows of 300, 1,000 and 4,000 keys:
//   128: 64 blocks 11, 18, 25 (19, 33, 50); 128: 20, 33, 67 (19, 34, 94); 250: 37, 64, 166 (21, 37, 102)
//    64: 128 blocks 11, 15, 28 (14, 25, 65); 250: 17, 27, 64 (15, 26, 70); 300: 21, 33, 80 (19, 33, 71)
//    32: 250 blocks 11, 18, 41 (13, 21, 56); 384: 15, 24, 58 (16, 27, 70); 500: 19, 30, 72 (16, 28, 74)
// Its keys are cut into parts until the chip holds no more workgroups at once, one per CU at head dim 128 (128 KB of stages), two
// below (32 x 32/8 heads x 8,192 keys x 128, window 2,048: 51.5 us at one per CU, 59 at two, 68 at four); of at least eight
// tiles, and of more where many rows have to be joined (a workgroup each: 4 x 1,024 rows x 64 over 1,000
// keys take 17 us in parts of eight tiles and 12 whole). 0: blocks of four row tiles.
int window_fwd_splits(const WindowParams& p, int D) {
  const int64_t slices = (int64_t)p.Z * p.Hk, rows = (int64_t)p.N * p.G;
  if (rows > 32 && slices * ((rows + 127) / 128) > (D == 128 ? 128 : D == 64 ? 256 : 400)) return 0;
  const int64_t blocks = slices * ((rows + 31) / 32), want = D == 128 ? 256 : 512;
  return (int)std::max<int64_t>(1, std::min<int64_t>(want / blocks, most_tiles(p) / std::max<int64_t>(8, slices * rows / 128)));
}

// Parts that the queries of dK / dV are cut into. `parts`, of every key block's: where all blocks together are at most half of
// what the chip holds at once (two workgroups a CU), as many as fill it, of at least 16 steps each (whole backward of 1 x 32/2
// x 4,096 x 64, causal, 1,364 -> 309 us; 1 x 8/1 x 8,192 x 128, window 1,024, 283 -> 184). `splits`, of those that hold first
// keys: each about as long as another block's part, or as an even share of all work over four workgroups per CU where that is
// more, so that all parts together stay near a thousand.
void window_bwd_parts(WindowParams& p, int D) {
  const int64_t rw = key_tiles(D), keys = 32 * rw, slices = (int64_t)p.Z * p.Hk;
  const int64_t all = (int64_t)p.G * ((p.N + 31) / 32);
  const int64_t list = std::min<int64_t>(all, (int64_t)p.G * (std::min<int64_t>(p.window, p.S) / 32 + rw + 1));
  const int64_t blocks = (p.S + keys - 1) / keys, first = std::min<int64_t>(blocks, (p.sinks + keys - 1) / keys);
  p.parts = (int32_t)std::max<int64_t>(1, std::min<int64_t>(512 / (slices * blocks), list / 16));
  p.splits = p.parts;
  if (p.sinks == 0) return;
  const int64_t share = slices * (first * all + (blocks - first) * list) / 1024;
  const int64_t part = std::max<int64_t>(std::max<int64_t>(list / p.parts, share), 32);
  p.splits = (int32_t)std::max<int64_t>(p.parts, std::min<int64_t>((all + part - 1) / part, 256));
}

int64_t window_bwd_part_floats(const WindowParams& p, int D) {
  const KeyBlocks kbs(key_tiles(D), p);
  return (int64_t)p.Z * p.Hk * kbs.first(kbs.parted()) * 2 * 32 * key_tiles(D) * D;
}

int launch_window_fwd(WindowParams p, int D, int dtype, hipStream_t st) { TATTN_WIN_SWITCH(fwd_d) }
int launch_window_bwd(WindowParams p, int D, int dtype, hipStream_t st) { TATTN_WIN_SWITCH(bwd_d) }

int launch_combine(const float* part, void* out, float* m, const int64_t so[3], int64_t slices, int Hk, int G, int N,
                   int splits, int D, int dtype, hipStream_t st) {
  switch (D) {
#define TATTN_COMBINE(D_)                                                                               \
  case D_:                                                                                              \
    return dtype == 0 ? combine_d<f16, D_>(part, out, m, so, slices, Hk, G, N, splits, st)              \
                      : combine_d<bf16, D_>(part, out, m, so, slices, Hk, G, N, splits, st);
    TATTN_COMBINE(16) TATTN_COMBINE(32) TATTN_COMBINE(64) TATTN_COMBINE(128)
#undef TATTN_COMBINE
  }
  return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %d", D);
}

}  // namespace tattn
