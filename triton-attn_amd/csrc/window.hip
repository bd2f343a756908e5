// Attention over a sliding window and the first keys, 16-bit, forward and backward, on gfx950.
//
// The waves of a workgroup share row tiles and key tiles as in the kernels for few rows: NW = RW * CS waves own RW
// 32-row tiles; a step stages CS tiles of the other dimension by LDS DMA (buffer_load ... lds, swizzled rows) into one of
// two stages while the other is worked on; wave (rw, cs) works on tile cs of the step for row tile rw, and the CS partial
// results of a row tile are added through LDS at the end. What differs is the list of tiles: only those that some
// row of the workgroup sees are walked (TileList), only those at the ends of a row's window pay for masks, and a wave
// passes over tiles that none of its own rows sees.
//
// Rows that nobody in the workgroup sees (before the window, behind the last key) are fetched from beyond the end of
// the buffer, which reads as zero: whatever a cache holds there cannot reach a sum.
#include <algorithm>
#include <type_traits>

#include "window.h"

namespace tattn {
namespace {

template <int D, int NW, int CS>
struct WinRing {
  static constexpr int RB = Swz<D>::RB, TILE = 32 * RB, PIECES = TILE / 1024;
  static constexpr int HALF = CS * TILE;        // bytes of one tensor's tiles
  static constexpr int STAGE = 2 * HALF;
  static constexpr int PW = STAGE / 1024 / NW;  // 1 KB DMA pieces per wave and step
  static_assert(PW >= 1 && PW * NW * 1024 == STAGE && NW % 2 == 0, "whole pieces, one tensor per wave");
};

constexpr uint32_t kBeyond = 0x7fffffffu;  // byte offset past every slice: reads as zero

// DMA of tile pairs: the first half of the waves loads the first tensor, the other half the second.
template <int D, int NW, int CS>
struct WinLoader {
  using R = WinRing<D, NW, CS>;
  uint32_t go[R::PW];
  uint32_t tile_bytes;
  int base, g0, lane;
  bool second;
  __device__ __forceinline__ void init(int64_t sa, int64_t sb, int wu, int lane_) {
    lane = lane_;
    second = wu >= NW / 2;
    const int64_t st = second ? sb : sa;
    tile_bytes = uniform32((uint32_t)(st * 64));
    base = wu * R::PW * 1024;
    g0 = (wu * R::PW) % (CS * R::PIECES);
    constexpr int CPR = R::RB / 16;
#pragma unroll
    for (int i = 0; i < R::PW; ++i) {
      const int j = 64 * ((g0 + i) % R::PIECES) + lane;
      const int row = j / CPR, cc = ((j % CPR) ^ Swz<D>::f(row)) & (D / 8 - 1);
      go[i] = (uint32_t)(perm32(row) * st * 2 + cc * 16);
    }
  }
  // Which of the step's CS tiles piece i belongs to, and the row of that tile the lane fetches.
  __device__ __forceinline__ int slot(int i) const { return (g0 + i) / R::PIECES; }
  __device__ __forceinline__ int row(int i) const {
    return perm32((64 * ((g0 + i) % R::PIECES) + lane) / (R::RB / 16));
  }
  __device__ __forceinline__ void fetch(__amdgpu_buffer_rsrc_t rs, char* stage, int i, uint32_t off) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (TATTN_LDS void*)(stage + base + 1024 * i), 16, (int)off, 0, 0, 0);
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
  int p0, p1;    // positions of the workgroup's rows
  int top;       // last key any of them sees
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
    top = p1;
  }
};

template <typename T, int D>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t win_rsrc(const void* base, int64_t off, int64_t rows, int64_t stride) {
  return slice_rsrc((const T*)base + off, rows > 0 ? slice_bytes(rows, stride, D) : 0);
}

// K and V tiles of list entries [i0, i0 + CS) into `stage`; entries from i1 on are not fetched.
template <int D, int NW, int CS>
__device__ __forceinline__ void fetch_keys(const WinLoader<D, NW, CS>& ld, __amdgpu_buffer_rsrc_t rs, char* stage,
                                           const TileList& list, int i0, int i1, int top, int sinks) {
#pragma unroll
  for (int i = 0; i < WinRing<D, NW, CS>::PW; ++i) {
    const int at = i0 + ld.slot(i);
    if (at >= i1) continue;
    const int t = list.at(at);
    uint32_t o = ld.go[i] + (uint32_t)t * ld.tile_bytes;
    if (32 * t + 31 > top || (32 * t < list.lo && 32 * t + 31 >= sinks)) {
      const int key = 32 * t + ld.row(i);
      if (key > top || (key < list.lo && key >= sinks)) o = kBeyond;
    }
    ld.fetch(rs, stage, i, o);
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
  __shared__ float red[2][NW][32];

  const int tid = threadIdx.x;
  const int lane = tid & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(tid >> 6));
  const int rw = wu / CS, cs = wu % CS;
  const float c = p.c;
  int slice, blk, split = 0;
  if (!window_coord(p.Z * p.Hk, p.nblk * (SPLIT ? p.splits : 1), p.runs, slice, blk)) return;
  if (SPLIT) split = blk % p.splits, blk /= p.splits;
  WinRows b;
  b.init(p, slice, p.nblk - 1 - blk, RW);  // longest rows first
  TileList list;
  list.init(b.p0, b.p1, p.window, p.sinks);
  const int i0 = SPLIT ? (int)((int64_t)list.n * split / p.splits) : 0;
  const int i1 = SPLIT ? (int)((int64_t)list.n * (split + 1) / p.splits) : list.n;
  const int nsteps = (i1 - i0 + CS - 1) / CS;

  WinLoader<D, NW, CS> ld;
  ld.init(p.sk[2], p.sv[2], wu, lane);
  const __amdgpu_buffer_rsrc_t rs =
      ld.second ? win_rsrc<T, D>(p.v, b.z * p.sv[0] + b.hk * p.sv[1], b.len, p.sv[2])
                : win_rsrc<T, D>(p.k, b.z * p.sk[0] + b.hk * p.sk[1], b.len, p.sk[2]);
  auto issue = [&](char* stage, int step) __attribute__((always_inline)) {
    fetch_keys<D, NW, CS>(ld, rs, stage, list, i0 + step * CS, i1, b.top, p.sinks);
  };
  if (nsteps > 0) issue(s0, 0);

  const int tile0 = 32 * (b.tile0 + rw);
  const int row = tile0 + l32;
  const bool live = row < b.rows;
  const int n = (live ? row : 0) / p.G, g = (live ? row : 0) % p.G;
  const int pos = b.off + n;
  // The wave's positions; a wave without rows sees no tile.
  const int wp0 = b.off + tile0 / p.G, wp1 = tile0 < b.rows ? b.off + min(tile0 + 31, b.rows - 1) / p.G : -1;
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

  float mrow = kNoMax, lrow = 0.0f;
  f32x16 acc[DT];
#pragma unroll
  for (int u = 0; u < DT; ++u) acc[u] = f32x16{};

  // Tile t, staged in `st`. Probabilities against the running max as it stands; a lane whose 16 probabilities sum above
  // 2^12 (its first visible tile among them) sends the wave through the row max and a rescale. The branch is
  // one-sided (state updated first, undone inside): a two-sided one makes the allocator hold two copies of it.
  auto tile = [&](const char* st, int t, auto mask_tag) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
    const RowMask hide(pos, t, h2, p.window, p.sinks);
    f32x16 s = f32x16{};
#pragma unroll
    for (int sd = 0; sd < NSD; ++sd) s = Elt<T>::mfma(lds8<T>(st + at.nat[sd]), qop[sd], s);
    V8 x[2];
    auto probs = [&]() __attribute__((always_inline)) {
      float ps = 0.0f;
#pragma unroll
      for (int sg = 0; sg < 2; ++sg)
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const int r = 8 * sg + i;
          float e0 = fast_exp2(__builtin_fmaf(s[r], c, -mrow)), e1 = fast_exp2(__builtin_fmaf(s[r + 1], c, -mrow));
          if (MASK) {
            e0 = hide.hides(r) ? 0.0f : e0;
            e1 = hide.hides(r + 1) ? 0.0f : e1;
          }
          const V2 pr = H::pack(e0, e1);
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
      for (int r = 0; r < 16; ++r) mx = MASK && hide.hides(r) ? mx : __builtin_fmaxf(mx, s[r] * c);
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
      if (!tile_hidden(wp0, wp1, t, p.window, p.sinks)) {
        if (tile_masked(wp0, wp1, t, p.window, p.sinks)) tile(cur, t, std::true_type{});
        else tile(cur, t, std::false_type{});
      }
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
  static_assert(2 * PER >= NW, "partials fit the stages");
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
// O = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s, D / 4 lanes per row.
template <typename T, int D>
__global__ __launch_bounds__(256) void combine_kernel(const float* part, T* out, float* m, int64_t sz, int64_t sh, int64_t sn,
                                                      int64_t slices, int Hk, int G, int N, int splits) {
  typedef T V4 __attribute__((ext_vector_type(4)));
  constexpr int LPR = D / 4;
  const int rows = N * G;
  const int64_t r = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (r >= slices * rows) return;
  const int64_t slice = r / rows;
  const int row = (int)(r % rows), d0 = threadIdx.x % LPR * 4;
  const float* ml = part + slices * splits * rows * D;
  const int64_t first = slice * splits * rows + row;
  float mall = kNoMax;
  for (int s = 0; s < splits; ++s) mall = __builtin_fmaxf(mall, ml[(first + (int64_t)s * rows) * 2]);
  f32x4 x = f32x4{};
  float l = 0.0f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const int64_t at = first + (int64_t)s * rows;
    const float w = fast_exp2(ml[at * 2] - mall), ls = ml[at * 2 + 1];
    if (ls == 0.0f) continue;  // no visible key: the sums of such a part may not be there
    l = __builtin_fmaf(w, ls, l);
    const f32x4 y = *reinterpret_cast<const f32x4*>(part + at * D + d0);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(w, y[e], x[e]);
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
// Rows and key tiles as in the forward; computes delta = rowsum(dO * O) on the way and stores it for dK / dV.
template <typename T, int D, int RW, int CS, int OCC>
__global__ __launch_bounds__(RW * CS * 64, OCC) void window_dq_kernel(const WindowParams p) {
  using H = H16<T>;
  using V8 = typename H::V8;
  using V4 = typename H::V4;
  using V2 = typename H::V2;
  constexpr int NW = RW * CS, NSD = D / 16, DT = (D + 31) / 32;
  using R = WinRing<D, NW, CS>;
  __shared__ __attribute__((aligned(1024))) char s0[R::STAGE];
  __shared__ __attribute__((aligned(1024))) char s1[R::STAGE];

  const int tid = threadIdx.x;
  const int lane = tid & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(tid >> 6));
  const int rw = wu / CS, cs = wu % CS;
  const float c = p.c;
  int slice, blk;
  if (!window_coord(p.Z * p.Hk, p.nblk, p.runs, slice, blk)) return;
  WinRows b;
  b.init(p, slice, p.nblk - 1 - blk, RW);
  TileList list;
  list.init(b.p0, b.p1, p.window, p.sinks);
  const int nsteps = (list.n + CS - 1) / CS;

  WinLoader<D, NW, CS> ld;
  ld.init(p.sk[2], p.sv[2], wu, lane);
  const __amdgpu_buffer_rsrc_t rs =
      ld.second ? win_rsrc<T, D>(p.v, b.z * p.sv[0] + b.hk * p.sv[1], b.len, p.sv[2])
                : win_rsrc<T, D>(p.k, b.z * p.sk[0] + b.hk * p.sk[1], b.len, p.sk[2]);
  auto issue = [&](char* stage, int step) __attribute__((always_inline)) {
    fetch_keys<D, NW, CS>(ld, rs, stage, list, step * CS, list.n, b.top, p.sinks);
  };
  if (nsteps > 0) issue(s0, 0);

  const int tile0 = 32 * (b.tile0 + rw);
  const int row = tile0 + l32;
  const bool live = row < b.rows;
  const int n = (live ? row : 0) / p.G, g = (live ? row : 0) % p.G, h = b.hk * p.G + g;
  const int pos = b.off + n;
  const int wp0 = b.off + tile0 / p.G, wp1 = tile0 < b.rows ? b.off + min(tile0 + 31, b.rows - 1) / p.G : -1;
  const int64_t mrow = ((int64_t)b.z * p.H + h) * p.N + n;
  V8 qop[NSD], dop[NSD];
  float dl;
  {
    const T* qs = (const T*)p.q + b.z * p.sq[0] + h * p.sq[1] + n * p.sq[2] + 8 * h2;
    const T* ds = (const T*)p.dout + b.z * p.sd[0] + h * p.sd[1] + n * p.sd[2] + 8 * h2;
    const T* os = (const T*)p.o + b.z * p.so[0] + h * p.so[1] + n * p.so[2] + 8 * h2;
    float sd[NSD];
#pragma unroll
    for (int s = 0; s < NSD; ++s) {
      const V8 x = *reinterpret_cast<const V8*>(qs + 16 * s), y = *reinterpret_cast<const V8*>(ds + 16 * s);
      qop[s] = live ? x : V8{};
      dop[s] = live ? y : V8{};
      sd[s] = chunk_dot(*reinterpret_cast<const V8*>(os + 16 * s), y);
    }
    dl = row_delta(sd);
    if (live && h2 == 0 && cs == 0) p.delta[mrow] = dl;
    if (!live) dl = 0.0f;
  }
  const float nm = live ? -p.m[mrow] : 0.0f;
  WinOp<D> at;
  at.init(cs * R::TILE, lane);
  f32x16 dq[DT];
#pragma unroll
  for (int u = 0; u < DT; ++u) dq[u] = f32x16{};

  auto tile = [&](const char* st, int t, auto mask_tag) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
    const RowMask hide(pos, t, h2, p.window, p.sinks);
    f32x16 s = f32x16{}, dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) dp[r] = -dl;  // seeds dP - delta
#pragma unroll
    for (int sd = 0; sd < NSD; ++sd) {
      s = Elt<T>::mfma(lds8<T>(st + at.nat[sd]), qop[sd], s);
      dp = Elt<T>::mfma(lds8<T>(st + R::HALF + at.nat[sd]), dop[sd], dp);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = fast_exp2(__builtin_fmaf(s[r], c, nm)) * dp[r];
      if (MASK) s[r] = hide.hides(r) ? 0.0f : s[r];
    }
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
    if (i + 1 < nsteps) issue(nxt, i + 1);
    const int k = i * CS + cs;
    if (k < list.n) {
      const int t = list.at(k);
      if (!tile_hidden(wp0, wp1, t, p.window, p.sinks)) {
        if (tile_masked(wp0, wp1, t, p.window, p.sinks)) tile(cur, t, std::true_type{});
        else tile(cur, t, std::false_type{});
      }
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

  constexpr int PART = DT * 16 * 64 * 4;
  constexpr int PER = R::STAGE / PART;
  static_assert(2 * PER >= NW, "partials fit the stages");
  auto part = [&](int k) { return (TATTN_LDS float*)(k < PER ? s0 + k * PART : s1 + (k - PER) * PART); };
  {
    TATTN_LDS float* dst = part(wu) + lane;
#pragma unroll
    for (int u = 0; u < DT; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) dst[(16 * u + r) * 64] = dq[u][r];
  }
  __syncthreads();
  if (!live) return;
  T* orow = (T*)p.out + b.z * p.sout[0] + h * p.sout[1] + n * p.sout[2];
  for (int gr = cs; gr < DT * 4; gr += CS) {
    const int d0 = 8 * gr + 4 * h2;
    if (d0 < D) {
      f32x4 x = f32x4{};
#pragma unroll
      for (int k = 0; k < CS; ++k) {
        const TATTN_LDS float* src = part(rw * CS + k) + lane + 4 * gr * 64;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += src[64 * e];
      }
      V4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (T)(x[e] * p.scale);
      *reinterpret_cast<V4*>(orow + d0) = y;
    }
  }
}

// ---- dK / dV -------------------------------------------------------------------------------------
// A workgroup owns RW tiles of 32 keys and walks the query tiles that see any of them, head after head of
// the group: the sum over shared heads stays in registers. Key blocks that hold first keys are seen by every later query, an
// N / window-fold of the others' work: their list is cut into `splits` parts (WindowParams), which write float32 sums that
// window_first_keys_kernel adds in order.
template <int RW>
struct KeyBlocks {
  int sink_blocks, items;  // per slice: sink_blocks * splits parts, then the other blocks
  __host__ __device__ KeyBlocks(int S, int sinks, int splits) {
    const int blocks = (S + 32 * RW - 1) / (32 * RW);
    sink_blocks = splits > 1 ? (sinks + 32 * RW - 1) / (32 * RW) : 0;
    if (sink_blocks > blocks) sink_blocks = blocks;
    items = sink_blocks * splits + blocks - sink_blocks;
  }
};

template <typename T, int D, int RW, int CS, int OCC>
__global__ __launch_bounds__(RW * CS * 64, OCC) void window_dkdv_kernel(const WindowParams p) {
  using H = H16<T>;
  using V8 = typename H::V8;
  using V2 = typename H::V2;
  constexpr int NW = RW * CS, NSD = D / 16, DT = (D + 31) / 32;
  // At head dim 128 the accumulators take 128 registers: V's operands then stay in LDS.
  constexpr bool VLDS = D == 128;
  using R = WinRing<D, NW, CS>;
  __shared__ __attribute__((aligned(1024))) char s0[R::STAGE];
  __shared__ __attribute__((aligned(1024))) char s1[R::STAGE];
  __shared__ __attribute__((aligned(1024))) char sv[VLDS ? RW * R::TILE : 16];
  __shared__ __attribute__((aligned(16))) float md[NW][2][64];  // per wave and parity: M[32], -delta[32]

  const int tid = threadIdx.x;
  const int lane = tid & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(tid >> 6));
  const int rw = wu / CS, cs = wu % CS;
  const float c = p.c;
  const KeyBlocks<RW> kbs(p.S, p.sinks, p.splits);
  int slice, kb, split = 0;
  if (!window_coord(p.Z * p.Hk, kbs.items, p.runs, slice, kb)) return;
  const bool parted = kb < kbs.sink_blocks * p.splits;
  if (parted) split = kb % p.splits, kb /= p.splits;
  else kb = kb - kbs.sink_blocks * p.splits + kbs.sink_blocks;
  const int z = slice / p.Hk, hk = slice % p.Hk, off = p.S - p.N;
  const int k0 = 32 * RW * kb, k1 = k0 + 32 * RW - 1;
  // Queries that see a key of the block, as tiles of 32 of each head in turn.
  const int nlo = max(0, k0 - off);
  const int nhi = k0 < p.sinks ? p.N - 1 : min(p.N - 1, k1 + p.window - 1 - off);
  const int qt0 = nlo >> 5, nq = nhi < nlo ? 0 : (nhi >> 5) - qt0 + 1;
  const int total = nq * p.G;
  const int i0 = parted ? (int)((int64_t)total * split / p.splits) : 0;
  const int i1 = parted ? (int)((int64_t)total * (split + 1) / p.splits) : total;
  const int nsteps = (i1 - i0 + CS - 1) / CS;

  WinLoader<D, NW, CS> ld;
  ld.init(p.sq[2], p.sd[2], wu, lane);
  const char* qbase = ld.second ? (const char*)((const T*)p.dout + z * p.sd[0] + (int64_t)hk * p.G * p.sd[1])
                                : (const char*)((const T*)p.q + z * p.sq[0] + (int64_t)hk * p.G * p.sq[1]);
  const int64_t head_bytes = (ld.second ? p.sd[1] : p.sq[1]) * 2;
  const uint32_t qbytes = (uint32_t)slice_bytes(p.N, ld.second ? p.sd[2] : p.sq[2], D);
  auto issue = [&](char* stage, int step) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < R::PW; ++i) {
      const int k = i0 + step * CS + ld.slot(i);
      if (k >= i1) continue;
      const int g = k / nq, qt = qt0 + k % nq;
      // Rows past the head's last query lie past the end of its slice and read as zero.
      ld.fetch(slice_rsrc(qbase + g * head_bytes, qbytes), stage, i, ld.go[i] + (uint32_t)qt * ld.tile_bytes);
    }
  };
  if (nsteps > 0) issue(s0, 0);
  // Lanes 0-31 fetch M and lanes 32-63 delta of the wave's tile; zero past the end.
  const float* mdsrc = (h2 ? p.delta : p.m) + ((int64_t)z * p.H + hk * p.G) * p.N;
  auto md_load = [&](int step) {
    const int k = i0 + step * CS + cs;
    const int q = k < i1 ? 32 * (qt0 + k % nq) + l32 : p.N;
    const float x = q < p.N ? mdsrc[(int64_t)(k / nq) * p.N + q] : 0.0f;
    return h2 ? -x : x;
  };
  md[wu][0][lane] = nsteps > 0 ? md_load(0) : 0.0f;
  const int kt = kb * RW + rw, key = 32 * kt + l32;
  V8 kop[NSD], vop[VLDS ? 1 : NSD];
  {
    const T* ks = (const T*)p.k + z * p.sk[0] + hk * p.sk[1] + (int64_t)(key < p.S ? key : 0) * p.sk[2] + 8 * h2;
    const T* vs = (const T*)p.v + z * p.sv[0] + hk * p.sv[1] + (int64_t)(key < p.S ? key : 0) * p.sv[2] + 8 * h2;
#pragma unroll
    for (int s = 0; s < NSD; ++s) {
      const V8 a = *reinterpret_cast<const V8*>(ks + 16 * s);
      const V8 b = *reinterpret_cast<const V8*>(vs + 16 * s);
      kop[s] = key < p.S ? a : V8{};
      const V8 x = key < p.S ? b : V8{};
      if constexpr (VLDS) {
        if (cs == 0) *reinterpret_cast<TATTN_LDS V8*>((TATTN_LDS char*)sv + rw * R::TILE + Swz<D>::addr(l32, (16 * s + 8 * h2) * 2)) = x;
      } else {
        vop[s] = x;
      }
    }
  }
  WinOp<D> at;
  at.init(cs * R::TILE, lane);
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int u = 0; u < DT; ++u) dk[u] = dv[u] = f32x16{};

  auto tile = [&](const char* st, const float* mdw, int qt, auto mask_tag) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
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
      V8 vo;
      if constexpr (VLDS) vo = lds8<T>(sv + rw * R::TILE + at.nat[sd] - cs * R::TILE);
      else vo = vop[sd];
      dp = Elt<T>::mfma(lds8<T>(st + R::HALF + at.nat[sd]), vo, dp);
    }
    // Register r is query 32 qt + 8 h2 + 16 (r / 8) + r % 8 at position `off` further, the lane's key is `key`.
    const int first = off + 32 * qt + 8 * h2 - key;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = fast_exp2(__builtin_fmaf(s[r], c, -mv[r]));
      if (MASK) {
        const int gap = first + 16 * (r >> 3) + (r & 7);
        const bool hide = gap < 0 || (gap >= p.window && key >= p.sinks) || 16 * (r >> 3) + (r & 7) >= p.N - 32 * qt - 8 * h2;
        s[r] = hide ? 0.0f : s[r];
        dp[r] = hide ? 0.0f : dp[r];
      }
    }
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
      if (q1 >= wk0 && (q0 - wk1 < p.window || wk0 < p.sinks)) {
        if (q0 < wk1 || (q1 - wk0 >= p.window && wk1 >= p.sinks) || 32 * qt + 32 > p.N) tile(cur, md[wu][par], qt, std::true_type{});
        else tile(cur, md[wu][par], qt, std::false_type{});
      }
    }
    md[wu][par ^ 1][lane] = mdn;  // the wave's own rows: no barrier needed
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
  // A part's sums: [slice][sink block][split][dK, dV][32 RW keys][D] float32.
  float* fdst = p.part + (((int64_t)slice * kbs.sink_blocks + kb) * p.splits + split) * (2 * 32 * RW * D);
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
          if (parted) fpart[(32 * rw + in) * D + d] = x;
          else if (wk0 + in < p.S) dst[(int64_t)(wk0 + in) * stride + d] = (T)(x * mul);
        }
    }
  };
  reduce(dk, p.scale, (T*)p.dk + z * p.sdk[0] + hk * p.sdk[1], p.sdk[2], fdst);
  __syncthreads();
  reduce(dv, 1.0f, (T*)p.dv + z * p.sdv[0] + hk * p.sdv[1], p.sdv[2], fdst + 32 * RW * D);
}

// dK and dV of the key blocks whose queries were cut into parts.
template <typename T, int D, int RW>
__global__ __launch_bounds__(256) void window_first_keys_kernel(const WindowParams p) {
  const KeyBlocks<RW> kbs(p.S, p.sinks, p.splits);
  constexpr int BLOCK = 32 * RW * D;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t per = 2ll * BLOCK;
  if (i >= (int64_t)p.Z * p.Hk * kbs.sink_blocks * per) return;
  const int64_t block = i / per;
  const int e = (int)(i % per), which = e / BLOCK, in = e % BLOCK / D, d = e % D;
  const int slice = (int)(block / kbs.sink_blocks), kb = (int)(block % kbs.sink_blocks);
  const int key = 32 * RW * kb + in;
  if (key >= p.S) return;
  float x = 0.0f;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) x += p.part[(block * p.splits + s) * per + e];
  const int z = slice / p.Hk, hk = slice % p.Hk;
  if (which) ((T*)p.dv)[z * p.sdv[0] + hk * p.sdv[1] + (int64_t)key * p.sdv[2] + d] = (T)x;
  else ((T*)p.dk)[z * p.sdk[0] + hk * p.sdk[1] + (int64_t)key * p.sdk[2] + d] = (T)(x * p.scale);
}

// ---- launch ----------------------------------------------------------------------------------------
// Row tiles per workgroup and tiles of the other dimension per step.
template <int D> struct WinShape { static constexpr int RW = 2, CS = D == 128 ? 2 : 4; };
template <int D> struct KeyShape { static constexpr int RW = D == 128 ? 4 : 2, CS = D == 128 ? 2 : 4; };

int grid_of(int64_t slices, int64_t per_slice, unsigned* out) {
  const int64_t blocks = slices * per_slice + 8;
  if (blocks > 0x7ffffff) return set_error(TATTN_E_ARG, "grid too large: %lld workgroups", (long long)blocks);
  *out = (unsigned)((slices * per_slice + 7) / 8 * 8);
  return TATTN_OK;
}

// Whether consecutive blocks of a slice share an XCD: windows much shorter than the rows make blocks equal; else the
// later ones are longer, and only whole slices per XCD keep the XCDs level.
int in_runs(const WindowParams& p) { return ((int64_t)p.Z * p.Hk) % 8 == 0 || (int64_t)p.window * 4 <= p.S; }

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
  p.runs = in_runs(p);
  if (p.splits > 0) {
    p.nblk = (int)((rows + 31) / 32);
    if ((rc = grid_of(slices, (int64_t)p.nblk * p.splits, &blocks))) return rc;
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
  if ((rc = grid_of(slices, p.nblk, &blocks))) return rc;
  constexpr int OCC = D == 128 ? 2 : 4;
  window_fwd_kernel<T, D, S::RW, S::CS, OCC, false><<<dim3(blocks), dim3(S::RW * S::CS * 64), 0, st>>>(p);
  return check_launch("tattn_window_fwd");
}

template <typename T, int D>
int bwd_d(WindowParams p, hipStream_t st) {
  using S = WinShape<D>;
  using K = KeyShape<D>;
  const int64_t slices = (int64_t)p.Z * p.Hk, rows = (int64_t)p.N * p.G;
  const int splits = p.splits;
  unsigned blocks;
  int rc;
  p.runs = in_runs(p);
  p.nblk = (int)((rows + 32 * S::RW - 1) / (32 * S::RW));
  if ((rc = grid_of(slices, p.nblk, &blocks))) return rc;
  window_dq_kernel<T, D, S::RW, S::CS, D >= 64 ? 2 : 4><<<dim3(blocks), dim3(S::RW * S::CS * 64), 0, st>>>(p);
  if ((rc = check_launch("tattn_window_bwd"))) return rc;
  const KeyBlocks<K::RW> kbs(p.S, p.sinks, splits);
  if ((rc = grid_of(slices, kbs.items, &blocks))) return rc;
  window_dkdv_kernel<T, D, K::RW, K::CS, D >= 64 ? 2 : D == 32 ? 3 : 4><<<dim3(blocks), dim3(K::RW * K::CS * 64), 0, st>>>(p);
  if ((rc = check_launch("tattn_window_bwd")) || !kbs.sink_blocks) return rc;
  const int64_t n = slices * kbs.sink_blocks * 2 * 32 * K::RW * D;
  window_first_keys_kernel<T, D, K::RW><<<dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st>>>(p);
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
  constexpr int PER = 256 / (D / 4);
  combine_kernel<T, D><<<dim3((unsigned)((rows + PER - 1) / PER)), dim3(256), 0, st>>>(part, (T*)out, m, so[0], so[1], so[2],
                                                                                       slices, Hk, G, N, splits);
  return check_launch("combine");
}

}  // namespace

// Few rows: one row tile per workgroup, and its keys cut into parts until the chip has two workgroups per CU, each with
// at least eight tiles. 0: enough rows for the blocks of two row tiles.
int window_fwd_splits(const WindowParams& p) {
  const int64_t slices = (int64_t)p.Z * p.Hk, rows = (int64_t)p.N * p.G;
  if (slices * ((rows + 63) / 64) >= 256) return 0;
  const int64_t blocks = slices * ((rows + 31) / 32);
  return (int)std::max<int64_t>(1, std::min<int64_t>((512 + blocks - 1) / blocks, most_tiles(p) / 8));
}

// Parts of the first keys' dK and dV: each about as long as another key block's list, or as an even share of all
// work over four workgroups per CU where that is more.
int window_bwd_splits(const WindowParams& p, int D) {
  if (p.sinks == 0) return 1;
  const int64_t rw = D == 128 ? KeyShape<128>::RW : KeyShape<64>::RW, keys = 32 * rw;
  const int64_t all = (int64_t)p.G * ((p.N + 31) / 32);
  const int64_t list = std::min<int64_t>(all, (int64_t)p.G * (std::min<int64_t>(p.window, p.S) / 32 + rw + 1));
  const int64_t share = (int64_t)p.Z * p.Hk * ((p.S + keys - 1) / keys) * list / 1024;
  const int64_t part = std::max<int64_t>(std::max<int64_t>(list, share), 32);
  return (int)std::max<int64_t>(1, std::min<int64_t>((all + part - 1) / part, 256));
}

int64_t window_bwd_part_floats(const WindowParams& p, int D) {
  const int splits = window_bwd_splits(p, D);
  if (splits == 1) return 0;
  const int64_t rw = D == 128 ? KeyShape<128>::RW : KeyShape<64>::RW;
  const int64_t blocks = D == 128 ? KeyBlocks<KeyShape<128>::RW>(p.S, p.sinks, splits).sink_blocks
                                  : KeyBlocks<KeyShape<64>::RW>(p.S, p.sinks, splits).sink_blocks;
  return (int64_t)p.Z * p.Hk * blocks * splits * 2 * 32 * rw * D;
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
