// Attention over a sliding window and the first keys in float32, forward and backward, on gfx950's float32 matrix
// instruction.
//
//   v_mfma_f32_32x32x2f32: A lane holds A[m = lane % 32][k = lane / 32], B lane B[k = lane / 32][n = lane % 32]
//
// Four waves of a workgroup own a 32-row tile each (rows with all their heads, window.h; 32 keys for dK / dV) and walk the tiles
// of the other dimension that any of them sees, staged one at a time through registers into LDS, the next one's loads in
// flight meanwhile. The order of d within a dot product is free: lane half h owns d from h D / 2 on, so that a
// 16-byte LDS read feeds four instructions. Tiles are read in perm32 order, which gives a lane's 16 results the
// keys (or queries) kappa(r, h): what the second product needs as its operand, with no lane exchange and no rounding.
// Bound by the matrix instruction: 2,048 multiply-adds in 64 cycles, 157 TFLOP/s in all. 4 x 16 x 4,096 x 64 at window 1,024
// takes 0.58 ms forward (104 TFLOP/s) and 2.9 ms backward (52 with the five products that count, 73 with its seven);
// 11 x 12/4 x 1,500 x 128 at window 512 0.51 and 1.9 ms. Keys are not split between workgroups, so few rows over many keys
// leave the chip partly idle (8 x 32/8 x 128, one query over a window of 4,096: 0.62 ms).
#include "window.h"

namespace tattn {
namespace {

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

// The rows of a workgroup of four row tiles and those of the wave.
struct Rows32 {
  int z, hk, off, len, rows, top, slice;
  int n, g, pos;
  bool ok, live;
  TileList list;
  WaveTiles sees;
  __device__ __forceinline__ void init(const WindowParams& p, int w, int l32) {
    int blk;
    ok = window_coord(p.Z * p.Hk, p.nblk, p.head, p.tail, slice, blk);
    if (!ok) return;
    blk = p.nblk - 1 - blk;  // longest rows first
    z = slice / p.Hk;
    hk = slice % p.Hk;
    len = p.lens ? min(max(p.lens[z], 0), p.S) : p.S;
    off = len - p.N;
    rows = p.N * p.G;
    const int p0 = off + 128 * blk / p.G;
    top = off + min(128 * blk + 127, rows - 1) / p.G;
    list.init(p0, top, off + min(128 * blk + 96, rows - 1) / p.G, p.window, p.sinks);
    const int tile0 = 128 * blk + 32 * w, row = tile0 + l32;
    live = row < rows;
    n = (live ? row : 0) / p.G;
    g = (live ? row : 0) % p.G;
    pos = off + n;
    sees.init(list, off + tile0 / p.G, tile0 < rows ? off + min(tile0 + 31, rows - 1) / p.G : -1, p.window, p.sinks);
  }
  // Whether entry i of the list has the key: some row of the workgroup sees it.
  __device__ __forceinline__ bool key(int i, int k, int sinks) const { return k <= top && (k >= list.low(i) || k < sinks); }
};

template <int D, int OCC>
__global__ __launch_bounds__(256, OCC) void window_fwd_f32_kernel(const WindowParams p) {
  using C = F32<D>;
  __shared__ __attribute__((aligned(16))) float ks[32 * C::LD], vs[32 * C::LD];
  const int lane = threadIdx.x & 63, h2 = lane >> 5, l32 = lane & 31;
  Rows32 b;
  b.init(p, (int)uniform32(threadIdx.x >> 6), l32);
  if (!b.ok) return;
  const float c = p.c, hidden = hidden_score(c);
  const float* K = (const float*)p.k + b.z * p.sk[0] + b.hk * p.sk[1];
  const float* V = (const float*)p.v + b.z * p.sv[0] + b.hk * p.sv[1];
  float q[C::H];
  own_row<D>((const float*)p.q + b.z * p.sq[0] + (b.hk * p.G + b.g) * p.sq[1] + b.n * p.sq[2], b.live, h2, q);
  float mrow = kNoMax, lrow = 0.0f;
  f32x16 acc[C::DT];
#pragma unroll
  for (int u = 0; u < C::DT; ++u) acc[u] = f32x16{};
  Tile32<D> kn, vn;
  auto load = [&](int i) {
    auto seen = [&](int key) { return b.key(i, key, p.sinks); };
    kn.load(K, p.sk[2], 32 * b.list.at(i), seen);
    vn.load(V, p.sv[2], 32 * b.list.at(i), seen);
  };
  if (b.list.n > 0) load(0);
  for (int i = 0; i < b.list.n; ++i) {
    __syncthreads();
    kn.store(ks);
    vn.store(vs);
    __syncthreads();
    if (i + 1 < b.list.n) load(i + 1);
    const int t = b.list.at(i);
    if (!b.sees.live(i, t)) continue;
    f32x16 s = rows_dot<D>(ks, q, f32x16{}, l32, h2);
    if (b.sees.masked(t)) RowMask(b.pos, t, h2, p.window, p.sinks).hide(s, hidden);
    float mx = kNoMax;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = __builtin_fmaxf(mx, s[r] * c);
    const float cand = max_halves(mx);
    const float mnew = cand > mrow + kRescaleLog2 ? cand : mrow, alpha = fast_exp2(mrow - mnew);
    if (__builtin_amdgcn_ballot_w64(mnew != mrow)) {
#pragma unroll
      for (int u = 0; u < C::DT; ++u) acc[u] *= alpha;
    }
    mrow = mnew;
    float ps = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = fast_exp2(__builtin_fmaf(s[r], c, -mnew));
      ps += s[r];
    }
    lrow = lrow * alpha + ps;
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int u = 0; u < C::DT; ++u) acc[u] = mfma2(cell<D>(vs, r, 32 * u + l32, h2), s[r], acc[u]);
  }
  const float lt = sum_halves(lrow), inv = lt == 0.0f ? 0.0f : 1.0f / lt;  // rows that see no key become 0
  if (!b.live) return;
  const int h = b.hk * p.G + b.g;
  float* orow = (float*)p.out + b.z * p.sout[0] + h * p.sout[1] + b.n * p.sout[2];
#pragma unroll
  for (int u = 0; u < C::DT; ++u)
#pragma unroll
    for (int gr = 0; gr < 4; ++gr) {
      const int d0 = 32 * u + 8 * gr + 4 * h2;
      if (d0 >= D) continue;
      f32x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = acc[u][4 * gr + e] * inv;
      *reinterpret_cast<f32x4*>(orow + d0) = y;
    }
  if (h2 == 0 && p.m) p.m[((int64_t)b.z * p.H + h) * p.N + b.n] = mrow + __log2f(lt);
}

template <int D, int OCC>
__global__ __launch_bounds__(256, OCC) void window_dq_f32_kernel(const WindowParams p) {
  using C = F32<D>;
  __shared__ __attribute__((aligned(16))) float ks[32 * C::LD], vs[32 * C::LD];
  const int lane = threadIdx.x & 63, h2 = lane >> 5, l32 = lane & 31;
  Rows32 b;
  b.init(p, (int)uniform32(threadIdx.x >> 6), l32);
  if (!b.ok) return;
  const float c = p.c, hidden = hidden_score(c);
  const float* K = (const float*)p.k + b.z * p.sk[0] + b.hk * p.sk[1];
  const float* V = (const float*)p.v + b.z * p.sv[0] + b.hk * p.sv[1];
  const int h = b.hk * p.G + b.g;
  const int64_t mrow = ((int64_t)b.z * p.H + h) * p.N + b.n;
  float q[C::H], go[C::H];
  own_row<D>((const float*)p.q + b.z * p.sq[0] + h * p.sq[1] + b.n * p.sq[2], b.live, h2, q);
  own_row<D>((const float*)p.dout + b.z * p.sd[0] + h * p.sd[1] + b.n * p.sd[2], b.live, h2, go);
  float dl = 0.0f;
  {
    const float* o = (const float*)p.o + b.z * p.so[0] + h * p.so[1] + b.n * p.so[2] + h2 * C::H;
#pragma unroll
    for (int j = 0; j < C::H; ++j) dl = __builtin_fmaf(o[j], go[j], dl);
    dl = b.live ? sum_halves(dl) : 0.0f;
    if (b.live && h2 == 0) p.delta[mrow] = -dl;
  }
  const float nm = b.live ? -p.m[mrow] : 0.0f;
  f32x16 dq[C::DT];
#pragma unroll
  for (int u = 0; u < C::DT; ++u) dq[u] = f32x16{};
  Tile32<D> kn, vn;
  auto load = [&](int i) {
    auto seen = [&](int key) { return b.key(i, key, p.sinks); };
    kn.load(K, p.sk[2], 32 * b.list.at(i), seen);
    vn.load(V, p.sv[2], 32 * b.list.at(i), seen);
  };
  if (b.list.n > 0) load(0);
  for (int i = 0; i < b.list.n; ++i) {
    __syncthreads();
    kn.store(ks);
    vn.store(vs);
    __syncthreads();
    if (i + 1 < b.list.n) load(i + 1);
    const int t = b.list.at(i);
    if (!b.sees.live(i, t)) continue;
    f32x16 s = rows_dot<D>(ks, q, f32x16{}, l32, h2), dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) dp[r] = -dl;
    dp = rows_dot<D>(vs, go, dp, l32, h2);
    if (b.sees.masked(t)) RowMask(b.pos, t, h2, p.window, p.sinks).hide(s, hidden);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = fast_exp2(__builtin_fmaf(s[r], c, nm)) * dp[r];
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int u = 0; u < C::DT; ++u) dq[u] = mfma2(cell<D>(ks, r, 32 * u + l32, h2), s[r], dq[u]);
  }
  if (!b.live) return;
  float* orow = (float*)p.out + b.z * p.sout[0] + h * p.sout[1] + b.n * p.sout[2];
#pragma unroll
  for (int u = 0; u < C::DT; ++u)
#pragma unroll
    for (int gr = 0; gr < 4; ++gr) {
      const int d0 = 32 * u + 8 * gr + 4 * h2;
      if (d0 >= D) continue;
      f32x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = dq[u][4 * gr + e] * p.scale;
      *reinterpret_cast<f32x4*>(orow + d0) = y;
    }
}

// A workgroup owns 128 keys and walks the query tiles that see any of them, head after head of the group.
template <int D>
__global__ __launch_bounds__(256, 1) void window_dkdv_f32_kernel(const WindowParams p) {
  using C = F32<D>;
  __shared__ __attribute__((aligned(16))) float qs[32 * C::LD], gs[32 * C::LD];
  __shared__ __attribute__((aligned(16))) float md[2][32];  // M, -delta
  const int tid = threadIdx.x, lane = tid & 63, h2 = lane >> 5, l32 = lane & 31, w = (int)uniform32(tid >> 6);
  int slice, kb;
  if (!window_coord(p.Z * p.Hk, p.nblk, p.head, p.tail, slice, kb)) return;
  const int z = slice / p.Hk, hk = slice % p.Hk, off = p.S - p.N;
  const int k0 = 128 * kb, k1 = k0 + 127;
  const int nlo = max(0, k0 - off), nhi = k0 < p.sinks ? p.N - 1 : min(p.N - 1, k1 + p.window - 1 - off);
  const int qt0 = nlo >> 5, nq = nhi < nlo ? 0 : (nhi >> 5) - qt0 + 1, total = nq * p.G;
  const float c = p.c, hidden = hidden_score(c);
  const int wk0 = k0 + 32 * w, wk1 = wk0 + 31, key = wk0 + l32;
  const bool seen = key < p.S && (key < p.sinks || off - key < p.window);  // what lies at another key is taken as zero
  float k[C::H], v[C::H];
  own_row<D>((const float*)p.k + z * p.sk[0] + hk * p.sk[1] + (int64_t)(key < p.S ? key : 0) * p.sk[2], seen, h2, k);
  own_row<D>((const float*)p.v + z * p.sv[0] + hk * p.sv[1] + (int64_t)(key < p.S ? key : 0) * p.sv[2], seen, h2, v);
  f32x16 dk[C::DT], dv[C::DT];
#pragma unroll
  for (int u = 0; u < C::DT; ++u) dk[u] = dv[u] = f32x16{};
  Tile32<D> qn, gn;
  float mn = 0.0f;
  auto load = [&](int i) {
    const int h = hk * p.G + i / nq, first = 32 * (qt0 + i % nq);
    auto in = [&](int n) { return n < p.N; };
    qn.load((const float*)p.q + z * p.sq[0] + h * p.sq[1], p.sq[2], first, in);
    gn.load((const float*)p.dout + z * p.sd[0] + h * p.sd[1], p.sd[2], first, in);
    if (tid < 64) mn = first + l32 < p.N ? (h2 ? p.delta : p.m)[((int64_t)z * p.H + h) * p.N + first + l32] : 0.0f;
  };
  if (total > 0) load(0);
  for (int i = 0; i < total; ++i) {
    __syncthreads();
    qn.store(qs);
    gn.store(gs);
    if (tid < 64) md[h2][l32] = mn;
    __syncthreads();
    const int qt = qt0 + i % nq, q0 = off + 32 * qt, q1 = q0 + 31;
    if (i + 1 < total) load(i + 1);
    if (wk0 >= p.S || q1 < wk0 || (q0 - wk1 >= p.window && wk0 >= p.sinks)) continue;
    f32x16 s = rows_dot<D>(qs, k, f32x16{}, l32, h2), dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) dp[r] = md[1][kappa(r, h2)];
    dp = rows_dot<D>(gs, v, dp, l32, h2);
    if (q0 < wk1 || (q1 - wk0 >= p.window && wk1 >= p.sinks) || 32 * qt + 32 > p.N)
      ColMask(q0 - key, key, p.N - 32 * qt, h2, p.window, p.sinks).hide(s, hidden);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = fast_exp2(__builtin_fmaf(s[r], c, -md[0][kappa(r, h2)]));
      dp[r] *= s[r];
    }
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int u = 0; u < C::DT; ++u) {
        dv[u] = mfma2(s[r], cell<D>(gs, r, 32 * u + l32, h2), dv[u]);
        dk[u] = mfma2(dp[r], cell<D>(qs, r, 32 * u + l32, h2), dk[u]);
      }
  }
  float* dko = (float*)p.dk + z * p.sdk[0] + hk * p.sdk[1];
  float* dvo = (float*)p.dv + z * p.sdv[0] + hk * p.sdv[1];
#pragma unroll
  for (int u = 0; u < C::DT; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = wk0 + 8 * (r >> 2) + 4 * h2 + (r & 3), d = 32 * u + l32;
      if (row >= p.S || d >= D) continue;
      dko[(int64_t)row * p.sdk[2] + d] = dk[u][r] * p.scale;
      dvo[(int64_t)row * p.sdv[2] + d] = dv[u][r];
    }
}

template <int D>
int fwd_d(WindowParams p, hipStream_t st) {
  unsigned blocks;
  p.nblk = (int)(((int64_t)p.N * p.G + 127) / 128);
  p.tail = window_row_tail(p, 128, p.nblk);
  if (int rc = window_grid((int64_t)p.Z * p.Hk, p.nblk, p.tail, &blocks)) return rc;
  window_fwd_f32_kernel<D, D == 128 ? 1 : 2><<<dim3(blocks), dim3(256), 0, st>>>(p);
  return check_launch("tattn_window_fwd");
}

template <int D>
int bwd_d(WindowParams p, hipStream_t st) {
  unsigned blocks;
  int rc;
  p.nblk = (int)(((int64_t)p.N * p.G + 127) / 128);
  p.tail = window_row_tail(p, 128, p.nblk);
  if ((rc = window_grid((int64_t)p.Z * p.Hk, p.nblk, p.tail, &blocks))) return rc;
  window_dq_f32_kernel<D, D == 128 ? 1 : 2><<<dim3(blocks), dim3(256), 0, st>>>(p);
  if ((rc = check_launch("tattn_window_bwd"))) return rc;
  p.nblk = (p.S + 127) / 128;
  p.tail = window_key_tail(p, 128, p.nblk);
  if ((rc = window_grid((int64_t)p.Z * p.Hk, p.nblk, p.tail, &blocks))) return rc;
  window_dkdv_f32_kernel<D><<<dim3(blocks), dim3(256), 0, st>>>(p);
  return check_launch("tattn_window_bwd");
}

}  // namespace

int launch_window_f32(const WindowParams& p, int D, bool bwd, hipStream_t st) {
  switch (D) {
    case 16: return bwd ? bwd_d<16>(p, st) : fwd_d<16>(p, st);
    case 32: return bwd ? bwd_d<32>(p, st) : fwd_d<32>(p, st);
    case 64: return bwd ? bwd_d<64>(p, st) : fwd_d<64>(p, st);
    case 128: return bwd ? bwd_d<128>(p, st) : fwd_d<128>(p, st);
  }
  return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %d", D);
}

}  // namespace tattn
