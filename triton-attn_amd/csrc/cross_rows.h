// Attention over keys of another length where rows are few: device code of the kernels of cross.hip and prefix.hip.
//
// The waves of a workgroup share 32 rows, and each takes its own key tiles by itself, staged by LDS DMA into LDS of its own: no
// barrier until their partial results are added.
#pragma once

#include <type_traits>

#include "cross.h"

namespace tattn {
namespace {

// Workgroups of rows_block that a CU holds: 64 KB of tiles at head dim 128, 128 registers below.
constexpr int rows_occ(int D) { return D == 128 ? 2 : 4; }

// LDS of a rows_block: W / H tiles of K, and of V, in each of H arrays.
template <int D, int W, int H>
struct RowsBuf {
  char *k[H], *v[H];
  float (*red)[W][32];
};

// Which halves of a word of two values are not finite: bits 15 of the sum, into which only exponents of ones carry.
template <typename T>
__device__ __forceinline__ uint32_t exponent_carry(uint32_t w) {
  constexpr uint32_t E = std::is_same_v<T, f16> ? 0x7c007c00u : 0x7f807f80u;
  return (w & E) + (0x80008000u - E);
}
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) { return exponent_carry<T>(w) & 0x80008000u; }

// A tile of V in LDS of which rows see some keys and others do not: a hidden key's probability is 0, but 0 times what is not finite is
// not. Where there is any such value, the sums that see it (register r of the lane's row sees keys up to `last`) become NaN, and
// the tile holds a zero in its place. The check takes up to 3% of a call of many queries (8 sequences x 256 queries x 32/8 heads x 128 behind
// 1,024 keys, with 512 of their own: 89 us, 87 without); single tokens see all keys and do without.
template <typename T, int D, int DT>
__device__ __forceinline__ void shield_values(char* vt, const CrossOp<D>& at, f32x16 (&acc)[DT], int last, int t, int lane) {
  using V8 = typename H16<T>::V8;
  TATTN_LDS char* mine = (TATTN_LDS char*)vt + 16 * lane;
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < CrossTile<D>::PIECES; ++i) {
    const u32x4 w = *reinterpret_cast<const TATTN_LDS u32x4*>(mine + 1024 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) any |= exponent_carry<T>(w[e]);
  }
  if (!__builtin_amdgcn_ballot_w64((any & 0x80008000u) != 0)) return;
  const int h2 = lane >> 5, hi = last - 32 * t - 8 * h2;
  V8 seen[2];
#pragma unroll
  for (int r = 0; r < 16; ++r) seen[r >> 3][r & 7] = 16 * (r >> 3) + (r & 7) <= hi ? (T)1.0f : (T)0.0f;
#pragma unroll
  for (int u = 0; u < DT; ++u) {
    f32x16 count = f32x16{};
#pragma unroll
    for (int sg = 0; sg < 2; ++sg) {
      const u32x4 w = __builtin_bit_cast(u32x4, at.template tr<T>(vt, sg, u, lane));
      V8 ones;
#pragma unroll
      for (int e = 0; e < 8; ++e) ones[e] = not_finite<T>(w[e / 2]) >> (e % 2 * 16 + 15) & 1 ? (T)1.0f : (T)0.0f;
      count = Elt<T>::mfma(ones, seen[sg], count);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[u][i] = count[i] > 0.0f ? __builtin_nanf("") : acc[u][i];
  }
#pragma unroll
  for (int i = 0; i < CrossTile<D>::PIECES; ++i) {
    u32x4 w = *reinterpret_cast<const TATTN_LDS u32x4*>(mine + 1024 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] &= ~((not_finite<T>(w[e]) >> 15) * 0xffffu);
    *reinterpret_cast<TATTN_LDS u32x4*>(mine + 1024 * i) = w;
  }
}

// The part `split` of the keys for 32 rows of a slice. CAUSAL: query n is at position len - N + n and sees no key after it.
template <typename T, int D, int W, bool CAUSAL, int H>
__device__ __forceinline__ void rows_block(const CrossParams& p, int slice, int blk, int split, const RowsBuf<D, W, H>& buf) {
  using V4 = typename H16<T>::V4;
  using V8 = typename H16<T>::V8;
  using Tile = CrossTile<D>;
  constexpr int NSD = D / 16, DT = (D + 31) / 32, PIECES = Tile::PIECES;
  const int tid = threadIdx.x;
  const int lane = tid & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(tid >> 6));
  const CrossSlice sl(p, slice);
  const int tiles = (sl.len + 31) >> 5;
  const int i0 = (int)((int64_t)tiles * split / p.splits), i1 = (int)((int64_t)tiles * (split + 1) / p.splits);
  const int rows = p.B * p.G * p.N;
  const float c = p.c, hidden = hidden_score(c);

  const __amdgpu_buffer_rsrc_t krs = rows_rsrc<T, D>(p.k, sl.zs * p.sk[0] + sl.hk * p.sk[1], sl.len, p.sk[2]);
  const __amdgpu_buffer_rsrc_t vrs = rows_rsrc<T, D>(p.v, sl.zs * p.sv[0] + sl.hk * p.sv[1], sl.len, p.sv[2]);
  const uint32_t kb = uniform32((uint32_t)(p.sk[2] * 64)), vb = uniform32((uint32_t)(p.sv[2] * 64));
  uint32_t gk[PIECES], gv[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    gk[i] = Tile::source(i, lane, p.sk[2]);
    gv[i] = Tile::source(i, lane, p.sv[2]);
  }
  constexpr int PER = W / H;
  auto* red = buf.red;
  auto fetch_k = [&](char* kt, int t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) dma16(krs, kt + 1024 * i, gk[i] + (uint32_t)t * kb);
  };
  auto fetch_v = [&](char* vt, int t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) dma16(vrs, vt + 1024 * i, gv[i] + (uint32_t)t * vb);
  };
  int t = i0 + wu;
  // What a wave does with its own tiles is written out for each array that they may lie in: only of a known array does the compiler
  // see that a load into it does not concern reads of another.
  auto own = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < H; ++a)
      if (H == 1 || wu / PER == a) f(buf.k[a] + wu % PER * Tile::BYTES, buf.v[a] + wu % PER * Tile::BYTES);
  };
  if (t < i1)
    own([&](char* kt, char* vt) __attribute__((always_inline)) {
      fetch_k(kt, t);
      fetch_v(vt, t);
    });

  const int row = 32 * blk + l32;
  V8 qop[NSD];
  int last = sl.len - 1;  // key that the lane's row sees
  {
    const bool live = row < rows;
    const CrossRow r(p, sl, live ? row : 0);
    if (CAUSAL) last = sl.len - p.N + r.n;
    const T* src = (const T*)p.q + r.at(p.sq) + 8 * h2;
#pragma unroll
    for (int s = 0; s < NSD; ++s) {
      const V8 x = *reinterpret_cast<const V8*>(src + 16 * s);
      qop[s] = live ? x : V8{};
    }
  }
  // Tiles from here on hold keys that some row does not see.
  const int masked = (CAUSAL ? max(0, sl.len - p.N + 1) : sl.len) >> 5;
  CrossOp<D> at;
  at.init(lane);

  float mrow = kNoMax, lrow = 0.0f;
  f32x16 acc[DT];
#pragma unroll
  for (int u = 0; u < DT; ++u) acc[u] = f32x16{};

  // A wave has one tile of each: K of the next tile is on its way from the end of this one's scores on, V from the end of its products
  // on. (Past the last tile it comes again, so that as many loads are in flight in every step.) Probabilities are taken against
  // the running max as it stands; a lane whose 16 sum above 2^12 (its first tile among them) sends the wave through the row max
  // and a rescale, a one-sided branch (two-sided ones make the compiler hold the accumulators twice).
  auto step = [&](char* kt, char* vt) __attribute__((always_inline)) {
    const int after = t + W < i1 ? t + W : t;
    wave_landed<PIECES>();  // V is still in flight
    f32x16 s = f32x16{};
#pragma unroll
    for (int sd = 0; sd < NSD; ++sd) s = Elt<T>::mfma(lds8<T>(kt + at.nat[sd]), qop[sd], s);
    reads_done();
    fetch_k(kt, after);
    if (t >= masked) hide_after(s, last, t, h2, hidden);
    V8 x[2];
    const float ps = tile_probs<T>(s, x, c, -mrow), before = lrow;
    lrow += ps;
    if (__builtin_amdgcn_ballot_w64(!(ps <= 4096.0f))) {
      const float mnew = moved_max(s, c, mrow), alpha = fast_exp2(mrow - mnew);
      mrow = mnew;
      lrow = before * alpha + tile_probs<T>(s, x, c, -mnew);
#pragma unroll
      for (int u = 0; u < DT; ++u) acc[u] *= alpha;
    }
    wave_landed<PIECES>();  // the next K is still in flight
    if (CAUSAL && p.N > 1 && t >= masked) shield_values<T, D, DT>(vt, at, acc, last, t, lane);
#pragma unroll
    for (int sg = 0; sg < 2; ++sg)
#pragma unroll
      for (int u = 0; u < DT; ++u) acc[u] = Elt<T>::mfma(at.template tr<T>(vt, sg, u, lane), x[sg], acc[u]);
    reads_done();
    fetch_v(vt, after);
    t += W;
  };
  own([&](char* kt, char* vt) __attribute__((always_inline)) {
    while (t < i1) step(kt, vt);  // (as a plain loop body it takes 30 more registers)
  });
  wave_landed<0>();

  // The waves' results through LDS.
  {
    const float lsum = sum_halves(lrow);
    if (h2 == 0) {
      red[0][wu][l32] = mrow;
      red[1][wu][l32] = lsum;
    }
  }
  constexpr int PART = DT * 16 * 64;  // floats of one wave's rows: two tiles of K or V
  static_assert(PART * 4 == 2 * Tile::BYTES && PER % 2 == 0, "the buffers hold the rows of every wave");
  const bool parted = p.splits > 1 || p.joined;
  auto part = [&](int k) {
    char* base = buf.k[0];
#pragma unroll
    for (int a = 0; a < 2 * H; ++a)
      if (k / (PER / 2) == a) base = a % 2 ? buf.v[a / 2] : buf.k[a / 2];
    return (TATTN_LDS float*)base + k % (PER / 2) * PART + lane;
  };
  __syncthreads();  // every wave is done with its tiles, nothing is in flight
  float mall = kNoMax, lall = 0.0f;
#pragma unroll
  for (int k = 0; k < W; ++k) mall = __builtin_fmaxf(mall, red[0][k][l32]);
#pragma unroll
  for (int k = 0; k < W; ++k) lall += fast_exp2(red[0][k][l32] - mall) * red[1][k][l32];
  float wgt = fast_exp2(mrow - mall);
  if (!parted) wgt = lall == 0.0f ? 0.0f : wgt / lall;  // no keys: zeros
  TATTN_LDS float* dst = part(wu);
#pragma unroll
  for (int u = 0; u < DT; ++u)
#pragma unroll
    for (int i = 0; i < 16; ++i) dst[(16 * u + i) * 64] = acc[u][i] * wgt;
  __syncthreads();
  if (row < rows) {
    const CrossRow r(p, sl, row);
    T* orow = (T*)p.out + r.at(p.sout);
    const int64_t prow = ((int64_t)slice * p.splits + split) * rows + row;
    for (int g = wu; g < DT * 4; g += W) {  // four consecutive columns per register group
      const int d0 = 8 * g + 4 * h2;
      if (d0 >= D) continue;
      f32x4 x = f32x4{};
#pragma unroll
      for (int k = 0; k < W; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += part(k)[(4 * g + e) * 64];
      if (parted) {
        *reinterpret_cast<f32x4*>(p.part + prow * D + d0) = x;
      } else {
        V4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (T)x[e];
        *reinterpret_cast<V4*>(orow + d0) = y;
      }
    }
    if (wu == 0 && h2 == 0) {
      if (parted) {
        float* ml = p.part + (int64_t)p.Zs * p.Hk * p.splits * rows * D + prow * 2;
        ml[0] = mall;
        ml[1] = lall;
      } else if (p.m) {
        p.m[r.index(p)] = mall + __log2f(lall);
      }
    }
  }
}

}  // namespace
}  // namespace tattn
