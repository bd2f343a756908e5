// Attention over keys of another length where there are many rows: device code of the kernels of cross_fwd.hip and prefix.hip.
//
// A workgroup's NW waves own 32 QT rows each and walk the keys together, 32 a step. Step i issues S_{i+1} = K_{i+1} Q^T and
// O^T += V_{i-1}^T P_{i-1}^T, neither of which waits for its softmax, and turns S_i into P_i meanwhile. Probabilities are taken
// against the running max as it stands (seeded from the first tile), and only a lane whose 16 sum above 2^12 sends its wave
// through the row max, a rescale and S_i again.
//
// Tiles come by LDS DMA into a ring of four stages, each an array of its own (a DMA into one does not alias reads of another):
// stage (i + 3) % 4 is filled in step i with K_{i+3} and V_{i+1}, so step i reads both its tiles from stage (i + 1) % 4, and the
// slow path K_i from stage i % 4. One barrier per step. Half of the waves fetch K, the others V.
#pragma once

#include "cross.h"

namespace tattn {
namespace {

template <typename T, int D, int NW, int QT>
__device__ __forceinline__ void pipe_block(const CrossParams& p, int slice, int blk, int split, char* st0, char* st1, char* st2,
                                           char* st3) {
  using V8 = typename H16<T>::V8;
  using Tile = CrossTile<D>;
  constexpr int NSD = D / 16, DT = (D + 31) / 32, HALF = Tile::BYTES;
  constexpr int CPW = 2 * Tile::PIECES / NW;  // pieces that a wave fetches in a step
  static_assert(CPW >= 1 && CPW * NW == 2 * Tile::PIECES && NW % 2 == 0, "whole pieces, one tensor per wave");
  auto stage = [&](int s) __attribute__((always_inline)) -> char* { return s == 0 ? st0 : s == 1 ? st1 : s == 2 ? st2 : st3; };

  const int tid = threadIdx.x;
  const int lane = tid & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(tid >> 6));
  const float c = p.c;
  const CrossSlice sl(p, slice);
  const int tiles = (sl.len + 31) >> 5;
  const int i0 = (int)((int64_t)tiles * split / p.splits), i1 = (int)((int64_t)tiles * (split + 1) / p.splits);
  const int nsteps = i1 - i0, left = sl.len - 32 * i0;  // keys from the part's first on
  const int rows = p.B * p.G * p.N, row0 = 32 * QT * (blk * NW + wu);

  const bool second = wu >= NW / 2;
  const int64_t kvs = second ? p.sv[2] : p.sk[2];
  const __amdgpu_buffer_rsrc_t rs = second ? rows_rsrc<T, D>(p.v, sl.zs * p.sv[0] + sl.hk * p.sv[1], sl.len, p.sv[2])
                                           : rows_rsrc<T, D>(p.k, sl.zs * p.sk[0] + sl.hk * p.sk[1], sl.len, p.sk[2]);
  const uint32_t step_bytes = uniform32((uint32_t)(kvs * 64));
  const int piece0 = wu % (NW / 2) * CPW, base = (second ? HALF : 0) + 1024 * piece0;
  uint32_t go[CPW];
#pragma unroll
  for (int i = 0; i < CPW; ++i) go[i] = Tile::source(piece0 + i, lane, kvs) + (uint32_t)i0 * step_bytes;
  auto fetch = [&](char* st, int t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < CPW; ++i) dma16(rs, st + base + 1024 * i, go[i] + (uint32_t)t * step_bytes);
  };
  // The tiles of step i: K_{i+3}, or V_{i+1}.
  const int ahead = second ? 1 : 3;

  if (!second) {
    fetch(st0, 0);
    fetch(st1, 1);
    fetch(st2, 2);
  } else {
    fetch(st2, 0);
  }
  for (int o = tid * 16; o < HALF; o += NW * 64 * 16) st16(st1 + HALF + o, u32x4{});  // read in step 0 with all-zero P

  V8 qop[QT][NSD];
#pragma unroll
  for (int j = 0; j < QT; ++j) {
    const int row = row0 + 32 * j + l32;
    const CrossRow r(p, sl, row < rows ? row : 0);
    const T* src = (const T*)p.q + r.at(p.sq) + 8 * h2;
#pragma unroll
    for (int s = 0; s < NSD; ++s) {
      const V8 x = *reinterpret_cast<const V8*>(src + 16 * s);
      qop[j][s] = row < rows ? x : V8{};
    }
  }
  CrossOp<D> at;
  at.init(lane);

  float mrow[QT], lrow[QT];
  f32x16 acc[DT][QT];
#pragma unroll
  for (int j = 0; j < QT; ++j) {
    lrow[j] = 0.0f;
#pragma unroll
    for (int u = 0; u < DT; ++u) acc[u][j] = f32x16{};
  }
  auto qk = [&](f32x16 (&s)[QT], const char* st) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < QT; ++j) s[j] = f32x16{};
#pragma unroll
    for (int sd = 0; sd < NSD; ++sd) {
      const V8 ka = lds8<T>(st + at.nat[sd]);
#pragma unroll
      for (int j = 0; j < QT; ++j) s[j] = Elt<T>::mfma(ka, qop[j][sd], s[j]);
    }
  };
  auto pv = [&](const V8 (&x)[QT][2], const char* st) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < DT; ++u)
#pragma unroll
      for (int sg = 0; sg < 2; ++sg) {
        const V8 va = at.template tr<T>(st + HALF, sg, u, lane);
#pragma unroll
        for (int j = 0; j < QT; ++j) acc[u][j] = Elt<T>::mfma(va, x[j][sg], acc[u][j]);
      }
  };
  const float hidden = hidden_score(c);
  // Keys past the last of a tile with `there` of them.
  auto hide = [&](f32x16 (&s)[QT], int there) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < QT; ++j) hide_after(s[j], there - 1, 0, h2, hidden);
  };

  // Stage i % 4 holds K_i, of whose keys `there` are left.
  auto softmax = [&](f32x16 (&s)[QT], V8 (&x)[QT][2], const char* st, int there, auto mask_tag) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
    if constexpr (MASK) hide(s, there);
    float before[QT];
    bool over = false;
#pragma unroll
    for (int j = 0; j < QT; ++j) {
      const float ps = tile_probs<T>(s[j], x[j], c, -mrow[j]);
      before[j] = lrow[j];
      lrow[j] += ps;
      over |= !(ps <= 4096.0f);
    }
    if (__builtin_amdgcn_ballot_w64(over)) {
      qk(s, st);
      if constexpr (MASK) hide(s, there);
#pragma unroll
      for (int j = 0; j < QT; ++j) {
        const float mnew = moved_max(s[j], c, mrow[j]), alpha = fast_exp2(mrow[j] - mnew);
        mrow[j] = mnew;
        lrow[j] = before[j] * alpha + tile_probs<T>(s[j], x[j], c, -mnew);
#pragma unroll
        for (int u = 0; u < DT; ++u) acc[u][j] *= alpha;
      }
    }
  };
  auto step_end = [&]() __attribute__((always_inline)) {
    wave_landed<CPW>();
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
  };

  all_landed_barrier();
  f32x16 sa[QT], sb[QT];
  V8 pa[QT][2], pb[QT][2];
#pragma unroll
  for (int j = 0; j < QT; ++j) {
    pa[j][0] = pa[j][1] = V8{};
    mrow[j] = kNoMax;
  }
  if (nsteps > 0) {
    qk(sa, st0);
    f32x16 seen[QT];
#pragma unroll
    for (int j = 0; j < QT; ++j) seen[j] = sa[j];
    if (left < 32) hide(seen, left);
#pragma unroll
    for (int j = 0; j < QT; ++j) mrow[j] = moved_max(seen[j], c, kNoMax);
  }
  auto step = [&](int i, f32x16 (&s0)[QT], f32x16 (&s1)[QT], const V8 (&x0)[QT][2], V8 (&x1)[QT][2], int st, auto mask_tag)
                  __attribute__((always_inline)) {
    fetch(stage((st + 3) & 3), i + ahead);
    pv(x0, stage((st + 1) & 3));
    qk(s1, stage((st + 1) & 3));
    softmax(s0, x1, stage(st), left - 32 * i, mask_tag);
    step_end();
  };
  const int n_full = min(nsteps, left >> 5);
  int i = 0;
  for (; i + 3 < n_full; i += 4) {
    step(i, sa, sb, pa, pb, 0, std::false_type{});
    step(i + 1, sb, sa, pb, pa, 1, std::false_type{});
    step(i + 2, sa, sb, pa, pb, 2, std::false_type{});
    step(i + 3, sb, sa, pb, pa, 3, std::false_type{});
  }
  for (; i < nsteps; ++i) {
    step(i, sa, sb, pa, pb, i & 3, std::true_type{});
#pragma unroll
    for (int j = 0; j < QT; ++j) {
      sa[j] = sb[j];
      pa[j][0] = pb[j][0];
      pa[j][1] = pb[j][1];
    }
  }
  if (nsteps > 0) pv(pa, stage((nsteps + 1) & 3));
  wave_landed<0>();  // nothing is in flight when the workgroup's LDS is released

#pragma unroll
  for (int j = 0; j < QT; ++j) {
    const float lt = sum_halves(lrow[j]);
    const int row = row0 + 32 * j + l32;
    if (row >= rows) continue;
    f32x16 o[DT];
#pragma unroll
    for (int u = 0; u < DT; ++u) o[u] = acc[u][j];
    const CrossRow r(p, sl, row);
    if (p.splits > 1 || p.joined) {
      const int64_t prow = ((int64_t)slice * p.splits + split) * rows + row;
      store_row_t<float, D>(p.part + prow * D, o, 1.0f, h2);
      if (h2 == 0) {
        float* ml = p.part + (int64_t)p.Zs * p.Hk * p.splits * rows * D + prow * 2;
        ml[0] = mrow[j];
        ml[1] = lt;
      }
    } else {
      store_row_t<T, D>((T*)p.out + r.at(p.sout), o, lt == 0.0f ? 0.0f : 1.0f / lt, h2);  // no keys: zeros
      if (h2 == 0 && p.m) p.m[r.index(p)] = mrow[j] + __log2f(lt);
    }
  }
}

}  // namespace
}  // namespace tattn
