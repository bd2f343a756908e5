// Attention over few keys (a short text that many image tokens read), 16-bit, forward and the whole backward, on gfx950.
//
// K and V of a slice stay in LDS as NT tiles of 32 keys, and every wave walks row tiles of its own with no barrier. All scores
// of a row are in its lane (lane = row, two halves of the keys) before any is turned into a probability, so the softmax takes
// its exact max and sum. The backward needs neither M nor O then: with p the probabilities, delta = sum_j p_j dP_j, dS = p (dP
// - delta), dQ = dS K scale; P and dS go through the wave's own LDS rows once to be read transposed, dV += P^T dO, dK += dS^T
// Q, which stay in registers over all of a wave's rows. Five products run, of which all count, and q and dO are read once. The
// four waves' dK and dV are added through LDS, and the parts that a slice's rows are cut into by cross_sum_kernel, in order.
//
// Roundings: P and dS as operands, once. In float16 dS is scaled by the power of two that the largest norms of dO and v allow
// (|dS| <= 2 |dO| |v|); where a later tile has larger rows, what was summed is scaled down with it.
//
// Bound by bytes forward, and by the chain of products of the one wave that a SIMD holds backward (dK and dV of 96 keys take 192
// registers); cross_short_pipe.hip has the form for two row tiles in a step. us, keys not in a cache: 16 x 8 x 4,096 over 77 x 64 fp16
// forward 39 (134 MB), backward 76 (201 MB, 35 as a copy) and 5 for the sum; over 128 x 64 45 and 114; over 64 x 128 fp16 60
// and 170 (some registers spill; bf16, which needs no factor on dS, 120; by the kernels for many keys 300 and 267).
#include <algorithm>
#include <type_traits>

#include "cross_short.h"

namespace tattn {
namespace {

template <typename T, int D, int NT>
__global__ __launch_bounds__(kShortWaves * 64, 2) void short_fwd_kernel(const CrossParams p) {
  using V8 = typename H16<T>::V8;
  using V4 = typename H16<T>::V4;
  using Tile = CrossTile<D>;
  constexpr int NSD = D / 16, DT = (D + 31) / 32, CPR = D / 8;
  __shared__ __attribute__((aligned(1024))) char kv[2 * NT * Tile::BYTES];
  __shared__ __attribute__((aligned(1024))) char ost[kShortWaves * Tile::BYTES];
  __shared__ __attribute__((aligned(16))) float mask[32 * NT];
  const int lane = threadIdx.x & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(threadIdx.x >> 6));
  const ShortRows b(p, p.nblk);
  if (!b.ok) return;
  const CrossSlice sl(p, b.slice);
  const float c = __builtin_fabsf(p.c);
  const uint32_t sign = p.c < 0.0f ? 0x80008000u : 0;
  u32x4 next[NSD];
  auto load = [&](int t) __attribute__((always_inline)) {
    const int row = 32 * t + l32;
    load_rows<T, D>((const T*)p.q, CrossRow(p, sl, row < b.rows ? row : 0).at(p.sq), h2, next);
  };
  int t = b.t0 + wu;
  if (t < b.t1) load(t);
  stage_mask<NT>(sl, mask);
  stage_keys<T, D, NT>(p, sl, kv, wu, lane);
  CrossOp<D> at;
  at.init(lane);
  char* mine = ost + wu * Tile::BYTES;
  for (; t < b.t1; t += kShortWaves) {
    V8 q[NSD];
#pragma unroll
    for (int s = 0; s < NSD; ++s) q[s] = signed_rows<V8>(next[s], sign);
    if (t + kShortWaves < b.t1) load(t + kShortWaves);
    f32x16 s[NT];
    float mx = kNoMax;
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      s[k] = masked_start(mask, k, h2);
#pragma unroll
      for (int sd = 0; sd < NSD; ++sd) s[k] = Elt<T>::mfma(lds8<T>(kv + k * Tile::BYTES + at.nat[sd]), q[sd], s[k]);
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = __builtin_fmaxf(mx, s[k][r]);
    }
    const float m = __builtin_fmaxf(max_halves(mx) * c, kNoMax);  // finite where no key is seen, too
    float l = 0.0f, le = 0.0f;  // of the rounded probabilities, for O, and as they are, for M
    f32x16 o[DT];
#pragma unroll
    for (int u = 0; u < DT; ++u) o[u] = f32x16{};
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      V8 x[2];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[k][r] = fast_exp2(__builtin_fmaf(s[k][r], c, -m));
        le += s[k][r];
      }
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const auto pr = H16<T>::pack(s[k][r], s[k][r + 1]);
        l = H16<T>::sum2(pr, l);
        x[r >> 3][r & 7] = pr[0];
        x[r >> 3][(r & 7) + 1] = pr[1];
      }
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int u = 0; u < DT; ++u) o[u] = Elt<T>::mfma(at.template tr<T>(kv + (NT + k) * Tile::BYTES, g, u, lane), x[g], o[u]);
    }
    l = sum_halves(l);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no keys: zeros
    if (p.m) {
      const int row = 32 * t + l32;
      le = sum_halves(le);
      if (row < b.rows && h2 == 0) p.m[CrossRow(p, sl, row).index(p)] = m + __log2f(le);
    }
    // Whole rows out through the wave's own LDS rows.
#pragma unroll
    for (int u = 0; u < DT; ++u)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d0 = 32 * u + 8 * g + 4 * h2;
        if (d0 >= D) continue;
        V4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (T)(o[u][4 * g + e] * inv);
        *reinterpret_cast<TATTN_LDS V4*>((TATTN_LDS char*)mine + Swz<D>::addr(l32, 2 * d0)) = y;
      }
#pragma unroll
    for (int i = 0; i < (32 * CPR + 63) / 64; ++i) {
      const int j = 64 * i + lane, in = j / CPR, cc = j % CPR, row = 32 * t + in;
      if (in >= 32 || row >= b.rows) continue;
      const u32x4 v = *reinterpret_cast<const TATTN_LDS u32x4*>((const TATTN_LDS char*)mine + Swz<D>::addr(in, 16 * cc));
      st16((T*)p.out + CrossRow(p, sl, row).at(p.sout) + 8 * cc, v);
    }
  }
}

template <typename T, int D, int NT, int OCC>
__global__ __launch_bounds__(kShortWaves * 64, OCC) void short_bwd_kernel(const CrossParams p) {
  using V8 = typename H16<T>::V8;
  using Tile = CrossTile<D>;
  using Pt = Swz<32>;  // rows of a tile of P or dS: 32 keys
  constexpr int NSD = D / 16, DT = (D + 31) / 32, TB = Tile::BYTES;
  constexpr bool LIFT = std::is_same_v<T, f16>;
  constexpr bool AHEAD = NT * DT < 8;                    // registers for the next tile's rows
  constexpr int WAVE = 2 * TB + 2 * 32 * Pt::RB;         // Q, dO, P and dS of a wave
  constexpr int SPACE = 2 * NT * TB + kShortWaves * WAVE;
  static_assert(kShortWaves * short_part(D) <= SPACE, "the waves' sums fit");
  __shared__ __attribute__((aligned(1024))) char smem[SPACE];
  __shared__ __attribute__((aligned(16))) float mask[32 * NT];
  const int tid = threadIdx.x, lane = tid & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(tid >> 6));
  const ShortRows b(p, p.parts);
  if (!b.ok) return;
  const CrossSlice sl(p, b.slice);
  const float c = __builtin_fabsf(p.c);
  const uint32_t sign = p.c < 0.0f ? 0x80008000u : 0;
  char *kv = smem, *qt = smem + 2 * NT * TB + wu * WAVE, *gt = qt + TB, *pt = gt + TB, *st = pt + 32 * Pt::RB;

  u32x4 nq[NSD], ng[NSD];
  auto load = [&](int t) __attribute__((always_inline)) {
    const int row = 32 * t + l32;
    const bool live = row < b.rows;
    const CrossRow r(p, sl, live ? row : 0);
    load_rows<T, D>((const T*)p.q, r.at(p.sq), h2, nq);
    load_rows<T, D>((const T*)p.dout, r.at(p.sd), h2, ng);
    if (!live) {  // contributes nothing
#pragma unroll
      for (int s = 0; s < NSD; ++s) nq[s] = ng[s] = u32x4{};
    }
  };
  int t = b.t0 + wu;
  if (AHEAD && t < b.t1) load(t);
  stage_mask<NT>(sl, mask);
  stage_keys<T, D, NT>(p, sl, kv, wu, lane);
  CrossOp<D> at;
  at.init(lane);
  int plo, phi;  // transposed reads of P and dS: operand lane = key
  tr_addrs<32>(0, 0, lane, plo, phi);

  int ev = 0;  // exponent of the largest norm of v
  if constexpr (LIFT) {
    uint32_t top = 0;
    for (int k = 0; k < NT; ++k) {
      float norm = 0.0f;
#pragma unroll
      for (int s = 0; s < NSD; ++s) {
        const V8 v = lds8<T>(kv + (NT + k) * TB + at.nat[s]);
        norm += chunk_dot(v, v);
      }
      top = max(top, max_wave(__builtin_bit_cast(uint32_t, sum_halves(norm))));
    }
    ev = norm_exponent(top);
  }
  int lift = 40;  // dS is scaled by 2^lift

  f32x16 dk[NT][DT], dv[NT][DT];
#pragma unroll
  for (int k = 0; k < NT; ++k)
#pragma unroll
    for (int u = 0; u < DT; ++u) dk[k][u] = dv[k][u] = f32x16{};

  if (sl.len == 0) {  // zeros: no row sees a key
    for (; t < b.t1; t += kShortWaves) {
      const int row = 32 * t + l32;
      if (row >= b.rows) continue;
      T* dst = (T*)p.out + CrossRow(p, sl, row).at(p.sout);
#pragma unroll
      for (int s = 0; s < NSD; ++s) st16(dst + 16 * s + 8 * h2, u32x4{});
    }
  }
  for (; t < b.t1; t += kShortWaves) {
    if (!AHEAD) load(t);
    V8 q[NSD], g[NSD];
#pragma unroll
    for (int s = 0; s < NSD; ++s) {
      q[s] = signed_rows<V8>(nq[s], sign);
      g[s] = __builtin_bit_cast(V8, ng[s]);
      const int a = Swz<D>::addr(perm32(l32), (16 * s + 8 * h2) * 2);
      *reinterpret_cast<TATTN_LDS u32x4*>((TATTN_LDS char*)qt + a) = nq[s];
      *reinterpret_cast<TATTN_LDS u32x4*>((TATTN_LDS char*)gt + a) = ng[s];
    }
    if (AHEAD && t + kShortWaves < b.t1) load(t + kShortWaves);
    float up = 1.0f;
    if constexpr (LIFT) {
      float norm = 0.0f;
#pragma unroll
      for (int s = 0; s < NSD; ++s) norm += chunk_dot(g[s], g[s]);
      const int e = norm_exponent(max_wave(__builtin_bit_cast(uint32_t, sum_halves(norm))));
      // |dS| < 2^(e + ev + 3); rows with an infinity or a NaN, which spoil their own results, ask for nothing.
      const int most = e >= 30 || ev >= 30 ? 0 : 12 - e - ev;
      if (most < lift) {
        const float down = unlift_of(lift - most);  // 2^(most - lift)
        lift = most;
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
          for (int u = 0; u < DT; ++u) dk[k][u] *= down;
      }
      up = unlift_of(-lift);
    }
    // All scores and dP of the rows (lane = row, register r = key kappa(r, h2)).
    f32x16 s[NT], dp[NT];
    float mx = kNoMax;
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      s[k] = masked_start(mask, k, h2);
      dp[k] = f32x16{};
#pragma unroll
      for (int sd = 0; sd < NSD; ++sd) {
        s[k] = Elt<T>::mfma(lds8<T>(kv + k * TB + at.nat[sd]), q[sd], s[k]);
        dp[k] = Elt<T>::mfma(lds8<T>(kv + (NT + k) * TB + at.nat[sd]), g[sd], dp[k]);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = __builtin_fmaxf(mx, s[k][r]);
    }
    const float m = max_halves(mx) * c;
    float l = 0.0f, dl = 0.0f;
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[k][r] = fast_exp2(__builtin_fmaf(s[k][r], c, -m));
        l += s[k][r];
        dl = __builtin_fmaf(s[k][r], dp[k][r], dl);
      }
    l = sum_halves(l);
    const float inv = 1.0f / l;
    // dS 2^lift = p (dP inv - delta inv) 2^lift with p before its division by l.
    const float by = inv * up, off = -sum_halves(dl) * inv * by;
    f32x16 dq[DT];
#pragma unroll
    for (int u = 0; u < DT; ++u) dq[u] = f32x16{};
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      V8 pp[2], ds[2];
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        float x[2], y[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[e] = s[k][r + e] * inv;
          y[e] = s[k][r + e] * __builtin_fmaf(dp[k][r + e], by, off);
        }
        const auto ph = H16<T>::pack(x[0], x[1]), dh = H16<T>::pack(y[0], y[1]);
        pp[r >> 3][r & 7] = ph[0];
        pp[r >> 3][(r & 7) + 1] = ph[1];
        ds[r >> 3][r & 7] = dh[0];
        ds[r >> 3][(r & 7) + 1] = dh[1];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int a = Pt::addr(perm32(l32), (16 * i + 8 * h2) * 2);
        *reinterpret_cast<TATTN_LDS V8*>((TATTN_LDS char*)pt + a) = pp[i];
        *reinterpret_cast<TATTN_LDS V8*>((TATTN_LDS char*)st + a) = ds[i];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int u = 0; u < DT; ++u) dq[u] = Elt<T>::mfma(at.template tr<T>(kv + k * TB, i, u, lane), ds[i], dq[u]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const V8 pa = tr_pair<T>(pt + 16 * i * Pt::RB, plo, phi), da = tr_pair<T>(st + 16 * i * Pt::RB, plo, phi);
#pragma unroll
        for (int u = 0; u < DT; ++u) {
          dv[k][u] = Elt<T>::mfma(pa, at.template tr<T>(gt, i, u, lane), dv[k][u]);
          dk[k][u] = Elt<T>::mfma(da, at.template tr<T>(qt, i, u, lane), dk[k][u]);
        }
      }
    }
    const int row = 32 * t + l32;
    if (row < b.rows)
      store_row_t<T, D>((T*)p.out + CrossRow(p, sl, row).at(p.sout), dq, p.scale * (LIFT ? unlift_of(lift) : 1.0f), h2);
  }

  short_sums<T, D, NT, DT>(p, sl, b, smem, dk, dv, LIFT ? unlift_of(lift) : 1.0f);
}

template <typename T, int D, int NT>
int short_d(const CrossParams& p, bool bwd, hipStream_t st) {
  unsigned blocks;
  int rc;
  if ((rc = cross_grid(p.slices(), bwd ? p.parts : p.nblk, kShortWaves * 64, &blocks))) return rc;
  if (!bwd) {
    short_fwd_kernel<T, D, NT><<<dim3(blocks), dim3(kShortWaves * 64), 0, st>>>(p);
    return check_launch("tattn_cross_fwd");
  }
  if constexpr (NT <= cross_short_tiles(D, true)) {
    if constexpr (cross_short_piped(D, NT)) rc = launch_cross_short_pipe(p, D, std::is_same_v<T, f16> ? 0 : 2, st);
    else {
      short_bwd_kernel<T, D, NT, cross_short_occ(D, NT)><<<dim3(blocks), dim3(kShortWaves * 64), 0, st>>>(p);
      rc = check_launch("tattn_cross_bwd");
    }
    if (rc || p.parts == 1) return rc;
    return launch_cross_sum(p, D, std::is_same_v<T, f16> ? 0 : 2, true, 32 * NT, st);
  }
  return set_error(TATTN_E_ARG, "too many keys: %d", p.S);
}

template <typename T, int D>
int short_nt(const CrossParams& p, bool bwd, hipStream_t st) {
  switch ((p.S + 31) / 32) {
    case 1: return short_d<T, D, 1>(p, bwd, st);
    case 2: return short_d<T, D, 2>(p, bwd, st);
    case 3: return short_d<T, D, 3>(p, bwd, st);
    case 4: return short_d<T, D, 4>(p, bwd, st);
  }
  return set_error(TATTN_E_ARG, "too many keys: %d", p.S);
}

}  // namespace

int launch_cross_short(const CrossParams& p, int D, int dtype, bool bwd, hipStream_t st) {
  switch (D) {
    case 16: return dtype == 0 ? short_nt<f16, 16>(p, bwd, st) : short_nt<bf16, 16>(p, bwd, st);
    case 32: return dtype == 0 ? short_nt<f16, 32>(p, bwd, st) : short_nt<bf16, 32>(p, bwd, st);
    case 64: return dtype == 0 ? short_nt<f16, 64>(p, bwd, st) : short_nt<bf16, 64>(p, bwd, st);
    case 128: return dtype == 0 ? short_nt<f16, 128>(p, bwd, st) : short_nt<bf16, 128>(p, bwd, st);
  }
  return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %d", D);
}

}  // namespace tattn
