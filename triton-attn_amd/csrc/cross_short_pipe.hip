// Attention over few keys, 16-bit backward where a SIMD holds one wave and there are registers and LDS for two row tiles in a step, on
// gfx950. The mathematics, roundings and layout of cross_short.hip. Step i turns the scores and dP of tile i into P and dS while the
// products of tile i - 1 with them (dV, dK) run, then issues dQ_i and the scores and dP of tile i + 1: none waits for what it follows.
//
// 16 x 8 x 4,096 rows x 64, keys not in a cache, us, one tile in a step and two: 77 keys (fp16) 86 and 76, 60 (bf16) 70 and 57;
// 16 x 16 x 4,096 over 128 x 32 147 and 131. With two and 128 keys x 64 registers spill, and two waves on a SIMD, where their sums
// fit, are as fast by one tile each.
#include <type_traits>

#include "cross_short.h"

namespace tattn {
namespace {

template <typename T, int D, int NT>
__global__ __launch_bounds__(kShortWaves * 64, 1) void short_pipe_kernel(const CrossParams p) {
  using V8 = typename H16<T>::V8;
  using Tile = CrossTile<D>;
  using Pt = Swz<32>;  // rows of a tile of P or dS: 32 keys
  constexpr int NSD = D / 16, DT = (D + 31) / 32, TB = Tile::BYTES;
  constexpr bool LIFT = std::is_same_v<T, f16>;
  constexpr int PB = 32 * Pt::RB, WAVE = 4 * TB + 2 * NT * PB;  // Q and dO of two tiles, P and dS of a wave
  constexpr int SPACE = 2 * NT * TB + kShortWaves * WAVE;
  static_assert(kShortWaves * short_part(D) <= SPACE, "the waves' sums fit");
  __shared__ __attribute__((aligned(1024))) char smem[SPACE];
  __shared__ __attribute__((aligned(16))) float mask[32 * NT];
  const int lane = threadIdx.x & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(threadIdx.x >> 6));
  const ShortRows b(p, p.parts);
  if (!b.ok) return;
  const CrossSlice sl(p, b.slice);
  const float c = __builtin_fabsf(p.c);
  const uint32_t sign = p.c < 0.0f ? 0x80008000u : 0;
  char *kv = smem, *pt = smem + 2 * NT * TB + wu * WAVE, *st = pt + NT * PB, *qt = st + NT * PB;

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
  load(t);
  for (int i = lane; i < WAVE / 16; i += 64) st16(pt + 16 * i, u32x4{});  // read by the first tile's step
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
  // All scores and dP of the loaded rows (lane = row, register r = key kappa(r, h2)); the rows go to LDS as well, to `tile`.
  f32x16 s[NT], dp[NT];
  int most = 0;  // power of two that keeps the rows' dS finite
  // Where it is less than that of the rows before, what was summed is scaled down with it.
  auto follow = [&]() __attribute__((always_inline)) {
    if constexpr (LIFT)
      if (most < lift) {
        const float down = unlift_of(lift - most);  // 2^(most - lift)
        lift = most;
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
          for (int u = 0; u < DT; ++u) dk[k][u] *= down;
      }
  };
  auto scores = [&](char* tile) __attribute__((always_inline)) {
    V8 q[NSD], g[NSD];
#pragma unroll
    for (int i = 0; i < NSD; ++i) {
      q[i] = signed_rows<V8>(nq[i], sign);
      g[i] = __builtin_bit_cast(V8, ng[i]);
      const int a = Swz<D>::addr(perm32(l32), (16 * i + 8 * h2) * 2);
      *reinterpret_cast<TATTN_LDS u32x4*>((TATTN_LDS char*)tile + a) = nq[i];
      *reinterpret_cast<TATTN_LDS u32x4*>((TATTN_LDS char*)tile + TB + a) = ng[i];
    }
    if constexpr (LIFT) {
      float norm = 0.0f;
#pragma unroll
      for (int i = 0; i < NSD; ++i) norm += chunk_dot(g[i], g[i]);
      const int e = norm_exponent(max_wave(__builtin_bit_cast(uint32_t, sum_halves(norm))));
      // |dS| < 2^(e + ev + 3); rows with an infinity or a NaN, which spoil their own results, ask for nothing.
      most = e >= 30 || ev >= 30 ? 0 : 12 - e - ev;
    }
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      s[k] = masked_start(mask, k, h2);
      dp[k] = f32x16{};
#pragma unroll
      for (int sd = 0; sd < NSD; ++sd) {
        s[k] = Elt<T>::mfma(lds8<T>(kv + k * TB + at.nat[sd]), q[sd], s[k]);
        dp[k] = Elt<T>::mfma(lds8<T>(kv + (NT + k) * TB + at.nat[sd]), g[sd], dp[k]);
      }
    }
  };
  // dV += P^T dO, dK += dS^T Q of the rows that lie in LDS.
  auto sums_of_rows = [&](const char* tile) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int o = k * PB + 16 * i * Pt::RB;
        const V8 pa = tr_pair<T>(pt + o, plo, phi), da = tr_pair<T>(st + o, plo, phi);
#pragma unroll
        for (int u = 0; u < DT; ++u) {
          dv[k][u] = Elt<T>::mfma(pa, at.template tr<T>(tile + TB, i, u, lane), dv[k][u]);
          dk[k][u] = Elt<T>::mfma(da, at.template tr<T>(tile, i, u, lane), dk[k][u]);
        }
      }
  };
  int other = 2 * TB;  // of the tiles in LDS: not the one that is turned into P and dS
  if (t < b.t1) {
    scores(qt);
    load(t + kShortWaves);
  }
  for (; t < b.t1; t += kShortWaves) {
    float mx = kNoMax;
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = __builtin_fmaxf(mx, s[k][r]);
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
    sums_of_rows(qt + other);  // of the last tile
    follow();
    l = sum_halves(l);
    const float inv = 1.0f / l;
    // dS 2^lift = p (dP inv - delta inv) 2^lift with p before its division by l.
    const float by = LIFT ? inv * unlift_of(-lift) : inv, off = -sum_halves(dl) * inv * by;
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
        const int a = k * PB + Pt::addr(perm32(l32), (16 * i + 8 * h2) * 2);
        *reinterpret_cast<TATTN_LDS V8*>((TATTN_LDS char*)pt + a) = pp[i];
        *reinterpret_cast<TATTN_LDS V8*>((TATTN_LDS char*)st + a) = ds[i];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int u = 0; u < DT; ++u) dq[u] = Elt<T>::mfma(at.template tr<T>(kv + k * TB, i, u, lane), ds[i], dq[u]);
    }
    const float scale = p.scale * (LIFT ? unlift_of(lift) : 1.0f);
    scores(qt + other);  // of the next tile; past the last one of no meaning
    load(t + 2 * kShortWaves);
    other = 2 * TB - other;
    const int row = 32 * t + l32;
    if (row < b.rows)
      store_row_t<T, D>((T*)p.out + CrossRow(p, sl, row).at(p.sout), dq, scale, h2);
  }
  sums_of_rows(qt + other);
  short_sums<T, D, NT, DT>(p, sl, b, smem, dk, dv, LIFT ? unlift_of(lift) : 1.0f);
}

template <typename T, int D, int NT>
int pipe_nt(const CrossParams& p, hipStream_t st) {
  unsigned blocks;
  if (int rc = cross_grid(p.slices(), p.parts, kShortWaves * 64, &blocks)) return rc;
  short_pipe_kernel<T, D, NT><<<dim3(blocks), dim3(kShortWaves * 64), 0, st>>>(p);
  return check_launch("tattn_cross_bwd");
}

template <typename T>
int pipe_t(const CrossParams& p, int D, hipStream_t st) {
  const int nt = (p.S + 31) / 32;
  if (D == 16 && nt == 4) return pipe_nt<T, 16, 4>(p, st);
  if (D == 32 && nt == 4) return pipe_nt<T, 32, 4>(p, st);
  if (D == 64 && nt == 2) return pipe_nt<T, 64, 2>(p, st);
  if (D == 64 && nt == 3) return pipe_nt<T, 64, 3>(p, st);
  return set_error(TATTN_E_ARG, "no kernel for %d keys of head dim %d", p.S, D);
}

}  // namespace

int launch_cross_short_pipe(const CrossParams& p, int D, int dtype, hipStream_t st) {
  return dtype == 0 ? pipe_t<f16>(p, D, st) : pipe_t<bf16>(p, D, st);
}

}  // namespace tattn
