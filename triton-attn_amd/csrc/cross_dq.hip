// Attention over keys of another length, 16-bit backward, on gfx950: dQ, and delta on the way. cross_bwd.hip has the mathematics,
// the schedule and the roundings.
//
// Traced: 4 x 16 x 4,096 over 4,096 x 64 fp16 425 us (970 TF of its three products), 2 x 16 x 4,096 over 4,096 x 128 bf16 419
// (985; by single waves, which have a SIMD each, 530).
#include <algorithm>
#include <type_traits>

#include "cross_bwd.h"

namespace tattn {
namespace {

// Whether a sum of the lane's row, whose columns lie in both halves of the wave, is not finite.
template <int DT>
__device__ __forceinline__ bool row_overflowed(const f32x16 (&dq)[DT], int l32) {
  float zero = 0.0f;  // times every sum: NaN where one is not finite
#pragma unroll
  for (int u = 0; u < DT; ++u)
#pragma unroll
    for (int g = 0; g < 16; ++g) zero = __builtin_fmaf(dq[u][g], 0.0f, zero);
  const uint64_t bad = __builtin_amdgcn_ballot_w64(zero != 0.0f);
  return ((bad | bad >> 32) >> l32 & 1) != 0;
}

// What dS of a row in float16 is scaled by, 2^lift, in the next try after one that was not finite; false: there is none. First up where
// dO is small (small_gradient_lift), then as it is, then down so far that it is finite whatever the values: |dS| <= |dO| (|v| + |o|) <
// 2^(exponent + 1) 2^21, as norms of at most 128 values of float16 stay below 2^20. A row of dO that is not finite has one try.
__device__ __forceinline__ bool next_lift(bool overflowed, int exponent, int& lift) {
  if (!overflowed || lift < 0 || exponent >= 30 || (lift == 0 && exponent <= -7)) return false;
  lift = lift > 0 ? 0 : -(exponent + 7);
  return true;
}

// A wave takes 32 rows.
template <typename T, int D, int NW, int OCC>
__global__ __launch_bounds__(NW * 64, OCC) void cross_dq_kernel(const CrossParams p) {
  using V8 = typename H16<T>::V8;
  using B = BwdPipe<D>;
  constexpr int NSD = B::NSD, DT = B::DT, STAGE = B::DQ_STAGE;
  constexpr bool LIFT = std::is_same_v<T, f16>;
  // dS as a sum of two halves up to head dim 32. With few columns the error of delta, which comes from the rounded O, adds to that of
  // a rounded dS: dQ is then 1.55 (head dim 16) and 1.5 times (32) as far off as its last rounding leaves it (1.45 at 64 and 128), and
  // 1.1 times with two halves, at 111 us for 77 and 125 for 92 (4 x 16 x 2,048 over 2,048).
  constexpr int NE = D <= 32 ? 4 : 2;
  __shared__ __attribute__((aligned(16))) char smem[B::NST * STAGE];
  __shared__ uint32_t norms[2][LIFT ? NW : 1];  // per wave: largest squared norm, |delta|

  const int tid = threadIdx.x;
  const int lane = tid & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(tid >> 6));
  const float c = p.c;
  int slice, blk;
  if (!cross_coord(p, p.nblk * p.splits, slice, blk)) return;
  const int split = blk % p.splits;
  blk /= p.splits;
  const CrossSlice sl(p, slice);
  const int tiles = (sl.len + 31) >> 5;
  const int i0 = (int)((int64_t)tiles * split / p.splits), i1 = (int)((int64_t)tiles * (split + 1) / p.splits);
  const int nsteps = i1 - i0, rows = p.G * p.N;

  const __amdgpu_buffer_rsrc_t krs = rows_rsrc<T, D>(p.k, sl.zs * p.sk[0] + sl.hk * p.sk[1], sl.len, p.sk[2]);
  const __amdgpu_buffer_rsrc_t vrs = rows_rsrc<T, D>(p.v, sl.zs * p.sv[0] + sl.hk * p.sv[1], sl.len, p.sv[2]);
  const uint32_t kb = uniform32((uint32_t)(p.sk[2] * 64)), vb = uniform32((uint32_t)(p.sv[2] * 64));
  StepRows<D, NW * 64> next, second;
  next.init(tid, p.sk[2], p.sv[2]);
  second = next;
  next.load(krs, vrs, (uint32_t)i0 * kb, (uint32_t)i0 * vb);
  second.load(krs, vrs, (uint32_t)(i0 + 1) * kb, (uint32_t)(i0 + 1) * vb);

  const int row = 32 * (blk * NW + wu) + l32;
  const bool live = row < rows;
  const CrossRow r(p, sl, live ? row : 0);
  V8 qop[NSD], dop[NSD];
  float dl;
  int lift = 0, exponent = 0;  // dS is scaled by 2^lift; of the norm of the row of dO
  uint32_t top = 0;
  {
    const T* qs = (const T*)p.q + r.at(p.sq) + 8 * h2;
    const T* ds = (const T*)p.dout + r.at(p.sd) + 8 * h2;
    const T* os = (const T*)p.o + r.at(p.so) + 8 * h2;
    float sd[NSD], norm = 0.0f;
#pragma unroll
    for (int s = 0; s < NSD; ++s) {
      const V8 x = *reinterpret_cast<const V8*>(qs + 16 * s), y = *reinterpret_cast<const V8*>(ds + 16 * s);
      qop[s] = live ? x : V8{};
      dop[s] = live ? y : V8{};
      sd[s] = chunk_dot(*reinterpret_cast<const V8*>(os + 16 * s), y);
      if (LIFT) norm += chunk_dot(dop[s], dop[s]);
    }
    dl = row_delta(sd);
    if (!live) dl = 0.0f;
    if (live && h2 == 0 && split == 0) p.delta[(int64_t)slice * rows + row] = -dl;
    if constexpr (LIFT) {
      const uint32_t bits = __builtin_bit_cast(uint32_t, sum_halves(norm));
      exponent = norm_exponent(bits);
      lift = small_gradient_lift(exponent, 60);
      top = max_wave(bits);  // NaN above all
      norms[0][wu] = top;
      norms[1][wu] = max_wave(__builtin_bit_cast(uint32_t, __builtin_fabsf(dl)));
    }
  }
  const float m = live ? p.m[r.index(p)] : 0.0f;
  float nm = live ? (float)lift - m : 0.0f;
  CrossOp<D> at;
  at.init(lane);
  f32x16 dq[DT];

  // S^T and dP^T - delta of a stage's 32 keys (lane = row, register r = key kappa(r, h2)).
  auto first = [&](f32x16& s, f32x16& dp, int st) __attribute__((always_inline)) {
    const char* base = smem + st * STAGE;
    s = f32x16{};
#pragma unroll
    for (int i = 0; i < 16; ++i) dp[i] = -dl;
#pragma unroll
    for (int sd = 0; sd < NSD; ++sd) {
      s = Elt<T>::mfma(lds8<T>(base + at.nat[sd]), qop[sd], s);
      dp = Elt<T>::mfma(lds8<T>(base + B::TILE + at.nat[sd]), dop[sd], dp);
    }
  };
  auto grad = [&](const V8 (&ds)[NE], int st) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int u = 0; u < DT; ++u) {
        const V8 ka = at.template tr<T>(smem + st * STAGE, g, u, lane);
#pragma unroll
        for (int e = g; e < NE; e += 2) dq[u] = Elt<T>::mfma(ka, ds[e], dq[u]);
      }
  };
  auto dsv = [&](const f32x16& s, const f32x16& dp, V8 (&ds)[NE], int left, auto mask_tag) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        float x[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int g = 8 * a + i + e;
          float pr = fast_exp2(__builtin_fmaf(s[g], c, nm));
          if constexpr (MASK) pr = kappa(g, h2) >= left ? 0.0f : pr;
          x[e] = pr * dp[g];
        }
        const auto y = H16<T>::pack(x[0], x[1]);
        ds[a][i] = y[0];
        ds[a][i + 1] = y[1];
        if constexpr (NE == 4) {
          const auto low = H16<T>::pack(x[0] - (float)y[0], x[1] - (float)y[1]);
          ds[2 + a][i] = low[0];
          ds[2 + a][i + 1] = low[1];
        }
      }
  };

  next.clear(smem + 3 * STAGE, tid);  // read by the first step together with all-zero dS
  next.store(smem, tid);
  second.store(smem + STAGE, tid);
  __syncthreads();
  if constexpr (LIFT) {
    if (tid < 2 && split == 0) {  // for dK / dV
      top = norms[tid][0];
#pragma unroll
      for (int k = 1; k < NW; ++k) top = max(top, norms[tid][k]);
      p.norms[2 * ((int64_t)slice * p.nblk + blk) + tid] = __builtin_bit_cast(float, top);
    }
  }
  // Steps whose 32 keys are all there.
  const int n_full = min(nsteps, (sl.len >> 5) - i0);
  for (;;) {
#pragma unroll
    for (int u = 0; u < DT; ++u) dq[u] = f32x16{};
    f32x16 sa, da, sb, db;
    V8 ea[NE] = {}, eb[NE];
    if (nsteps > 0) first(sa, da, 0);
    auto step = [&](int i, int st, f32x16& s0, f32x16& d0, f32x16& s1, f32x16& d1, const V8 (&e0)[NE], V8 (&e1)[NE], auto mask_tag)
                    __attribute__((always_inline)) {
      next.load(krs, vrs, (uint32_t)(i0 + i + 2) * kb, (uint32_t)(i0 + i + 2) * vb);
      first(s1, d1, (st + 1) & 3);
      grad(e0, (st + 3) & 3);
      dsv(s0, d0, e1, sl.len - 32 * (i0 + i), mask_tag);
      next.store(smem + ((st + 2) & 3) * STAGE, tid);
      __syncthreads();
    };
    int i = 0;
    for (; i + 3 < n_full; i += 4) {
      step(i, 0, sa, da, sb, db, ea, eb, std::false_type{});
      step(i + 1, 1, sb, db, sa, da, eb, ea, std::false_type{});
      step(i + 2, 2, sa, da, sb, db, ea, eb, std::false_type{});
      step(i + 3, 3, sb, db, sa, da, eb, ea, std::false_type{});
    }
    for (; i < nsteps; ++i) {
      step(i, i & 3, sa, da, sb, db, ea, eb, std::true_type{});
      sa = sb;
      da = db;
#pragma unroll
      for (int e = 0; e < NE; ++e) ea[e] = eb[e];
    }
    if (nsteps > 0) grad(ea, (nsteps - 1) & 3);
    if (!LIFT) break;
    const bool again = live && next_lift(row_overflowed(dq, l32), exponent, lift);
    if (!__syncthreads_or(again)) break;
    nm = live ? (float)lift - m : 0.0f;
    next.clear(smem + 3 * STAGE, tid);
    next.load(krs, vrs, (uint32_t)i0 * kb, (uint32_t)i0 * vb);
    next.store(smem, tid);
    next.load(krs, vrs, (uint32_t)(i0 + 1) * kb, (uint32_t)(i0 + 1) * vb);
    next.store(smem + STAGE, tid);
    __syncthreads();
  }
  if (!live) return;
  const float unlift = LIFT ? unlift_of(lift) : 1.0f;
  if (p.splits > 1)
    store_row_t<float, D>(p.part + (((int64_t)slice * p.splits + split) * rows + row) * D, dq, unlift, h2);
  else
    store_row_t<T, D>((T*)p.out + r.at(p.sout), dq, p.scale * unlift, h2);
}

// Head dim 128: Q, dO and dQ of 32 rows take more registers than a wave has if another is to share its SIMD. So two waves take a
// tile of rows, each with half of the operands. Over each 32-key step
//   wave j     (role A): S^T = K Q^T, P = 2^(S c - M), into LDS in float32
//   wave j + 4 (role B): dP^T - delta = V dO^T - delta, dS = P (dP - delta), dQ^T += K^T dS^T
// In step i A issues S_{i+1} and turns S_i into P_i; B turns P_{i-1} and dP_{i-1} into dS, adds to dQ and issues dP_i.
template <typename T, int D>
__global__ __launch_bounds__(512, 2) void cross_dq_pair_kernel(const CrossParams p) {
  using V8 = typename H16<T>::V8;
  using B = BwdPipe<D>;
  constexpr int NP = 4, NSD = B::NSD, DT = B::DT, STAGE = B::DQ_STAGE;
  constexpr int XB = 32 * 32 * 4;  // P of a pair
  constexpr bool LIFT = std::is_same_v<T, f16>;
  __shared__ __attribute__((aligned(16))) char smem[B::NST * STAGE];
  __shared__ __attribute__((aligned(16))) char xbuf[2 * NP * XB];
  __shared__ uint32_t norms[2][NP];  // per pair: largest squared norm, |delta|
  __shared__ float lifts[NP][32];

  const int tid = threadIdx.x;
  const int lane = tid & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(tid >> 6));
  const int pr = wu % NP;
  const bool role_b = wu >= NP;
  const float c = p.c;
  int slice, blk;
  if (!cross_coord(p, p.nblk * p.splits, slice, blk)) return;
  const int split = blk % p.splits;
  blk /= p.splits;
  const CrossSlice sl(p, slice);
  const int tiles = (sl.len + 31) >> 5;
  const int i0 = (int)((int64_t)tiles * split / p.splits), i1 = (int)((int64_t)tiles * (split + 1) / p.splits);
  const int nsteps = i1 - i0, rows = p.G * p.N;

  const __amdgpu_buffer_rsrc_t krs = rows_rsrc<T, D>(p.k, sl.zs * p.sk[0] + sl.hk * p.sk[1], sl.len, p.sk[2]);
  const __amdgpu_buffer_rsrc_t vrs = rows_rsrc<T, D>(p.v, sl.zs * p.sv[0] + sl.hk * p.sv[1], sl.len, p.sv[2]);
  const uint32_t kb = uniform32((uint32_t)(p.sk[2] * 64)), vb = uniform32((uint32_t)(p.sv[2] * 64));
  StepRows<D, 512> next, second;
  next.init(tid, p.sk[2], p.sv[2]);
  second = next;
  next.load(krs, vrs, (uint32_t)i0 * kb, (uint32_t)i0 * vb);
  second.load(krs, vrs, (uint32_t)(i0 + 1) * kb, (uint32_t)(i0 + 1) * vb);

  const int row = 32 * (blk * NP + pr) + l32;
  const bool live = row < rows;
  const CrossRow r(p, sl, live ? row : 0);
  V8 op[NSD];  // Q (A) or dO (B)
  {
    const T* src = role_b ? (const T*)p.dout + r.at(p.sd) + 8 * h2 : (const T*)p.q + r.at(p.sq) + 8 * h2;
#pragma unroll
    for (int s = 0; s < NSD; ++s) {
      const V8 x = *reinterpret_cast<const V8*>(src + 16 * s);
      op[s] = live ? x : V8{};
    }
  }
  int lift = 0, exponent = 0;  // dS is scaled by 2^lift; of the norm of the row of dO
  float dl = 0.0f;
  if (role_b) {
    const T* os = (const T*)p.o + r.at(p.so) + 8 * h2;
    float sd[NSD], norm = 0.0f;
#pragma unroll
    for (int s = 0; s < NSD; ++s) {
      sd[s] = chunk_dot(*reinterpret_cast<const V8*>(os + 16 * s), op[s]);
      if (LIFT) norm += chunk_dot(op[s], op[s]);
    }
    dl = row_delta(sd);
    if (!live) dl = 0.0f;
    if (live && h2 == 0 && split == 0) p.delta[(int64_t)slice * rows + row] = -dl;
    if constexpr (LIFT) {
      const uint32_t bits = __builtin_bit_cast(uint32_t, sum_halves(norm));
      exponent = norm_exponent(bits);
      lift = small_gradient_lift(exponent, 60);
      lifts[pr][l32] = (float)lift;
      norms[0][pr] = max_wave(bits);  // NaN above all
      norms[1][pr] = max_wave(__builtin_bit_cast(uint32_t, __builtin_fabsf(dl)));
    }
  }
  const float m = live ? p.m[r.index(p)] : 0.0f;
  CrossOp<D> at;
  at.init(lane);

  next.clear(smem + 3 * STAGE, tid);  // read by the first step together with all-zero dS
  next.store(smem, tid);
  second.store(smem + STAGE, tid);
  __syncthreads();
  float nm = -m;
  if constexpr (LIFT) {
    if (tid < 2 && split == 0) {  // for dK / dV
      uint32_t top = norms[tid][0];
#pragma unroll
      for (int k = 1; k < NP; ++k) top = max(top, norms[tid][k]);
      p.norms[2 * ((int64_t)slice * p.nblk + blk) + tid] = __builtin_bit_cast(float, top);
    }
    nm = live ? lifts[pr][l32] - m : 0.0f;
  }
  // Steps whose 32 keys are all there.
  const int n_full = min(nsteps, (sl.len >> 5) - i0);
  char* xpair = xbuf + pr * XB;

  // A: S^T, B: dP^T - delta of a stage's 32 keys (lane = row, register r = key kappa(r, h2)).
  auto first = [&](f32x16& s, int st, auto role_tag) __attribute__((always_inline)) {
    constexpr bool RB_ = decltype(role_tag)::value;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = RB_ ? -dl : 0.0f;
    const char* tile = smem + st * STAGE + (RB_ ? B::TILE : 0);
#pragma unroll
    for (int sd = 0; sd < NSD; ++sd) s = Elt<T>::mfma(lds8<T>(tile + at.nat[sd]), op[sd], s);
  };
  auto probs = [&](const f32x16& s, int odd, int left, auto mask_tag) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
    TATTN_LDS char* x = (TATTN_LDS char*)xpair + odd * (NP * XB) + 16 * lane;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = fast_exp2(__builtin_fmaf(s[4 * a + e], c, nm));
        if constexpr (MASK) v[e] = kappa(4 * a + e, h2) >= left ? 0.0f : v[e];
      }
      *reinterpret_cast<TATTN_LDS f32x4*>(x + 1024 * a) = v;
    }
  };
  auto dsv = [&](const f32x16& dp, V8 (&ds)[2], int odd) __attribute__((always_inline)) {
    const TATTN_LDS char* x = (const TATTN_LDS char*)xpair + odd * (NP * XB) + 16 * lane;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const f32x4 v = *reinterpret_cast<const TATTN_LDS f32x4*>(x + 1024 * a);
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const auto y = H16<T>::pack(v[e] * dp[4 * a + e], v[e + 1] * dp[4 * a + e + 1]);
        ds[a >> 1][4 * (a & 1) + e] = y[0];
        ds[a >> 1][4 * (a & 1) + e + 1] = y[1];
      }
    }
  };
  f32x16 dq[DT];
  auto grad = [&](const V8 (&ds)[2], int st) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int u = 0; u < DT; ++u) dq[u] = Elt<T>::mfma(at.template tr<T>(smem + st * STAGE, g, u, lane), ds[g], dq[u]);
  };

  auto run = [&](auto role_tag) __attribute__((always_inline)) {
    constexpr bool RB_ = decltype(role_tag)::value;
    f32x16 sa = f32x16{}, sb = f32x16{};  // A: S of this step and the next; B: dP (sa)
    V8 ds[2];
    if (!RB_ && nsteps > 0) first(sa, 0, role_tag);
    auto step = [&](int i, int st, f32x16& x0, f32x16& x1, auto mask_tag) __attribute__((always_inline)) {
      next.load(krs, vrs, (uint32_t)(i0 + i + 2) * kb, (uint32_t)(i0 + i + 2) * vb);
      if constexpr (!RB_) {
        first(x1, (st + 1) & 3, role_tag);
        probs(x0, i & 1, sl.len - 32 * (i0 + i), mask_tag);
      } else {
        if (i > 0) {
          dsv(sa, ds, (i - 1) & 1);
          grad(ds, (st + 3) & 3);
        }
        first(sa, st, role_tag);
      }
      next.store(smem + ((st + 2) & 3) * STAGE, tid);
      __syncthreads();
    };
    int i = 0;
    for (; i + 3 < n_full; i += 4) {
      step(i, 0, sa, sb, std::false_type{});
      step(i + 1, 1, sb, sa, std::false_type{});
      step(i + 2, 2, sa, sb, std::false_type{});
      step(i + 3, 3, sb, sa, std::false_type{});
    }
    for (; i < nsteps; ++i) {
      step(i, i & 3, sa, sb, std::true_type{});
      if constexpr (!RB_) sa = sb;
    }
    if (RB_ && nsteps > 0) {
      dsv(sa, ds, (nsteps - 1) & 1);
      grad(ds, (nsteps - 1) & 3);
    }
  };
  for (;;) {
#pragma unroll
    for (int u = 0; u < DT; ++u) dq[u] = f32x16{};
    if (role_b) run(std::true_type{});
    else run(std::false_type{});
    if (!LIFT) break;
    const bool again = role_b && live && next_lift(row_overflowed(dq, l32), exponent, lift);
    if (again) lifts[pr][l32] = (float)lift;  // A has read it
    if (!__syncthreads_or(again)) break;
    nm = live ? lifts[pr][l32] - m : 0.0f;
    next.clear(smem + 3 * STAGE, tid);
    next.load(krs, vrs, (uint32_t)i0 * kb, (uint32_t)i0 * vb);
    next.store(smem, tid);
    next.load(krs, vrs, (uint32_t)(i0 + 1) * kb, (uint32_t)(i0 + 1) * vb);
    next.store(smem + STAGE, tid);
    __syncthreads();
  }
  if (!live || !role_b) return;
  const float unlift = LIFT ? unlift_of(lift) : 1.0f;
  if (p.splits > 1)
    store_row_t<float, D>(p.part + (((int64_t)slice * p.splits + split) * rows + row) * D, dq, unlift, h2);
  else
    store_row_t<T, D>((T*)p.out + r.at(p.sout), dq, p.scale * unlift, h2);
}

}  // namespace

int launch_cross_dq(const CrossParams& p, int D, int dtype, hipStream_t st) {
  unsigned blocks;
  const dim3 block(cross_dq_threads(D));
  if (int rc = cross_grid(p.slices(), (int64_t)p.nblk * p.splits, (int)block.x, &blocks)) return rc;
  const dim3 grid(blocks);
  switch (D) {
#define TATTN_DQ(D_)                                                           \
  case D_:                                                                     \
    if (dtype == 0) cross_dq_kernel<f16, D_, 4, 2><<<grid, block, 0, st>>>(p); \
    else cross_dq_kernel<bf16, D_, 4, 2><<<grid, block, 0, st>>>(p);           \
    break;
    TATTN_DQ(16) TATTN_DQ(32) TATTN_DQ(64)
#undef TATTN_DQ
    case 128:
      if (dtype == 0) cross_dq_pair_kernel<f16, 128><<<grid, block, 0, st>>>(p);
      else cross_dq_pair_kernel<bf16, 128><<<grid, block, 0, st>>>(p);
      break;
    default: return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %d", D);
  }
  return check_launch("tattn_cross_bwd");
}

}  // namespace tattn
