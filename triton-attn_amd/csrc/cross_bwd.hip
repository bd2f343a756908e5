// Attention over keys of another length, 16-bit backward, on gfx950.
//
//   P = 2^(S c - M),  dS = P (dP - delta),  dP = dO V^T,  delta = rowsum(dO * O)
//   dQ = dS K scale,  dK = dS^T Q scale,  dV = P^T dO,  the last two summed over the query heads of a key head
//
// Two kernels, no atomics: `cross_dq_kernel` (cross_dq.hip) owns rows and walks the keys (it also computes delta),
// `cross_dkdv_kernel` owns keys and walks the rows of all heads. A wave keeps 32 rows (keys) in registers. Per step of 32 keys
// (rows) it issues the first products of the next step and the second products of the one before, none of which wait for the
// step's exponentials. Tiles come through registers into a ring of four LDS stages, one barrier per step. Where there are too
// few blocks to fill the chip, the walked dimension is cut into parts, whose float32 sums `cross_sum_kernel` adds in order.
//
// Keys at or past len are fetched as zeros and get zero gradients.
//
// Roundings: P and dS are rounded to the element type as operands of the second products, everything else is float32. In
// float16 dS is scaled by a power of two first: up where dO is small (small_gradient_lift), down where dS would pass the type.
//
// Bound by the issue of matrix and vector instructions. Traced, dK / dV: 4 x 16 x 4,096 over 4,096 x 64 fp16 581 us (946 TF of its four
// products), 2 x 16 x 4,096 over 4,096 x 128 bf16, one wave on a SIMD, 560 (982).
#include <algorithm>
#include <type_traits>

#include "cross_bwd.h"

namespace tattn {
namespace {

// ---- dK / dV -------------------------------------------------------------------------------------
// What dS of a block of keys is scaled by, 2^by, the same for the workgroup: up by the largest norm of the slice's rows of dO, and up or
// down so far that the largest |dS| stays finite, |dS| <= |dO| |v| + |delta|. Values that are not finite ask for nothing.
template <int NW, typename V8, int N>
__device__ __forceinline__ int keys_lift(const CrossParams& p, int slice, const V8 (&v)[N], int wu, int lane, uint32_t (&share)[NW]) {
  const u32x2* norms = reinterpret_cast<const u32x2*>(p.norms) + (int64_t)slice * p.nblk;
  u32x2 top = u32x2{};
  for (int i = lane; i < p.nblk; i += 64) {
    const u32x2 a = norms[i];
    top[0] = max(top[0], a[0]);
    top[1] = max(top[1], a[1]);
  }
  const int row = norm_exponent(max_wave(top[0]));
  float norm = 0.0f;
#pragma unroll
  for (int s = 0; s < N; ++s) norm += chunk_dot(v[s], v[s]);
  share[wu] = max_wave(__builtin_bit_cast(uint32_t, sum_halves(norm)));
  __syncthreads();
  uint32_t most = share[0];
#pragma unroll
  for (int k = 1; k < NW; ++k) most = max(most, share[k]);
  const int key = norm_exponent(uniform32(most)), delta = (int)(max_wave(top[1]) >> 23) - 127;
  // |dS| < 2^(row + key + 2) + 2^(delta + 1)
  return row >= 30 || key >= 30 || delta >= 127 ? 0 : min(small_gradient_lift(row, 15), min(12 - row - key, 13 - delta));
}

template <typename T, int D, int NW, int OCC>
__global__ __launch_bounds__(NW * 64, OCC) void cross_dkdv_kernel(const CrossParams p) {
  using V8 = typename H16<T>::V8;
  using B = BwdPipe<D>;
  constexpr int NSD = B::NSD, DT = B::DT, STAGE = B::DKDV_STAGE, KEYS = 32 * NW;
  constexpr bool LIFT = std::is_same_v<T, f16>;
  __shared__ __attribute__((aligned(16))) char smem[B::NST * STAGE];
  __shared__ uint32_t share[NW];

  const int tid = threadIdx.x;
  const int lane = tid & 63, h2 = lane >> 5, l32 = lane & 31;
  const int wu = (int)uniform32((uint32_t)(tid >> 6));
  const float c = p.c;
  int slice, item;
  if (!cross_coord(p, p.kblk * p.parts, slice, item)) return;
  const int kbi = item / p.parts, part = item % p.parts;
  const CrossSlice sl(p, slice);
  const int kw0 = KEYS * kbi + 32 * wu, key = kw0 + l32;
  const bool idle = kw0 >= sl.len;
  // The rows' tiles, head after head.
  const int nq = (p.N + 31) >> 5, total = KEYS * kbi < sl.len ? nq * p.G : 0;
  const int i0 = (int)((int64_t)total * part / p.parts), i1 = (int)((int64_t)total * (part + 1) / p.parts);
  const int nsteps = i1 - i0;

  const int64_t row0 = (int64_t)slice * p.G * p.N;
  const T* qbase = (const T*)p.q + sl.zs * p.sq[0] + (int64_t)sl.hk * p.G * p.sq[1];
  const T* obase = (const T*)p.dout + sl.zs * p.sd[0] + (int64_t)sl.hk * p.G * p.sd[1];
  const uint32_t qbytes = (uint32_t)slice_bytes(p.N, p.sq[2], D), obytes = (uint32_t)slice_bytes(p.N, p.sd[2], D);
  const uint32_t qb = uniform32((uint32_t)(p.sq[2] * 64)), ob = uniform32((uint32_t)(p.sd[2] * 64));
  StepRows<D, NW * 64> next, second;
  next.init(tid, p.sq[2], p.sd[2]);
  second = next;
  const bool md_loader = tid < 64;  // lanes 0-31 of wave 0 stage M, lanes 32-63 -delta
  float md_next, md_second;
  // The tile to be loaded next; past the last one rows are read as zeros.
  int fg = i0 / nq, fq = i0 % nq, left = nsteps;
  auto load = [&](StepRows<D, NW * 64>& to, float& md) __attribute__((always_inline)) {
    const bool more = left > 0;
    const __amdgpu_buffer_rsrc_t qrs = slice_rsrc(qbase + fg * p.sq[1], more ? qbytes : 0);
    const __amdgpu_buffer_rsrc_t ors = slice_rsrc(obase + fg * p.sd[1], more ? obytes : 0);
    to.load(qrs, ors, (uint32_t)fq * qb, (uint32_t)fq * ob);
    const int64_t head = row0 + (int64_t)fg * p.N;
    const __amdgpu_buffer_rsrc_t mrs = slice_rsrc(p.m + head, more ? (uint64_t)p.N * 4 : 0);
    const __amdgpu_buffer_rsrc_t drs = slice_rsrc(p.delta + head, more ? (uint64_t)p.N * 4 : 0);
    const int at = (32 * fq + l32) * 4;
    const uint32_t a = __builtin_amdgcn_raw_buffer_load_b32(mrs, at, 0, 0), b = __builtin_amdgcn_raw_buffer_load_b32(drs, at, 0, 0);
    md = __builtin_bit_cast(float, h2 ? b : a);
    --left;
    if (++fq == nq) fq = 0, ++fg;
  };
  load(next, md_next);
  load(second, md_second);

  V8 kop[NSD], vop[NSD];
  {
    const T* ks = (const T*)p.k + sl.zs * p.sk[0] + sl.hk * p.sk[1] + (int64_t)(key < sl.len ? key : 0) * p.sk[2] + 8 * h2;
    const T* vs = (const T*)p.v + sl.zs * p.sv[0] + sl.hk * p.sv[1] + (int64_t)(key < sl.len ? key : 0) * p.sv[2] + 8 * h2;
#pragma unroll
    for (int s = 0; s < NSD; ++s) {
      const V8 a = *reinterpret_cast<const V8*>(ks + 16 * s), b = *reinterpret_cast<const V8*>(vs + 16 * s);
      kop[s] = key < sl.len ? a : V8{};
      vop[s] = key < sl.len ? b : V8{};
    }
  }
  // Up, P is scaled with dS, through M. Down, dS alone, through V and delta: P would lose its precision. V then falls below the
  // normal range only by as much as |dO| is large: dP is off by 2^(row - 32) |dO| |v| or less (row as in keys_lift, 19 at most).
  int by = 0;
  if constexpr (LIFT) {
    by = keys_lift<NW>(p, slice, vop, wu, lane, share);
    if (by < 0) {
      const float down = unlift_of(-by);
#pragma unroll
      for (int s = 0; s < NSD; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) vop[s][i] = (T)((float)vop[s][i] * down);
    }
  }
  const float lift = h2 ? 0.0f : (float)max(by, 0), down = h2 ? unlift_of(max(-by, 0)) : 1.0f;
  auto store = [&](const StepRows<D, NW * 64>& from, float md, int st) __attribute__((always_inline)) {
    from.store(smem + st * STAGE, tid);
    if (md_loader) *reinterpret_cast<float*>(smem + st * STAGE + 2 * B::TILE + 4 * tid) = __builtin_fmaf(md, down, -lift);
  };
  CrossOp<D> at;
  at.init(lane);
  const int mo = 2 * B::TILE + 32 * h2;  // M of queries 8 h2 .. (bytes); -delta at +128
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int u = 0; u < DT; ++u) dk[u] = dv[u] = f32x16{};

  auto first = [&](f32x16& s, f32x16& dp, int st) __attribute__((always_inline)) {
    const char* base = smem + st * STAGE;
    const TATTN_LDS char* nd = (const TATTN_LDS char*)base + mo + 128;
    s = f32x16{};
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const f32x4 x = *reinterpret_cast<const TATTN_LDS f32x4*>(nd + 64 * (a >> 1) + 16 * (a & 1));
#pragma unroll
      for (int e = 0; e < 4; ++e) dp[4 * a + e] = x[e];
    }
#pragma unroll
    for (int sd = 0; sd < NSD; ++sd) {
      s = Elt<T>::mfma(lds8<T>(base + at.nat[sd]), kop[sd], s);
      dp = Elt<T>::mfma(lds8<T>(base + B::TILE + at.nat[sd]), vop[sd], dp);
    }
  };
  auto grad = [&](const V8 (&pp)[2], const V8 (&ds)[2], int st) __attribute__((always_inline)) {
    const char* base = smem + st * STAGE;
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int u = 0; u < DT; ++u) {
        dv[u] = Elt<T>::mfma(pp[g], at.template tr<T>(base + B::TILE, g, u, lane), dv[u]);
        dk[u] = Elt<T>::mfma(ds[g], at.template tr<T>(base, g, u, lane), dk[u]);
      }
  };
  auto probs = [&](const f32x16& s, const f32x16& dp, V8 (&pp)[2], V8 (&ds)[2], int st) __attribute__((always_inline)) {
    const TATTN_LDS char* base = (const TATTN_LDS char*)smem + st * STAGE + mo;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const f32x4 m = *reinterpret_cast<const TATTN_LDS f32x4*>(base + 64 * (a >> 1) + 16 * (a & 1));
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = fast_exp2(__builtin_fmaf(s[4 * a + e], c, -m[e]));
        y[e] = x[e] * dp[4 * a + e];
      }
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const auto ph = H16<T>::pack(x[e], x[e + 1]), dh = H16<T>::pack(y[e], y[e + 1]);
        pp[a >> 1][4 * (a & 1) + e] = ph[0];
        pp[a >> 1][4 * (a & 1) + e + 1] = ph[1];
        ds[a >> 1][4 * (a & 1) + e] = dh[0];
        ds[a >> 1][4 * (a & 1) + e + 1] = dh[1];
      }
    }
  };

  next.clear(smem + 3 * STAGE, tid);  // read by the first step together with all-zero P and dS
  store(next, md_next, 0);
  store(second, md_second, 1);
  __syncthreads();
  f32x16 sa, da, sb, db;
  V8 pa[2] = {}, ea[2] = {}, pb[2], eb[2];
  if (nsteps > 0 && !idle) first(sa, da, 0);
  auto step = [&](int st, f32x16& s0, f32x16& d0, f32x16& s1, f32x16& d1, const V8 (&p0)[2], const V8 (&e0)[2], V8 (&p1)[2],
                  V8 (&e1)[2]) __attribute__((always_inline)) {
    load(next, md_next);
    if (!idle) {
      first(s1, d1, (st + 1) & 3);
      grad(p0, e0, (st + 3) & 3);
      probs(s0, d0, p1, e1, st);
    }
    store(next, md_next, (st + 2) & 3);
    __syncthreads();
  };
  int i = 0;
  for (; i + 3 < nsteps; i += 4) {
    step(0, sa, da, sb, db, pa, ea, pb, eb);
    step(1, sb, db, sa, da, pb, eb, pa, ea);
    step(2, sa, da, sb, db, pa, ea, pb, eb);
    step(3, sb, db, sa, da, pb, eb, pa, ea);
  }
  for (; i < nsteps; ++i) {
    step(i & 3, sa, da, sb, db, pa, ea, pb, eb);
    sa = sb;
    da = db;
#pragma unroll
    for (int a = 0; a < 2; ++a) pa[a] = pb[a], ea[a] = eb[a];
  }
  if (nsteps > 0 && !idle) grad(pa, ea, (nsteps - 1) & 3);

  // C register r of a lane: key 8 (r / 4) + 4 h2 + r % 4 of the tile, column 32 u + l32. Keys past len get zeros: what
  // their lanes hold is of no meaning. Parts go out as float32 sums, tiles in rows through LDS, free after the barrier.
  const float unlift = unlift_of(by), unlift_v = unlift_of(max(by, 0));
  if (p.parts > 1) {
    float* dst = p.kpart + (((int64_t)slice * p.kblk + kbi) * p.parts + part) * (2 * KEYS * D) + 32 * wu * D;
#pragma unroll
    for (int u = 0; u < DT; ++u)
#pragma unroll
      for (int g = 0; g < 16; ++g) {
        const int in = 8 * (g >> 2) + 4 * h2 + (g & 3), d = 32 * u + l32;
        if (d >= D) continue;
        const bool seen = kw0 + in < sl.len;
        dst[in * D + d] = seen ? dk[u][g] * unlift : 0.0f;
        dst[KEYS * D + in * D + d] = seen ? dv[u][g] * unlift_v : 0.0f;
      }
    return;
  }
  __syncthreads();
  constexpr int RB = B::RB, CPR = D / 8;
  static_assert(NW * 32 * RB <= B::NST * STAGE, "store blocks fit the ring");
  char* wb = smem + wu * 32 * RB;
  auto rows_out = [&](const f32x16 (&a)[DT], float mul, T* dst, int64_t stride) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < DT; ++u)
      if (32 * u + l32 < D) {
#pragma unroll
        for (int g = 0; g < 16; ++g) {
          const int in = 8 * (g >> 2) + 4 * h2 + (g & 3);
          *reinterpret_cast<TATTN_LDS T*>((TATTN_LDS char*)wb + in * RB + (32 * u + l32) * 2) = (T)(kw0 + in < sl.len ? a[u][g] * mul : 0.0f);
        }
      }
#pragma unroll
    for (int i = 0; i < (32 * CPR + 63) / 64; ++i) {
      const int j = 64 * i + lane, in = j / CPR, cc = j % CPR;
      if (in >= 32) break;
      const u32x4 v = *reinterpret_cast<const TATTN_LDS u32x4*>((const TATTN_LDS char*)wb + in * RB + 16 * cc);
      if (kw0 + in < p.S) st16(dst + (int64_t)(kw0 + in) * stride + 8 * cc, v);
    }
  };
  rows_out(dk, p.scale * unlift, (T*)p.dk + sl.zs * p.sdk[0] + sl.hk * p.sdk[1], p.sdk[2]);
  rows_out(dv, unlift_v, (T*)p.dv + sl.zs * p.sdv[0] + sl.hk * p.sdv[1], p.sdv[2]);
}

// ---- sums of parts -------------------------------------------------------------------------------
// dQ (which = 0), or dK and dV: four consecutive columns a thread.
template <typename T, int D, bool KEYS>
__global__ __launch_bounds__(256) void cross_sum_kernel(const CrossParams p, int block) {
  typedef T V4 __attribute__((ext_vector_type(4)));
  const int64_t i = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x), cell = i / D;
  const int d = (int)(i % D);
  f32x4 x = f32x4{};
  T* dst;
  float mul = p.scale;
  if constexpr (KEYS) {  // cells: [slice][key block][dK, dV][key]
    const int64_t kb = cell / (2 * block);
    if (kb >= (int64_t)p.Zs * p.Hk * p.kblk) return;
    const int in = (int)(cell % (2 * block)), which = in / block, key = (int)(kb % p.kblk) * block + in % block;
    const int slice = (int)(kb / p.kblk), zs = slice / p.Hk, hk = slice % p.Hk;
    if (key >= p.S) return;
    const float* src = p.kpart + (kb * p.parts * 2 * block + in) * D + d;
#pragma unroll 4
    for (int s = 0; s < p.parts; ++s) x += *reinterpret_cast<const f32x4*>(src + (int64_t)s * 2 * block * D);
    dst = which ? (T*)p.dv + zs * p.sdv[0] + hk * p.sdv[1] + key * p.sdv[2] : (T*)p.dk + zs * p.sdk[0] + hk * p.sdk[1] + key * p.sdk[2];
    if (which) mul = 1.0f;
  } else {  // cells: [slice][row]
    const int rows = p.G * p.N;
    const int64_t slice = cell / rows;
    if (slice >= (int64_t)p.Zs * p.Hk) return;
    const int row = (int)(cell % rows), g = row / p.N;
    const float* src = p.part + (slice * p.splits * rows + row) * D + d;
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) x += *reinterpret_cast<const f32x4*>(src + (int64_t)s * rows * D);
    dst = (T*)p.out + slice / p.Hk * p.sout[0] + (slice % p.Hk * p.G + g) * p.sout[1] + (int64_t)(row % p.N) * p.sout[2];
  }
  V4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (T)(x[e] * mul);
  *reinterpret_cast<V4*>(dst + d) = y;
}

template <typename T, int D>
int sum_d(const CrossParams& p, bool keys, int block, hipStream_t st) {
  const int64_t blocks = cross_sum_blocks(p, D, keys, block);
  if (int rc = check_grid(blocks, 256)) return rc;
  if (keys) cross_sum_kernel<T, D, true><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(p, block);
  else cross_sum_kernel<T, D, false><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(p, 0);
  return check_launch("tattn_cross_bwd");
}

// ---- launch --------------------------------------------------------------------------------------
constexpr int kRowTiles = 4;  // row tiles of a dQ workgroup
// Key tiles of a dK / dV workgroup. Eight take 145 us where four take 121 (whole backward, 16 x 8 x 4,096 over 77 x 64), 184 for 175
// (8 x 16 x 1,024 over 375 to 1,500 x 64), 1,012 for 995 (4 x 16 x 4,096 over 4,096 x 64).
constexpr int kKeyTiles = 4;
constexpr int bwd_occ(int D) { return D == 128 ? 1 : 2; }

// Rows that lie at one stride, whatever head they belong to, are walked as one head's: no tile holds the end of a head. (Not where
// heads share an address: rows past the last would be read as it.)
CrossParams walked(const CrossParams& p, int D) {
  CrossParams w = p;
  const int64_t rows = (int64_t)p.G * p.N, sq = p.N == 1 ? p.sq[1] : p.sq[2], sd = p.N == 1 ? p.sd[1] : p.sd[2];
  const bool one = p.G > 1 && p.sq[1] == p.N * sq && p.sd[1] == p.N * sd && sq >= D && sd >= D && rows < (1 << 30) &&
                   (rows + 256) * std::max(sq, sd) * 2 < 0x7fffff00ll;
  if (!one) return w;
  w.N = (int32_t)rows;
  w.G = 1;
  w.H = p.Hk;
  w.sq[1] = rows * sq;
  w.sd[1] = rows * sd;
  w.sq[2] = sq;
  w.sd[2] = sd;
  return w;
}

template <typename T, int D>
int bwd_d(const CrossParams& p, hipStream_t st) {
  unsigned blocks;
  int rc;
  if (cross_short(p, D, std::is_same_v<T, f16> ? 0 : 2, true)) return launch_cross_short(p, D, std::is_same_v<T, f16> ? 0 : 2, true, st);
  if ((rc = launch_cross_dq(p, D, std::is_same_v<T, f16> ? 0 : 2, st))) return rc;
  if (p.splits > 1 && (rc = sum_d<T, D>(p, false, 0, st))) return rc;
  if ((rc = cross_grid(p.slices(), (int64_t)p.kblk * p.parts, 64 * kKeyTiles, &blocks))) return rc;
  cross_dkdv_kernel<T, D, kKeyTiles, bwd_occ(D)><<<dim3(blocks), dim3(64 * kKeyTiles), 0, st>>>(walked(p, D));
  if ((rc = check_launch("tattn_cross_bwd")) || p.parts == 1) return rc;
  return sum_d<T, D>(p, true, 32 * kKeyTiles, st);
}

}  // namespace

// Blocks are cut into parts while all of them together leave half of the chip's places empty (two workgroups a CU, one at head dim
// 128, dQ in float32 of up to two row tiles four times as many of one wave); a part has at least 8 tiles of keys or 16 of rows, in
// float32, where a tile takes eight times as long, three.
int cross_bwd_plan(CrossParams& p, int D, int dtype) {
  unsigned launched;
  int rc;
  const int64_t slices = p.slices(), places = 256 * bwd_occ(D), keys = 32 * kKeyTiles;
  if (cross_short(p, D, dtype, true)) {  // row tiles of a slice in as many parts as the chip holds at once, two a wave at least
    const int nt = (p.S + 31) / 32;
    p.nblk = p.splits = p.kblk = 1;
    p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(256 * cross_short_occ(D, nt) / slices, (p.rows() + 31) / 32 / 8));
    if ((rc = cross_grid(slices, p.parts, 256, &launched)) || p.parts == 1) return rc;
    return check_grid(cross_sum_blocks(p, D, true, 32 * nt), 256);
  }
  p.waves = dtype == 1 && p.rows() <= 64 ? 1 : kRowTiles;
  p.nblk = (int)((p.rows() + 32 * p.waves - 1) / (32 * p.waves));
  p.kblk = (int)((p.S + keys - 1) / keys);
  const int64_t rt = (int64_t)p.G * ((p.N + 31) / 32), kt = ((int64_t)p.S + 31) / 32;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(places * kRowTiles / p.waves / (slices * p.nblk), kt / (dtype == 1 ? 3 : 8)));
  p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(places / (slices * p.kblk), rt / (dtype == 1 ? 3 : 16)));
  if ((rc = cross_grid(slices, (int64_t)p.nblk * p.splits, dtype == 1 ? 64 * p.waves : cross_dq_threads(D), &launched)) ||
      (rc = cross_grid(slices, (int64_t)p.kblk * p.parts, 256, &launched)) ||
      (p.splits > 1 && (rc = check_grid(cross_sum_blocks(p, D, false, 0), 256))))
    return rc;
  return p.parts > 1 ? check_grid(cross_sum_blocks(p, D, true, keys), 256) : TATTN_OK;
}

namespace {
int64_t even(int64_t x) { return (x + 3) / 4 * 4; }
}  // namespace

int64_t cross_bwd_floats(const CrossParams& p, int D, int dtype) {
  const int64_t rows = p.slices() * p.rows();
  if (cross_short(p, D, dtype, true)) return p.parts > 1 ? p.slices() * p.parts * 2 * ((p.S + 31) / 32 * 32) * D : 4;
  return even(rows) + (dtype == 0 ? even(2 * p.slices() * p.nblk) : 0) + (p.splits > 1 ? rows * p.splits * D : 0) +
         (p.parts > 1 ? p.slices() * p.kblk * p.parts * 2 * 32 * kKeyTiles * D : 0);
}

void cross_bwd_workspace(CrossParams& p, int D, int dtype, float* work) {
  const int64_t rows = p.slices() * p.rows();
  if (cross_short(p, D, dtype, true)) {
    p.kpart = work;
    return;
  }
  p.delta = work;
  p.norms = p.delta + even(rows);
  p.part = p.norms + (dtype == 0 ? even(2 * p.slices() * p.nblk) : 0);
  p.kpart = p.part + (p.splits > 1 ? rows * p.splits * D : 0);
}

int launch_cross_bwd(const CrossParams& p, int D, int dtype, hipStream_t st) {
  switch (D) {
    case 16: return dtype == 0 ? bwd_d<f16, 16>(p, st) : bwd_d<bf16, 16>(p, st);
    case 32: return dtype == 0 ? bwd_d<f16, 32>(p, st) : bwd_d<bf16, 32>(p, st);
    case 64: return dtype == 0 ? bwd_d<f16, 64>(p, st) : bwd_d<bf16, 64>(p, st);
    case 128: return dtype == 0 ? bwd_d<f16, 128>(p, st) : bwd_d<bf16, 128>(p, st);
  }
  return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %d", D);
}

int launch_cross_sum(const CrossParams& p, int D, int dtype, bool keys, int block, hipStream_t st) {
#define TATTN_SUM(D_)                                              \
  case D_:                                                         \
    return dtype == 0   ? sum_d<f16, D_>(p, keys, block, st)       \
           : dtype == 2 ? sum_d<bf16, D_>(p, keys, block, st)      \
                        : sum_d<float, D_>(p, keys, block, st);
  switch (D) { TATTN_SUM(16) TATTN_SUM(32) TATTN_SUM(64) TATTN_SUM(128) }
#undef TATTN_SUM
  return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %d", D);
}

}  // namespace tattn
