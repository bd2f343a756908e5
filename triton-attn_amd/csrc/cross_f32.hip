// Attention over keys of another length in float32, forward and backward, on gfx950's float32 matrix instruction
// (f32_tiles.h). The rows, keys and parts of cross.h; four waves of a workgroup own a 32-row tile each (32 keys for dK / dV) and
// walk the tiles of the other dimension, staged one at a time through registers into LDS, the next one's loads in flight meanwhile. Up
// to two row tiles are a workgroup of one wave each, over more parts of the keys: all SIMDs then have a tile to work on.
// Nothing is rounded below float32.
//
// Bound by the matrix instruction, 64 cycles for 32 x 32 x 2 (154 TF as a large product reaches it), and by the other vector
// work, which does not overlap it even where a SIMD has two waves. Traced, 4 x 16 x 1,024 over 1,024 x 64: forward 149 us (116
// TF), dQ 208 (124), dK / dV 272 (126; with one wave on a SIMD, as the compiler would have it for 276 registers, a fifth more).
// 4 x 8 x 1,024 over 1,024 x 128, one wave on a SIMD: 154 (112), 215 (120) and 301 (114). One query of each of 16 x 8 heads
// over 8,192 x 128, whole calls: forward 264 us (4.1 TB/s; 607 with the workgroups of four), with gradients 1,304 (2,164).
#include "cross.h"
#include "f32_tiles.h"

namespace tattn {
namespace {

// A 32-row tile on its way from memory to LDS, by NT threads; rows past the buffer's end are zeros. Offsets of 32 bits, one addition a
// load: with 64-bit addresses and a check of each row the loads are half of a step's vector instructions (157, 216 and 289 us at 64).
template <int D, int NT>
struct RowTile32 {
  using C = F32<D>;
  static constexpr int CPT = (32 * C::CPR + NT - 1) / NT;
  uint32_t off[CPT];
  u32x4 x[CPT];
  __device__ __forceinline__ void init(int64_t stride) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int ch = threadIdx.x + NT * i;
      off[i] = (uint32_t)(ch / C::CPR * stride * 4 + 16 * (ch % C::CPR));
    }
  }
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t from) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) x[i] = rsrc_load(rs, off[i] + from);
  }
  __device__ __forceinline__ void store(float* lds) const {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int ch = threadIdx.x + NT * i, row = ch / C::CPR;
      if (32 * C::CPR % NT == 0 || row < 32)
        *reinterpret_cast<TATTN_LDS u32x4*>((TATTN_LDS float*)lds + row * C::LD + 4 * (ch % C::CPR)) = x[i];
    }
  }
};
template <int D>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows32_rsrc(const void* base, int64_t off, int64_t rows, int64_t stride) {
  return slice_rsrc((const float*)base + off, rows > 0 ? slice_bytes(rows, 2 * stride, 2 * D) : 0);
}

// The rows of a workgroup of NW row tiles and the lane's, and the part of the keys that is walked.
template <int NW>
struct CrossRows32 {
  int slice, blk, split, row, rows, i0, i1;
  bool ok, live;
  __device__ __forceinline__ CrossRows32(const CrossParams& p, int w, int l32) {
    ok = cross_coord(p, p.nblk * p.splits, slice, blk);
    if (!ok) return;
    split = blk % p.splits;
    blk /= p.splits;
    rows = p.B * p.G * p.N;
    row = 32 * (NW * blk + w) + l32;
    live = row < rows;
    const int tiles = (CrossSlice(p, slice).len + 31) >> 5;
    i0 = (int)((int64_t)tiles * split / p.splits);
    i1 = (int)((int64_t)tiles * (split + 1) / p.splits);
  }
};

template <int D, int NW, int OCC>
__global__ __launch_bounds__(64 * NW, OCC) void cross_fwd_f32_kernel(const CrossParams p) {
  using C = F32<D>;
  __shared__ __attribute__((aligned(16))) float ks[32 * C::LD], vs[32 * C::LD];
  const int lane = threadIdx.x & 63, h2 = lane >> 5, l32 = lane & 31;
  const CrossRows32<NW> b(p, (int)uniform32(threadIdx.x >> 6), l32);
  if (!b.ok) return;
  const CrossSlice sl(p, b.slice);
  const CrossRow r(p, sl, b.live ? b.row : 0);
  const float c = p.c, hidden = hidden_score(c);
  const __amdgpu_buffer_rsrc_t krs = rows32_rsrc<D>(p.k, sl.zs * p.sk[0] + sl.hk * p.sk[1], sl.len, p.sk[2]);
  const __amdgpu_buffer_rsrc_t vrs = rows32_rsrc<D>(p.v, sl.zs * p.sv[0] + sl.hk * p.sv[1], sl.len, p.sv[2]);
  const uint32_t kb = uniform32((uint32_t)(p.sk[2] * 128)), vb = uniform32((uint32_t)(p.sv[2] * 128));
  float q[C::H];
  own_row<D>((const float*)p.q + r.at(p.sq), b.live, h2, q);
  float mrow = kNoMax, lrow = 0.0f;
  f32x16 acc[C::DT];
#pragma unroll
  for (int u = 0; u < C::DT; ++u) acc[u] = f32x16{};
  RowTile32<D, 64 * NW> kn, vn;
  kn.init(p.sk[2]);
  vn.init(p.sv[2]);
  auto load = [&](int t) {
    kn.load(krs, (uint32_t)t * kb);
    vn.load(vrs, (uint32_t)t * vb);
  };
  if (b.i0 < b.i1) load(b.i0);
  for (int t = b.i0; t < b.i1; ++t) {
    __syncthreads();
    kn.store(ks);
    vn.store(vs);
    __syncthreads();
    if (t + 1 < b.i1) load(t + 1);
    f32x16 s = rows_dot<D>(ks, q, f32x16{}, l32, h2);
    if (32 * t + 32 > sl.len) hide_after(s, sl.len - 1, t, h2, hidden);
    const float mnew = moved_max(s, c, mrow), alpha = fast_exp2(mrow - mnew);
    if (__builtin_amdgcn_ballot_w64(mnew != mrow)) {
#pragma unroll
      for (int u = 0; u < C::DT; ++u) acc[u] *= alpha;
    }
    mrow = mnew;
    float ps = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = fast_exp2(__builtin_fmaf(s[i], c, -mnew));
      ps += s[i];
    }
    lrow = lrow * alpha + ps;
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int u = 0; u < C::DT; ++u) acc[u] = mfma2(cell<D>(vs, i, 32 * u + l32, h2), s[i], acc[u]);
  }
  const float lt = sum_halves(lrow);
  if (!b.live) return;
  if (p.splits > 1) {
    const int64_t prow = ((int64_t)b.slice * p.splits + b.split) * b.rows + b.row;
    store_row_t<float, D>(p.part + prow * D, acc, 1.0f, h2);
    if (h2 == 0) {
      float* ml = p.part + (int64_t)p.Zs * p.Hk * p.splits * b.rows * D + prow * 2;
      ml[0] = mrow;
      ml[1] = lt;
    }
    return;
  }
  store_row_t<float, D>((float*)p.out + r.at(p.sout), acc, lt == 0.0f ? 0.0f : 1.0f / lt, h2);  // no keys: zeros
  if (h2 == 0 && p.m) p.m[r.index(p)] = mrow + __log2f(lt);
}

template <int D, int NW, int OCC>
__global__ __launch_bounds__(64 * NW, OCC) void cross_dq_f32_kernel(const CrossParams p) {
  using C = F32<D>;
  __shared__ __attribute__((aligned(16))) float ks[32 * C::LD], vs[32 * C::LD];
  const int lane = threadIdx.x & 63, h2 = lane >> 5, l32 = lane & 31;
  const CrossRows32<NW> b(p, (int)uniform32(threadIdx.x >> 6), l32);
  if (!b.ok) return;
  const CrossSlice sl(p, b.slice);
  const CrossRow r(p, sl, b.live ? b.row : 0);
  const float c = p.c, hidden = hidden_score(c);
  const __amdgpu_buffer_rsrc_t krs = rows32_rsrc<D>(p.k, sl.zs * p.sk[0] + sl.hk * p.sk[1], sl.len, p.sk[2]);
  const __amdgpu_buffer_rsrc_t vrs = rows32_rsrc<D>(p.v, sl.zs * p.sv[0] + sl.hk * p.sv[1], sl.len, p.sv[2]);
  const uint32_t kb = uniform32((uint32_t)(p.sk[2] * 128)), vb = uniform32((uint32_t)(p.sv[2] * 128));
  float q[C::H], go[C::H];
  own_row<D>((const float*)p.q + r.at(p.sq), b.live, h2, q);
  own_row<D>((const float*)p.dout + r.at(p.sd), b.live, h2, go);
  float dl = 0.0f;
  {
    const float* o = (const float*)p.o + r.at(p.so) + h2 * C::H;
#pragma unroll
    for (int j = 0; j < C::H; ++j) dl = __builtin_fmaf(o[j], go[j], dl);
    dl = b.live ? sum_halves(dl) : 0.0f;
    if (b.live && h2 == 0 && b.split == 0) p.delta[(int64_t)b.slice * b.rows + b.row] = -dl;
  }
  const float nm = b.live ? -p.m[r.index(p)] : 0.0f;
  f32x16 dq[C::DT];
#pragma unroll
  for (int u = 0; u < C::DT; ++u) dq[u] = f32x16{};
  RowTile32<D, 64 * NW> kn, vn;
  kn.init(p.sk[2]);
  vn.init(p.sv[2]);
  auto load = [&](int t) {
    kn.load(krs, (uint32_t)t * kb);
    vn.load(vrs, (uint32_t)t * vb);
  };
  if (b.i0 < b.i1) load(b.i0);
  for (int t = b.i0; t < b.i1; ++t) {
    __syncthreads();
    kn.store(ks);
    vn.store(vs);
    __syncthreads();
    if (t + 1 < b.i1) load(t + 1);
    f32x16 s = rows_dot<D>(ks, q, f32x16{}, l32, h2), dp;
#pragma unroll
    for (int i = 0; i < 16; ++i) dp[i] = -dl;
    dp = rows_dot<D>(vs, go, dp, l32, h2);
    if (32 * t + 32 > sl.len) hide_after(s, sl.len - 1, t, h2, hidden);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = fast_exp2(__builtin_fmaf(s[i], c, nm)) * dp[i];
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int u = 0; u < C::DT; ++u) dq[u] = mfma2(cell<D>(ks, i, 32 * u + l32, h2), s[i], dq[u]);
  }
  if (!b.live) return;
  if (p.splits > 1)
    store_row_t<float, D>(p.part + (((int64_t)b.slice * p.splits + b.split) * b.rows + b.row) * D, dq, 1.0f, h2);
  else
    store_row_t<float, D>((float*)p.out + r.at(p.sout), dq, p.scale, h2);
}

// A workgroup owns 128 keys and walks the rows' tiles, head after head of the group.
template <int D, int OCC>
__global__ __launch_bounds__(256, OCC) void cross_dkdv_f32_kernel(const CrossParams p) {
  using C = F32<D>;
  __shared__ __attribute__((aligned(16))) float qs[32 * C::LD], gs[32 * C::LD];
  __shared__ __attribute__((aligned(16))) float md[2][32];  // M, -delta
  const int tid = threadIdx.x, lane = tid & 63, h2 = lane >> 5, l32 = lane & 31, w = (int)uniform32(tid >> 6);
  int slice, item;
  if (!cross_coord(p, p.kblk * p.parts, slice, item)) return;
  const int kb = item / p.parts, part = item % p.parts;
  const CrossSlice sl(p, slice);
  const int nq = (p.N + 31) >> 5, total = 128 * kb < sl.len ? nq * p.G : 0;
  const int i0 = (int)((int64_t)total * part / p.parts), i1 = (int)((int64_t)total * (part + 1) / p.parts);
  const float c = p.c;
  const int wk0 = 128 * kb + 32 * w, key = wk0 + l32;
  const bool seen = key < sl.len;
  float k[C::H], v[C::H];
  own_row<D>((const float*)p.k + sl.zs * p.sk[0] + sl.hk * p.sk[1] + (int64_t)(seen ? key : 0) * p.sk[2], seen, h2, k);
  own_row<D>((const float*)p.v + sl.zs * p.sv[0] + sl.hk * p.sv[1] + (int64_t)(seen ? key : 0) * p.sv[2], seen, h2, v);
  f32x16 dk[C::DT], dv[C::DT];
#pragma unroll
  for (int u = 0; u < C::DT; ++u) dk[u] = dv[u] = f32x16{};
  RowTile32<D, 256> qn, gn;
  qn.init(p.sq[2]);
  gn.init(p.sd[2]);
  const uint32_t qb = uniform32((uint32_t)(p.sq[2] * 128)), ob = uniform32((uint32_t)(p.sd[2] * 128));
  float mn = 0.0f;
  auto load = [&](int i) {
    const int g = i / nq, first = 32 * (i % nq);
    qn.load(rows32_rsrc<D>(p.q, sl.zs * p.sq[0] + (sl.hk * p.G + g) * p.sq[1], p.N, p.sq[2]), (uint32_t)(i % nq) * qb);
    gn.load(rows32_rsrc<D>(p.dout, sl.zs * p.sd[0] + (sl.hk * p.G + g) * p.sd[1], p.N, p.sd[2]), (uint32_t)(i % nq) * ob);
    if (tid < 64) mn = first + l32 < p.N ? (h2 ? p.delta : p.m)[((int64_t)slice * p.G + g) * p.N + first + l32] : 0.0f;
  };
  if (i0 < i1) load(i0);
  for (int i = i0; i < i1; ++i) {
    __syncthreads();
    qn.store(qs);
    gn.store(gs);
    if (tid < 64) md[h2][l32] = mn;
    __syncthreads();
    if (i + 1 < i1) load(i + 1);
    if (wk0 >= sl.len) continue;
    f32x16 s = rows_dot<D>(qs, k, f32x16{}, l32, h2), dp;
#pragma unroll
    for (int e = 0; e < 16; ++e) dp[e] = md[1][kappa(e, h2)];
    dp = rows_dot<D>(gs, v, dp, l32, h2);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[e] = fast_exp2(__builtin_fmaf(s[e], c, -md[0][kappa(e, h2)]));
      dp[e] *= s[e];
    }
#pragma unroll
    for (int e = 0; e < 16; ++e)
#pragma unroll
      for (int u = 0; u < C::DT; ++u) {
        dv[u] = mfma2(s[e], cell<D>(gs, e, 32 * u + l32, h2), dv[u]);
        dk[u] = mfma2(dp[e], cell<D>(qs, e, 32 * u + l32, h2), dk[u]);
      }
  }
  // Keys past len get zeros: what their lanes hold is of no meaning.
  float* part_out = p.kpart + (((int64_t)slice * p.kblk + kb) * p.parts + part) * (2 * 128 * D) + 32 * w * D;
  float* dko = (float*)p.dk + sl.zs * p.sdk[0] + sl.hk * p.sdk[1];
  float* dvo = (float*)p.dv + sl.zs * p.sdv[0] + sl.hk * p.sdv[1];
#pragma unroll
  for (int u = 0; u < C::DT; ++u)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int in = 8 * (e >> 2) + 4 * h2 + (e & 3), d = 32 * u + l32;
      if (d >= D) continue;
      const bool there = wk0 + in < sl.len;
      if (p.parts > 1) {
        part_out[in * D + d] = there ? dk[u][e] : 0.0f;
        part_out[128 * D + in * D + d] = there ? dv[u][e] : 0.0f;
      } else if (wk0 + in < p.S) {
        dko[(int64_t)(wk0 + in) * p.sdk[2] + d] = there ? dk[u][e] * p.scale : 0.0f;
        dvo[(int64_t)(wk0 + in) * p.sdv[2] + d] = there ? dv[u][e] : 0.0f;
      }
    }
}

template <int D>
int fwd_d(const CrossParams& p, hipStream_t st) {
  unsigned blocks;
  int rc;
  if ((rc = cross_grid(p.slices(), (int64_t)p.nblk * p.splits, 64 * p.waves, &blocks))) return rc;
  if (p.waves == 1) cross_fwd_f32_kernel<D, 1, cross_f32_occ(D)><<<dim3(blocks), dim3(64), 0, st>>>(p);
  else cross_fwd_f32_kernel<D, 4, cross_f32_occ(D)><<<dim3(blocks), dim3(256), 0, st>>>(p);
  if ((rc = check_launch("tattn_cross_fwd")) || p.splits == 1) return rc;
  return launch_cross_combine_f32(p, D, st);
}

template <int D>
int bwd_d(const CrossParams& p, hipStream_t st) {
  unsigned blocks;
  int rc;
  if ((rc = cross_grid(p.slices(), (int64_t)p.nblk * p.splits, 64 * p.waves, &blocks))) return rc;
  if (p.waves == 1) cross_dq_f32_kernel<D, 1, cross_f32_occ(D)><<<dim3(blocks), dim3(64), 0, st>>>(p);
  else cross_dq_f32_kernel<D, 4, cross_f32_occ(D)><<<dim3(blocks), dim3(256), 0, st>>>(p);
  if ((rc = check_launch("tattn_cross_bwd")) || (p.splits > 1 && (rc = launch_cross_sum(p, D, 1, false, 0, st)))) return rc;
  if ((rc = cross_grid(p.slices(), (int64_t)p.kblk * p.parts, 256, &blocks))) return rc;
  cross_dkdv_f32_kernel<D, cross_f32_occ(D)><<<dim3(blocks), dim3(256), 0, st>>>(p);
  if ((rc = check_launch("tattn_cross_bwd")) || p.parts == 1) return rc;
  return launch_cross_sum(p, D, 1, true, 128, st);
}

}  // namespace

int launch_cross_f32(const CrossParams& p, int D, bool bwd, hipStream_t st) {
  switch (D) {
    case 16: return bwd ? bwd_d<16>(p, st) : fwd_d<16>(p, st);
    case 32: return bwd ? bwd_d<32>(p, st) : fwd_d<32>(p, st);
    case 64: return bwd ? bwd_d<64>(p, st) : fwd_d<64>(p, st);
    case 128: return bwd ? bwd_d<128>(p, st) : fwd_d<128>(p, st);
  }
  return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %d", D);
}

}  // namespace tattn
