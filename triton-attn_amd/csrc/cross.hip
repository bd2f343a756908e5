// Attention over keys of another length, 16-bit forward, on gfx950: few rows, the choice between the kernels, and the sum of parts.
//
//   O = softmax(c' Q K^T) V over the first len keys, one pass over the keys with the running max and sum of the softmax
//
// Few rows: cross_rows.h. Many: cross_pipe.h. Few keys: cross_short.hip. The keys are cut into parts where workgroups are few, and
// combine_kernel joins the parts in order.
//
// Few rows are bound by the keys' bytes. One token of each sequence, keys not in a cache, us (as a copy): 32 x 32/8 over 375 to
// 1,500 x 128 28 (22), 64 x 32/8 over 1,024 x 128 50 (47), 64 x 32/8 over 1,024 to 4,096 x 64 66 (59), 1 x 32 over 131,072 x
// 128 367 (377).
//
// Roundings: P is rounded to the element type, as the matrix instruction takes it, and its sum is taken from the rounded values.
// Scores, maxima, sums and accumulators are float32.
#include <algorithm>
#include <type_traits>

#include "cross_rows.h"

namespace tattn {
namespace {

template <typename T, int D, int W, int OCC>
__global__ __launch_bounds__(W * 64, OCC) void cross_rows_kernel(const CrossParams p) {
  __shared__ __attribute__((aligned(1024))) char kbuf[W * CrossTile<D>::BYTES];
  __shared__ __attribute__((aligned(1024))) char vbuf[W * CrossTile<D>::BYTES];
  __shared__ float red[2][W][32];
  int slice, blk;
  if (!cross_coord(p, p.nblk * p.splits, slice, blk)) return;
  rows_block<T, D, W, false, 1>(p, slice, blk / p.splits, blk % p.splits, {{kbuf}, {vbuf}, red});
}

// ---- rows whose keys were cut into parts ---------------------------------------------------------
struct CombineParams {
  const float* part[2];  // of the slices' rows; of each sequence's own rows, or null
  int32_t splits[2];
  void* out;
  float* m;
  const int32_t* lens;  // own keys of each sequence: rows at positions below 0 become 0
  int64_t st[3];
  int64_t slices;
  int32_t Hk, B, G, N, S;
  int32_t dealt;  // groups of lanes that a row's parts are dealt to
};

// O = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s. D / 4 lanes hold a row's columns; `dealt` such groups share a row's parts
// and are added in order through LDS.
template <typename T, int D>
__global__ __launch_bounds__(256) void combine_kernel(const CombineParams p) {
  typedef T V4 __attribute__((ext_vector_type(4)));
  constexpr int LPR = D / 4, GROUPS = 256 / LPR;
  __shared__ __attribute__((aligned(16))) float sums[GROUPS][D];
  __shared__ float ml[GROUPS][2];
  const int tid = threadIdx.x, g = tid / LPR, d0 = tid % LPR * 4, deal = g % p.dealt;
  const int rows = p.B * p.G * p.N;
  const int64_t i = (int64_t)blockIdx.x * (GROUPS / p.dealt) + g / p.dealt;
  const bool live = i < p.slices * rows;
  const int64_t slice = live ? i / rows : 0;
  const int row = live ? (int)(i % rows) : 0, b = row / (p.G * p.N), rest = row % (p.G * p.N);
  const int64_t zs = slice / p.Hk, hk = slice % p.Hk, z = zs * p.B + b;
  const int n = rest % p.N;
  float m = kNoMax, l = 0.0f;
  f32x4 x = f32x4{};
  auto add = [&](float ms, float ls, f32x4 y) __attribute__((always_inline)) {
    const float mn = __builtin_fmaxf(m, ms), a = fast_exp2(m - mn), w = fast_exp2(ms - mn);
    m = mn;
    l = l * a + ls * w;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = x[e] * a + y[e] * w;
  };
  auto take = [&](const float* part, int splits, int first, int64_t slices, int64_t slice, int rows, int row) __attribute__((always_inline)) {
    const float* tail = part + slices * splits * rows * D;
#pragma unroll 4
    for (int s = first; s < splits; s += p.dealt) {
      const int64_t at = (slice * splits + s) * rows + row;
      const f32x2 v = *reinterpret_cast<const f32x2*>(tail + 2 * at);
      add(v[0], v[1], *reinterpret_cast<const f32x4*>(part + at * D + d0));
    }
  };
  if (live) {
    take(p.part[0], p.splits[0], deal, p.slices, slice, rows, row);
    if (p.part[1]) take(p.part[1], p.splits[1], deal, p.slices * p.B, z * p.Hk + hk, p.G * p.N, rest);
  }
  if (p.dealt > 1) {
    *reinterpret_cast<f32x4*>(&sums[g][d0]) = x;
    if (d0 == 0) ml[g][0] = m, ml[g][1] = l;
    __syncthreads();
    if (deal > 0) return;
    for (int k = 1; k < p.dealt; ++k) add(ml[g + k][0], ml[g + k][1], *reinterpret_cast<const f32x4*>(&sums[g + k][d0]));
  }
  if (!live) return;
  if (p.lens && min(max(p.lens[z], 0), p.S) - p.N + n < 0) l = 0.0f;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  V4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (T)(l == 0.0f ? 0.0f : x[e] * inv);
  const int64_t h = hk * p.G + rest / p.N;
  *reinterpret_cast<V4*>((T*)p.out + z * p.st[0] + h * p.st[1] + n * p.st[2] + d0) = y;
  if (p.m && d0 == 0) p.m[(z * p.Hk * p.G + h) * p.N + n] = m + __log2f(l);
}

template <typename T, int D>
int combine(CombineParams p, hipStream_t st, const char* what) {
  const int64_t blocks = combine_blocks(p.slices * p.B * p.G * p.N, std::max(p.splits[0], p.part[1] ? p.splits[1] : 0), D, p.dealt);
  if (int rc = check_grid(blocks, 256)) return rc;
  combine_kernel<T, D><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(p);
  return check_launch(what);
}

CombineParams combine_params(const CrossParams& p) {
  CombineParams c{};
  c.part[0] = p.part;
  c.splits[0] = p.splits;
  c.out = p.out;
  c.m = p.m;
  for (int i = 0; i < 3; ++i) c.st[i] = p.sout[i];
  c.slices = p.slices();
  c.Hk = p.Hk; c.B = p.B; c.G = p.G; c.N = p.N;
  return c;
}

template <typename T, int D>
int combine_cross(const CrossParams& p, hipStream_t st) { return combine<T, D>(combine_params(p), st, "tattn_cross_fwd"); }

template <typename T, int D>
int combine_prefix(const PrefixParams& p, hipStream_t st) {
  CombineParams c = combine_params(p.pre);
  c.part[1] = p.own.part;
  c.splits[1] = p.own.splits;
  c.lens = p.own.lens;
  c.S = p.own.S;
  return combine<T, D>(c, st, "tattn_prefix_attention");
}

template <typename T, int D>
int fwd_d(const CrossParams& p, hipStream_t st) {
  unsigned blocks;
  int rc;
  if (cross_short(p, D, std::is_same_v<T, f16> ? 0 : 2, false)) return launch_cross_short(p, D, std::is_same_v<T, f16> ? 0 : 2, false, st);
  if (p.pipe) {
    if ((rc = launch_cross_pipe(p, D, std::is_same_v<T, f16> ? 0 : 2, st)) || p.splits == 1) return rc;
    return combine_cross<T, D>(p, st);
  }
  if ((rc = cross_grid(p.slices(), (int64_t)p.nblk * p.splits, 64 * p.waves, &blocks))) return rc;
  if (p.waves == 8) cross_rows_kernel<T, D, 8, rows_occ(D)><<<dim3(blocks), dim3(512), 0, st>>>(p);
  else cross_rows_kernel<T, D, 4, rows_occ(D)><<<dim3(blocks), dim3(256), 0, st>>>(p);
  if ((rc = check_launch("tattn_cross_fwd")) || p.splits == 1) return rc;
  return combine_cross<T, D>(p, st);
}

}  // namespace

// Up to two row tiles: one per workgroup (rows_block; in float32 of one wave). More: blocks of cross_pipe_rows (128 in
// float32). Keys are cut into parts until the chip holds no more workgroups at once, of at least eight tiles (in float32, where
// a tile takes eight times as long, three).
int cross_fwd_plan(CrossParams& p, int D, int dtype) {
  unsigned launched;
  // Few keys: a slice's row tiles in as many parts as the chip holds workgroups, of four tiles for a wave at least. us at 512, 768 and
  // 1,024: 16 x 8 x 4,096 over 77 x 64 41, 39, 44; over 64 x 128 57, 62, 59; 16 x 16 x 4,096 over 77 x 32 51, 49, 45.
  if (cross_short(p, D, dtype, false)) {
    const int64_t tiles = (p.rows() + 31) / 32, places = 256 * (D == 128 ? 2 : D == 64 ? 3 : 4);
    p.nblk = (int)std::max<int64_t>(1, std::min<int64_t>(places / p.slices(), tiles / 16));
    p.splits = 1;
    return cross_grid(p.slices(), p.nblk, 256, &launched);
  }
  const int64_t tiles = ((int64_t)p.S + 31) / 32;
  p.pipe = dtype != 1 && p.rows() > 64;
  p.waves = dtype == 1 && p.rows() <= 64 ? 1 : 4;
  const int64_t block = dtype == 1 ? 32 * p.waves : p.pipe ? cross_pipe_rows(D) : 32;
  p.nblk = (int)((p.rows() + block - 1) / block);
  const int64_t blocks = p.slices() * p.nblk, want = 256 * (dtype == 1 ? cross_f32_occ(D) * 4 / p.waves : p.pipe ? 2 : rows_occ(D));
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want / blocks, tiles / (dtype == 1 ? 3 : 8)));
  // Eight waves share the rows before the keys are cut: fewer parts to join, or none (32 x 32/8 over 375 to 1,500 x 128, one
  // token: 22.5 us for 24.6, keys in the cache).
  if (!p.pipe && dtype != 1 && p.splits > 1) {
    p.waves = 8;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want / 2 / blocks, tiles / 16));
  }
  return cross_grid(p.slices(), (int64_t)p.nblk * p.splits, 64 * p.waves, &launched);
}

#define TATTN_CROSS_SWITCH(FN)                                                   \
  switch (D) {                                                                   \
    case 16: return dtype == 0 ? FN<f16, 16>(p, st) : FN<bf16, 16>(p, st);       \
    case 32: return dtype == 0 ? FN<f16, 32>(p, st) : FN<bf16, 32>(p, st);       \
    case 64: return dtype == 0 ? FN<f16, 64>(p, st) : FN<bf16, 64>(p, st);       \
    case 128: return dtype == 0 ? FN<f16, 128>(p, st) : FN<bf16, 128>(p, st);    \
  }                                                                              \
  return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %d", D);

int launch_cross_fwd(const CrossParams& p, int D, int dtype, hipStream_t st) { TATTN_CROSS_SWITCH(fwd_d) }
int launch_prefix_combine(const PrefixParams& p, int D, int dtype, hipStream_t st) { TATTN_CROSS_SWITCH(combine_prefix) }
int launch_cross_combine_f32(const CrossParams& p, int D, hipStream_t st) {
  switch (D) {
    case 16: return combine_cross<float, 16>(p, st);
    case 32: return combine_cross<float, 32>(p, st);
    case 64: return combine_cross<float, 64>(p, st);
    case 128: return combine_cross<float, 128>(p, st);
  }
  return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %d", D);
}

}  // namespace tattn
