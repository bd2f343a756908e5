// Attention over keys of another length, 16-bit forward, and one step behind a shared prefix, on gfx950.
//
//   O = softmax(c' Q K^T) V over the first len keys, one pass over the keys with the running max and sum of the softmax
//
// Few rows (`rows_block`): the waves of a workgroup share 32 rows, and each takes its own key tiles by itself, staged by LDS DMA
// into LDS of its own: no barrier until their partial results are added. The keys are cut into parts where rows are few, and
// `combine_kernel` joins the parts in order.
//
// Roundings: P is rounded to the element type, as the matrix instruction takes it, and its sum is taken from the rounded values.
// Scores, maxima, sums and accumulators are float32.
#include <algorithm>
#include <type_traits>

#include "cross.h"

namespace tattn {
namespace {

// The part `split` of the keys for 32 rows of a slice. CAUSAL: query n is at position len - N + n and sees no key after it.
template <typename T, int D, int W, bool CAUSAL>
__device__ __forceinline__ void rows_block(const CrossParams& p, int slice, int blk, int split, char* kbuf, char* vbuf,
                                           float (*red)[W][32]) {
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
  char *kt = kbuf + wu * Tile::BYTES, *vt = vbuf + wu * Tile::BYTES;
  auto fetch_k = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) dma16(krs, kt + 1024 * i, gk[i] + (uint32_t)t * kb);
  };
  auto fetch_v = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) dma16(vrs, vt + 1024 * i, gv[i] + (uint32_t)t * vb);
  };
  int t = i0 + wu;
  if (t < i1) {
    fetch_k(t);
    fetch_v(t);
  }

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
  auto step = [&]() __attribute__((always_inline)) {
    const int after = t + W < i1 ? t + W : t;
    wave_landed<PIECES>();  // V is still in flight
    f32x16 s = f32x16{};
#pragma unroll
    for (int sd = 0; sd < NSD; ++sd) s = Elt<T>::mfma(lds8<T>(kt + at.nat[sd]), qop[sd], s);
    reads_done();
    fetch_k(after);
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
#pragma unroll
    for (int sg = 0; sg < 2; ++sg)
#pragma unroll
      for (int u = 0; u < DT; ++u) acc[u] = Elt<T>::mfma(at.template tr<T>(vt, sg, u, lane), x[sg], acc[u]);
    reads_done();
    fetch_v(after);
    t += W;
  };
  while (t < i1) step();  // (as a plain loop body it takes 30 more registers)
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
  static_assert(PART * 4 == 2 * Tile::BYTES && W % 2 == 0, "the buffers hold the rows of every wave");
  const bool parted = p.splits > 1 || p.joined;
  auto part = [&](int k) { return (TATTN_LDS float*)(k < W / 2 ? kbuf : vbuf) + k % (W / 2) * PART + lane; };
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

template <typename T, int D, int W, int OCC>
__global__ __launch_bounds__(W * 64, OCC) void cross_rows_kernel(const CrossParams p) {
  __shared__ __attribute__((aligned(1024))) char kbuf[W * CrossTile<D>::BYTES];
  __shared__ __attribute__((aligned(1024))) char vbuf[W * CrossTile<D>::BYTES];
  __shared__ float red[2][W][32];
  int slice, blk;
  if (!cross_coord(p, p.nblk * p.splits, slice, blk)) return;
  rows_block<T, D, W, false>(p, slice, blk / p.splits, blk % p.splits, kbuf, vbuf, red);
}

// Workgroups over the prefix, the row blocks that read one part of it on one XCD, whose L2 hands it to the others.
__host__ __device__ inline int64_t prefix_blocks(const CrossParams& p) { return ((int64_t)p.Zs * p.Hk * p.splits + 7) / 8 * 8 * p.nblk; }

// The prefix's parts first, which are the longer ones, then each sequence's own keys.
template <typename T, int D, int OCC>
__global__ __launch_bounds__(4 * 64, OCC) void prefix_rows_kernel(const PrefixParams p) {
  __shared__ __attribute__((aligned(1024))) char kbuf[4 * CrossTile<D>::BYTES];
  __shared__ __attribute__((aligned(1024))) char vbuf[4 * CrossTile<D>::BYTES];
  __shared__ float red[2][4][32];
  const int total = (int)prefix_blocks(p.pre);
  int i = blockIdx.x;
  if (i < total) {
    const int l = i >> 3, unit = 8 * (l / p.pre.nblk) + (i & 7), slice = unit / p.pre.splits;
    if (slice < p.pre.Zs * p.pre.Hk)
      rows_block<T, D, 4, false>(p.pre, slice, l % p.pre.nblk, unit % p.pre.splits, kbuf, vbuf, red);
    return;
  }
  i -= total;
  const int per = p.own.nblk * p.own.splits, blk = i % per;
  rows_block<T, D, 4, true>(p.own, i / per, blk / p.own.splits, blk % p.own.splits, kbuf, vbuf, red);
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
  constexpr int GROUPS = 256 / (D / 4);
  const int most = std::max(p.splits[0], p.part[1] ? p.splits[1] : 0);
  for (p.dealt = 1; p.dealt < GROUPS && 4 * p.dealt < most; p.dealt *= 2) {}
  const int64_t rows = p.slices * p.B * p.G * p.N, per = GROUPS / p.dealt, blocks = (rows + per - 1) / per;
  if (blocks > 0x7fffffff) return set_error(TATTN_E_ARG, "grid too large: %lld rows", (long long)rows);
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

// Workgroups of rows_block that a CU holds: 64 KB of tiles at head dim 128, 128 registers below.
constexpr int rows_occ(int D) { return D == 128 ? 2 : 4; }

template <typename T, int D>
int fwd_d(const CrossParams& p, hipStream_t st) {
  unsigned blocks;
  int rc;
  if (cross_short(p, D, std::is_same_v<T, f16> ? 0 : 2, false)) return launch_cross_short(p, D, std::is_same_v<T, f16> ? 0 : 2, false, st);
  if (p.pipe) {
    if ((rc = launch_cross_pipe(p, D, std::is_same_v<T, f16> ? 0 : 2, st)) || p.splits == 1) return rc;
    return combine_cross<T, D>(p, st);
  }
  if ((rc = cross_grid(p.slices(), (int64_t)p.nblk * p.splits, &blocks))) return rc;
  if (p.waves == 8) cross_rows_kernel<T, D, 8, rows_occ(D)><<<dim3(blocks), dim3(512), 0, st>>>(p);
  else cross_rows_kernel<T, D, 4, rows_occ(D)><<<dim3(blocks), dim3(256), 0, st>>>(p);
  if ((rc = check_launch("tattn_cross_fwd")) || p.splits == 1) return rc;
  return combine_cross<T, D>(p, st);
}

template <typename T, int D>
int prefix_d(const PrefixParams& p, hipStream_t st) {
  int rc;
  const int64_t blocks = prefix_blocks(p.pre) + p.own.slices() * p.own.nblk * p.own.splits;
  if (blocks > 0x7ffffff) return set_error(TATTN_E_ARG, "grid too large: %lld workgroups", (long long)blocks);
  prefix_rows_kernel<T, D, rows_occ(D)><<<dim3((unsigned)blocks), dim3(4 * 64), 0, st>>>(p);
  if ((rc = check_launch("tattn_prefix_attention"))) return rc;
  CombineParams c = combine_params(p.pre);
  c.part[1] = p.own.part;
  c.splits[1] = p.own.splits;
  c.lens = p.own.lens;
  c.S = p.own.S;
  return combine<T, D>(c, st, "tattn_prefix_attention");
}

}  // namespace

// Up to two row tiles: one per workgroup (rows_block). More: blocks of cross_pipe_rows. Keys are cut into parts until the chip
// holds no more workgroups at once, of at least eight tiles (in float32, where a tile takes eight times as long, three).
void cross_fwd_plan(CrossParams& p, int D, int dtype) {
  if (cross_short(p, D, dtype, false)) {  // row tiles of a slice in parts, four a workgroup for a wave at least
    const int64_t tiles = (p.rows() + 31) / 32;
    p.nblk = (int)std::max<int64_t>(1, std::min<int64_t>(1024 / p.slices(), tiles / 16));
    p.splits = 1;
    return;
  }
  const int64_t tiles = ((int64_t)p.S + 31) / 32;
  p.pipe = dtype != 1 && p.rows() > 64;
  const int64_t block = dtype == 1 ? 128 : p.pipe ? cross_pipe_rows(D) : 32;
  p.nblk = (int)((p.rows() + block - 1) / block);
  const int64_t blocks = p.slices() * p.nblk, want = 256 * (p.pipe ? 2 : rows_occ(D));
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want / blocks, tiles / (dtype == 1 ? 3 : 8)));
  p.waves = 4;
  if (!p.pipe && dtype != 1 && p.splits > 1) {  // eight waves share the rows before the keys are cut: fewer parts to join, or none
    p.waves = 8;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want / 2 / blocks, tiles / 16));
  }
}

// Parts of the prefix as long as an even share of all tiles over the places that the chip has, those of a sequence's own keys half
// of that, as later workgroups fill the places that fall free; none has less than eight tiles. us at shares of (prefix, own) (1/2, 1/2),
// (1, 1/2), (1, 1), (3/2, 1/2):
//   64 requests x 32/8 x 128, prefix 8,192, up to 1,024 own keys   49, 44, 44, 68
//   8 x 16 samples x 16/4 x 128, prefix 4,096, up to 2,048          81, 77, 83, 77
//   128 x 16 x 5 queries x 128, prefix 8,192, up to 64               90, 85, 85, 86
void prefix_plan(PrefixParams& p, int D) {
  const int64_t pt = std::max<int64_t>(1, ((int64_t)p.pre.S + 31) / 32), ot = std::max<int64_t>(1, ((int64_t)p.own.S + 31) / 32);
  p.pre.nblk = (int)((p.pre.rows() + 31) / 32);
  p.own.nblk = (int)((p.own.rows() + 31) / 32);
  const int64_t share = (p.pre.slices() * p.pre.nblk * pt + p.own.slices() * p.own.nblk * ot) / (256 * rows_occ(D));
  const int64_t shared = std::max<int64_t>(8, share), own = std::max<int64_t>(8, share / 2);
  p.pre.splits = (int)((pt + shared - 1) / shared);
  p.own.splits = (int)((ot + own - 1) / own);
  p.pre.joined = p.own.joined = 1;
}
int64_t prefix_floats(const PrefixParams& p, int D) {
  return cross_part_floats(p.pre.slices(), p.pre.rows(), p.pre.splits, D) + cross_part_floats(p.own.slices(), p.own.rows(), p.own.splits, D);
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
int launch_prefix(const PrefixParams& p, int D, int dtype, hipStream_t st) { TATTN_CROSS_SWITCH(prefix_d) }
int launch_cross_combine(const CrossParams& p, int D, int dtype, hipStream_t st) {
  if (dtype == 1) {
    switch (D) {
      case 16: return combine_cross<float, 16>(p, st);
      case 32: return combine_cross<float, 32>(p, st);
      case 64: return combine_cross<float, 64>(p, st);
      case 128: return combine_cross<float, 128>(p, st);
    }
  }
  TATTN_CROSS_SWITCH(combine_cross)
}

}  // namespace tattn
