// Attention of one token per request over a paged cache in 4 bits, on gfx950.
//
// Bound by the cache's bytes: 17/32 D for a key and as many for a value, read once for up to 16 query heads that share
// them, whose rows are the columns of 16 x 16 x 32 matrix instructions (unused columns cost nothing that bounds the kernel).
//   v_mfma_f32_16x16x32: A lane holds A[m = lane % 16][k = 8 (lane / 16) + i], B lane B[k = 8 (lane / 16) + i][n = lane % 16],
//   C lane holds C[m = 4 (lane / 16) + r][n = lane % 16], r < 4
// A wave takes 32 keys at a time, alone. Lane (l, g) = (lane % 16, lane / 16) loads a quarter row, codes of K and of V and
// their exponent, of two keys, 8 (l / 4) + 4 a + l % 4 of the tile for a = 0, 1, converts two codes an instruction
// (v_cvt_scalef32_pk, which also applies the block's power of two), and
//   S^T = K Q^T     two 16-key tiles. K's codes become operands in the lane that loaded them: the order of d within a dot
//                   product is free, so a lane group owns a quarter of d, for Q as well. With the keys above, a lane's
//                   8 scores are those of keys 8 g .. 8 g + 7: the B operand of
//   O^T += V^T P^T  V's values go through the wave's own 32 rows of LDS, swizzled, and come back transposed.
// The next tile's codes and the page numbers of the one after are on their way meanwhile; waves meet only at the end. A
// workgroup of four waves takes `chunk` consecutive tiles of one request and key head; requests of many tiles are cut into
// equal chunks, whatever their lengths, and joined by combine_kernel. 64 requests of up to 16,384 tokens with 32/8 heads x 128
// take 147-153 us, 4.7-4.9 TB/s of the cache's bytes, where a kernel that only reads has 6.3 (32 x 32 x 16 instructions, with
// twice the unused columns: 163 us).
//
// Roundings: K and V are what the cache holds, exact in either type; P is rounded to it as the second product's operand, its sum
// taken from the rounded values; scores, maxima, sums and accumulators are float32 (relative to 64 bits, in norm, in bf16:
// 2.3e-3, a float32 computation rounded once 1.7e-3).
#include <algorithm>

#include "fp4.h"
#include "window.h"

namespace tattn {
namespace {

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

constexpr int kRows = 16;  // query heads per workgroup

template <int D>
struct C4 {
  static constexpr int W = D / 32;   // words of codes in a quarter row, and matrix instructions over d
  static constexpr int DT = D / 16;  // 16-row tiles of O^T
  static constexpr int RB = 2 * D;   // bytes of a row of V in LDS
  static constexpr int TILE = 32 * RB;
  // Chunk swizzle of V's rows: the 16 rows that a lane group writes at one chunk, and the 16 rows x 32 bytes of a
  // transposed read, spread over all banks.
  static __device__ __forceinline__ int f(int row) {
    if constexpr (D == 128) return (row & 3) | (((row >> 3) & 3) << 2);
    else if constexpr (D == 64) return ((row >> 1) & 1) | (((row >> 3) & 3) << 1);
    else return (row >> 3) & 3;
  }
  static __device__ __forceinline__ int addr(int row, int byte) { return row * RB + ((((byte >> 4) ^ f(row)) << 4) | (byte & 15)); }
};

// Exponents of a lane's two keys: a byte each, or at head dim 64 those of the eight rows around them in one load, from which
// byte `pick` of either half is the lane's (two loads fewer per tile: 104 -> 91 us for 64 x 16,384 x 32/8; at 32 it gains nothing).
template <int D>
struct Scales {
  static constexpr bool WIDE = D == 64;
  uint32_t x[WIDE ? 4 : 2];
  __device__ __forceinline__ void load(const uint8_t* p) {
    typedef uint32_t U4 __attribute__((ext_vector_type(4), aligned(4)));
    if constexpr (WIDE) {
      const U4 a = *reinterpret_cast<const U4*>(p);
      x[0] = a[0], x[1] = a[1], x[2] = a[2], x[3] = a[3];
    } else {
      x[0] = p[0], x[1] = p[4 * (D / 32)];
    }
  }
  __device__ __forceinline__ void hide(int a) {
    if constexpr (WIDE) x[2 * a] = x[2 * a + 1] = 0x7f7f7f7fu;
    else x[a] = 127;
  }
  __device__ __forceinline__ float of(int a, uint32_t pick) const {
    uint32_t e = x[a];
    if constexpr (WIDE) e = __builtin_amdgcn_perm(x[2 * a + 1], x[2 * a], 0x0c0c0c00u | pick);  // 0x0c: a zero byte
    return __builtin_bit_cast(float, e << 23);
  }
};

// The lane's quarter rows of its two keys of a tile.
template <int D>
struct Codes {
  uint32_t k[2 * C4<D>::W], v[2 * C4<D>::W];
  Scales<D> scale[2];     // exponents of K and of V
  bool ok[2];             // the key is visible and its page is one of the cache's
};

template <int W>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* x) {
  if constexpr (W == 4) {
    const u32x4 a = *reinterpret_cast<const u32x4*>(p);
    x[0] = a[0], x[1] = a[1], x[2] = a[2], x[3] = a[3];
  } else {
    const u32x2 a = *reinterpret_cast<const u32x2*>(p);
    x[0] = a[0], x[1] = a[1];
  }
}

// Half rows of two keys as loaded (lanes 0-31 of the first key, the others of the second) -> a quarter row of either.
template <int W>
__device__ __forceinline__ void quarters(uint32_t (&x)[2 * W]) {
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const auto y = __builtin_amdgcn_permlane32_swap(x[i], x[W + i], false, false);
    x[i] = y[0];
    x[W + i] = y[1];
  }
}

// Eight codes as values.
template <typename T>
__device__ __forceinline__ typename H16<T>::V8 values8(uint32_t codes, float scale) {
  return __builtin_bit_cast(typename H16<T>::V8,
                            u32x4{Fp4<T>::template unpack<0>(codes, scale), Fp4<T>::template unpack<1>(codes, scale),
                                  Fp4<T>::template unpack<2>(codes, scale), Fp4<T>::template unpack<3>(codes, scale)});
}

// Over the four lanes that hold a column's rows.
__device__ __forceinline__ float max_groups(float x) { return max_halves(__builtin_fmaxf(x, __shfl_xor(x, 16))); }
__device__ __forceinline__ float sum_groups(float x) { return sum_halves(x + __shfl_xor(x, 16)); }

template <typename T, int D>
__global__ __launch_bounds__(256, D == 128 ? 3 : 4) void cache4_attention_kernel(const Cache4AttnParams p) {
  using H = H16<T>;
  using V8 = typename H::V8;
  using V4 = typename H::V4;
  using V2 = typename H::V2;
  using C = C4<D>;
  // Below head dim 128 a lane loads half a row of one of its two keys and swaps a quarter with the lane 32 away: half as many
  // loads, each twice as wide (64 x 16,384 x 32/8 x 64: 90 -> 85 us; 112 x 11,401 x 3 x 32: 63 -> 32).
  constexpr bool HALVES = D < 128;
  __shared__ __attribute__((aligned(1024))) char smem[4 * C::TILE];
  __shared__ float red[2][4][kRows];

  const int tid = threadIdx.x;
  const int lane = tid & 63, g = lane >> 4, l16 = lane & 15;
  const int w = (int)uniform32((uint32_t)(tid >> 6));
  const int units = p.R * p.Hk * p.groups;  // requests x key heads x groups of up to 16 query heads
  const int unit = blockIdx.x % units, chunk = blockIdx.x / units;
  const int rg = unit % p.groups, hk = unit / p.groups % p.Hk, r = unit / p.groups / p.Hk;
  const int row = kRows * rg + l16;  // of the key head's G
  const bool live = row < p.G;

  const int len = min(max(p.lens[r], 0), p.most);
  const int pos = len - 1;
  TileList list;
  list.init(pos, pos, pos, p.window, p.sinks);
  const int i0 = chunk * p.chunk, i1 = min(list.n, i0 + p.chunk);
  const int64_t slice = (int64_t)r * p.Hk + hk;
  const int64_t prow = (slice * p.splits + chunk) * p.G + row;
  float* ml = p.part + (int64_t)p.R * p.Hk * p.splits * p.G * D + prow * 2;
  if (i0 >= i1 && p.splits > 1) {  // nothing here: an empty part
    if (w == 0 && g == 0 && live) ml[0] = kNoMax, ml[1] = 0.0f;
    return;
  }

  const int quarter = HALVES ? 2 * (g & 1) + (g >> 1) : g;  // of d, that the lane's group owns
  V8 qop[C::W];
  {
    const T* src = (const T*)p.q + r * p.sq[0] + (hk * p.G + (live ? row : 0)) * p.sq[1] + quarter * (D / 4);
#pragma unroll
    for (int s = 0; s < C::W; ++s) {
      const V8 x = *reinterpret_cast<const V8*>(src + 8 * s);
      qop[s] = live ? x : V8{};
    }
  }
  const float c = p.c, hidden = hidden_score(c);
  const int32_t* table = p.tables + r * p.table_stride;
  const int in_page = (1 << p.shift) - 1;
  const int key0 = 8 * (l16 >> 2) + (l16 & 3);  // the lane's keys of a tile: key0 and key0 + 4
  // Byte offsets are (page number) * (bytes of a page) + what follows; a tile starts a page, or lies within one.
  const uint32_t page_rows = (uint32_t)p.Hk * 2 << p.shift;
  const uint8_t* codes = p.codes + ((int64_t)hk * 2 << p.shift) * (D / 2) + (HALVES ? (g & 1) * (D / 4) + 2 * D * (g >> 1) : g * (D / 8));
  const uint8_t* scales = p.scales + ((int64_t)hk * 2 << p.shift) * (D / 32) + (D == 128 ? g : 0);
  const uint32_t pick = 2 * (l16 & 3) + (quarter >> 1);

  // The page of the lane's keys in list entry i (pages hold multiples of 16 keys: both lie in one; -1 where both are
  // hidden), and which of them are visible.
  auto page_of = [&](int i, bool (&see)[2]) __attribute__((always_inline)) {
    const int t = list.at(min(i, i1 - 1));
    const bool inner = i < i1 && 32 * t + 31 <= pos && (32 * t >= list.lo || 32 * t + 31 < p.sinks);
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const int key = 32 * t + key0 + 4 * a;
      see[a] = inner || (i < i1 && key <= pos && (key >= list.lo || key < p.sinks));
    }
    return see[0] || see[1] ? table[(32 * t + key0) >> p.shift] : -1;
  };
  auto load = [&](int i, int page, const bool (&see)[2]) __attribute__((always_inline)) {
    Codes<D> x;
    const bool held = (uint32_t)page < (uint32_t)p.pages;
    const uint64_t at = (uint64_t)(held ? (uint32_t)page : 0u) * page_rows + (uint32_t)((32 * list.at(min(i, i1 - 1)) + key0) & in_page);
    const uint8_t* pc = codes + at * (D / 2);
    const uint8_t* ps = scales + (Scales<D>::WIDE ? at & ~(uint64_t)7 : at) * (D / 32);
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      x.ok[a] = held && see[a];
      if constexpr (!HALVES) {
        load_words<C::W>(pc + 4 * a * (D / 2), x.k + a * C::W);
        load_words<C::W>(pc + 4 * a * (D / 2) + ((D / 2) << p.shift), x.v + a * C::W);
      }
    }
    if constexpr (HALVES) {
      load_words<2 * C::W>(pc, x.k);
      load_words<2 * C::W>(pc + ((D / 2) << p.shift), x.v);
    }
#pragma unroll
    for (int v = 0; v < 2; ++v) x.scale[v].load(ps + (v ? (D / 32) << p.shift : 0));
    return x;
  };

  char* vrows = smem + w * C::TILE;
  // Transposed reads: lane s of a group at row 8 g + s / 4 (+ 4 for the second read), column 4 (s % 4) of 16.
  int lo[C::DT], hi[C::DT];
#pragma unroll
  for (int u = 0; u < C::DT; ++u) {
    lo[u] = C::addr(8 * g + (l16 >> 2), 32 * u + 8 * (l16 & 3));
    hi[u] = C::addr(8 * g + 4 + (l16 >> 2), 32 * u + 8 * (l16 & 3));
  }
  float mrow = kNoMax, lrow = 0.0f;
  f32x4 acc[C::DT];
#pragma unroll
  for (int u = 0; u < C::DT; ++u) acc[u] = f32x4{};

  auto tile = [&](Codes<D>& x) __attribute__((always_inline)) {
    const uint64_t see0 = __builtin_amdgcn_ballot_w64(x.ok[0]), see1 = __builtin_amdgcn_ballot_w64(x.ok[1]);
    if ((see0 | see1) == 0) return;
    if constexpr (HALVES) {
      quarters<C::W>(x.k);
      quarters<C::W>(x.v);
    }
    if ((see0 & see1) != ~0ull) {  // what lies at a hidden key's place reaches nothing
#pragma unroll
      for (int a = 0; a < 2; ++a)
        if (!x.ok[a]) {
#pragma unroll
          for (int i = 0; i < C::W; ++i) x.k[a * C::W + i] = x.v[a * C::W + i] = 0;
          x.scale[0].hide(a);
          x.scale[1].hide(a);
        }
    }
    f32x4 s[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      s[a] = f32x4{};
      const float scale = x.scale[0].of(a, pick);
#pragma unroll
      for (int i = 0; i < C::W; ++i) s[a] = mfma16(values8<T>(x.k[a * C::W + i], scale), qop[i], s[a]);
    }
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const float scale = x.scale[1].of(a, pick);
#pragma unroll
      for (int i = 0; i < C::W; ++i)
        *reinterpret_cast<TATTN_LDS V8*>((TATTN_LDS char*)vrows + C::addr(key0 + 4 * a, quarter * (D / 2) + 16 * i)) = values8<T>(x.v[a * C::W + i], scale);
    }
    if ((see0 & see1) != ~0ull) {  // row m of tile a is lane m's key a: the lane's scores are rows 4 g + e
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const uint32_t bits = (uint32_t)(a ? see1 : see0) >> (4 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[a][e] = bits >> e & 1 ? s[a][e] : hidden;
      }
    }
    V8 pr;
    auto probs = [&]() __attribute__((always_inline)) {
      float ps = 0.0f;
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const V2 two = H::pack(fast_exp2(__builtin_fmaf(s[a][e], c, -mrow)), fast_exp2(__builtin_fmaf(s[a][e + 1], c, -mrow)));
          ps = H::sum2(two, ps);
          pr[4 * a + e] = two[0];
          pr[4 * a + e + 1] = two[1];
        }
      return ps;
    };
    // Probabilities against the running max as it stands; a sum above 2^12 (the first visible tile among them) sends the
    // wave through the row max and a rescale. One-sided: state first, undone inside.
    const float lprev = lrow;
    const float ps = probs();
    lrow += ps;
    if (__builtin_amdgcn_ballot_w64(!(ps <= 4096.0f))) {
      float mx = kNoMax;
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = __builtin_fmaxf(mx, s[a][e] * c);
      const float cand = max_groups(mx);
      const float mnew = cand > mrow + kRescaleLog2 ? cand : mrow;
      const float alpha = fast_exp2(mrow - mnew);
      mrow = mnew;
      const float again = probs();
      lrow = lprev * alpha + again;
#pragma unroll
      for (int u = 0; u < C::DT; ++u) acc[u] *= alpha;
    }
#pragma unroll
    for (int u = 0; u < C::DT; ++u) acc[u] = mfma16(tr_pair<T>(vrows, lo[u], hi[u]), pr, acc[u]);
  };

  int i = i0 + w;
  if (i < i1) {
    bool see[2];
    int page = page_of(i, see);
    Codes<D> x = load(i, page, see);
    page = page_of(i + 4, see);
    for (; i < i1; i += 8) {
      Codes<D> y = load(i + 4, page, see);
      page = page_of(i + 8, see);
      tile(x);
      if (i + 4 >= i1) break;
      x = load(i + 8, page, see);
      page = page_of(i + 12, see);
      tile(y);
    }
  }

  // Join the four waves: register e of tile u is column d = 16 u + 4 g + e of row l16; wave w adds tiles w, w + 4, ...
  const float lt = sum_groups(lrow);
  if (g == 0) {
    red[0][w][l16] = mrow;
    red[1][w][l16] = lt;
  }
  __syncthreads();
  float mall = kNoMax, lall = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) mall = __builtin_fmaxf(mall, red[0][k][l16]);
#pragma unroll
  for (int k = 0; k < 4; ++k) lall += fast_exp2(red[0][k][l16] - mall) * red[1][k][l16];
  const bool parts = p.splits > 1;
  float wgt = fast_exp2(mrow - mall);
  if (!parts) wgt = lall == 0.0f ? 0.0f : wgt / lall;
  static_assert(C::DT * 1024 == C::TILE, "a wave's sums fit its rows of V");
#pragma unroll
  for (int u = 0; u < C::DT; ++u) *reinterpret_cast<TATTN_LDS f32x4*>((TATTN_LDS char*)vrows + 1024 * u + 16 * lane) = acc[u] * wgt;
  __syncthreads();
  T* orow = (T*)p.out + r * p.so[0] + (hk * p.G + row) * p.so[1];
  for (int u = w; u < C::DT; u += 4) {
    f32x4 x = f32x4{};
#pragma unroll
    for (int k = 0; k < 4; ++k) x += *reinterpret_cast<const TATTN_LDS f32x4*>((const TATTN_LDS char*)smem + k * C::TILE + 1024 * u + 16 * lane);
    const int d0 = 16 * u + 4 * g;
    if (!live) continue;
    if (parts) {
      *reinterpret_cast<f32x4*>(p.part + prow * D + d0) = x;
    } else {
      V4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (T)x[e];
      *reinterpret_cast<V4*>(orow + d0) = y;
    }
  }
  if (parts && w == 0 && g == 0 && live) ml[0] = mall, ml[1] = lall;
}

template <typename T, int D>
int run(const Cache4AttnParams& p, hipStream_t st) {
  const int64_t blocks = (int64_t)p.R * p.Hk * p.groups * p.splits;
  if (blocks > 0x7ffffff) return set_error(TATTN_E_ARG, "grid too large: %lld workgroups", (long long)blocks);
  cache4_attention_kernel<T, D><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(p);
  const int rc = check_launch("tattn_cache4_attention");
  if (rc || p.splits == 1) return rc;
  const int64_t so[3] = {p.so[0], p.so[1], 0};
  return launch_combine(p.part, p.out, nullptr, so, (int64_t)p.R * p.Hk, p.Hk, p.G, 1, p.splits, D,
                        std::is_same_v<T, bf16> ? 2 : 0, st);
}

}  // namespace

void cache4_chunks(Cache4AttnParams& p) {
  const int64_t seen = std::min<int64_t>(p.most, (int64_t)p.window + p.sinks + 31);
  const int64_t tiles = std::max<int64_t>(1, (seen + 31) / 32 + 1), units = (int64_t)p.R * p.Hk * p.groups;
  int64_t chunk = tiles * units / 512;
  chunk = std::min<int64_t>(64, std::max<int64_t>(4, (chunk + 3) / 4 * 4));
  p.chunk = (int32_t)chunk;
  p.splits = (int32_t)((tiles + chunk - 1) / chunk);
}

int launch_cache4_attention(const Cache4AttnParams& p, int D, int dtype, hipStream_t st) {
  const bool h = dtype == 0;
  switch (D) {
    case 32: return h ? run<f16, 32>(p, st) : run<bf16, 32>(p, st);
    case 64: return h ? run<f16, 64>(p, st) : run<bf16, 64>(p, st);
    case 128: return h ? run<f16, 128>(p, st) : run<bf16, 128>(p, st);
  }
  return set_error(TATTN_E_ARG, "head dim must be 32, 64 or 128, got %d", D);
}

}  // namespace tattn
