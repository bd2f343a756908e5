// Attention of one token per request over a paged cache in 4 bits, on gfx950.
//
// Bound by the cache's bytes: 17/32 D for a key and as many for a value, read once for all G query heads that share
// them, whose rows fill the 32 columns of a matrix instruction (unused columns cost nothing that bounds the kernel).
// A wave takes 32 keys at a time, alone: lane (key, half of d) loads that half row's codes of K and of V,
// converts two codes an instruction (v_cvt_scalef32_pk, which also applies the block's power of two), and
//   S^T = K Q^T     K's codes become operands in the lane that loaded them: the order of d within a dot product is
//                   free, so each lane half owns one contiguous half of d, for Q as well
//   O^T += V^T P^T  V's values go through the wave's own 32 rows of LDS, swizzled, and come back transposed
// The next tile's codes and the page numbers of the one after are on their way meanwhile; waves meet only at the end. A
// workgroup of four waves takes `chunk` consecutive tiles of one request and key head; requests of many tiles are cut into
// equal chunks, whatever their lengths, and joined by combine_kernel.
#include <algorithm>

#include "fp4.h"
#include "window.h"

namespace tattn {
namespace {

template <int D>
struct C4 {
  static constexpr int W = D / 16;              // words of codes per lane and tensor: half a row
  static constexpr int NSD = D / 16, DT = (D + 31) / 32;
  static constexpr int BLOCKS = D >= 64 ? D / 64 : 1;  // blocks of 32 values in half a row (D = 32: half a block)
  static constexpr int TILE = 32 * Swz<D>::RB;
  static constexpr int MERGE = 4 * 16 * 64 * 4;  // one 32-row d tile of every wave
  static constexpr int LDS = 4 * TILE > MERGE ? 4 * TILE : MERGE;
};

// One tile's codes of the lane's key and half of d.
template <int D>
struct Codes {
  uint32_t k[C4<D>::W], v[C4<D>::W];
  uint32_t ks, vs;  // exponents, a byte per block
  bool ok;          // the key is visible and its page is one of the cache's
};

template <int W>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&x)[W]) {
  if constexpr (W == 2) {
    const u32x2 a = *reinterpret_cast<const u32x2*>(p);
    x[0] = a[0], x[1] = a[1];
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const u32x4 a = *reinterpret_cast<const u32x4*>(p + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i + j] = a[j];
    }
  }
}

// Eight codes as values.
template <typename T>
__device__ __forceinline__ typename H16<T>::V8 values8(uint32_t codes, float scale) {
  return __builtin_bit_cast(typename H16<T>::V8,
                            u32x4{Fp4<T>::template unpack<0>(codes, scale), Fp4<T>::template unpack<1>(codes, scale),
                                  Fp4<T>::template unpack<2>(codes, scale), Fp4<T>::template unpack<3>(codes, scale)});
}

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void cache4_attention_kernel(const Cache4AttnParams p) {
  using H = H16<T>;
  using V8 = typename H::V8;
  using V4 = typename H::V4;
  using V2 = typename H::V2;
  using C = C4<D>;
  __shared__ __attribute__((aligned(1024))) char smem[C::LDS];
  __shared__ float red[2][4][32];

  const int tid = threadIdx.x;
  const int lane = tid & 63, h2 = lane >> 5, l32 = lane & 31;
  const int w = (int)uniform32((uint32_t)(tid >> 6));
  const int units = p.R * p.Hk * p.groups;  // requests x key heads x groups of up to 32 query heads
  const int unit = blockIdx.x % units, chunk = blockIdx.x / units;
  const int rg = unit % p.groups, hk = unit / p.groups % p.Hk, r = unit / p.groups / p.Hk;
  const int row = 32 * rg + l32;  // of the key head's G
  const bool live = row < p.G;

  const int len = min(max(p.lens[r], 0), p.most);
  const int pos = len - 1;
  TileList list;
  list.init(pos, pos, p.window, p.sinks);
  const int i0 = chunk * p.chunk, i1 = min(list.n, i0 + p.chunk);
  const int64_t slice = (int64_t)r * p.Hk + hk;
  const int64_t prow = (slice * p.splits + chunk) * p.G + row;
  float* ml = p.part + (int64_t)p.R * p.Hk * p.splits * p.G * D + prow * 2;
  if (i0 >= i1 && p.splits > 1) {  // nothing here: an empty part
    if (w == 0 && h2 == 0 && live) ml[0] = kNoMax, ml[1] = 0.0f;
    return;
  }

  V8 qop[C::NSD];
  {
    const T* src = (const T*)p.q + r * p.sq[0] + (hk * p.G + (live ? row : 0)) * p.sq[1] + h2 * (D / 2);
#pragma unroll
    for (int s = 0; s < C::NSD; ++s) {
      const V8 x = *reinterpret_cast<const V8*>(src + 8 * s);
      qop[s] = live ? x : V8{};
    }
  }
  const float c = p.c;
  const int32_t* table = p.tables + r * p.table_stride;
  const int page = 1 << p.shift;
  const int in_tile = perm32(l32);  // the lane's key of a tile, so that S^T comes out in the order of P^T's operand

  // Page of the lane's key in list entry i; -1 where the key is hidden.
  auto page_of = [&](int i) __attribute__((always_inline)) {
    const int key = 32 * list.at(min(i, i1 - 1)) + in_tile;
    const bool see = i < i1 && key <= pos && (key >= list.lo || key < p.sinks);
    return see ? table[key >> p.shift] : -1;
  };
  auto load = [&](int i, int pg) __attribute__((always_inline)) {
    Codes<D> x;
    const int key = 32 * list.at(min(i, i1 - 1)) + in_tile;
    x.ok = (uint32_t)pg < (uint32_t)p.pages;
    const int64_t at = (((int64_t)(x.ok ? pg : 0) * p.Hk + hk) * 2 << p.shift) + (x.ok ? key & (page - 1) : 0);
    const uint8_t* codes = p.codes + at * (D / 2) + h2 * (D / 4);
    load_words(codes, x.k);
    load_words(codes + ((D / 2) << p.shift), x.v);
    const uint8_t* sc = p.scales + at * (D / 32) + (D >= 64 ? h2 * (D / 64) : 0);
    const uint8_t* sv = sc + ((D / 32) << p.shift);
    if constexpr (D == 128) {
      x.ks = *reinterpret_cast<const uint16_t*>(sc);
      x.vs = *reinterpret_cast<const uint16_t*>(sv);
    } else {
      x.ks = *sc;
      x.vs = *sv;
    }
    return x;
  };

  TATTN_LDS char* vrows = (TATTN_LDS char*)(smem + w * C::TILE);
  int lo[C::DT], hi[C::DT];
#pragma unroll
  for (int u = 0; u < C::DT; ++u) tr_addrs<D>(0, u, lane, lo[u], hi[u]);
  float mrow = kNoMax, lrow = 0.0f;
  f32x16 acc[C::DT];
#pragma unroll
  for (int u = 0; u < C::DT; ++u) acc[u] = f32x16{};

  auto tile = [&](Codes<D>& x) __attribute__((always_inline)) {
    const uint64_t see = __builtin_amdgcn_ballot_w64(x.ok);  // both halves alike: bit m is row m of S^T
    if (see == 0) return;
    const bool masked = see != ~0ull;
    if (masked && !x.ok) {
      // What lies at a hidden key's place reaches nothing.
#pragma unroll
      for (int i = 0; i < C::W; ++i) x.k[i] = x.v[i] = 0;
      x.ks = x.vs = 0x7f7f;
    }
    f32x16 s = f32x16{};
#pragma unroll
    for (int i = 0; i < C::NSD; ++i) {
      const float scale = __builtin_bit_cast(float, ((x.ks >> (8 * (i / 4))) & 255) << 23);
      s = Elt<T>::mfma(values8<T>(x.k[i], scale), qop[i], s);
    }
#pragma unroll
    for (int i = 0; i < C::W; ++i) {
      const float scale = __builtin_bit_cast(float, ((x.vs >> (8 * (i / 4))) & 255) << 23);
      *reinterpret_cast<TATTN_LDS V8*>(vrows + Swz<D>::addr(l32, h2 * D + 16 * i)) = values8<T>(x.v[i], scale);
    }
    // Bit 8 (r / 4) + r % 4 of the half's mask: whether register r's key is visible.
    const uint32_t bits = (uint32_t)see >> (4 * h2);
    V8 pr[2];
    auto probs = [&]() __attribute__((always_inline)) {
      float ps = 0.0f;
#pragma unroll
      for (int sg = 0; sg < 2; ++sg)
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const int a = 8 * sg + i;
          float e0 = fast_exp2(__builtin_fmaf(s[a], c, -mrow)), e1 = fast_exp2(__builtin_fmaf(s[a + 1], c, -mrow));
          if (masked) {
            e0 = bits >> (8 * (a / 4) + a % 4) & 1 ? e0 : 0.0f;
            e1 = bits >> (8 * ((a + 1) / 4) + (a + 1) % 4) & 1 ? e1 : 0.0f;
          }
          const V2 two = H::pack(e0, e1);
          ps = H::sum2(two, ps);
          pr[sg][i] = two[0];
          pr[sg][i + 1] = two[1];
        }
      return ps;
    };
    const float lprev = lrow;
    const float ps = probs();
    lrow += ps;
    if (__builtin_amdgcn_ballot_w64(!(ps <= 4096.0f))) {
      float mx = kNoMax;
#pragma unroll
      for (int a = 0; a < 16; ++a) mx = bits >> (8 * (a / 4) + a % 4) & 1 ? __builtin_fmaxf(mx, s[a] * c) : mx;
      const float cand = max_halves(mx);
      const float mnew = cand > mrow + kRescaleLog2 ? cand : mrow;
      const float alpha = fast_exp2(mrow - mnew);
      mrow = mnew;
      const float again = probs();
      lrow = lprev * alpha + again;
#pragma unroll
      for (int u = 0; u < C::DT; ++u) acc[u] *= alpha;
    }
#pragma unroll
    for (int sg = 0; sg < 2; ++sg)
#pragma unroll
      for (int u = 0; u < C::DT; ++u)
        acc[u] = Elt<T>::mfma(tr_pair<T>((const char*)smem + w * C::TILE + 16 * sg * Swz<D>::RB, lo[u], hi[u]), pr[sg], acc[u]);
  };

  int i = i0 + w;
  if (i < i1) {
    Codes<D> cur = load(i, page_of(i));
    int pg = page_of(i + 4);
    for (; i < i1; i += 4) {
      Codes<D> nxt = load(i + 4, pg);
      pg = page_of(i + 8);
      tile(cur);
      cur = nxt;
    }
  }

  // Join the four waves, one 32-row tile of d at a time; wave w adds four of its columns for every row.
  const float lt = sum_halves(lrow);
  if (h2 == 0) {
    red[0][w][l32] = mrow;
    red[1][w][l32] = lt;
  }
  __syncthreads();
  float mall = kNoMax, lall = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) mall = __builtin_fmaxf(mall, red[0][k][l32]);
#pragma unroll
  for (int k = 0; k < 4; ++k) lall += fast_exp2(red[0][k][l32] - mall) * red[1][k][l32];
  const bool parts = p.splits > 1;
  float wgt = fast_exp2(mrow - mall);
  if (!parts) wgt = lall == 0.0f ? 0.0f : wgt / lall;
  T* orow = (T*)p.out + r * p.so[0] + (hk * p.G + row) * p.so[1];
#pragma unroll
  for (int u = 0; u < C::DT; ++u) {
    TATTN_LDS float* mine = (TATTN_LDS float*)smem + w * 1024 + lane;
#pragma unroll
    for (int a = 0; a < 16; ++a) mine[a * 64] = acc[u][a] * wgt;
    __syncthreads();
    f32x4 x = f32x4{};
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += ((TATTN_LDS float*)smem + k * 1024 + lane)[(4 * w + e) * 64];
    const int d0 = 32 * u + 8 * w + 4 * h2;
    if (live) {
      if (parts) {
        *reinterpret_cast<f32x4*>(p.part + prow * D + d0) = x;
      } else {
        V4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (T)x[e];
        *reinterpret_cast<V4*>(orow + d0) = y;
      }
    }
    __syncthreads();
  }
  if (parts && w == 0 && h2 == 0 && live) ml[0] = mall, ml[1] = lall;
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
  int64_t chunk = tiles * units / 1024;
  chunk = std::min<int64_t>(128, std::max<int64_t>(4, (chunk + 3) / 4 * 4));
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
