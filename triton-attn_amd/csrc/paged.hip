// Pages of a key/value cache on gfx950: which page and slot every new token gets, and the tokens'
// keys and values into and out of a cache held in 4 bits.
#include "common.h"
#include "fp4.h"
#include "ops.h"

namespace tattn {
namespace {

// ---- pages and slots ---------------------------------------------------------------------------
// Request r holds len_r tokens and adds new_r. Its pages up to ceil(len_r / page) are in its table row;
// the next need_r = ceil((len_r + new_r) / page) - ceil(len_r / page) come from the free list, in request
// order: page i of them is free[sum of need before r + i]. A token at position p lies in slot
// row[p / page] * page + p % page.
//
// Both sums run over the requests before r, so every workgroup walks the requests from the first
// on (1,024 per round, four a thread, 8 bytes each, out of L2 after the first) until it has
// passed its own 1,024 tokens. That repeats a few hundred nanoseconds of scanning per workgroup
// and needs no second launch, no flag between workgroups and no workspace. Each fresh page starts with
// a new token (the request had filled the pages before), so the thread of that token writes its table entry,
// and reads for older pages never meet a write. Latency-bound: 4.7 us for 256 requests of one token, 8.7 us for 64
// requests of 2,048, less than the call takes on the host.
constexpr int kTokens = 1024;  // tokens per workgroup
constexpr int kRound = 1024;   // requests per round

// Exclusive sum over the workgroup's 256 threads; `total` is the sum of all.
__device__ __forceinline__ int64_t scan_exclusive(int64_t x, int64_t* part, int64_t& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int64_t s = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t y = __shfl_up(s, d);
    if (lane >= d) s += y;
  }
  if (lane == 63) part[w] = s;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < w) before += part[i];
    total += part[i];
  }
  __syncthreads();
  return before + s - x;
}

__global__ __launch_bounds__(256) void page_tables_kernel(const TablesParams p) {
  __shared__ int64_t part[4];
  __shared__ int32_t first[kRound + 1];  // first token of the round's requests
  __shared__ int32_t held[kRound];       // tokens they hold
  __shared__ int64_t page0[kRound];      // where their fresh pages start in the free list
  const int tid = threadIdx.x;
  const int page = 1 << p.shift;
  const int64_t lo = (int64_t)blockIdx.x * kTokens, hi = lo + kTokens < p.T ? lo + kTokens : p.T;
  const bool lead = blockIdx.x == 0;

  int64_t tokens = 0, pages = 0;  // of the requests before the round
  for (int r0 = 0; r0 < p.R && (lead || tokens < hi); r0 += kRound) {
    int64_t add[4];
    int32_t len[4];
    int64_t sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + 4 * tid + i;
      len[i] = r < p.R ? p.lens[r] : 0;
      const int32_t a = r < p.R ? p.add[r] : 0;
      len[i] = len[i] > 0 ? len[i] : 0;
      add[i] = a > 0 ? a : 0;
      sum += add[i];
    }
    int64_t round_tokens, round_pages;
    int64_t at = tokens + scan_exclusive(sum, part, round_tokens);
    int64_t need[4], start[5];
    sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      start[i] = at < p.T ? at : p.T;  // tokens past the list's end are not placed
      at += add[i];
      start[i + 1] = at < p.T ? at : p.T;
      const int64_t have = ((int64_t)len[i] + page - 1) >> p.shift;
      const int64_t want = ((int64_t)len[i] + (start[i + 1] - start[i]) + page - 1) >> p.shift;
      const int64_t end = want < p.P ? want : p.P;  // a table row holds P pages
      need[i] = end > have ? end - have : 0;
      sum += need[i];
    }
    int64_t pg = pages + scan_exclusive(sum, part, round_pages);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = 4 * tid + i;
      first[j] = (int32_t)start[i];
      if (j == kRound - 1) first[kRound] = (int32_t)start[4];
      held[j] = len[i];
      page0[j] = pg;
      pg += need[i];
      if (lead && r0 + j < p.R) p.starts[r0 + j] = (int32_t)start[i];
    }
    __syncthreads();
    const int64_t from = first[0] > lo ? first[0] : lo, to = first[kRound] < hi ? first[kRound] : hi;
    for (int64_t t = from + tid; t < to; t += 256) {
      int a = 0, b = kRound;  // first[a] <= t < first[b]
      while (b - a > 1) {
        const int m = (a + b) >> 1;
        if (first[m] <= t) a = m;
        else b = m;
      }
      const int64_t pos = (int64_t)held[a] + (t - first[a]);
      const int64_t have = ((int64_t)held[a] + page - 1) >> p.shift, idx = pos >> p.shift;
      int32_t* row = p.tables + (int64_t)(r0 + a) * p.table_stride;
      int32_t pageno = -1;
      if (idx < p.P) {
        if (idx < have) {
          pageno = row[idx];
        } else {
          const int64_t f = page0[a] + (idx - have);
          if (f < p.F) pageno = p.free_pages[f];
          if ((pos & (page - 1)) == 0) row[idx] = pageno;
        }
      }
      p.slots[t] = pageno < 0 ? -1 : ((int64_t)pageno << p.shift) + (pos & (page - 1));
      p.positions[t] = (int32_t)(pos < 0x7fffffff ? pos : 0x7fffffff);
    }
    tokens += round_tokens;
    pages += round_pages;
    __syncthreads();
  }
  const int64_t end = tokens < p.T ? tokens : p.T;
  for (int64_t t = (end > lo ? end : lo) + tid; t < hi; t += 256) {  // behind the last request
    p.slots[t] = -1;
    p.positions[t] = 0;
  }
  if (lead && tid == 0) {
    p.starts[p.R] = (int32_t)end;
    p.taken[0] = (int32_t)(pages < 0x7fffffff ? pages : 0x7fffffff);
  }
}

// ---- cache in 4 bits -----------------------------------------------------------------------------
// A block of 32 values along d is held as e2m1 codes times 2^e: e is the smallest exponent at which
// the block's largest magnitude rounds to 6 or less, e = floor(log2 amax) - 2, one more where amax / 2^e
// is 7 or more (7 lies between 6 and the missing 8 and would go to 8), and at most the exponent at which
// 6 * 2^e is finite in the element type (larger magnitudes become 6 * 2^e). v_cvt_scalef32_pk_fp4 divides by
// 2^e and rounds to nearest even in one instruction; every step is exact but that rounding. A block with
// an infinity or a NaN is held as NaN (exponent byte 255); magnitudes below 2^-120 count as zero, which
// keeps every held value a normal number of the element type's exponent range.
//
// Bound by bytes: 16 values a thread (two 16-byte loads, one 8-byte store), a workgroup takes one head of
// 2048 / D consecutive tokens, keys and values, so that its codes and exponents fill whole lines of a page. 16,384 tokens
// of 8 heads x 128 in bf16 are written in 13.6-14.5 us and read in 16.5 (5.9-6.2 and 5.1 TB/s of their 85 MB; a kernel that copies has
// 5.7, one that writes 6.0).

// Row x of a workgroup's 256 / (D / 16) rows: token, K (0) or V (1), and the thread's 16 values.
template <int D>
struct Rows {
  static constexpr int TPR = D / 16, TB = 128 / TPR;  // threads per row, tokens per workgroup
  int64_t slot;
  int t, kv, c;
  bool live;
  __device__ __forceinline__ void init(const Cache4Params& p) {
    const int row = threadIdx.x / TPR;
    c = threadIdx.x % TPR;
    kv = row / TB;
    t = blockIdx.x / p.H * TB + row % TB;
    live = t < p.T;
    slot = live ? p.slots[t] : -1;
  }
  // Row of the cache (token and kv of this head) as an index into its [.., page] dimension.
  __device__ __forceinline__ int64_t cache_row(const Cache4Params& p, int h) const {
    const int64_t pageno = slot >> p.shift, in = slot & ((1ll << p.shift) - 1);
    return (((pageno * p.H + h) * 2 + kv) << p.shift) + in;
  }
};

template <typename T, int D>
__global__ __launch_bounds__(256) void cache4_write_kernel(const Cache4Params p) {
  using F = Fp4<T>;
  Rows<D> r;
  r.init(p);
  const int h = blockIdx.x % p.H;
  const bool in = r.slot >= 0 && r.slot < p.total;
  u32x4 x[2] = {};
  if (in) {
    const T* src = (const T*)(r.kv ? p.v : p.k) + (int64_t)r.t * (r.kv ? p.sv[0] : p.sk[0]) + h * (r.kv ? p.sv[1] : p.sk[1]) + 16 * r.c;
    x[0] = ld16(src);
    x[1] = ld16(src + 8);
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w = x[i >> 2][i & 3];
    const uint32_t a = w & 0x7fff, b = (w >> 16) & 0x7fff;
    top = max(top, max(a, b));
  }
  top = max(top, (uint32_t)__shfl_xor((int)top, 1));  // the block's other half
  const uint32_t bits = F::exponent(top);
  uint32_t e = (bits >> 23) - 2 + ((bits & 0x7fffff) >= 0x600000 ? 1 : 0);
  const bool nan = top >= F::kInf, zero = (bits >> 23) < 7;  // below 2^-120
  e = nan ? 255 : zero ? 1 : min(e, F::kTop);
  const float scale = __builtin_bit_cast(float, (nan ? 127u : e) << 23);
  uint32_t codes[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    codes[i] = F::template pack<0>(codes[i], x[i][0], scale);
    codes[i] = F::template pack<1>(codes[i], x[i][1], scale);
    codes[i] = F::template pack<2>(codes[i], x[i][2], scale);
    codes[i] = F::template pack<3>(codes[i], x[i][3], scale);
    if (nan || zero) codes[i] = 0;
  }
  if (!in) return;
  const int64_t row = r.cache_row(p, h);
  *reinterpret_cast<u32x2*>(p.codes + row * (D / 2) + 8 * r.c) = u32x2{codes[0], codes[1]};
  if ((r.c & 1) == 0) p.scales[row * (D / 32) + (r.c >> 1)] = (uint8_t)e;
}

template <typename T, int D>
__global__ __launch_bounds__(256) void cache4_read_kernel(const Cache4Params p) {
  using F = Fp4<T>;
  Rows<D> r;
  r.init(p);
  if (!r.live) return;
  const int h = blockIdx.x % p.H;
  u32x4 x[2] = {};
  if (r.slot >= 0 && r.slot < p.total) {
    const int64_t row = r.cache_row(p, h);
    const u32x2 c = *reinterpret_cast<const u32x2*>(p.codes + row * (D / 2) + 8 * r.c);
    const uint32_t e = p.scales[row * (D / 32) + (r.c >> 1)];
    const float scale = __builtin_bit_cast(float, e << 23);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[i] = u32x4{F::template unpack<0>(c[i], scale), F::template unpack<1>(c[i], scale),
                   F::template unpack<2>(c[i], scale), F::template unpack<3>(c[i], scale)};
    }
  }
  T* dst = (T*)(r.kv ? p.vo : p.ko) + ((int64_t)r.t * p.H + h) * D + 16 * r.c;
  st16(dst, x[0]);
  st16(dst + 8, x[1]);
}

template <typename T, int D>
int launch_cache4(const Cache4Params& p, bool write, hipStream_t st) {
  const int64_t blocks = ((int64_t)p.T + Rows<D>::TB - 1) / Rows<D>::TB * p.H;
  if (blocks > 0x7fffffff) return set_error(TATTN_E_ARG, "grid too large: %lld workgroups", (long long)blocks);
  if (write) cache4_write_kernel<T, D><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(p);
  else cache4_read_kernel<T, D><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(p);
  return check_launch(write ? "tattn_cache4_write" : "tattn_cache4_read");
}

int dispatch_cache4(const Cache4Params& p, int D, int dtype, bool write, hipStream_t st) {
  const bool h = dtype == 0;
  switch (D) {
    case 32: return h ? launch_cache4<f16, 32>(p, write, st) : launch_cache4<bf16, 32>(p, write, st);
    case 64: return h ? launch_cache4<f16, 64>(p, write, st) : launch_cache4<bf16, 64>(p, write, st);
    case 128: return h ? launch_cache4<f16, 128>(p, write, st) : launch_cache4<bf16, 128>(p, write, st);
  }
  return set_error(TATTN_E_ARG, "head dim must be 32, 64 or 128, got %d", D);
}

}  // namespace

int launch_page_tables(const TablesParams& p, hipStream_t st) {
  const unsigned blocks = p.T > 0 ? (unsigned)(((int64_t)p.T + kTokens - 1) / kTokens) : 1u;
  page_tables_kernel<<<dim3(blocks), dim3(256), 0, st>>>(p);
  return check_launch("tattn_page_tables");
}

int launch_cache4_write(const Cache4Params& p, int D, int dtype, hipStream_t st) {
  return dispatch_cache4(p, D, dtype, true, st);
}
int launch_cache4_read(const Cache4Params& p, int D, int dtype, hipStream_t st) {
  return dispatch_cache4(p, D, dtype, false, st);
}

}  // namespace tattn
