// One step of sequences behind a shared prefix, on gfx950: attention of their newest tokens to the prefix, read once for all rows of
// its group, and to each sequence's own keys, in one launch. Both write parts, joined in order by combine_kernel of cross.hip.
#include <algorithm>
#include <type_traits>

#include "cross_pipe.h"
#include "cross_rows.h"

namespace tattn {
namespace {

// Workgroups that a CU holds: at head dim 64 registers for rows walked together.
constexpr int prefix_occ(int D) { return D == 64 ? 3 : rows_occ(D); }

// Workgroups over the prefix, the row blocks that read one part of it on one XCD, whose L2 hands it to the others.
__host__ __device__ inline int64_t prefix_blocks(const CrossParams& p) { return ((int64_t)p.Zs * p.Hk * p.splits + 7) / 8 * 8 * p.nblk; }

// All of a launch.
int64_t prefix_launch(const PrefixParams& p) { return prefix_blocks(p.pre) + p.own.slices() * p.own.nblk * p.own.splits; }

// The prefix's parts first, then each sequence's own keys.
template <typename T, int D>
__global__ __launch_bounds__(4 * 64, prefix_occ(D)) void prefix_kernel(const PrefixParams p) {
  constexpr int STAGE = 2 * CrossTile<D>::BYTES;
  __shared__ __attribute__((aligned(1024))) char st0[STAGE], st1[STAGE], st2[STAGE], st3[STAGE];
  __shared__ float red[2][4][32];
  const int total = (int)prefix_blocks(p.pre);
  int i = blockIdx.x;
  if (i < total) {
    const int l = i >> 3, unit = 8 * (l / p.pre.nblk) + (i & 7), slice = unit / p.pre.splits;
    if (slice >= p.pre.Zs * p.pre.Hk) return;
    if (p.pre.pipe) pipe_block<T, D, 4, 1>(p.pre, slice, l % p.pre.nblk, unit % p.pre.splits, st0, st1, st2, st3);
    else rows_block<T, D, 4, false, 2>(p.pre, slice, l % p.pre.nblk, unit % p.pre.splits, {{st0, st1}, {st2, st3}, red});
    return;
  }
  i -= total;
  const int per = p.own.nblk * p.own.splits, blk = i % per;
  rows_block<T, D, 4, true, 2>(p.own, i / per, blk / p.own.splits, blk % p.own.splits, {{st0, st1}, {st2, st3}, red});
}

template <typename T, int D>
int prefix_d(const PrefixParams& p, hipStream_t st) {
  const int64_t blocks = prefix_launch(p);
  if (int rc = check_grid(blocks, 256)) return rc;
  prefix_kernel<T, D><<<dim3((unsigned)blocks), dim3(4 * 64), 0, st>>>(p);
  const int rc = check_launch("tattn_prefix_attention");
  return rc ? rc : launch_prefix_combine(p, D, std::is_same_v<T, f16> ? 0 : 2, st);
}

}  // namespace

// More than 32 rows behind a prefix are walked by all waves together, 128 a workgroup: each part of the prefix is then read once for
// them. Parts are as long as an even share of all tiles over the places that the chip has (a workgroup over a sequence's own keys
// counts eight tiles more, for what it costs besides), those of own keys three quarters of that; none has less than eight tiles,
// nor less than sixteen where rows are walked together. us, keys not in a cache, at shares of (prefix, own):
//                                                            32 rows a workgroup (1, 1/2)   (1, 1/2)   (1, 3/4)   (1, 1)   (3/2, 1)
//   64 requests x 32/8 x 128, prefix 8,192, up to 1,024 own keys                       60         52         53       52         62
//   8 x 16 samples x 16/4 x 128, prefixes to 4,096, up to 2,048                         79         79         79       81         81
//   64 requests x 32/8 x 64, prefix 8,192, up to 1,024                                  38         31         31       32         35
//   256 requests x 32/8 x 128, prefix 4,096, up to 256                                  78         60         60       60         60
//   128 x 16 x 5 queries x 128, prefix 8,192, up to 64                                  99         73         73       73         72
//   8 requests x 32/8 x 128 (32 rows), prefix 32,768, up to 512                         40         39         39       37         41
//   2 x 32 requests x 16/8 x 128, prefixes of 2,000, up to 500                           -         33         29       29         37
int prefix_plan(PrefixParams& p, int D) {
  const int64_t pt = std::max<int64_t>(1, ((int64_t)p.pre.S + 31) / 32), ot = std::max<int64_t>(1, ((int64_t)p.own.S + 31) / 32);
  p.pre.pipe = p.pre.rows() > 32;
  const int64_t block = p.pre.pipe ? 128 : 32;
  p.pre.nblk = (int)((p.pre.rows() + block - 1) / block);
  p.own.nblk = (int)((p.own.rows() + 31) / 32);
  const int64_t share = (p.pre.slices() * p.pre.nblk * pt + p.own.slices() * p.own.nblk * (ot + 8)) / (256 * prefix_occ(D));
  const int64_t shared = std::max<int64_t>(p.pre.pipe ? 16 : 8, share), own = std::max<int64_t>(8, share * 3 / 4);
  p.pre.splits = (int)((pt + shared - 1) / shared);
  p.own.splits = (int)((ot + own - 1) / own);
  p.pre.joined = p.own.joined = 1;
  const int rc = check_grid(prefix_launch(p), 256);
  if (rc) return rc;
  int32_t dealt;
  return check_grid(combine_blocks(p.pre.slices() * p.pre.rows(), std::max(p.pre.splits, p.own.splits), D, dealt), 256);
}
int64_t prefix_floats(const PrefixParams& p, int D) {
  return cross_part_floats(p.pre.slices(), p.pre.rows(), p.pre.splits, D) + cross_part_floats(p.own.slices(), p.own.rows(), p.own.splits, D);
}

int launch_prefix(const PrefixParams& p, int D, int dtype, hipStream_t st) {
  switch (D) {
    case 16: return dtype == 0 ? prefix_d<f16, 16>(p, st) : prefix_d<bf16, 16>(p, st);
    case 32: return dtype == 0 ? prefix_d<f16, 32>(p, st) : prefix_d<bf16, 32>(p, st);
    case 64: return dtype == 0 ? prefix_d<f16, 64>(p, st) : prefix_d<bf16, 64>(p, st);
    case 128: return dtype == 0 ? prefix_d<f16, 128>(p, st) : prefix_d<bf16, 128>(p, st);
  }
  return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %d", D);
}

}  // namespace tattn
