// Attention over keys of another length, 16-bit forward where there are many rows, on gfx950.
// cross_pipe.h has the schedule.
//
// Bound by the issue of matrix and vector instructions, as far as the card's clock goes under them. us (rate), whole calls:
//   1 x 32/8 x 8,192 rows over 16,384 x 128 bf16   1,836 (1,196 TF; an 8,192^3 product reaches 1,208 to 1,357)
//   4 x 32/8 x 4,096 over 4,096 x 128 bf16           940 (1,169 TF)
//   4 x 16 x 4,096 over 4,096 x 64 fp16              272 (1,010 TF): twice the exponentials for a product
// Eight waves take 1,782, 941 and 271, and 79 us where four take 53 (8 x 16 x 1,024 over 375 to 1,500 x 64: fewer, larger blocks).
#include <algorithm>
#include <type_traits>

#include "cross_pipe.h"

namespace tattn {
namespace {

template <typename T, int D, int NW, int QT, int OCC>
__global__ __launch_bounds__(NW * 64, OCC) void cross_pipe_kernel(const CrossParams p) {
  constexpr int STAGE = 2 * CrossTile<D>::BYTES;
  __shared__ __attribute__((aligned(1024))) char st0[STAGE], st1[STAGE], st2[STAGE], st3[STAGE];
  int slice, blk;
  if (!cross_coord(p, p.nblk * p.splits, slice, blk)) return;
  pipe_block<T, D, NW, QT>(p, slice, blk / p.splits, blk % p.splits, st0, st1, st2, st3);
}

template <typename T, int D>
int pipe_d(const CrossParams& p, hipStream_t st) {
  constexpr int NW = cross_pipe_waves(D);
  unsigned blocks;
  if (int rc = cross_grid(p.slices(), (int64_t)p.nblk * p.splits, 64 * NW, &blocks)) return rc;
  cross_pipe_kernel<T, D, NW, cross_pipe_tiles(D), 2><<<dim3(blocks), dim3(NW * 64), 0, st>>>(p);
  return check_launch("tattn_cross_fwd");
}

}  // namespace

int launch_cross_pipe(const CrossParams& p, int D, int dtype, hipStream_t st) {
  switch (D) {
    case 16: return dtype == 0 ? pipe_d<f16, 16>(p, st) : pipe_d<bf16, 16>(p, st);
    case 32: return dtype == 0 ? pipe_d<f16, 32>(p, st) : pipe_d<bf16, 32>(p, st);
    case 64: return dtype == 0 ? pipe_d<f16, 64>(p, st) : pipe_d<bf16, 64>(p, st);
    case 128: return dtype == 0 ? pipe_d<f16, 128>(p, st) : pipe_d<bf16, 128>(p, st);
  }
  return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %d", D);
}

}  // namespace tattn
