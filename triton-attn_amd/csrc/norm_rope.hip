// Root-mean-square norm of every query and key head and the position rotation, in one pass, and
// its gradients, on gfx950.
//
//   y = x r w,  r = 1 / sqrt(mean(x^2) + eps);  (a, b) of y -> (a cos - b sin, b cos + a sin)
//   with t the gradient turned back by the same angles: dw = sum over rows of t x r,
//   u = t w,  dx = r (u - x r mean(u x r))
//
// The pairs are (i, i + D/2), or (2i, 2i + 1) when interleaved. Everything is float32 between the
// load and the one rounding of each result.
//
// Bound by bytes: x in and y out, or x and dy in and dx out (r is computed again: reading it back would
// save a reduction that hides behind the loads). A row belongs to D / 2 elements / 16 bytes lanes; a
// lane holds 16 bytes of the row's lower half and the 16 bytes D/2 further, so either kind of pair lies in one lane
// and the row's sum takes at most four lane swaps. A lane group takes up to four heads of one token, whose
// position, cosines, sines and weights it loads once, and has all their loads in flight together. At 4 x 32/8 x 4,096 x 128
// in bf16 the forward takes 61-65 us (5.3-5.5 TB/s) and the backward 104 and 5 us (4.8 TB/s), in float32 124 (5.5) and
// 203 us (5.0); a kernel that copies has 5.7 TB/s.
#include <type_traits>

#include "norm_rope.h"

namespace tattn {
namespace {

// Column sums of the partial rows [first, first + rows): 16 columns a workgroup, 16 rows at a time.
template <typename W>
__global__ __launch_bounds__(256) void norm_rope_dw_kernel(const float* partial, W* qw, W* kw, int D, int rows_q, int rows_k) {
  __shared__ float s[16][16];
  const int col = threadIdx.x & 15, row = threadIdx.x >> 4;
  const int per = D / 16;
  const bool is_k = (int)blockIdx.x >= per;
  const int d = ((int)blockIdx.x - (is_k ? per : 0)) * 16 + col;
  const int first = is_k ? rows_q : 0, rows = is_k ? rows_k : rows_q;
  float a = 0.0f;
#pragma unroll 8
  for (int i = row; i < rows; i += 16) a += partial[(int64_t)(first + i) * D + d];
  s[row][col] = a;
  __syncthreads();
  if (row == 0) {
#pragma unroll
    for (int i = 1; i < 16; ++i) a += s[i][col];
    (is_k ? kw : qw)[d] = (W)a;
  }
}

template <typename T, int D>
int fwd_d(const NormRopeParams& p, bool interleaved, hipStream_t st) {
  constexpr uint32_t GROUPS = 256 / RowCfg<T, D>::LPR;
  const dim3 grid((p.units_q + p.units_k + GROUPS - 1) / GROUPS), block(256);
  if (interleaved) norm_rope_fwd_kernel<T, D, true, NormRopeParams, true><<<grid, block, 0, st>>>(p);
  else norm_rope_fwd_kernel<T, D, false, NormRopeParams, true><<<grid, block, 0, st>>>(p);
  return check_launch("tattn_norm_rope_fwd");
}

template <typename T, int D>
int bwd_d(NormRopeParams p, bool interleaved, hipStream_t st) {
  norm_rope_bwd_blocks<T, D>(p);
  const dim3 grid(p.blocks_q + p.blocks_k), block(kBwdThreads);
  if (interleaved) norm_rope_bwd_kernel<T, D, true, NormRopeParams><<<grid, block, 0, st>>>(p);
  else norm_rope_bwd_kernel<T, D, false, NormRopeParams><<<grid, block, 0, st>>>(p);
  int rc = check_launch("tattn_norm_rope_bwd");
  if (rc || !p.partial) return rc;
  return launch_norm_rope_dw(p, D, std::is_same_v<T, float> ? 1 : std::is_same_v<T, f16> ? 0 : 2, st);
}

template <typename T>
int run(const NormRopeParams& p, int D, bool interleaved, bool bwd, hipStream_t st) {
  switch (D) {
    case 16: return bwd ? bwd_d<T, 16>(p, interleaved, st) : fwd_d<T, 16>(p, interleaved, st);
    case 32: return bwd ? bwd_d<T, 32>(p, interleaved, st) : fwd_d<T, 32>(p, interleaved, st);
    case 64: return bwd ? bwd_d<T, 64>(p, interleaved, st) : fwd_d<T, 64>(p, interleaved, st);
    case 128: return bwd ? bwd_d<T, 128>(p, interleaved, st) : fwd_d<T, 128>(p, interleaved, st);
  }
  return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %d", D);
}

}  // namespace

// The workgroups' sums of the weights' gradients, in the weights' type.
int launch_norm_rope_dw(const NormRopeParams& p, int D, int dtype, hipStream_t st) {
  const dim3 cols(2 * D / 16), block(256);
  if (p.wide_w || dtype == 1)
    norm_rope_dw_kernel<float><<<cols, block, 0, st>>>(p.partial, (float*)p.dqw, (float*)p.dkw, D, p.blocks_q, p.blocks_k);
  else if (dtype == 0)
    norm_rope_dw_kernel<f16><<<cols, block, 0, st>>>(p.partial, (f16*)p.dqw, (f16*)p.dkw, D, p.blocks_q, p.blocks_k);
  else
    norm_rope_dw_kernel<bf16><<<cols, block, 0, st>>>(p.partial, (bf16*)p.dqw, (bf16*)p.dkw, D, p.blocks_q, p.blocks_k);
  return check_launch("tattn_norm_rope_bwd");
}

int launch_norm_rope(const NormRopeParams& p, int D, int dtype, bool interleaved, bool bwd, hipStream_t st) {
  if (dtype == 0) return run<f16>(p, D, interleaved, bwd, st);
  if (dtype == 2) return run<bf16>(p, D, interleaved, bwd, st);
  return run<float>(p, D, interleaved, bwd, st);
}

}  // namespace tattn
