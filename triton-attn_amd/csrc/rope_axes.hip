// Rotation of query and key heads by positions on several axes (time, height, width), with or without their norms, and the
// gradients, on gfx950. The mathematics and the layout of norm_rope.hip; a pair's angle is that of its own axis's position.
// Without norms the rotation is linear: the gradient turns dy back by the same kernel and reads no x.
//
// Bound by bytes: x in and y out. The angles of a token are looked up once for four heads; their tables stay in the caches. Forward
// and gradients with their launches, us (floor of a copy): 2 x 24 + 24 heads x 21,601 x 128 bf16 393 (376); 16 x 16 + 16 x 4,097 x 64 fp16
// with norms 269 (239).
#include <type_traits>

#include "norm_rope.h"

namespace tattn {
namespace {

template <typename T, int D, bool NORM>
int turn_d(const RopeAxesParams& p, bool interleaved, hipStream_t st, const char* what) {
  constexpr uint32_t GROUPS = 256 / RowCfg<T, D>::LPR;
  const dim3 grid((p.units_q + p.units_k + GROUPS - 1) / GROUPS), block(256);
  if (interleaved) norm_rope_fwd_kernel<T, D, true, RopeAxesParams, NORM><<<grid, block, 0, st>>>(p);
  else norm_rope_fwd_kernel<T, D, false, RopeAxesParams, NORM><<<grid, block, 0, st>>>(p);
  return check_launch(what);
}

template <typename T, int D>
int run_d(RopeAxesParams p, bool interleaved, bool bwd, hipStream_t st) {
  if (!bwd) return p.qw ? turn_d<T, D, true>(p, interleaved, st, "tattn_rope_axes_fwd") : turn_d<T, D, false>(p, interleaved, st, "tattn_rope_axes_fwd");
  if (!p.qw) return turn_d<T, D, false>(p, interleaved, st, "tattn_rope_axes_bwd");
  norm_rope_bwd_blocks<T, D>(p);
  const dim3 grid(p.blocks_q + p.blocks_k), block(kBwdThreads);
  if (interleaved) norm_rope_bwd_kernel<T, D, true, RopeAxesParams><<<grid, block, 0, st>>>(p);
  else norm_rope_bwd_kernel<T, D, false, RopeAxesParams><<<grid, block, 0, st>>>(p);
  const int rc = check_launch("tattn_rope_axes_bwd");
  return rc || !p.partial ? rc : launch_norm_rope_dw(p, D, std::is_same_v<T, float> ? 1 : std::is_same_v<T, f16> ? 0 : 2, st);
}

template <typename T>
int run(const RopeAxesParams& p, int D, bool interleaved, bool bwd, hipStream_t st) {
  switch (D) {
    case 16: return run_d<T, 16>(p, interleaved, bwd, st);
    case 32: return run_d<T, 32>(p, interleaved, bwd, st);
    case 64: return run_d<T, 64>(p, interleaved, bwd, st);
    case 128: return run_d<T, 128>(p, interleaved, bwd, st);
  }
  return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %d", D);
}

}  // namespace

int launch_rope_axes(const RopeAxesParams& p, int D, int dtype, bool interleaved, bool bwd, hipStream_t st) {
  if (dtype == 0) return run<f16>(p, D, interleaved, bwd, st);
  if (dtype == 2) return run<bf16>(p, D, interleaved, bwd, st);
  return run<float>(p, D, interleaved, bwd, st);
}

}  // namespace tattn
