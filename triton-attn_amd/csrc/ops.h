// Host-side launchers of the operators around attention: page bookkeeping, the cache in 4 bits,
// norms with rotation, window attention, attention over other lengths and shared prefixes. Arguments are checked by the entry points (abi_ops.hip).
#pragma once

#include <algorithm>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch.h"

namespace tattn {

// The current device runs these kernels: TATTN_OK or an error code with its message.
int require_device();

struct TablesParams {
  const int32_t* lens;
  const int32_t* add;
  int32_t* tables;
  const int32_t* free_pages;
  int64_t* slots;
  int32_t* positions;
  int32_t* starts;
  int32_t* taken;
  int64_t table_stride;
  int32_t R, P, F, T;
  int32_t shift;  // log2 of the page size
};
int launch_page_tables(const TablesParams& p, hipStream_t st);

// The cache in 4 bits: codes [pages, heads, 2, page, d / 2], scales [pages, heads, 2, page, d / 32].
struct Cache4Params {
  uint8_t* codes;
  uint8_t* scales;
  const void* k;  // written: [T, heads, d] with the strides below
  const void* v;
  void* ko;  // read: [T, heads, d] contiguous
  void* vo;
  const int64_t* slots;
  int64_t sk[2], sv[2];  // (token, head) strides of k and v in elements
  int64_t total;         // slots of the cache
  int32_t T, H;
  int32_t shift;  // log2 of the page size
};
int launch_cache4_write(const Cache4Params& p, int D, int dtype, hipStream_t st);
int launch_cache4_read(const Cache4Params& p, int D, int dtype, hipStream_t st);

// Norm and rotation of q [Z, H, N, D] and k [Z, Hk, N, D]; strides (z, h, n) in elements, unit d stride.
constexpr int kNormRopeRows = 512;  // most workgroups of the backward: rows of its workspace
struct NormRopeParams {
  const void* q;
  const void* k;
  const void* qw;
  const void* kw;
  const float* cos;  // [P, D / 2]
  const float* sin;
  const int32_t* positions;  // [N] or [Z, N]; null: n
  const void* gq;            // backward: gradients of the outputs
  const void* gk;
  void* qo;  // outputs; backward: gradients of q and k
  void* ko;
  void* dqw;
  void* dkw;
  float* partial;  // [kNormRopeRows, D]; null: no weight gradients
  int64_t sq[3], sk[3], sqo[3], sko[3], sgq[3], sgk[3];
  int64_t pos_stride;  // of z
  int32_t Z, H, Hk, N, P;
  int32_t wide_w;  // weights are float32 (else the tensors' type)
  float eps;
  uint32_t per_q, per_k;      // lane groups' work units per token
  uint32_t units_q, units_k;
  int32_t blocks_q, blocks_k;
};
int launch_norm_rope(const NormRopeParams& p, int D, int dtype, bool interleaved, bool bwd, hipStream_t st);
int launch_norm_rope_dw(const NormRopeParams& p, int D, int dtype, hipStream_t st);

// The same with several axes: positions [axes, N] or [axes, Z, N], an axis for each pair; the norm is left out without weights.
constexpr uint32_t kNoAxis = 15;
struct RopeAxesParams : NormRopeParams {
  alignas(4) uint8_t axes[32];  // four bits a pair, the first in the low ones; kNoAxis: not turned
  int64_t axis_stride;
  int32_t quads;  // pairs 4 i .. 4 i + 3 share an axis
  float sign;     // without norms: -1 turns back
};
int launch_rope_axes(const RopeAxesParams& p, int D, int dtype, bool interleaved, bool bwd, hipStream_t st);

// Attention over a window and the first keys (window.h). q, o, do, dq: [Z, H, N, D]; k, v, dk, dv: [Z, Hk, S, D].
struct WindowParams {
  const void* q;
  const void* k;
  const void* v;
  const void* o;  // backward: the forward's output
  const void* dout;
  void* out;  // forward: O; backward: dQ
  void* dk;
  void* dv;
  float* m;      // [Z, H, N] base-2 log-sum-exp, or null
  float* delta;  // [Z, H, N]
  float* norms;  // fp16 backward: [Z, Hk, window_norm_blocks, 2], largest squared norm of dO's rows, largest |delta|
  const int32_t* lens;  // [Z] keys of each sequence, or null: S
  float* part;          // partial rows of a split forward, see window_part_floats; partial dK, dV of the first keys
  int64_t sq[3], sk[3], sv[3], so[3], sd[3], sout[3], sdk[3], sdv[3];
  int32_t Z, H, Hk, G, N, S;
  int32_t window, sinks;
  int32_t nblk;
  int32_t splits;  // forward: parts of a row's keys; backward: parts of the first keys' queries
  int32_t parts;   // backward: parts of the other keys' queries
  int32_t head, tail;  // blocks of a slice that are placed first and last (window_coord)
  float c, scale;
};

// Partial rows of a forward split `splits` ways: for each split and row D sums, then its max and sum.
inline int64_t window_part_floats(int64_t slices, int64_t rows, int64_t splits, int64_t D) {
  return slices * rows * splits * (D + 2);
}
// Blocks of 128 rows (queries with their heads) of a slice, as dQ's workgroups take them.
__host__ __device__ inline int window_norm_blocks(int64_t N, int64_t G) { return (int)((N * G + 127) / 128); }
int window_fwd_splits(const WindowParams& p, int D);  // 0: no parts and two row tiles per workgroup
void window_bwd_parts(WindowParams& p, int D);  // sets splits and parts
int64_t window_bwd_part_floats(const WindowParams& p, int D);
// How many of a slice's `blocks` row blocks (of `rows` rows with their heads) or key blocks (of `keys` keys) are placed last
// (window_coord): those that the ends of the sequence make shorter, queries before a whole window and keys that fewer than a
// window of queries follow, where they are a fifth of all or more. At 4 x 16 x 4,096 x 64, window 1,024, the last workgroups
// then end together (forward 109 -> 101 us, dQ 133 -> 125, dK / dV 215 -> 203), causal 2 x 16/8 x 8,192 x 128 gains 3% and 1.5%;
// a few such blocks gain nothing and can fill a round of their own (32,768 x 16/4 x 64, window 128: backward 159 -> 167 us).
inline int window_tail(int64_t few, int64_t blocks) { return few * 5 >= blocks ? (int)(few < blocks ? few : blocks) : 0; }
inline int window_row_tail(const WindowParams& p, int rows, int blocks) {
  const int64_t head = std::max<int64_t>(0, std::min<int64_t>((int64_t)p.window - (p.S - p.N), p.N));
  return window_tail((head * p.G + rows - 1) / rows, blocks);
}
inline int window_key_tail(const WindowParams& p, int keys, int blocks) {
  return window_tail((std::min<int64_t>(p.window, p.S) + keys - 1) / keys, blocks);
}
// Workgroups of a launch over `slices` slices of `blocks` blocks, `apart` of them placed first or last (window_coord).
inline int window_grid(int64_t slices, int64_t blocks, int64_t apart, unsigned* out) {
  const int64_t n = (slices * (blocks - apart) + 7) / 8 * 8 + slices * apart;
  if (n > 0x7ffffff) return set_error(TATTN_E_ARG, "grid too large: %lld workgroups", (long long)n);
  *out = (unsigned)n;
  return TATTN_OK;
}
int launch_window_fwd(WindowParams p, int D, int dtype, hipStream_t st);  // 16-bit
int launch_window_bwd(WindowParams p, int D, int dtype, hipStream_t st);
int launch_window_f32(const WindowParams& p, int D, bool bwd, hipStream_t st);  // no parts, no workspace
// O of rows whose keys were split: part as laid out above, out [slices / Hk, H, N, D] with strides (z, h, n).
int launch_combine(const float* part, void* out, float* m, const int64_t so[3], int64_t slices, int Hk, int G, int N,
                   int splits, int D, int dtype, hipStream_t st);

// Attention over keys of another length (cross.h). q, o, do, dq: [Zs B, H, N, D]; k, v, dk, dv: [Zs, Hk, S, D].
struct CrossParams {
  const void* q;
  const void* k;
  const void* v;
  const void* o;  // backward: the forward's output
  const void* dout;
  void* out;  // forward: O; backward: dQ
  void* dk;
  void* dv;
  float* m;             // [Zs B, H, N] base-2 log-sum-exp, or null
  float* delta;         // backward: [slices, rows], minus rowsum(dO * O)
  float* norms;         // fp16 backward: [slices, nblk, 2], largest squared norm of dO's rows, largest |delta|
  const int32_t* lens;  // [Zs] keys that each sequence (or group) sees, or null: S
  float* part;          // forward: partial rows, see cross_part_floats; backward: partial dQ
  float* kpart;         // backward: partial dK, dV
  int64_t sq[3], sk[3], sv[3], so[3], sd[3], sout[3], sdk[3], sdv[3];
  int32_t Zs, B, H, Hk, G, N, S;
  int32_t nblk, splits;   // row blocks of a slice, parts of their keys
  int32_t joined;         // forward: results are parts even where there is one
  int32_t waves;          // of a workgroup: forward where rows are few, dQ in float32
  int32_t pipe;           // forward: row blocks of cross_pipe_rows rows, walked by all waves together
  int32_t kblk, parts;    // backward: key blocks of a slice, parts of their rows
  float c, scale;
  int64_t slices() const { return (int64_t)Zs * Hk; }
  int64_t rows() const { return (int64_t)B * G * N; }  // of a slice
};
// Partial rows of a forward split `splits` ways: for each slice, part and row D sums, then for each its max and sum; in whole chunks
// of 16 bytes, so that another region may lie behind.
inline int64_t cross_part_floats(int64_t slices, int64_t rows, int64_t splits, int64_t D) {
  return (slices * rows * splits * (D + 2) + 3) / 4 * 4;
}
// Whether slices are dealt out to the XCDs (cross_coord): an eighth of the places at most is left idle.
__host__ __device__ inline bool cross_dealt(int64_t slices) { return ((slices + 7) / 8 * 8 - slices) * 8 <= slices; }
// A launch holds fewer than 2^32 threads.
inline int check_grid(int64_t blocks, int threads) {
  if (blocks > 0xffffffffll / threads)
    return set_error(TATTN_E_ARG, "grid too large: %lld workgroups of %d threads", (long long)blocks, threads);
  return TATTN_OK;
}
inline int cross_grid(int64_t slices, int64_t blocks, int threads, unsigned* out) {
  const int rc = window_grid(cross_dealt(slices) ? (slices + 7) / 8 * 8 : slices, blocks, 0, out);
  return rc ? rc : check_grid(*out, threads);
}
// Set nblk, splits and waves, and for the backward kblk and parts; refuse what its launches would not hold.
int cross_fwd_plan(CrossParams& p, int D, int dtype);
int cross_bwd_plan(CrossParams& p, int D, int dtype);
// Workgroups that join the parts of so many rows, `most` parts a row at most; `dealt` groups of lanes share a row's parts.
inline int64_t combine_blocks(int64_t rows, int most, int D, int32_t& dealt) {
  const int groups = 256 / (D / 4);
  for (dealt = 1; dealt < groups && 4 * dealt < most; dealt *= 2) {}
  const int64_t per = groups / dealt;
  return (rows + per - 1) / per;
}
inline int64_t cross_sum_blocks(const CrossParams& p, int D, bool keys, int block) {
  return ((keys ? p.slices() * p.kblk * 2 * block * D / 4 : p.slices() * p.rows() * D / 4) + 255) / 256;
}
int64_t cross_bwd_floats(const CrossParams& p, int D, int dtype);  // workspace of a planned backward
void cross_bwd_workspace(CrossParams& p, int D, int dtype, float* work);  // lays out delta, norms, part and kpart
int launch_cross_fwd(const CrossParams& p, int D, int dtype, hipStream_t st);
int launch_cross_pipe(const CrossParams& p, int D, int dtype, hipStream_t st);  // without the joining of parts
// Waves of a workgroup of the forward for many rows, and row tiles of each.
constexpr int cross_pipe_waves(int D) { return 4; }
constexpr int cross_pipe_tiles(int D) { return D == 128 ? 1 : 2; }
constexpr int cross_pipe_rows(int D) { return 32 * cross_pipe_waves(D) * cross_pipe_tiles(D); }
int launch_cross_bwd(const CrossParams& p, int D, int dtype, hipStream_t st);
// Up to four tiles of keys (backward two at head dim 128, for the registers of a wave): cross_short.hip.
constexpr int cross_short_tiles(int D, bool bwd) { return D == 128 && bwd ? 2 : 4; }
constexpr int cross_short_occ(int D, int tiles) { return tiles * ((D + 31) / 32) <= 3 ? 2 : 1; }  // waves per SIMD of the backward
inline bool cross_short(const CrossParams& p, int D, int dtype, bool bwd) { return dtype != 1 && p.S <= 32 * cross_short_tiles(D, bwd); }
// Backward with two row tiles in a step: cross_short_pipe.hip.
constexpr bool cross_short_piped(int D, int tiles) { return D < 128 && tiles * ((D + 31) / 32) >= 4 && tiles * ((D + 31) / 32) < 8; }
int launch_cross_short(const CrossParams& p, int D, int dtype, bool bwd, hipStream_t st);
int launch_cross_short_pipe(const CrossParams& p, int D, int dtype, hipStream_t st);
constexpr int cross_dq_threads(int D) { return D == 128 ? 512 : 256; }
int launch_cross_dq(const CrossParams& p, int D, int dtype, hipStream_t st);  // 16-bit; dQ (its parts) and delta
constexpr int cross_f32_occ(int D) { return D == 128 ? 1 : 2; }  // waves per SIMD in float32
int launch_cross_f32(const CrossParams& p, int D, bool bwd, hipStream_t st);
int launch_cross_combine_f32(const CrossParams& p, int D, hipStream_t st);  // joins the parts of a forward in float32
// Adds the parts of dQ, or of dK and dV for key blocks of `block` keys.
int launch_cross_sum(const CrossParams& p, int D, int dtype, bool keys, int block, hipStream_t st);

// One step behind a shared prefix: `pre` holds a group's rows (B sequences) over the prefix, `own` each sequence's over its
// keys, causal. Both write parts (own.part lies behind pre.part), which are joined.
struct PrefixParams {
  CrossParams pre, own;
};
int prefix_plan(PrefixParams& p, int D);  // as the plans above
int64_t prefix_floats(const PrefixParams& p, int D);
int launch_prefix(const PrefixParams& p, int D, int dtype, hipStream_t st);
int launch_prefix_combine(const PrefixParams& p, int D, int dtype, hipStream_t st);

// One token per request over the cache in 4 bits.
struct Cache4AttnParams {
  const void* q;  // [R, H, D], strides (r, h)
  void* out;
  const uint8_t* codes;
  const uint8_t* scales;
  const int32_t* tables;
  const int32_t* lens;
  float* part;  // window_part_floats(R * Hk, G, splits, D)
  int64_t sq[2], so[2];
  int64_t table_stride;
  int32_t R, Hk, G, pages;
  int32_t groups;  // of 16 query heads of a key head
  int32_t shift;   // log2 of the page size
  int32_t most;    // tokens that a table row holds
  int32_t window, sinks;
  int32_t chunk, splits;  // key tiles per workgroup, workgroups per request and key head
  float c;
};
void cache4_chunks(Cache4AttnParams& p);  // sets chunk and splits
int launch_cache4_attention(const Cache4AttnParams& p, int D, int dtype, hipStream_t st);

}  // namespace tattn
