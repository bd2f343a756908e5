/*
 * tattn: fused attention (FlashAttention-2 style) for AMD Instinct MI355X (gfx950).
 *
 * C ABI of libtattn_hip.so. Every entry point enqueues hand-written HIP kernels on the
 * caller's stream and returns immediately: no host synchronisation, no device allocation.
 * The caller owns every buffer (outputs and the float32 M / delta workspaces).
 *
 * Layouts. q, k, v, o, do, dq, dk, dv are [Z, H, N, D] tensors of one element type
 * (TATTN_F16, TATTN_BF16 or TATTN_F32). Strides are in ELEMENTS, four per tensor, ordered
 * (z, h, n, d). The d stride must be 1, rows must be 16-byte aligned. M and delta are
 * float32 [Z, H, N], contiguous. Head dims: 16, 32, 64, 128.
 *
 * Numerics (the reference's rounding points are kept): scores are scaled by
 * sm_scale * log2(e) and exponentiated in base 2 with float32 softmax state; P and dS are
 * rounded to the element type only as MFMA operands; M = max + log2(sum) per query row.
 *
 * Return value: 0 on success, a TATTN_E* code otherwise; tattn_last_error() then gives a
 * per-thread message.
 */
#ifndef TATTN_H
#define TATTN_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TATTN_ABI_VERSION 4

/* TATTN_BF16 has no counterpart in the reference, which accepts fp16 and fp32 only
 * (src/tattn/api.py:55-56); it runs the fp16 kernels with bf16 MFMAs and bf16 rounding points. */
enum tattn_dtype { TATTN_F16 = 0, TATTN_F32 = 1, TATTN_BF16 = 2 };
enum tattn_kernel { TATTN_K_FWD = 0, TATTN_K_BWD_DKDV = 1, TATTN_K_BWD_DQ = 2 };
enum tattn_status {
  TATTN_OK = 0,
  TATTN_E_ARG = 1,      /* bad shape, dtype, head dim, stride or null pointer */
  TATTN_E_CONFIG = 2,   /* tile config id out of range for this kernel/dim/dtype */
  TATTN_E_LAUNCH = 3,   /* the HIP runtime refused the launch */
  TATTN_E_DEVICE = 4    /* current device is not a gfx950 */
};

/* One entry of the gfx950 tile table. */
typedef struct tattn_config {
  int32_t block_m;      /* query rows per workgroup */
  int32_t block_n;      /* key rows per workgroup (bwd dK/dV) or per inner step */
  int32_t waves;        /* wavefronts (64 lanes) per workgroup */
  int32_t tiles;        /* 32-row MFMA tiles each wave owns */
  int32_t lds_bytes;    /* LDS the workgroup uses */
  int32_t kind;         /* 0 generic kernel, 1 software-pipelined, 2 persistent (falls back to the
                           pipelined kernel of the same tiles where a problem does not fit it),
                           3 dK/dV with paired waves (two waves per 32-key tile, split roles) */
  int32_t ring;         /* persistent forward: K/V tiles in flight (LDS ring depth); else 0 */
} tattn_config;

/* ABI version of the loaded library; equals TATTN_ABI_VERSION of this header. */
int tattn_abi_version(void);

/* Message of the last failed call on this thread ("" if none). */
const char* tattn_last_error(void);

/* 1 if the current HIP device is gfx950 and the kernels can run on it, else 0. */
int tattn_device_supported(void);

/*
 * Forward: o = softmax(q k^T * sm_scale [causal mask]) v, m = per-row base-2 log-sum-exp.
 * Replaces `_forward` + `_fwd_kernel` of the reference
 * (src/tattn/api.py:78-99, src/tattn/kernels.py:57-148). Arbitrary z/h/n strides per tensor
 * (api.py:95-96); m is [Z,H,N] float32 contiguous (api.py:88), or NULL when no backward will
 * follow: the log-sum-exp is then not stored (the reference always stores it, api.py:88, 161).
 * config_id = -1 picks the kernel for the problem, from the table or outside it (tattn_picked);
 * otherwise an index into the TATTN_K_FWD table (the reference's `config=` override, api.py:69-75).
 */
int tattn_fwd(const void* q, const void* k, const void* v, void* o, float* m,
              const int64_t q_strides[4], const int64_t k_strides[4],
              const int64_t v_strides[4], const int64_t o_strides[4],
              int64_t Z, int64_t H, int64_t N, int64_t D, int dtype, int causal,
              float sm_scale, int config_id, void* stream);

/*
 * delta[z,h,i] = sum_d o[z,h,i,d] * do[z,h,i,d] in float32.
 * Replaces `_bwd_preprocess` (src/tattn/kernels.py:324-337, launched at api.py:122).
 * o and do share `strides` (the reference makes them contiguous, api.py:111).
 */
int tattn_bwd_preprocess(const void* o, const void* dout, float* delta, const int64_t strides[4],
                         int64_t Z, int64_t H, int64_t N, int64_t D, int dtype, void* stream);

/*
 * dK, dV for every key block, looping over query blocks; no atomics.
 * Replaces `_bwd_dkdv_kernel` (src/tattn/kernels.py:151-239, launched at api.py:124-142).
 * q, k, v, do, dk, dv share one layout `strides` (kernels.py:180-181, api.py:111-114).
 */
int tattn_bwd_dkdv(const void* q, const void* k, const void* v, const void* dout,
                   void* dk, void* dv, const float* m, const float* delta,
                   const int64_t strides[4], int64_t Z, int64_t H, int64_t N, int64_t D,
                   int dtype, int causal, float sm_scale, int config_id, void* stream);

/*
 * dQ for every query block, looping over key blocks; no atomics.
 * Replaces `_bwd_dq_kernel` (src/tattn/kernels.py:242-321, launched at api.py:143-145).
 */
int tattn_bwd_dq(const void* q, const void* k, const void* v, const void* dout, void* dq,
                 const float* m, const float* delta, const int64_t strides[4], int64_t Z,
                 int64_t H, int64_t N, int64_t D, int dtype, int causal, float sm_scale,
                 int config_id, void* stream);

/*
 * The whole backward in stream order (preprocess, dK/dV, dQ: src/tattn/api.py:102-146), in one to
 * three launches; the same bits as the three entry points above with the same picks.
 * delta is caller-owned float32 [Z,H,N] scratch. config_id applies to both dK/dV and dQ
 * (as the reference's `config=` does, api.py:124-145); -1 picks per kernel.
 */
int tattn_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout,
              void* dq, void* dk, void* dv, const float* m, float* delta,
              const int64_t strides[4], int64_t Z, int64_t H, int64_t N, int64_t D,
              int dtype, int causal, float sm_scale, int config_id, void* stream);

/*
 * tattn_bwd with the gradients in a layout of their own: q, k, v, o and do share `strides`, dq, dk
 * and dv share `grad_strides`. The backward then reads activations where they lie (a token-major
 * view, say) and writes contiguous gradients, where the reference first copies its inputs
 * contiguous (api.py:111). Same results bit for bit as tattn_bwd on contiguous copies, unless rows
 * overlap or lie so far apart that the launch goes to kernels that contiguous copies do not need.
 */
int tattn_bwd_layouts(const void* q, const void* k, const void* v, const void* o, const void* dout,
                      void* dq, void* dk, void* dv, const float* m, float* delta,
                      const int64_t strides[4], const int64_t grad_strides[4],
                      int64_t Z, int64_t H, int64_t N, int64_t D, int dtype, int causal,
                      float sm_scale, int config_id, void* stream);

/*
 * tattn_bwd without the delta argument and without any allocation: delta lives in a static
 * device array of the library (16 MiB per GPU, held until the process ends), so the caller
 * passes only inputs and outputs. No counterpart in the reference: it is for callers that
 * cannot allocate device memory (code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc). Limit: Z*H*N <= 4,194,304 query rows, else TATTN_E_ARG and nothing
 * is enqueued. Every call on one GPU shares that GPU's array: calls that overlap on one GPU
 * (two streams, two threads) race on it and must be serialised by the caller.
 */
int tattn_bwd_noalloc(const void* q, const void* k, const void* v, const void* o, const void* dout,
                      void* dq, void* dk, void* dv, const float* m,
                      const int64_t strides[4], int64_t Z, int64_t H, int64_t N, int64_t D,
                      int dtype, int causal, float sm_scale, int config_id, void* stream);

/*
 * Tile table introspection (the gfx950 replacement of the reference's autotune config lists,
 * src/tattn/kernels.py:21-54): number of entries for (kernel, D, dtype), the entry itself, and
 * the table entry ranked first for a launch that fills the GPU with a batch x heads count that is a
 * multiple of 8 (the reference keys its autotuner on (N bucket, head dim, causal), kernels.py:57-61
 * and api.py:59-62). What a call with config_id -1 runs depends on the whole problem and may be a
 * kernel outside the table: tattn_picked.
 */
int tattn_num_configs(int kernel, int64_t D, int dtype);
int tattn_config_desc(int kernel, int64_t D, int dtype, int config_id, tattn_config* out);
int tattn_pick_config(int kernel, int64_t D, int dtype, int causal, int64_t N);

/* Kernels outside the table, as tattn_picked reports them. */
enum tattn_pick {
  TATTN_PICK_COOP = 1000,   /* 16-bit, few rows: the waves of a workgroup split the summed dimension */
  TATTN_PICK_PLANES = 1001, /* float32 on the 16-bit matrix cores, operands as three planes */
  TATTN_PICK_SHORT = 1002   /* 16-bit, N <= 128: whole slices in LDS, the whole backward in one launch */
};

/*
 * What a call with config_id -1 runs for a problem: a table index or a tattn_pick. Forward
 * (TATTN_K_FWD): strides of k and of v. Backward kernels, as tattn_bwd and its variants run them:
 * k_strides are the strides the inputs share, v_strides is not read. Null strides: contiguous
 * (v_strides: those of k). -1 for arguments the entry points refuse. Launches nothing.
 */
int tattn_picked(int kernel, const int64_t k_strides[4], const int64_t v_strides[4], int64_t Z, int64_t H,
                 int64_t N, int64_t D, int dtype, int causal, float sm_scale);

/*
 * Operators around attention. No counterpart in the reference. Pointers may be null where their
 * tensor has no elements; a call without work (no tokens, no requests) launches nothing and returns 0.
 *
 * Pages for the tokens that R requests add: request r holds lens[r] tokens, adds new_tokens[r], and its
 * pages are tables[r * table_stride ..] (P entries). Pages past ceil(lens[r] / page_size) come from
 * free_pages (F of them) in request order and are entered into the table. For the T tokens in request order:
 * slots (page * page_size + offset) and positions; starts[R + 1] is where each request's tokens begin and
 * taken[0] how many pages they need. A token without a page (free list or table row exhausted, or an
 * entry of the table below 0) has slot -1; tokens past T are not placed, entries of T behind the last request hold
 * slot -1, position 0. Negative lengths count as 0. page_size: a power of two, 16 to 1024. lens is not updated.
 */
int tattn_page_tables(const int32_t* lens, const int32_t* new_tokens, int32_t* tables, const int32_t* free_pages,
                      int64_t* slots, int32_t* positions, int32_t* starts, int32_t* taken, int64_t R, int64_t P,
                      int64_t table_stride, int64_t F, int64_t T, int64_t page_size, void* stream);

/*
 * A key/value cache in 4 bits (TATTN_F16 or TATTN_BF16 values; D = 32, 64 or 128). codes:
 * [pages, H, 2, page_size, D / 2] bytes (2: keys, values; an even d in the low four bits), e2m1: sign, two
 * exponent bits, one mantissa bit. scales: [pages, H, 2, page_size, D / 32] bytes, exponents biased by 127 of
 * the blocks of 32 values along d: the smallest at which the block's largest magnitude rounds to 6 or less (and
 * at which 6 * 2^e is finite in the element type); 255
 * marks a block that held an infinity or a NaN and reads as NaN. Magnitudes below 2^-120 count as zero.
 * write: k, v [T, H, D] with (token, head) strides in elements, unit d stride, 16-byte aligned rows,
 * into `slots`; read: what the cache holds for `slots`, contiguous [T, H, D]. Slots outside the cache (a batch's
 * padding has -1) are not written and read as zeros. No two tokens of a write may have one slot.
 */
int tattn_cache4_write(uint8_t* codes, uint8_t* scales, const void* k, const void* v, const int64_t* slots,
                       const int64_t k_strides[2], const int64_t v_strides[2], int64_t T, int64_t H, int64_t D,
                       int64_t pages, int64_t page_size, int dtype, void* stream);
int tattn_cache4_read(const uint8_t* codes, const uint8_t* scales, void* k, void* v, const int64_t* slots, int64_t T,
                      int64_t H, int64_t D, int64_t pages, int64_t page_size, int dtype, void* stream);

/*
 * Root-mean-square norm of every head of q [Z, H, N, D] and k [Z, Hk, N, D], its weights, and the position
 * rotation: y = x / sqrt(mean(x^2) + eps) * weight, then pairs (i, i + D / 2) of y, or (2i, 2i + 1) when
 * interleaved, turned by the angle whose cosine and sine are cos[position][i], sin[position][i] (float32
 * [P, D / 2], contiguous). positions: [N] (pos_stride 0) or one row per z, pos_stride apart; null: n. A position
 * outside [0, P) gives a row of NaN. dtype: any; D: 16, 32, 64, 128; w_dtype: dtype or TATTN_F32. Tensor strides
 * are (z, h, n, d) in elements, unit d stride, 16-byte aligned rows; everything is float32 up to one rounding per result.
 *
 * The backward gives dq, dk and, unless workspace is null, both weights' gradients in w_dtype (sums in a fixed
 * order, no atomics). workspace: float32 [TATTN_NORM_ROPE_ROWS, D]. Without tokens nothing is written.
 */
#define TATTN_NORM_ROPE_ROWS 512
int tattn_norm_rope_fwd(const void* q, const void* k, const void* q_weight, const void* k_weight, const float* cos,
                        const float* sin, const int32_t* positions, void* q_out, void* k_out, const int64_t q_strides[4],
                        const int64_t k_strides[4], const int64_t qo_strides[4], const int64_t ko_strides[4],
                        int64_t pos_stride, int64_t Z, int64_t H, int64_t Hk, int64_t N, int64_t D, int64_t P, int dtype,
                        int w_dtype, int interleaved, float eps, void* stream);
int tattn_norm_rope_bwd(const void* q, const void* k, const void* q_weight, const void* k_weight, const float* cos,
                        const float* sin, const int32_t* positions, const void* dq_out, const void* dk_out, void* dq,
                        void* dk, void* dq_weight, void* dk_weight, float* workspace, const int64_t q_strides[4],
                        const int64_t k_strides[4], const int64_t dqo_strides[4], const int64_t dko_strides[4],
                        const int64_t dq_strides[4], const int64_t dk_strides[4], int64_t pos_stride, int64_t Z, int64_t H,
                        int64_t Hk, int64_t N, int64_t D, int64_t P, int dtype, int w_dtype, int interleaved, float eps,
                        void* stream);

/*
 * Causal attention over a sliding window and the first keys, grouped heads: q, o [Z, H, N, D], k, v [Z, Hk, S, D],
 * H a multiple of Hk (query head h reads key head h / (H / Hk)), any dtype, D = 16, 32, 64 or 128.
 * The queries are the last N of len_z positions, len_z = lens[z] (clamped to [0, S]) or S where lens is null: query n
 * is at position len_z - N + n and sees key j <= position with position - j < window or j < sinks. Rows that see no
 * key (positions below 0) give zeros; keys that no query of a block sees are not read into any sum. Strides per tensor
 * (z, h, n, d) in elements, unit d stride, 16-byte aligned rows that do not overlap; a head spans less than 2 GiB.
 *
 * m: [Z, H, N] float32 base-2 log-sum-exp for the backward, or null. workspace: float32, 16-byte aligned, as many
 * as tattn_window_workspace gives for the same sizes (may be null where that is 0, and in TATTN_F32); calls that may
 * overlap need one each.
 * The backward (no lens, S >= N) sums dk and dv over the heads of a group, without atomics; delta: float32 scratch, 8-byte aligned, of
 * Z H N values, in TATTN_F16 of Z H N rounded up to an even number and 2 Z Hk ceil(N (H / Hk) / 128) more.
 */
int tattn_window_workspace(int backward, int64_t Z, int64_t H, int64_t Hk, int64_t N, int64_t S, int64_t D, int64_t window,
                           int64_t sinks, int64_t* floats);
/* What a 16-bit forward of these sizes runs: 0 for workgroups of four row tiles, otherwise one row tile per workgroup and the
 * number of parts that its keys are cut into; -1 for sizes that it refuses. */
int tattn_window_picked(int64_t Z, int64_t H, int64_t Hk, int64_t N, int64_t S, int64_t D, int64_t window, int64_t sinks);
int tattn_window_fwd(const void* q, const void* k, const void* v, void* o, float* m, const int32_t* lens, float* workspace,
                     const int64_t q_strides[4], const int64_t k_strides[4], const int64_t v_strides[4],
                     const int64_t o_strides[4], int64_t Z, int64_t H, int64_t Hk, int64_t N, int64_t S, int64_t D,
                     int64_t window, int64_t sinks, int dtype, float sm_scale, void* stream);
int tattn_window_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout, void* dq, void* dk,
                     void* dv, const float* m, float* delta, float* workspace, const int64_t q_strides[4],
                     const int64_t k_strides[4], const int64_t v_strides[4], const int64_t o_strides[4],
                     const int64_t do_strides[4], const int64_t dq_strides[4], const int64_t dk_strides[4],
                     const int64_t dv_strides[4], int64_t Z, int64_t H, int64_t Hk, int64_t N, int64_t S, int64_t D,
                     int64_t window, int64_t sinks, int dtype, float sm_scale, void* stream);

/*
 * Attention of one token per request over the cache in 4 bits: q, o [R, H, D] with (request, head) strides in elements, H a
 * multiple of the cache's Hk heads (head h reads key head h / (H / Hk)), D = 32, 64 or 128, dtype of the cache's values.
 * Request r sees its first lens[r] tokens (clamped to [0, width * page_size]) through tables[r * table_stride ..]
 * (width pages); with a window (0: none) only the last `window` of them and the first `sinks`. Pages that no visible token
 * lies in are not looked up; tokens on a page outside [0, pages) are hidden. A request that sees no token gives zeros.
 * workspace: float32, 16-byte aligned, as many as tattn_cache4_attention_workspace gives (null where 0).
 */
int tattn_cache4_attention_workspace(int64_t R, int64_t H, int64_t Hk, int64_t D, int64_t width, int64_t page_size,
                                     int64_t window, int64_t sinks, int64_t* floats);
int tattn_cache4_attention(const void* q, void* o, const uint8_t* codes, const uint8_t* scales, const int32_t* tables,
                           const int32_t* lens, float* workspace, const int64_t q_strides[2], const int64_t o_strides[2],
                           int64_t table_stride, int64_t R, int64_t H, int64_t Hk, int64_t D, int64_t width, int64_t pages,
                           int64_t page_size, int64_t window, int64_t sinks, int dtype, float sm_scale, void* stream);

/*
 * Attention over keys of another length, an encoder's states, without a causal mask, grouped heads: q, o [Z, H, N, D], k, v
 * [Z, Hk, S, D], H a multiple of Hk (query head h reads key head h / (H / Hk)), any dtype, D = 16, 32, 64 or 128. Every query of
 * sequence z sees its first lens[z] keys (clamped to [0, S]; lens null: S); where that is none, rows of o are zeros. What lies at
 * or past lens[z] reaches nothing. Strides per tensor (z, h, n, d) in elements, unit d stride, 16-byte aligned rows; rows of k
 * and v, and in the backward of all tensors, do not overlap and a head of them spans less than 2 GiB.
 *
 * m: [Z, H, N] float32 base-2 log-sum-exp for the backward, or null. workspace: float32, 16-byte aligned, as many as
 * tattn_cross_workspace gives for the same sizes (null where 0); calls that may overlap need one each.
 * The backward sums dk and dv over the heads of a group, without atomics; keys at or past lens[z] get zeros. Calls whose launches would
 * hold 2^32 threads or more are refused, by the workspace's functions too.
 */
int tattn_cross_workspace(int backward, int64_t Z, int64_t H, int64_t Hk, int64_t N, int64_t S, int64_t D, int dtype,
                          int64_t* floats);
int tattn_cross_fwd(const void* q, const void* k, const void* v, void* o, float* m, const int32_t* lens, float* workspace,
                    const int64_t q_strides[4], const int64_t k_strides[4], const int64_t v_strides[4],
                    const int64_t o_strides[4], int64_t Z, int64_t H, int64_t Hk, int64_t N, int64_t S, int64_t D, int dtype,
                    float sm_scale, void* stream);
int tattn_cross_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout, void* dq, void* dk, void* dv,
                    const float* m, const int32_t* lens, float* workspace, const int64_t q_strides[4],
                    const int64_t k_strides[4], const int64_t v_strides[4], const int64_t o_strides[4],
                    const int64_t do_strides[4], const int64_t dq_strides[4], const int64_t dk_strides[4],
                    const int64_t dv_strides[4], int64_t Z, int64_t H, int64_t Hk, int64_t N, int64_t S, int64_t D, int dtype,
                    float sm_scale, void* stream);

/*
 * Attention of the newest N tokens of sequences behind shared prefixes (TATTN_F16 or TATTN_BF16; D = 16, 32, 64 or 128): q, o
 * [groups * members, H, N, D], prefix_k, prefix_v [groups, Hk, P, D], k, v [groups * members, Hk, S, D]. Sequence z belongs to
 * group z / members. Its query n is at position lens[z] - N + n (lens clamped to [0, S]) of its own keys and sees all
 * prefix_lens[group] keys of the prefix (clamped to [0, P]; null: P) and its own keys up to its position; at a position below 0 it
 * sees nothing and its row is zeros. P and S may be 0. Strides and workspace as above (tattn_prefix_workspace).
 */
int tattn_prefix_workspace(int64_t groups, int64_t members, int64_t H, int64_t Hk, int64_t N, int64_t P, int64_t S, int64_t D,
                           int64_t* floats);
int tattn_prefix_attention(const void* q, const void* prefix_k, const void* prefix_v, const void* k, const void* v, void* o,
                           const int32_t* prefix_lens, const int32_t* lens, float* workspace, const int64_t q_strides[4],
                           const int64_t pk_strides[4], const int64_t pv_strides[4], const int64_t k_strides[4],
                           const int64_t v_strides[4], const int64_t o_strides[4], int64_t groups, int64_t members, int64_t H,
                           int64_t Hk, int64_t N, int64_t P, int64_t S, int64_t D, int dtype, float sm_scale, void* stream);

/*
 * The rotation of tattn_norm_rope_* by positions on several axes: pair i of a token is turned by the angle whose cosine and sine
 * are cos[x][i], sin[x][i] (float32 [R, D / 2], contiguous) with x the token's position on axis axes[i]. axes: host array of
 * D / 2 entries, each in [0, num_axes), num_axes <= 8, or -1 for a pair that stays as it is. positions: [num_axes, N] (pos_stride
 * 0) or [num_axes, Z, N], axis_stride and pos_stride apart. A position outside [0, R) makes the pairs of its axis NaN. Without
 * weights (both null) there is no norm: eps is not read, the backward reads no q and k and gives no gradients of weights.
 */
int tattn_rope_axes_fwd(const void* q, const void* k, const void* q_weight, const void* k_weight, const float* cos,
                        const float* sin, const int32_t* positions, const int32_t* axes, void* q_out, void* k_out,
                        const int64_t q_strides[4], const int64_t k_strides[4], const int64_t qo_strides[4],
                        const int64_t ko_strides[4], int64_t num_axes, int64_t axis_stride, int64_t pos_stride, int64_t Z,
                        int64_t H, int64_t Hk, int64_t N, int64_t D, int64_t R, int dtype, int w_dtype, int interleaved,
                        float eps, void* stream);
int tattn_rope_axes_bwd(const void* q, const void* k, const void* q_weight, const void* k_weight, const float* cos,
                        const float* sin, const int32_t* positions, const int32_t* axes, const void* dq_out,
                        const void* dk_out, void* dq, void* dk, void* dq_weight, void* dk_weight, float* workspace,
                        const int64_t q_strides[4], const int64_t k_strides[4], const int64_t dqo_strides[4],
                        const int64_t dko_strides[4], const int64_t dq_strides[4], const int64_t dk_strides[4],
                        int64_t num_axes, int64_t axis_stride, int64_t pos_stride, int64_t Z, int64_t H, int64_t Hk, int64_t N,
                        int64_t D, int64_t R, int dtype, int w_dtype, int interleaved, float eps, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TATTN_H */
