// C ABI of the operators around attention (declared in include/tattn.h): argument checks, then the
// launchers of ops.h.
#include <hip/hip_runtime.h>

#include "../../include/tattn.h"
#include "ops.h"

namespace tattn {
namespace {

bool aligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// A pointer that may be null only where the tensor has no elements.
int check_ptr(const char* name, const void* p, int64_t elements, unsigned align) {
  if (elements > 0 && !p) return set_error(TATTN_E_ARG, "%s is a null pointer", name);
  if (!aligned(p, align)) return set_error(TATTN_E_ARG, "%s must be %u-byte aligned", name, align);
  return TATTN_OK;
}

// Strides (in elements) of dimensions before the unit-stride d (given as the last of four): whole 16-byte rows.
int check_rows(const char* name, const int64_t* st, int n, int sz) {
  if (!st) return set_error(TATTN_E_ARG, "%s strides are null", name);
  if (n == 3 && st[3] != 1) return set_error(TATTN_E_ARG, "%s d stride must be 1, got %lld", name, (long long)st[3]);
  for (int i = 0; i < n; ++i)
    if (st[i] < 0 || (st[i] * sz) % 16 != 0)
      return set_error(TATTN_E_ARG, "%s stride %lld must be a multiple of %d elements", name, (long long)st[i], 16 / sz);
  return TATTN_OK;
}

int check_page(int64_t page_size, int32_t* shift) {
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))
    return set_error(TATTN_E_ARG, "page size must be a power of two from 16 to 1024, got %lld", (long long)page_size);
  *shift = __builtin_ctzll((unsigned long long)page_size);
  return TATTN_OK;
}

int check_count(const char* name, int64_t x) {
  if (x < 0 || x > 0x7fffffff - 4096) return set_error(TATTN_E_ARG, "%s out of range: %lld", name, (long long)x);
  return TATTN_OK;
}

int cache4_common(Cache4Params& p, const void* codes, const void* scales, const int64_t* slots, int64_t T, int64_t H,
                  int64_t D, int64_t pages, int64_t page_size, int dtype) {
  int rc;
  if (dtype != TATTN_F16 && dtype != TATTN_BF16)
    return set_error(TATTN_E_ARG, "dtype must be TATTN_F16 or TATTN_BF16, got %d", dtype);
  if (D != 32 && D != 64 && D != 128) return set_error(TATTN_E_ARG, "head dim must be 32, 64 or 128, got %lld", (long long)D);
  if ((rc = check_page(page_size, &p.shift)) || (rc = check_count("tokens", T)) || (rc = check_count("heads", H)) ||
      (rc = check_count("pages", pages)))
    return rc;
  if (H > 65536) return set_error(TATTN_E_ARG, "heads out of range: %lld", (long long)H);
  if ((rc = check_ptr("codes", codes, pages * H, 16)) || (rc = check_ptr("scales", scales, pages * H, 4)) ||
      (rc = check_ptr("slots", slots, T, 8)))
    return rc;
  p.codes = (uint8_t*)codes;
  p.scales = (uint8_t*)scales;
  p.slots = slots;
  p.T = (int32_t)T;
  p.H = (int32_t)H;
  p.total = pages * page_size;
  return TATTN_OK;
}

// Everything the norm's two directions share; no work is left when N or Z is 0.
int norm_rope_common(NormRopeParams& p, const void* q, const void* k, const void* qw, const void* kw, const float* cos,
                     const float* sin, const int32_t* positions, const int64_t* sq, const int64_t* sk, int64_t pos_stride,
                     int64_t Z, int64_t H, int64_t Hk, int64_t N, int64_t D, int64_t P, int dtype, int w_dtype, float eps) {
  int rc;
  if (dtype != TATTN_F16 && dtype != TATTN_F32 && dtype != TATTN_BF16) return set_error(TATTN_E_ARG, "unknown dtype %d", dtype);
  if (w_dtype != dtype && w_dtype != TATTN_F32) return set_error(TATTN_E_ARG, "weights must be of the tensors' dtype or float32");
  if (D != 16 && D != 32 && D != 64 && D != 128)
    return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %lld", (long long)D);
  if ((rc = check_count("batch", Z)) || (rc = check_count("heads", H)) || (rc = check_count("key heads", Hk)) ||
      (rc = check_count("length", N)) || (rc = check_count("table rows", P)))
    return rc;
  if (H < 1 || Hk < 1) return set_error(TATTN_E_ARG, "heads must be positive, got %lld and %lld", (long long)H, (long long)Hk);
  p.per_q = (uint32_t)((H + 3) / 4);
  p.per_k = (uint32_t)((Hk + 3) / 4);
  if (Z > 0 && N > 0 && (double)Z * (double)N * (double)(p.per_q + p.per_k) >= 2147483648.0)
    return set_error(TATTN_E_ARG, "too many tokens: %lld x %lld with %lld + %lld heads", (long long)Z, (long long)N,
                     (long long)H, (long long)Hk);
  const int64_t rows = Z * N;
  const int sz = dtype == TATTN_F32 ? 4 : 2;
  if ((rc = check_ptr("q", q, rows, 16)) || (rc = check_ptr("k", k, rows, 16)) || (rc = check_ptr("q_weight", qw, 1, 16)) ||
      (rc = check_ptr("k_weight", kw, 1, 16)) || (rc = check_ptr("cos", cos, P, 16)) || (rc = check_ptr("sin", sin, P, 16)) ||
      (rc = check_ptr("positions", positions, 0, 4)) || (rc = check_rows("q", sq, 3, sz)) || (rc = check_rows("k", sk, 3, sz)))
    return rc;
  if (rows > 0 && P < 1) return set_error(TATTN_E_ARG, "cos and sin have no rows");
  p.q = q; p.k = k; p.qw = qw; p.kw = kw; p.cos = cos; p.sin = sin; p.positions = positions;
  for (int i = 0; i < 3; ++i) p.sq[i] = sq[i], p.sk[i] = sk[i];
  p.pos_stride = pos_stride;
  p.Z = (int32_t)Z; p.H = (int32_t)H; p.Hk = (int32_t)Hk; p.N = (int32_t)N; p.P = (int32_t)P;
  p.wide_w = dtype != TATTN_F32 && w_dtype == TATTN_F32;
  p.eps = eps;
  p.units_q = (uint32_t)rows * p.per_q;
  p.units_k = (uint32_t)rows * p.per_k;
  return TATTN_OK;
}

// Window attention: sizes, window and first keys.
int window_common(WindowParams& p, int64_t Z, int64_t H, int64_t Hk, int64_t N, int64_t S, int64_t D, int64_t window,
                  int64_t sinks, bool lens) {
  int rc;
  if (D != 16 && D != 32 && D != 64 && D != 128)
    return set_error(TATTN_E_ARG, "head dim must be 16, 32, 64 or 128, got %lld", (long long)D);
  if ((rc = check_count("batch", Z)) || (rc = check_count("heads", H)) || (rc = check_count("length", N)) ||
      (rc = check_count("key length", S)))
    return rc;
  if (Z < 1 || H < 1 || N < 1 || S < 1) return set_error(TATTN_E_ARG, "sizes must be positive");
  if (Hk < 1 || H % Hk) return set_error(TATTN_E_ARG, "%lld heads do not share %lld key heads evenly", (long long)H, (long long)Hk);
  if (!lens && S < N) return set_error(TATTN_E_ARG, "%lld queries for %lld keys", (long long)N, (long long)S);
  if (window < 1) return set_error(TATTN_E_ARG, "window must be positive, got %lld", (long long)window);
  if (sinks < 0) return set_error(TATTN_E_ARG, "sinks must not be negative, got %lld", (long long)sinks);
  if ((double)H * (double)N > 1073741824.0 || (double)Z * (double)H * (double)((N + 31) / 32) > 67108864.0)
    return set_error(TATTN_E_ARG, "too many rows: %lld x %lld x %lld", (long long)Z, (long long)H, (long long)N);
  p.Z = (int32_t)Z; p.H = (int32_t)H; p.Hk = (int32_t)Hk; p.G = (int32_t)(H / Hk); p.N = (int32_t)N; p.S = (int32_t)S;
  p.window = (int32_t)(window < S ? window : S);
  p.sinks = (int32_t)(sinks < S ? sinks : S);
  return TATTN_OK;
}

// A tensor that the kernels read in tiles of 32 rows: strides (z, h, n), rows that do not overlap, slices that 31-bit
// byte offsets span with a step's rows to spare. A dimension of one row gets the stride of whole rows.
int check_tiles(const char* name, const void* ptr, const int64_t* st, int64_t rows, int64_t D, int dtype, int64_t (&out)[3]) {
  const int sz = dtype == TATTN_F32 ? 4 : 2;
  int rc;
  if ((rc = check_ptr(name, ptr, 1, 16)) || (rc = check_rows(name, st, 3, sz))) return rc;
  for (int i = 0; i < 3; ++i) out[i] = st[i];
  if (rows == 1) out[2] = D;
  if (out[2] < D) return set_error(TATTN_E_ARG, "%s rows overlap: stride %lld", name, (long long)out[2]);
  if (out[2] > (1ll << 24) || (rows + 256) * out[2] * sz >= 0x7fffff00ll)
    return set_error(TATTN_E_ARG, "a head of %s spans 2 GiB or more", name);
  return TATTN_OK;
}

// Scores to base-2 exponents. A scale of 0 becomes one so small that all exponents are 0 for finite scores below 1e22, because
// hidden keys are marked by scores whose scaled value is -inf.
float window_exponent_scale(float sm_scale) { return sm_scale == 0.0f ? 1.0e-30f : sm_scale * kLog2e; }

int check_dtype(int dtype) {
  if (dtype != TATTN_F16 && dtype != TATTN_F32 && dtype != TATTN_BF16) return set_error(TATTN_E_ARG, "unknown dtype %d", dtype);
  return TATTN_OK;
}

int check_16bit(int dtype) {
  if (dtype != TATTN_F16 && dtype != TATTN_BF16)
    return set_error(TATTN_E_ARG, "dtype must be TATTN_F16 or TATTN_BF16, got %d", dtype);
  return TATTN_OK;
}

int cache4_attn_common(Cache4AttnParams& p, int64_t R, int64_t H, int64_t Hk, int64_t D, int64_t width, int64_t page_size,
                       int64_t window, int64_t sinks) {
  int rc;
  if (D != 32 && D != 64 && D != 128) return set_error(TATTN_E_ARG, "head dim must be 32, 64 or 128, got %lld", (long long)D);
  if ((rc = check_page(page_size, &p.shift)) || (rc = check_count("requests", R)) || (rc = check_count("heads", H)) ||
      (rc = check_count("table width", width)))
    return rc;
  if (Hk < 1 || H < 1 || H > 65536 || H % Hk)
    return set_error(TATTN_E_ARG, "%lld heads do not share %lld key heads evenly", (long long)H, (long long)Hk);
  if (width * page_size > 0x7fffffff - 4096)
    return set_error(TATTN_E_ARG, "a table row of %lld pages holds 2^31 tokens or more", (long long)width);
  if (window < 0 || sinks < 0) return set_error(TATTN_E_ARG, "window and sinks must not be negative");
  p.R = (int32_t)R; p.Hk = (int32_t)Hk; p.G = (int32_t)(H / Hk); p.groups = (p.G + 15) / 16;
  if ((double)R * (double)Hk * p.groups > 67108864.0) return set_error(TATTN_E_ARG, "too many requests: %lld", (long long)R);
  p.most = (int32_t)(width * page_size);
  p.window = window == 0 || window > p.most ? p.most + 1 : (int32_t)window;
  p.sinks = (int32_t)(sinks < p.most ? sinks : p.most);
  cache4_chunks(p);
  return TATTN_OK;
}

}  // namespace
}  // namespace tattn

using namespace tattn;

extern "C" {

int tattn_page_tables(const int32_t* lens, const int32_t* new_tokens, int32_t* tables, const int32_t* free_pages,
                      int64_t* slots, int32_t* positions, int32_t* starts, int32_t* taken, int64_t R, int64_t P,
                      int64_t table_stride, int64_t F, int64_t T, int64_t page_size, void* stream) {
  TablesParams p{};
  int rc;
  if ((rc = check_page(page_size, &p.shift)) || (rc = check_count("requests", R)) || (rc = check_count("table width", P)) ||
      (rc = check_count("free pages", F)) || (rc = check_count("tokens", T)))
    return rc;
  if ((rc = check_ptr("lens", lens, R, 4)) || (rc = check_ptr("new_tokens", new_tokens, R, 4)) ||
      (rc = check_ptr("tables", tables, R * P, 4)) || (rc = check_ptr("free_pages", free_pages, F, 4)) ||
      (rc = check_ptr("slots", slots, T, 8)) || (rc = check_ptr("positions", positions, T, 4)) ||
      (rc = check_ptr("starts", starts, 1, 4)) || (rc = check_ptr("taken", taken, 1, 4)))
    return rc;
  if (R > 1 && table_stride < P) return set_error(TATTN_E_ARG, "table rows overlap: stride %lld", (long long)table_stride);
  if ((rc = require_device())) return rc;
  p.lens = lens; p.add = new_tokens; p.tables = tables; p.free_pages = free_pages;
  p.slots = slots; p.positions = positions; p.starts = starts; p.taken = taken;
  p.table_stride = table_stride;
  p.R = (int32_t)R; p.P = (int32_t)P; p.F = (int32_t)F; p.T = (int32_t)T;
  return launch_page_tables(p, (hipStream_t)stream);
}

int tattn_cache4_write(uint8_t* codes, uint8_t* scales, const void* k, const void* v, const int64_t* slots,
                       const int64_t k_strides[2], const int64_t v_strides[2], int64_t T, int64_t H, int64_t D,
                       int64_t pages, int64_t page_size, int dtype, void* stream) {
  Cache4Params p{};
  int rc;
  if ((rc = cache4_common(p, codes, scales, slots, T, H, D, pages, page_size, dtype))) return rc;
  if ((rc = check_ptr("k", k, T * H, 16)) || (rc = check_ptr("v", v, T * H, 16)) || (rc = check_rows("k", k_strides, 2, 2)) ||
      (rc = check_rows("v", v_strides, 2, 2)) || (rc = require_device()))
    return rc;
  if (T == 0 || H == 0 || pages == 0) return TATTN_OK;
  p.k = k; p.v = v;
  for (int i = 0; i < 2; ++i) p.sk[i] = k_strides[i], p.sv[i] = v_strides[i];
  return launch_cache4_write(p, (int)D, dtype, (hipStream_t)stream);
}

int tattn_cache4_read(const uint8_t* codes, const uint8_t* scales, void* k, void* v, const int64_t* slots, int64_t T,
                      int64_t H, int64_t D, int64_t pages, int64_t page_size, int dtype, void* stream) {
  Cache4Params p{};
  int rc;
  if ((rc = cache4_common(p, codes, scales, slots, T, H, D, pages, page_size, dtype))) return rc;
  if ((rc = check_ptr("k", k, T * H, 16)) || (rc = check_ptr("v", v, T * H, 16)) || (rc = require_device())) return rc;
  if (T == 0 || H == 0) return TATTN_OK;
  p.ko = k; p.vo = v;
  return launch_cache4_read(p, (int)D, dtype, (hipStream_t)stream);
}

int tattn_norm_rope_fwd(const void* q, const void* k, const void* q_weight, const void* k_weight, const float* cos,
                        const float* sin, const int32_t* positions, void* q_out, void* k_out, const int64_t q_strides[4],
                        const int64_t k_strides[4], const int64_t qo_strides[4], const int64_t ko_strides[4],
                        int64_t pos_stride, int64_t Z, int64_t H, int64_t Hk, int64_t N, int64_t D, int64_t P, int dtype,
                        int w_dtype, int interleaved, float eps, void* stream) {
  NormRopeParams p{};
  int rc;
  if ((rc = norm_rope_common(p, q, k, q_weight, k_weight, cos, sin, positions, q_strides, k_strides, pos_stride, Z, H, Hk,
                             N, D, P, dtype, w_dtype, eps)))
    return rc;
  const int sz = dtype == TATTN_F32 ? 4 : 2;
  if ((rc = check_ptr("q_out", q_out, Z * N, 16)) || (rc = check_ptr("k_out", k_out, Z * N, 16)) ||
      (rc = check_rows("q_out", qo_strides, 3, sz)) || (rc = check_rows("k_out", ko_strides, 3, sz)) || (rc = require_device()))
    return rc;
  if (Z == 0 || N == 0) return TATTN_OK;
  p.qo = q_out; p.ko = k_out;
  for (int i = 0; i < 3; ++i) p.sqo[i] = qo_strides[i], p.sko[i] = ko_strides[i];
  return launch_norm_rope(p, (int)D, dtype, interleaved != 0, false, (hipStream_t)stream);
}

int tattn_norm_rope_bwd(const void* q, const void* k, const void* q_weight, const void* k_weight, const float* cos,
                        const float* sin, const int32_t* positions, const void* dq_out, const void* dk_out, void* dq,
                        void* dk, void* dq_weight, void* dk_weight, float* workspace, const int64_t q_strides[4],
                        const int64_t k_strides[4], const int64_t dqo_strides[4], const int64_t dko_strides[4],
                        const int64_t dq_strides[4], const int64_t dk_strides[4], int64_t pos_stride, int64_t Z, int64_t H,
                        int64_t Hk, int64_t N, int64_t D, int64_t P, int dtype, int w_dtype, int interleaved, float eps,
                        void* stream) {
  NormRopeParams p{};
  int rc;
  if ((rc = norm_rope_common(p, q, k, q_weight, k_weight, cos, sin, positions, q_strides, k_strides, pos_stride, Z, H, Hk,
                             N, D, P, dtype, w_dtype, eps)))
    return rc;
  const int sz = dtype == TATTN_F32 ? 4 : 2;
  const int64_t rows = Z * N;
  if ((rc = check_ptr("dq_out", dq_out, rows, 16)) || (rc = check_ptr("dk_out", dk_out, rows, 16)) ||
      (rc = check_ptr("dq", dq, rows, 16)) || (rc = check_ptr("dk", dk, rows, 16)) ||
      (rc = check_rows("dq_out", dqo_strides, 3, sz)) || (rc = check_rows("dk_out", dko_strides, 3, sz)) ||
      (rc = check_rows("dq", dq_strides, 3, sz)) || (rc = check_rows("dk", dk_strides, 3, sz)))
    return rc;
  if (workspace) {
    if ((rc = check_ptr("dq_weight", dq_weight, 1, 2)) || (rc = check_ptr("dk_weight", dk_weight, 1, 2)) ||
        (rc = check_ptr("workspace", workspace, 1, 16)))
      return rc;
  } else if (dq_weight || dk_weight) {
    return set_error(TATTN_E_ARG, "weight gradients need the workspace");
  }
  if ((rc = require_device())) return rc;
  if (rows == 0) return TATTN_OK;
  p.gq = dq_out; p.gk = dk_out; p.qo = dq; p.ko = dk; p.dqw = dq_weight; p.dkw = dk_weight; p.partial = workspace;
  for (int i = 0; i < 3; ++i) {
    p.sqo[i] = dq_strides[i]; p.sko[i] = dk_strides[i]; p.sgq[i] = dqo_strides[i]; p.sgk[i] = dko_strides[i];
  }
  return launch_norm_rope(p, (int)D, dtype, interleaved != 0, true, (hipStream_t)stream);
}

int tattn_window_workspace(int backward, int64_t Z, int64_t H, int64_t Hk, int64_t N, int64_t S, int64_t D, int64_t window,
                           int64_t sinks, int64_t* floats) {
  WindowParams p{};
  int rc;
  if (!floats) return set_error(TATTN_E_ARG, "floats is a null pointer");
  if ((rc = window_common(p, Z, H, Hk, N, S, D, window, sinks, !backward))) return rc;
  if (backward) {
    window_bwd_parts(p, (int)D);
    *floats = window_bwd_part_floats(p, (int)D);
  } else {
    const int splits = window_fwd_splits(p, (int)D);
    *floats = splits > 1 ? window_part_floats(Z * Hk, N * p.G, splits, D) : 0;
  }
  return TATTN_OK;
}

int tattn_window_picked(int64_t Z, int64_t H, int64_t Hk, int64_t N, int64_t S, int64_t D, int64_t window, int64_t sinks) {
  WindowParams p{};
  if (window_common(p, Z, H, Hk, N, S, D, window, sinks, true)) return -1;
  return window_fwd_splits(p, (int)D);
}

int tattn_window_fwd(const void* q, const void* k, const void* v, void* o, float* m, const int32_t* lens, float* workspace,
                     const int64_t q_strides[4], const int64_t k_strides[4], const int64_t v_strides[4],
                     const int64_t o_strides[4], int64_t Z, int64_t H, int64_t Hk, int64_t N, int64_t S, int64_t D,
                     int64_t window, int64_t sinks, int dtype, float sm_scale, void* stream) {
  WindowParams p{};
  int rc;
  if ((rc = window_common(p, Z, H, Hk, N, S, D, window, sinks, lens != nullptr)) || (rc = check_dtype(dtype)) ||
      (rc = check_tiles("q", q, q_strides, N, D, dtype, p.sq)) || (rc = check_tiles("k", k, k_strides, S, D, dtype, p.sk)) ||
      (rc = check_tiles("v", v, v_strides, S, D, dtype, p.sv)) || (rc = check_tiles("o", o, o_strides, N, D, dtype, p.sout)) ||
      (rc = check_ptr("m", m, 0, 4)) || (rc = check_ptr("lens", lens, 0, 4)))
    return rc;
  p.splits = dtype == TATTN_F32 ? 0 : window_fwd_splits(p, (int)D);
  if ((rc = check_ptr("workspace", workspace, p.splits > 1, 16)) || (rc = require_device())) return rc;
  p.q = q; p.k = k; p.v = v; p.out = o; p.m = m; p.lens = lens; p.part = workspace;
  p.c = window_exponent_scale(sm_scale);
  p.scale = sm_scale;
  if (dtype == TATTN_F32) return launch_window_f32(p, (int)D, false, (hipStream_t)stream);
  return launch_window_fwd(p, (int)D, dtype, (hipStream_t)stream);
}

int tattn_window_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout, void* dq, void* dk,
                     void* dv, const float* m, float* delta, float* workspace, const int64_t q_strides[4],
                     const int64_t k_strides[4], const int64_t v_strides[4], const int64_t o_strides[4],
                     const int64_t do_strides[4], const int64_t dq_strides[4], const int64_t dk_strides[4],
                     const int64_t dv_strides[4], int64_t Z, int64_t H, int64_t Hk, int64_t N, int64_t S, int64_t D,
                     int64_t window, int64_t sinks, int dtype, float sm_scale, void* stream) {
  WindowParams p{};
  int rc;
  if ((rc = window_common(p, Z, H, Hk, N, S, D, window, sinks, false)) || (rc = check_dtype(dtype)) ||
      (rc = check_tiles("q", q, q_strides, N, D, dtype, p.sq)) || (rc = check_tiles("k", k, k_strides, S, D, dtype, p.sk)) ||
      (rc = check_tiles("v", v, v_strides, S, D, dtype, p.sv)) || (rc = check_tiles("o", o, o_strides, N, D, dtype, p.so)) ||
      (rc = check_tiles("do", dout, do_strides, N, D, dtype, p.sd)) || (rc = check_tiles("dq", dq, dq_strides, N, D, dtype, p.sout)) ||
      (rc = check_tiles("dk", dk, dk_strides, S, D, dtype, p.sdk)) || (rc = check_tiles("dv", dv, dv_strides, S, D, dtype, p.sdv)) ||
      (rc = check_ptr("m", m, 1, 4)) || (rc = check_ptr("delta", delta, 1, 8)))
    return rc;
  p.splits = p.parts = 1;
  if (dtype != TATTN_F32) window_bwd_parts(p, (int)D);
  if ((rc = check_ptr("workspace", workspace, p.splits > 1 || p.parts > 1, 16)) || (rc = require_device())) return rc;
  p.q = q; p.k = k; p.v = v; p.o = o; p.dout = dout; p.out = dq; p.dk = dk; p.dv = dv;
  p.m = const_cast<float*>(m);
  p.delta = delta;
  p.norms = delta + (Z * H * N + 1) / 2 * 2;
  p.part = workspace;
  p.c = window_exponent_scale(sm_scale);
  p.scale = sm_scale;
  if (dtype == TATTN_F32) return launch_window_f32(p, (int)D, true, (hipStream_t)stream);
  return launch_window_bwd(p, (int)D, dtype, (hipStream_t)stream);
}

int tattn_cache4_attention_workspace(int64_t R, int64_t H, int64_t Hk, int64_t D, int64_t width, int64_t page_size,
                                     int64_t window, int64_t sinks, int64_t* floats) {
  Cache4AttnParams p{};
  int rc;
  if (!floats) return set_error(TATTN_E_ARG, "floats is a null pointer");
  if ((rc = cache4_attn_common(p, R, H, Hk, D, width, page_size, window, sinks))) return rc;
  *floats = p.splits > 1 ? window_part_floats(R * Hk, p.G, p.splits, D) : 0;
  return TATTN_OK;
}

int tattn_cache4_attention(const void* q, void* o, const uint8_t* codes, const uint8_t* scales, const int32_t* tables,
                           const int32_t* lens, float* workspace, const int64_t q_strides[2], const int64_t o_strides[2],
                           int64_t table_stride, int64_t R, int64_t H, int64_t Hk, int64_t D, int64_t width, int64_t pages,
                           int64_t page_size, int64_t window, int64_t sinks, int dtype, float sm_scale, void* stream) {
  Cache4AttnParams p{};
  int rc;
  if ((rc = cache4_attn_common(p, R, H, Hk, D, width, page_size, window, sinks)) || (rc = check_16bit(dtype)) ||
      (rc = check_count("pages", pages)) || (rc = check_ptr("q", q, R, 16)) || (rc = check_ptr("o", o, R, 16)) ||
      (rc = check_rows("q", q_strides, 2, 2)) || (rc = check_rows("o", o_strides, 2, 2)) ||
      (rc = check_ptr("codes", codes, R, 16)) || (rc = check_ptr("scales", scales, R, 4)) ||
      (rc = check_ptr("tables", tables, R * width, 4)) || (rc = check_ptr("lens", lens, R, 4)) ||
      (rc = check_ptr("workspace", workspace, R > 0 && p.splits > 1, 16)))
    return rc;
  if (pages < 1) return set_error(TATTN_E_ARG, "the cache has no pages");
  if ((rc = require_device())) return rc;
  if (R == 0) return TATTN_OK;
  p.q = q; p.out = o; p.codes = codes; p.scales = scales; p.tables = tables; p.lens = lens; p.part = workspace;
  for (int i = 0; i < 2; ++i) p.sq[i] = q_strides[i], p.so[i] = o_strides[i];
  p.table_stride = table_stride;
  p.pages = (int32_t)pages;
  p.c = window_exponent_scale(sm_scale);
  return launch_cache4_attention(p, (int)D, dtype, (hipStream_t)stream);
}

}  // extern "C"
