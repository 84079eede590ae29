// C ABI of libtabicl_attn.so: argument checks, stride/layout translation from the reference's op
// signatures to the two kernel families, and the fit-time cache append kernel.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include "../../include/tabicl_attn.h"
#include "common.h"
#include "launch.h"
#include "paged.h"

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int launch_status(int err, const char* what) {
  if (err == 0) return 0;
  return fail(-err, "%s: HIP launch failed: %s", what, hipGetErrorString((hipError_t)err));
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
size_t esize(int32_t dtype) { return dtype == TABICL_DTYPE_BF16 ? 2 : 4; }
bool stride_ok(int64_t s, int32_t dtype) { return (s * (int64_t)esize(dtype)) % 16 == 0; }

// Shape rules of the small-head kernel: d = 16, h = 8, E = 128.
int smallhead_shape(const char* op, int64_t B, int64_t Lq, int64_t Lk, int64_t E, int32_t h,
                    int32_t dtype) {
  if (dtype != TABICL_DTYPE_BF16 && dtype != TABICL_DTYPE_F32)
    return fail(1, "%s: dtype code %d not supported", op, dtype);
  if (E != 128 || h != 8)
    return fail(1, "%s: needs E == 128 and h == 8 (head dim 16), got E=%lld h=%d", op,
                (long long)E, h);
  // no keys only where there is nothing to compute (no batch element or no query row: an empty
  // self-attention); the entry points return before any launch then
  const int64_t lk_min = B > 0 && Lq > 0 ? 1 : 0;
  if (B < 0 || Lq < 0 || Lk < lk_min || B > (1LL << 30) || Lq > (1LL << 30) || Lk > (1LL << 30))
    return fail(1, "%s: bad sizes B=%lld Lq=%lld Lk=%lld", op, (long long)B, (long long)Lq,
                (long long)Lk);
  return 0;
}

static_assert(TABICL_ROPE_SHARED_TABLES == TA_ROPE_SHARED, "shared-table RoPE flag");

// The rope code: none, or pairs / halves, optionally with TABICL_ROPE_SHARED_TABLES.
int rope_args(const char* op, int32_t rope, int32_t half, int32_t rot) {
  if (rope == TABICL_ROPE_NONE) return 0;
  rope &= ~TABICL_ROPE_SHARED_TABLES;
  if (rope != TABICL_ROPE_PAIRS && rope != TABICL_ROPE_HALVES)
    return fail(1, "%s: rope code %d not supported", op, rope);
  if (rot < 2 || rot > 16 || (rot & 1) || half * 2 != rot)
    return fail(1, "%s: rope needs even rot in [2, 16] and half == rot/2 (rot=%d half=%d)", op,
                rot, half);
  return 0;
}

template <typename T>
__global__ void cache_append_kernel(T* kc, T* vc, int64_t dst_sn, int64_t dst_sh, int64_t row0,
                                    const T* ks, const T* vs, int64_t src_sn, int64_t src_sh,
                                    int64_t src_st, int H, int T_rows, int D) {
  constexpr int EPC = 16 / sizeof(T);
  const int cpr = D / EPC;
  const int64_t total = (int64_t)gridDim.y * H * T_rows * cpr;  // gridDim.y = N
  const int n = blockIdx.y;
  for (int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; c < total / gridDim.y;
       c += (int64_t)gridDim.x * blockDim.x) {
    const int cc = (int)(c % cpr);
    const int64_t rowg = c / cpr;
    const int t = (int)(rowg % T_rows);
    const int h = (int)(rowg / T_rows);
    const int64_t so = n * src_sn + h * src_sh + t * src_st + cc * EPC;
    const int64_t dofs = n * dst_sn + h * dst_sh + (row0 + t) * D + cc * EPC;
    *(uint4*)(kc + dofs) = ldg16(ks + so);
    *(uint4*)(vc + dofs) = ldg16(vs + so);
  }
}

// Checks shared by the three backward entry points.
int bwd_common(const char* op, int64_t B, int64_t Lq, int64_t Lk, int64_t E, int32_t h, int32_t dtype,
               const float* bias, int64_t bias_b, const void* o, const void* dout, void* ws, int64_t ws_bytes) {
  int st = smallhead_shape(op, B, Lq, Lk, E, h, dtype);
  if (st) return st;
  if (bias && bias_b != 1 && bias_b != B)
    return fail(1, "%s: bias batch %lld must be 1 or B=%lld", op, (long long)bias_b, (long long)B);
  if (B > 0 && Lq > 0 && (!o || !dout || !aligned16(o) || !aligned16(dout)))
    return fail(1, "%s: o and dout must be 16-byte aligned device pointers", op);
  if (B > 0 && Lq > 0 && (!ws || !aligned16(ws) || ws_bytes < tabicl_launch_smallhead_bwd_ws_bytes(B, Lq)))
    return fail(1, "%s: workspace of %lld bytes (16-byte aligned) required", op,
                (long long)tabicl_launch_smallhead_bwd_ws_bytes(B, Lq));
  if (B * ((Lq + 127) / 128 + (Lk + 127) / 128) * 8 > (1LL << 31) - 1) return fail(1, "%s: grid too large", op);
  return 0;
}

// Argument checks shared by the ICL entry points (status 0 or 1 with the message set).
int icl_args(const char* op, const void* q, const void* k, const void* v, const int32_t* valid, int64_t valid_n,
             const float* key_bias, int64_t bias_n, int64_t bias_sn, const int32_t* q_len, int64_t q_len_n,
             const void* out, int64_t N, int64_t H, int64_t Tq, int64_t Tkv, int64_t D, const int64_t* strides,
             float scale, int32_t dtype) {
  if (dtype != TABICL_DTYPE_BF16 && dtype != TABICL_DTYPE_F32) return fail(1, "%s: dtype code %d not supported", op, dtype);
  if (key_bias) {
    if (bias_n != 1 && bias_n != N) return fail(1, "%s: key_bias must hold 1 or N rows", op);
    if (bias_n > 1 && bias_sn < Tkv) return fail(1, "%s: key_bias row stride %lld < Tkv", op, (long long)bias_sn);
    if (!aligned16(key_bias)) return fail(1, "%s: key_bias must be 16-byte aligned", op);
    if (!(scale > 0.f) || !(scale < 1e30f)) return fail(1, "%s: a key mask needs a positive finite scale", op);
  }
  if (D != 64) return fail(1, "%s: head dim must be 64, got %lld", op, (long long)D);
  if (N < 0 || H < 0 || Tq < 0 || Tkv < 1 || Tq > (1LL << 30) || Tkv > (1LL << 30)) return fail(1, "%s: bad sizes", op);
  if (valid && valid_n != 1 && valid_n != N) return fail(1, "%s: valid must hold 1 or N entries", op);
  if (q_len && q_len_n != 1 && q_len_n != N) return fail(1, "%s: q_len must hold 1 or N entries", op);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return fail(1, "%s: pointers must be 16-byte aligned", op);
  for (int i = 0; i < 12; ++i)
    if (strides[i] < 0 || !stride_ok(strides[i], dtype))
      return fail(1, "%s: strides must be non-negative multiples of 16 bytes", op);
  if (N * H * ((Tq + 127) / 128) > (1LL << 31) - 1) return fail(1, "%s: grid too large", op);
  return 0;
}

}  // namespace

extern "C" {

const char* tabicl_attn_last_error(void) { return g_err; }

const char* tabicl_attn_version(void) { return "tabicl_attn 0.1 gfx950"; }

int tabicl_attn_supported(int32_t op, int64_t Lq, int64_t Lk, int64_t E, int32_t h,
                          int32_t dtype) {
  if (dtype != TABICL_DTYPE_BF16 && dtype != TABICL_DTYPE_F32) return 0;
  if (Lq < 0 || Lk < 1 || Lq > (1LL << 30) || Lk > (1LL << 30)) return 0;
  switch (op) {
    case TABICL_OP_HX:
    case TABICL_OP_HXQ:
    case TABICL_OP_PK_SELF:
    case TABICL_OP_PK_CROSS:
      return E == 128 && h == 8;
    case TABICL_OP_ICL:
      return E == 64;
    default:
      return 0;
  }
}

int tabicl_hx_fwd(const void* q, const void* k, const void* v, const float* bias, int64_t bias_b,
                  void* out, int64_t B, int64_t Lq, int64_t Lk, int64_t E, int32_t h, int32_t dtype,
                  void* stream) {
  int st = smallhead_shape("hx_fwd", B, Lq, Lk, E, h, dtype);
  if (st) return st;
  if (bias && bias_b != 1 && bias_b != B)
    return fail(1, "hx_fwd: bias batch %lld must be 1 or B=%lld", (long long)bias_b, (long long)B);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || (bias && !aligned16(bias)))
    return fail(1, "hx_fwd: pointers must be 16-byte aligned");
  if (B == 0 || Lq == 0) return 0;
  return launch_status(
      tabicl_launch_smallhead(q, Lq * E, E, k, Lk * E, E, v, Lk * E, E, out, bias,
                              bias && bias_b == B ? Lk : 0, nullptr, 0, nullptr, nullptr, nullptr,
                              nullptr, 0, 0, 0, 1.0f, B, Lq, Lk, dtype, nullptr, 0,
                              (hipStream_t)stream),
      "hx_fwd");
}

int tabicl_hxq_fwd(const int32_t* valid, int64_t valid_n, const void* q, const void* kv, void* out,
                   int64_t B, int64_t Lq, int64_t Lk, int64_t E, int32_t h, int32_t dtype,
                   void* workspace, int64_t workspace_bytes, void* stream) {
  int st = smallhead_shape("hxq_fwd", B, Lq, Lk, E, h, dtype);
  if (st) return st;
  if (!valid || (valid_n != 1 && valid_n != B))
    return fail(1, "hxq_fwd: valid must hold 1 or B=%lld entries (got %lld)", (long long)B,
                (long long)valid_n);
  if (!aligned16(q) || !aligned16(kv) || !aligned16(out))
    return fail(1, "hxq_fwd: pointers must be 16-byte aligned");
  if (B == 0 || Lq == 0) return 0;
  const char* kvb = (const char*)kv;
  void* ws = workspace && aligned16(workspace) ? workspace : nullptr;
  return launch_status(
      tabicl_launch_smallhead(q, Lq * E, E, kvb, Lk * 2 * E, 2 * E, kvb + E * esize(dtype),
                              Lk * 2 * E, 2 * E, out, nullptr, 0, valid, valid_n, nullptr, nullptr,
                              nullptr, nullptr, 0, 0, 0, 1.0f, B, Lq, Lk, dtype, ws,
                              ws ? workspace_bytes : 0, (hipStream_t)stream),
      "hxq_fwd");
}

int tabicl_hxq_fwd_masked(const int32_t* valid, int64_t valid_n, const float* key_bias, int64_t bias_b,
                          const void* q, const void* kv, void* out, int64_t B, int64_t Lq, int64_t Lk, int64_t E,
                          int32_t h, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!key_bias) return tabicl_hxq_fwd(valid, valid_n, q, kv, out, B, Lq, Lk, E, h, dtype, workspace,
                                       workspace_bytes, stream);
  int st = smallhead_shape("hxq_fwd_masked", B, Lq, Lk, E, h, dtype);
  if (st) return st;
  if (valid && valid_n != 1 && valid_n != B)
    return fail(1, "hxq_fwd_masked: valid must hold 1 or B=%lld entries (got %lld)", (long long)B,
                (long long)valid_n);
  if (bias_b != 1 && bias_b != B)
    return fail(1, "hxq_fwd_masked: key_bias batch %lld must be 1 or B=%lld", (long long)bias_b, (long long)B);
  if (!aligned16(q) || !aligned16(kv) || !aligned16(out) || !aligned16(key_bias))
    return fail(1, "hxq_fwd_masked: pointers must be 16-byte aligned");
  if (B == 0 || Lq == 0) return 0;
  const char* kvb = (const char*)kv;
  void* ws = workspace && aligned16(workspace) ? workspace : nullptr;
  return launch_status(
      tabicl_launch_smallhead(q, Lq * E, E, kvb, Lk * 2 * E, 2 * E, kvb + E * esize(dtype), Lk * 2 * E, 2 * E, out,
                              key_bias, bias_b == B ? Lk : 0, valid, valid ? valid_n : 0, nullptr, nullptr,
                              nullptr, nullptr, 0, 0, 0, 1.0f, B, Lq, Lk, dtype, ws, ws ? workspace_bytes : 0,
                              (hipStream_t)stream),
      "hxq_fwd_masked");
}

int64_t tabicl_hxq_workspace_bytes(int64_t B, int64_t Lq, int64_t Lk, int64_t E, int32_t h,
                                   int32_t dtype) {
  if (E != 128 || h != 8 || B <= 0 || Lq <= 0 || Lk <= 0) return 0;
  if (dtype != TABICL_DTYPE_BF16 && dtype != TABICL_DTYPE_F32) return 0;
  // sized for tabicl_hxq_fwd_masked too (the prefix view of a key mask: 8 bytes per batch element)
  return tabicl_launch_smallhead_ws_bytes(B, Lq, Lk, dtype, true, 0);
}

int tabicl_pk_self_fwd(const void* qkv, const float* bias, int64_t bias_b, const float* cos_t,
                       const float* sin_t, void* out, int64_t B, int64_t L, int64_t E, int32_t h,
                       int32_t rope, int32_t half, int32_t rot, float scale, int32_t dtype,
                       void* stream) {
  int st = smallhead_shape("pk_self_fwd", B, L, L, E, h, dtype);
  if (st) return st;
  if ((st = rope_args("pk_self_fwd", rope, half, rot))) return st;
  if (rope && (!cos_t || !sin_t)) return fail(1, "pk_self_fwd: rope tables missing");
  if (bias && bias_b != 1 && bias_b != B)
    return fail(1, "pk_self_fwd: bias batch %lld must be 1 or B", (long long)bias_b);
  if (!aligned16(qkv) || !aligned16(out) || (rope && (!aligned16(cos_t) || !aligned16(sin_t))))
    return fail(1, "pk_self_fwd: pointers must be 16-byte aligned");
  if (B == 0 || L == 0) return 0;
  const char* base = (const char*)qkv;
  const size_t es = esize(dtype);
  return launch_status(
      tabicl_launch_smallhead(base, L * 3 * E, 3 * E, base + E * es, L * 3 * E, 3 * E,
                              base + 2 * E * es, L * 3 * E, 3 * E, out, bias,
                              bias && bias_b == B ? L : 0, nullptr, 0, cos_t, sin_t, cos_t, sin_t,
                              rope, half, rot, scale, B, L, L, dtype, nullptr, 0,
                              (hipStream_t)stream),
      "pk_self_fwd");
}

int tabicl_pk_cross_fwd(const void* q, int64_t q_b, const void* kv, const float* bias,
                        int64_t bias_b, const float* cq, const float* sq, const float* ck,
                        const float* sk, void* out, int64_t B, int64_t Lq, int64_t Lk, int64_t E,
                        int32_t h, int32_t rope, int32_t half, int32_t rot, float scale,
                        int32_t dtype, void* stream) {
  return tabicl_pk_cross_fwd_ragged(q, q_b, kv, bias, bias_b, cq, sq, ck, sk, out, B, Lq, Lk, E, h, rope, half,
                                    rot, scale, dtype, nullptr, 0, stream);
}

int tabicl_pk_cross_fwd_ragged(const void* q, int64_t q_b, const void* kv, const float* bias,
                               int64_t bias_b, const float* cq, const float* sq, const float* ck,
                               const float* sk, void* out, int64_t B, int64_t Lq, int64_t Lk, int64_t E,
                               int32_t h, int32_t rope, int32_t half, int32_t rot, float scale,
                               int32_t dtype, const int32_t* q_len, int64_t q_len_n, void* stream) {
  int st = smallhead_shape("pk_cross_fwd", B, Lq, Lk, E, h, dtype);
  if (st) return st;
  if ((st = rope_args("pk_cross_fwd", rope, half, rot))) return st;
  if (rope && (!cq || !sq || !ck || !sk)) return fail(1, "pk_cross_fwd: rope tables missing");
  if (q_b != 1 && q_b != B) return fail(1, "pk_cross_fwd: q batch must be 1 or B");
  if (q_len && q_len_n != 1 && q_len_n != B) return fail(1, "pk_cross_fwd: q_len must hold 1 or B entries");
  if (bias && bias_b != 1 && bias_b != B)
    return fail(1, "pk_cross_fwd: bias batch %lld must be 1 or B", (long long)bias_b);
  if (!aligned16(q) || !aligned16(kv) || !aligned16(out) ||
      (rope && (!aligned16(cq) || !aligned16(sq) || !aligned16(ck) || !aligned16(sk))))
    return fail(1, "pk_cross_fwd: pointers must be 16-byte aligned");
  if (B == 0 || Lq == 0) return 0;
  const char* kvb = (const char*)kv;
  return launch_status(
      tabicl_launch_smallhead(q, q_b == 1 && B > 1 ? 0 : Lq * E, E, kvb, Lk * 2 * E, 2 * E,
                              kvb + E * esize(dtype), Lk * 2 * E, 2 * E, out, bias,
                              bias && bias_b == B ? Lk : 0, nullptr, 0, cq, sq, ck, sk, rope, half,
                              rot, scale, B, Lq, Lk, dtype, nullptr, 0, (hipStream_t)stream, q_len,
                              q_len ? q_len_n : 0),
      "pk_cross_fwd");
}

int64_t tabicl_smallhead_bwd_workspace_bytes(int64_t B, int64_t Lq, int64_t E, int32_t h) {
  if (E != 128 || h != 8 || B < 0 || Lq < 0) return fail(-1, "smallhead_bwd_workspace_bytes: bad arguments");
  return tabicl_launch_smallhead_bwd_ws_bytes(B, Lq);
}

int tabicl_hx_bwd(const void* q, const void* k, const void* v, const float* bias, int64_t bias_b,
                  const void* o, const void* dout, void* dq, void* dk, void* dv, int64_t B, int64_t Lq,
                  int64_t Lk, int64_t E, int32_t h, int32_t dtype, void* workspace, int64_t workspace_bytes,
                  void* stream) {
  int st = bwd_common("hx_bwd", B, Lq, Lk, E, h, dtype, bias, bias_b, o, dout, workspace, workspace_bytes);
  if (st) return st;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv))
    return fail(1, "hx_bwd: pointers must be 16-byte aligned");
  if (B == 0 || Lk == 0) return 0;
  return launch_status(
      tabicl_launch_smallhead_bwd(q, Lq * E, E, k, Lk * E, E, v, Lk * E, E, o, dout, dq, Lq * E, E, dk, Lk * E, E,
                                  dv, Lk * E, E, bias, bias && bias_b == B ? Lk : 0, nullptr, nullptr, nullptr,
                                  nullptr, 0, 0, 0, 1.0f, B, Lq, Lk, dtype, workspace, workspace_bytes,
                                  (hipStream_t)stream),
      "hx_bwd");
}

int tabicl_pk_self_bwd(const void* qkv, const float* bias, int64_t bias_b, const float* cos_t,
                       const float* sin_t, const void* o, const void* dout, void* dqkv, int64_t B, int64_t L,
                       int64_t E, int32_t h, int32_t rope, int32_t half, int32_t rot, float scale, int32_t dtype,
                       void* workspace, int64_t workspace_bytes, void* stream) {
  int st = bwd_common("pk_self_bwd", B, L, L, E, h, dtype, bias, bias_b, o, dout, workspace, workspace_bytes);
  if (st) return st;
  if ((st = rope_args("pk_self_bwd", rope, half, rot))) return st;
  if (rope && (!cos_t || !sin_t)) return fail(1, "pk_self_bwd: rope tables missing");
  if (!aligned16(qkv) || !aligned16(dqkv) || (rope && (!aligned16(cos_t) || !aligned16(sin_t))))
    return fail(1, "pk_self_bwd: pointers must be 16-byte aligned");
  if (B == 0 || L == 0) return 0;
  const char* base = (const char*)qkv;
  char* dbase = (char*)dqkv;
  const size_t es = esize(dtype);
  return launch_status(
      tabicl_launch_smallhead_bwd(base, L * 3 * E, 3 * E, base + E * es, L * 3 * E, 3 * E, base + 2 * E * es,
                                  L * 3 * E, 3 * E, o, dout, dbase, L * 3 * E, 3 * E, dbase + E * es, L * 3 * E,
                                  3 * E, dbase + 2 * E * es, L * 3 * E, 3 * E, bias, bias && bias_b == B ? L : 0,
                                  cos_t, sin_t, cos_t, sin_t, rope, half, rot, scale, B, L, L, dtype, workspace,
                                  workspace_bytes, (hipStream_t)stream),
      "pk_self_bwd");
}

int tabicl_pk_cross_bwd(const void* q, int64_t q_b, const void* kv, const float* bias, int64_t bias_b,
                        const float* cq, const float* sq, const float* ck, const float* sk, const void* o,
                        const void* dout, void* dq, void* dkv, int64_t B, int64_t Lq, int64_t Lk, int64_t E,
                        int32_t h, int32_t rope, int32_t half, int32_t rot, float scale, int32_t dtype,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  int st = bwd_common("pk_cross_bwd", B, Lq, Lk, E, h, dtype, bias, bias_b, o, dout, workspace, workspace_bytes);
  if (st) return st;
  if ((st = rope_args("pk_cross_bwd", rope, half, rot))) return st;
  if (rope && (!cq || !sq || !ck || !sk)) return fail(1, "pk_cross_bwd: rope tables missing");
  if (q_b != 1 && q_b != B) return fail(1, "pk_cross_bwd: q batch must be 1 or B");
  if (rope && (!aligned16(cq) || !aligned16(sq) || !aligned16(ck) || !aligned16(sk)))
    return fail(1, "pk_cross_bwd: rope tables must be 16-byte aligned");
  if (!aligned16(q) || !aligned16(kv) || !aligned16(dq) || !aligned16(dkv))
    return fail(1, "pk_cross_bwd: pointers must be 16-byte aligned");
  if (B == 0 || Lk == 0) return 0;
  const char* kvb = (const char*)kv;
  char* dkvb = (char*)dkv;
  const size_t es = esize(dtype);
  return launch_status(
      tabicl_launch_smallhead_bwd(q, q_b == 1 && B > 1 ? 0 : Lq * E, E, kvb, Lk * 2 * E, 2 * E, kvb + E * es,
                                  Lk * 2 * E, 2 * E, o, dout, dq, Lq * E, E, dkvb, Lk * 2 * E, 2 * E,
                                  dkvb + E * es, Lk * 2 * E, 2 * E, bias, bias && bias_b == B ? Lk : 0, cq, sq,
                                  ck, sk, rope, half, rot, scale, B, Lq, Lk, dtype, workspace, workspace_bytes,
                                  (hipStream_t)stream),
      "pk_cross_bwd");
}

int tabicl_icl_fwd(const void* q, const void* k, const void* v, const int32_t* valid,
                   int64_t valid_n, void* out, int64_t N, int64_t H, int64_t Tq, int64_t Tkv,
                   int64_t D, int64_t q_sn, int64_t q_sh, int64_t q_st, int64_t k_sn, int64_t k_sh,
                   int64_t k_st, int64_t v_sn, int64_t v_sh, int64_t v_st, int64_t o_sn,
                   int64_t o_sh, int64_t o_st, float scale, int32_t dtype, void* workspace,
                   int64_t workspace_bytes, void* stream) {
  return tabicl_icl_fwd_ragged(q, k, v, valid, valid_n, nullptr, 0, out, N, H, Tq, Tkv, D, q_sn, q_sh, q_st, k_sn,
                               k_sh, k_st, v_sn, v_sh, v_st, o_sn, o_sh, o_st, scale, dtype, workspace,
                               workspace_bytes, stream);
}

int tabicl_icl_fwd_ragged(const void* q, const void* k, const void* v, const int32_t* valid,
                          int64_t valid_n, const int32_t* q_len, int64_t q_len_n, void* out, int64_t N,
                          int64_t H, int64_t Tq, int64_t Tkv, int64_t D, int64_t q_sn, int64_t q_sh,
                          int64_t q_st, int64_t k_sn, int64_t k_sh, int64_t k_st, int64_t v_sn,
                          int64_t v_sh, int64_t v_st, int64_t o_sn, int64_t o_sh, int64_t o_st,
                          float scale, int32_t dtype, void* workspace, int64_t workspace_bytes,
                          void* stream) {
  return tabicl_icl_fwd_masked(q, k, v, valid, valid_n, nullptr, 0, 0, q_len, q_len_n, out, N, H, Tq, Tkv, D, q_sn,
                               q_sh, q_st, k_sn, k_sh, k_st, v_sn, v_sh, v_st, o_sn, o_sh, o_st, scale, dtype,
                               workspace, workspace_bytes, stream);
}

int tabicl_icl_fwd_ragged_listed(const void* q, const void* k, const void* v, const int32_t* valid,
                                 int64_t valid_n, const int32_t* q_len, int64_t q_len_n, void* out, int64_t N,
                                 int64_t H, int64_t Tq, int64_t Tkv, int64_t D, int64_t q_sn, int64_t q_sh,
                                 int64_t q_st, int64_t k_sn, int64_t k_sh, int64_t k_st, int64_t v_sn,
                                 int64_t v_sh, int64_t v_st, int64_t o_sn, int64_t o_sh, int64_t o_st,
                                 float scale, int32_t dtype, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  const int64_t strides[12] = {q_sn, q_sh, q_st, k_sn, k_sh, k_st, v_sn, v_sh, v_st, o_sn, o_sh, o_st};
  int st = icl_args("icl_fwd_ragged_listed", q, k, v, valid, valid_n, nullptr, 0, 0, q_len, q_len_n, out, N, H, Tq,
                    Tkv, D, strides, scale, dtype);
  if (st || N == 0 || H == 0 || Tq == 0) return st;
  if (!q_len) return fail(1, "icl_fwd_ragged_listed: q_len is required");
  return launch_status(
      tabicl_launch_icl_fwd(q, k, v, valid, valid ? valid_n : 0, out, N, H, Tq, Tkv, 64, q_sn, q_sh, q_st, k_sn,
                            k_sh, k_st, v_sn, v_sh, v_st, o_sn, o_sh, o_st, scale, dtype,
                            workspace && aligned16(workspace) ? workspace : nullptr, workspace_bytes,
                            (hipStream_t)stream, q_len, q_len_n, nullptr, 0, 0, 1),
      "icl_fwd_ragged_listed");
}

int tabicl_icl_ragged_plan(const int32_t* q_len, int64_t q_len_n, int64_t N, int64_t H, int64_t Tq, int64_t Tkv,
                           int64_t D, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  if (N < 0 || H < 0 || Tq < 0 || Tkv < 0) return fail(1, "icl_ragged_plan: negative size");
  if (D != 64) return fail(1, "icl_ragged_plan: D must be 64");
  if (dtype != 0 && dtype != 1) return fail(1, "icl_ragged_plan: dtype must be 0 (bf16) or 1 (fp32)");
  if (!q_len || (q_len_n != 1 && q_len_n != N)) return fail(1, "icl_ragged_plan: q_len [1 or N] is required");
  if (N == 0 || H == 0 || Tq == 0 || Tkv == 0) return 0;
  if (workspace && !aligned16(workspace)) return fail(1, "icl_ragged_plan: workspace must be 16-byte aligned");
  // the list goes where the call puts it: the kernels need no q / k / v / out here, only their sizes
  return launch_status(
      tabicl_launch_icl_fwd(nullptr, nullptr, nullptr, nullptr, 0, nullptr, N, H, Tq, Tkv, 64, 0, 0, 0, 0, 0, 0, 0,
                            0, 0, 0, 0, 0, 1.0f, dtype, workspace, workspace ? workspace_bytes : 0,
                            (hipStream_t)stream, q_len, q_len_n, nullptr, 0, 0, 2),
      "icl_ragged_plan");
}

int tabicl_icl_fwd_masked(const void* q, const void* k, const void* v, const int32_t* valid, int64_t valid_n,
                          const float* key_bias, int64_t bias_n, int64_t bias_sn, const int32_t* q_len,
                          int64_t q_len_n, void* out, int64_t N, int64_t H, int64_t Tq, int64_t Tkv, int64_t D,
                          int64_t q_sn, int64_t q_sh, int64_t q_st, int64_t k_sn, int64_t k_sh, int64_t k_st,
                          int64_t v_sn, int64_t v_sh, int64_t v_st, int64_t o_sn, int64_t o_sh, int64_t o_st,
                          float scale, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const int64_t strides[12] = {q_sn, q_sh, q_st, k_sn, k_sh, k_st, v_sn, v_sh, v_st, o_sn, o_sh, o_st};
  int st = icl_args("icl_fwd", q, k, v, valid, valid_n, key_bias, bias_n, bias_sn, q_len, q_len_n, out, N, H, Tq,
                    Tkv, D, strides, scale, dtype);
  if (st || N == 0 || H == 0 || Tq == 0) return st;
  return launch_status(
      tabicl_launch_icl_fwd(q, k, v, valid, valid ? valid_n : 0, out, N, H, Tq, Tkv, 64, q_sn, q_sh,
                            q_st, k_sn, k_sh, k_st, v_sn, v_sh, v_st, o_sn, o_sh, o_st, scale,
                            dtype, workspace && aligned16(workspace) ? workspace : nullptr,
                            workspace_bytes, (hipStream_t)stream, q_len, q_len ? q_len_n : 0, key_bias,
                            key_bias ? bias_n : 0, key_bias ? bias_sn : 0),
      "icl_fwd");
}

int64_t tabicl_icl_bwd_workspace_bytes(int64_t N, int64_t H, int64_t Tq) {
  if (N < 0 || H < 0 || Tq < 0) return fail(-1, "icl_bwd_workspace_bytes: bad sizes");
  return tabicl_launch_icl_bwd_ws_bytes(N, H, Tq);
}

int tabicl_icl_bwd(const void* q, const void* k, const void* v, const int32_t* valid, int64_t valid_n,
                   const float* key_bias, int64_t bias_n, int64_t bias_sn, const void* o, const void* dout,
                   const float* stat, void* dq, void* dk, void* dv, int64_t N, int64_t H, int64_t Tq, int64_t Tkv,
                   int64_t D, float scale, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  // contiguous [N, H, T, 64] tensors: the strides the shared checks take
  const int64_t sq[3] = {H * Tq * D, Tq * D, D}, sk[3] = {H * Tkv * D, Tkv * D, D};
  const int64_t strides[12] = {sq[0], sq[1], sq[2], sk[0], sk[1], sk[2], sk[0], sk[1], sk[2], sq[0], sq[1], sq[2]};
  int st = icl_args("icl_bwd", q, k, v, valid, valid_n, key_bias, bias_n, bias_sn, nullptr, 0, o, N, H, Tq, Tkv, D,
                    strides, scale, dtype);
  if (st) return st;
  if (!(scale > 0.f) || !(scale < 1e30f)) return fail(1, "icl_bwd: scale must be positive and finite");
  if (!aligned16(dout) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv) || !aligned16(stat))
    return fail(1, "icl_bwd: pointers must be 16-byte aligned");
  if (stat && key_bias) return fail(1, "icl_bwd: forward statistics are taken for calls without a key mask only");
  if (N * H * ((Tkv + 63) / 64) > (1LL << 31) - 1 || N * H * ((Tq + 63) / 64) > (1LL << 31) - 1)
    return fail(1, "icl_bwd: grid too large");
  if (N == 0 || H == 0) return 0;
  if (!workspace || !aligned16(workspace) || workspace_bytes < tabicl_launch_icl_bwd_ws_bytes(N, H, Tq))
    return fail(1, "icl_bwd: workspace of %lld bytes (16-byte aligned) required",
                (long long)tabicl_launch_icl_bwd_ws_bytes(N, H, Tq));
  return launch_status(tabicl_launch_icl_bwd(q, k, v, valid, valid ? valid_n : 0, key_bias, key_bias ? bias_n : 0,
                                             key_bias ? bias_sn : 0, o, dout, stat, dq, dk, dv, N, H, Tq, Tkv, scale,
                                             dtype, workspace, workspace_bytes, (hipStream_t)stream),
                       "icl_bwd");
}

int tabicl_icl_fwd_stats(const void* q, const void* k, const void* v, const int32_t* valid, int64_t valid_n,
                         void* out, float* stat, int64_t N, int64_t H, int64_t Tq, int64_t Tkv, int64_t D,
                         int64_t q_sn, int64_t q_sh, int64_t q_st, int64_t k_sn, int64_t k_sh, int64_t k_st,
                         int64_t v_sn, int64_t v_sh, int64_t v_st, int64_t o_sn, int64_t o_sh, int64_t o_st,
                         float scale, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const int64_t strides[12] = {q_sn, q_sh, q_st, k_sn, k_sh, k_st, v_sn, v_sh, v_st, o_sn, o_sh, o_st};
  int st = icl_args("icl_fwd_stats", q, k, v, valid, valid_n, nullptr, 0, 0, nullptr, 0, out, N, H, Tq, Tkv, D,
                    strides, scale, dtype);
  if (st || N == 0 || H == 0 || Tq == 0) return st;
  if (!stat || !aligned16(stat)) return fail(1, "icl_fwd_stats: stat ([N, H, Tq, 2] fp32, 16-byte aligned) is required");
  return launch_status(
      tabicl_launch_icl_fwd(q, k, v, valid, valid ? valid_n : 0, out, N, H, Tq, Tkv, 64, q_sn, q_sh, q_st, k_sn,
                            k_sh, k_st, v_sn, v_sh, v_st, o_sn, o_sh, o_st, scale, dtype,
                            workspace && aligned16(workspace) ? workspace : nullptr, workspace_bytes,
                            (hipStream_t)stream, nullptr, 0, nullptr, 0, 0, 0, stat),
      "icl_fwd_stats");
}

int tabicl_icl_fwd_noalloc(const void* q, const void* k, const void* v, const int32_t* valid, int64_t valid_n,
                           const float* key_bias, int64_t bias_n, int64_t bias_sn, const int32_t* q_len,
                           int64_t q_len_n, void* out, int64_t N, int64_t H, int64_t Tq, int64_t Tkv, int64_t D,
                           int64_t q_sn, int64_t q_sh, int64_t q_st, int64_t k_sn, int64_t k_sh, int64_t k_st,
                           int64_t v_sn, int64_t v_sh, int64_t v_st, int64_t o_sn, int64_t o_sh, int64_t o_st,
                           float scale, int32_t dtype, void* stream) {
  const int64_t strides[12] = {q_sn, q_sh, q_st, k_sn, k_sh, k_st, v_sn, v_sh, v_st, o_sn, o_sh, o_st};
  int st = icl_args("icl_fwd_noalloc", q, k, v, valid, valid_n, key_bias, bias_n, bias_sn, q_len, q_len_n, out, N, H,
                    Tq, Tkv, D, strides, scale, dtype);
  if (st || N == 0 || H == 0 || Tq == 0) return st;
  const int64_t need = tabicl_launch_icl_noalloc_min_bytes(N, H, Tq, D, dtype);
  if (need > TABICL_ICL_SCRATCH_BYTES)
    return fail(1, "icl_fwd_noalloc: the call needs %lld bytes of scratch, more than the library's %lld (use "
                "tabicl_icl_fwd with a workspace)", (long long)need, (long long)TABICL_ICL_SCRATCH_BYTES);
  return launch_status(
      tabicl_launch_icl_fwd_noalloc(q, k, v, valid, valid ? valid_n : 0, out, N, H, Tq, Tkv, q_sn, q_sh, q_st, k_sn,
                                    k_sh, k_st, v_sn, v_sh, v_st, o_sn, o_sh, o_st, scale, dtype, (hipStream_t)stream,
                                    q_len, q_len ? q_len_n : 0, key_bias, key_bias ? bias_n : 0,
                                    key_bias ? bias_sn : 0),
      "icl_fwd_noalloc");
}

int64_t tabicl_icl_noalloc_scratch_bytes(void) { return TABICL_ICL_SCRATCH_BYTES; }

int64_t tabicl_icl_workspace_bytes(int64_t N, int64_t H, int64_t Tq, int64_t Tkv, int64_t D,
                                   int32_t dtype) {
  if ((dtype != TABICL_DTYPE_BF16 && dtype != TABICL_DTYPE_F32) || D != 64 || N < 0 || H < 0 ||
      Tq < 0 || Tkv < 1)
    return fail(-1, "icl_workspace_bytes: bad arguments");
  if (N == 0 || H == 0 || Tq == 0) return 0;
  return tabicl_launch_icl_ws_bytes(N, H, Tq, Tkv, 64, dtype);
}

int tabicl_hxf_fwd(const int32_t* valid, int64_t valid_n, const void* qf, int64_t q_b, const void* x, void* out,
                   int64_t B, int64_t hq, int64_t Lk, int64_t E, int32_t dtype, void* workspace,
                   int64_t workspace_bytes, void* stream) {
  if (!valid) return fail(1, "hxf_fwd: valid is required");
  return tabicl_hxf_fwd_masked(valid, valid_n, nullptr, 0, qf, q_b, x, out, B, hq, Lk, E, dtype, workspace,
                               workspace_bytes, stream);
}

int tabicl_hxf_fwd_masked(const int32_t* valid, int64_t valid_n, const float* key_bias, int64_t bias_b,
                          const void* qf, int64_t q_b, const void* x, void* out, int64_t B, int64_t hq, int64_t Lk,
                          int64_t E, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  if (dtype != TABICL_DTYPE_BF16 && dtype != TABICL_DTYPE_F32)
    return fail(1, "hxf_fwd: dtype code %d not supported", dtype);
  if (key_bias && bias_b != 1 && bias_b != B) return fail(1, "hxf_fwd: key_bias must hold 1 or B rows");
  if (key_bias && !aligned16(key_bias)) return fail(1, "hxf_fwd: key_bias must be 16-byte aligned");
  if (E != 128) return fail(1, "hxf_fwd: needs E == 128, got %lld", (long long)E);
  if (B < 0 || hq < 0 || Lk < 1 || B > (1LL << 30) || hq > (1LL << 30) || Lk > (1LL << 30))
    return fail(1, "hxf_fwd: bad sizes B=%lld hq=%lld Lk=%lld", (long long)B, (long long)hq, (long long)Lk);
  if (q_b != 1 && q_b != B) return fail(1, "hxf_fwd: qf batch must be 1 or B");
  if (valid && valid_n != 1 && valid_n != B)
    return fail(1, "hxf_fwd: valid must hold 1 or B=%lld entries", (long long)B);
  if (!aligned16(qf) || !aligned16(x) || !aligned16(out)) return fail(1, "hxf_fwd: pointers must be 16-byte aligned");
  if (B == 0 || hq == 0) return 0;
  if (B * ((hq + 127) / 128) * 4 > (1LL << 31) - 1) return fail(1, "hxf_fwd: grid too large");
  return launch_status(
      tabicl_launch_icl_fwd(qf, x, x, valid, valid ? valid_n : 0, out, B, 1, hq, Lk, 128,
                            q_b == 1 && B > 1 ? 0 : hq * E, 0, E, Lk * E, 0, E, Lk * E, 0, E, hq * E, 0, E, 1.0f,
                            dtype, workspace && aligned16(workspace) ? workspace : nullptr, workspace_bytes,
                            (hipStream_t)stream, nullptr, 0, key_bias, key_bias ? bias_b : 0,
                            key_bias && bias_b > 1 ? Lk : 0),
      "hxf_fwd");
}

int64_t tabicl_hxf_workspace_bytes(int64_t B, int64_t hq, int64_t Lk, int64_t E, int32_t dtype) {
  if ((dtype != TABICL_DTYPE_BF16 && dtype != TABICL_DTYPE_F32) || E != 128 || B < 0 || hq < 0 || Lk < 1)
    return fail(-1, "hxf_workspace_bytes: bad arguments");
  if (B == 0 || hq == 0) return 0;
  return tabicl_launch_icl_ws_bytes(B, 1, hq, Lk, 128, dtype);
}

int tabicl_icl_cache_append(void* k_cache, void* v_cache, int64_t dst_sn, int64_t dst_sh,
                            int64_t row0, int64_t cap, const void* k_src, const void* v_src,
                            int64_t src_sn, int64_t src_sh, int64_t src_st, int64_t N, int64_t H,
                            int64_t T, int64_t D, int32_t dtype, void* stream) {
  if (dtype != TABICL_DTYPE_BF16 && dtype != TABICL_DTYPE_F32)
    return fail(1, "icl_cache_append: dtype code %d not supported", dtype);
  if (D < 1 || (D * (int64_t)esize(dtype)) % 16) return fail(1, "icl_cache_append: bad head dim");
  if (row0 < 0 || T < 0 || row0 + T > cap)
    return fail(1, "icl_cache_append: rows [%lld, %lld) exceed capacity %lld", (long long)row0,
                (long long)(row0 + T), (long long)cap);
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_src) || !aligned16(v_src))
    return fail(1, "icl_cache_append: pointers must be 16-byte aligned");
  const int64_t s[5] = {dst_sn, dst_sh, src_sn, src_sh, src_st};
  for (int i = 0; i < 5; ++i)
    if (s[i] < 0 || !stride_ok(s[i], dtype))
      return fail(1, "icl_cache_append: strides must be non-negative multiples of 16 bytes");
  if (N == 0 || H == 0 || T == 0) return 0;
  if (N > 65535) return fail(1, "icl_cache_append: N too large");
  const int64_t per_n = H * T * (D * (int64_t)esize(dtype) / 16);
  int64_t gx = (per_n + 255) / 256;
  if (gx > 65536) gx = 65536;
  hipStream_t s0 = (hipStream_t)stream;
  if (dtype == TABICL_DTYPE_BF16)
    hipLaunchKernelGGL(cache_append_kernel<bf16>, dim3((unsigned)gx, (unsigned)N), dim3(256), 0, s0,
                       (bf16*)k_cache, (bf16*)v_cache, dst_sn, dst_sh, row0, (const bf16*)k_src,
                       (const bf16*)v_src, src_sn, src_sh, src_st, (int)H, (int)T, (int)D);
  else
    hipLaunchKernelGGL(cache_append_kernel<float>, dim3((unsigned)gx, (unsigned)N), dim3(256), 0, s0,
                       (float*)k_cache, (float*)v_cache, dst_sn, dst_sh, row0, (const float*)k_src,
                       (const float*)v_src, src_sn, src_sh, src_st, (int)H, (int)T, (int)D);
  return launch_status((int)hipGetLastError(), "icl_cache_append");
}

}  // extern "C"

int tabicl_layer_norm(const void* x, const void* residual, void* x_out, const float* weight, const float* bias,
                      void* out, int64_t rows, int64_t width, float eps, int32_t in_dtype, int32_t out_dtype,
                      void* stream) {
  if (rows < 0) return fail(1, "layer_norm: negative row count");
  if (width != 128 && width != 512) return fail(1, "layer_norm: width %lld not supported (128 or 512)", (long long)width);
  if ((in_dtype != 0 && in_dtype != 1) || (out_dtype != 0 && out_dtype != 1))
    return fail(1, "layer_norm: dtypes must be 0 (bf16) or 1 (fp32)");
  if (!(eps > 0.f)) return fail(1, "layer_norm: eps must be positive");
  if (rows == 0) return 0;
  if (!x || !out || !aligned16(x) || !aligned16(out) || (weight && !aligned16(weight)) || (bias && !aligned16(bias)))
    return fail(1, "layer_norm: x, out, weight and bias must be 16-byte aligned device pointers");
  if (residual && (!x_out || !aligned16(residual) || !aligned16(x_out)))
    return fail(1, "layer_norm: with a residual, x_out (16-byte aligned) receives x + residual");
  return launch_status(tabicl_launch_layer_norm(x, residual, residual ? x_out : nullptr, weight, bias, out, rows, width,
                                                eps, in_dtype, out_dtype, (hipStream_t)stream),
                       "layer_norm");
}

static int layer_args(const char* op, int64_t rows, int32_t dtype, float eps, const void* live, int64_t group_rows) {
  if (dtype != 0 && dtype != 1) return fail(1, "%s: dtype must be 0 (bf16) or 1 (fp32)", op);
  if (rows < 0 || rows > 0xffffffffLL) return fail(1, "%s: %lld rows not supported", op, (long long)rows);
  if (!(eps > 0.f)) return fail(1, "%s: eps must be positive", op);
  if (live && (group_rows < 1 || group_rows > 0xffffffffLL)) return fail(1, "%s: group_rows must be positive", op);
  return 0;
}

int tabicl_layer_proj(const void* x, const float* ln_weight, const float* ln_bias, float eps, const void* weight,
                      const void* bias, void* out, int64_t rows, int64_t n_out, int32_t dtype, int32_t* live,
                      int64_t group_rows, float skip, void* ws, int64_t ws_bytes, void* stream) {
  int st = layer_args("layer_proj", rows, dtype, eps, live, group_rows);
  if (st) return st;
  if (n_out != 128 && n_out != 256 && n_out != 384)
    return fail(1, "layer_proj: n_out %lld not supported (128, 256 or 384)", (long long)n_out);
  if (rows == 0) return 0;
  if (!x || !weight || !out || !aligned16(x) || !aligned16(weight) || !aligned16(out))
    return fail(1, "layer_proj: x, weight and out must be 16-byte aligned device pointers");
  if (ws && !aligned16(ws)) return fail(1, "layer_proj: the workspace must be 16-byte aligned");
  return launch_status(tabicl_launch_layer_proj(x, ln_weight, ln_bias, eps, weight, bias, out, rows, n_out, dtype, live,
                                                group_rows, skip, ws, ws_bytes, (hipStream_t)stream),
                       "layer_proj");
}

int tabicl_layer_tail(const void* attn, const void* x, const void* out_weight, const void* out_bias,
                      const float* ln_weight, const float* ln_bias, float eps, const void* w1, const void* b1,
                      const void* w2, const void* b2, void* out, int64_t rows, int32_t dtype, const int32_t* live,
                      int64_t group_rows, float skip, void* ws, int64_t ws_bytes, void* stream) {
  int st = layer_args("layer_tail", rows, dtype, eps, live, group_rows);
  if (st) return st;
  if (rows == 0) return 0;
  const void* ptrs[] = {attn, x, out_weight, w1, w2, out};
  for (const void* ptr : ptrs)
    if (!ptr || !aligned16(ptr))
      return fail(1, "layer_tail: attn, x, out and the weight matrices must be 16-byte aligned device pointers");
  if (ws && !aligned16(ws)) return fail(1, "layer_tail: the workspace must be 16-byte aligned");
  if ((ws ? ws_bytes : 0) < tabicl_launch_layer_ws_bytes(0, rows, dtype))
    return fail(1, "layer_tail: workspace of %lld bytes required", (long long)tabicl_launch_layer_ws_bytes(0, rows, dtype));
  return launch_status(tabicl_launch_layer_tail(attn, x, out_weight, out_bias, ln_weight, ln_bias, eps, w1, b1, w2, b2,
                                                out, rows, dtype, live, group_rows, skip, ws, ws_bytes, (hipStream_t)stream),
                       "layer_tail");
}

int64_t tabicl_layer_workspace_bytes(int64_t n_out, int64_t rows, int32_t dtype) {
  return tabicl_launch_layer_ws_bytes(n_out, rows, dtype);
}

int tabicl_ln_linear(const float* x, const float* ln_weight, const float* ln_bias, float eps, const void* weight,
                     const void* bias, void* out, int64_t rows, int64_t n_out, int32_t gelu, void* stream) {
  if (rows < 0 || rows > (1ll << 30)) return fail(1, "ln_linear: %lld rows not supported", (long long)rows);
  if (n_out < 128 || n_out > 8192 || n_out % 128)
    return fail(1, "ln_linear: n_out %lld must be a multiple of 128 up to 8192", (long long)n_out);
  if (!(eps > 0.f)) return fail(1, "ln_linear: eps must be positive");
  if (rows == 0) return 0;
  if (!x || !weight || !out || !aligned16(x) || !aligned16(weight) || !aligned16(out))
    return fail(1, "ln_linear: x, weight and out must be 16-byte aligned device pointers");
  return launch_status(tabicl_launch_ln_linear(x, ln_weight, ln_bias, eps, weight, bias, out, rows, n_out, gelu,
                                               (hipStream_t)stream),
                       "ln_linear");
}

int tabicl_linear_residual(const void* x, const void* weight, const void* bias, const float* residual, float* out,
                           int64_t rows, int64_t k, void* stream) {
  if (rows < 0 || rows > (1ll << 30)) return fail(1, "linear_residual: %lld rows not supported", (long long)rows);
  if (k != 512 && k != 1024) return fail(1, "linear_residual: k %lld must be 512 or 1024", (long long)k);
  if (rows == 0) return 0;
  if (!x || !weight || !residual || !out || !aligned16(x) || !aligned16(weight) || !aligned16(residual) || !aligned16(out))
    return fail(1, "linear_residual: x, weight, residual and out must be 16-byte aligned device pointers");
  return launch_status(tabicl_launch_linear_residual(x, weight, bias, residual, out, rows, k, (hipStream_t)stream),
                       "linear_residual");
}

int tabicl_icl_block_tail(const void* attn, const float* x, const void* out_weight, const void* out_bias,
                          const float* ln_weight, const float* ln_bias, float eps, const void* w1, const void* b1,
                          const void* w2, const void* b2, void* h, float* out, int64_t rows, void* stream) {
  // Host-bound where it is used (rows <= 8192): one call in place of three and the slices of the packed projection
  // gone, together with a cheaper route check: cached query of 8 x 60 rows 1497 -> 1322 us.
  if (rows > 0 && (const float*)out == x) return fail(1, "icl_block_tail: out must not be x");
  // checks before the first launch what the later ones would refuse
  if (rows > 0 && (!w1 || !w2 || !h || !out || !aligned16(w1) || !aligned16(w2) || !aligned16(h) || !(eps > 0.f)))
    return fail(1, "icl_block_tail: w1, w2, h and out must be 16-byte aligned device pointers, eps positive");
  int st = tabicl_linear_residual(attn, out_weight, out_bias, x, out, rows, 512, stream);
  if (st) return st;
  st = tabicl_ln_linear(out, ln_weight, ln_bias, eps, w1, b1, h, rows, 1024, 1, stream);
  if (st) return st;
  return tabicl_linear_residual(h, w2, b2, out, out, rows, 1024, stream);
}

int tabicl_column_embed(const float* x, const int64_t* real_features, const void* weight, const void* bias, void* out,
                        int64_t B, int64_t T, int64_t H, int64_t reserve, float skip, int32_t dtype, void* stream) {
  if (dtype != 0 && dtype != 1) return fail(1, "column_embed: dtype must be 0 (bf16) or 1 (fp32)");
  if (B < 0 || T < 0 || H < 1 || reserve < 0 || T > (1ll << 30) || H > (1ll << 20) || B * (H + reserve) > 65535)
    return fail(1, "column_embed: bad sizes B=%lld T=%lld H=%lld", (long long)B, (long long)T, (long long)H);
  if (B == 0 || T == 0) return 0;
  if (!x || !weight || !out || !aligned16(out)) return fail(1, "column_embed: bad pointers (out 16-byte aligned)");
  return launch_status(tabicl_launch_column_embed(x, real_features, weight, bias, out, B, T, H, reserve, skip, dtype,
                                                  (hipStream_t)stream),
                       "column_embed");
}

namespace {

constexpr int64_t PAGED_MAX_ROWS = 1LL << 30;  // rows of a sequence: row numbers and their sums stay in 32 bits

// The pool part of the paged entry points' arguments, checked and packed (status 0 or 1 with the message set).
int paged_pool(const char* op, PagedPool* c, const void* k_pages, const void* v_pages, int64_t pages, int64_t page_sp,
               int64_t page_rows, const int32_t* table, int64_t table_sn, int64_t max_pages, const int32_t* lengths,
               int64_t N, int64_t H, int64_t D, int32_t dtype, int64_t cell = 0) {
  if (!cell) cell = (int64_t)esize(dtype);  // bytes of a value in the pool
  if (dtype != TABICL_DTYPE_BF16 && dtype != TABICL_DTYPE_F32) return fail(1, "%s: dtype code %d not supported", op, dtype);
  if (D != 32 && D != 64 && D != 128) return fail(1, "%s: head dim must be 32, 64 or 128, got %lld", op, (long long)D);
  if (page_rows < 16 || page_rows > (1 << 20) || (page_rows & (page_rows - 1)))
    return fail(1, "%s: page_rows must be a power of two from 16 to 2^20, got %lld", op, (long long)page_rows);
  if (N < 0 || N > 65535 || H < 1 || H > 1024) return fail(1, "%s: needs 0 <= N <= 65535 and 1 <= H <= 1024", op);
  if (pages < 0 || pages > 0x7fffffffLL || max_pages < 0 || max_pages > PAGED_MAX_ROWS / page_rows || table_sn < 0)
    return fail(1, "%s: bad page counts (pages %lld, max_pages %lld)", op, (long long)pages, (long long)max_pages);
  if (page_sp < H * page_rows * D || page_sp * cell % 16 || (pages && page_sp > (1LL << 60) / pages))
    return fail(1, "%s: the page stride must be a multiple of 16 bytes and at least H * page_rows * D", op);
  if (N > 0 && (!lengths || (max_pages > 0 && !table))) return fail(1, "%s: table and lengths are required", op);
  if (!aligned16(k_pages) || !aligned16(v_pages)) return fail(1, "%s: pools must be 16-byte aligned", op);
  if (pages > 0 && (!k_pages || !v_pages)) return fail(1, "%s: pools are required", op);
  c->k = (void*)k_pages;
  c->v = (void*)v_pages;
  c->pages = pages;
  c->page_sp = page_sp;
  c->H = (int)H;
  c->D = (int)D;
  c->shift = __builtin_ctzll((unsigned long long)page_rows);
  c->table = table;
  c->table_sn = table_sn;
  c->max_pages = (int)max_pages;
  c->lengths = lengths;
  return 0;
}

int paged_attn_sizes(const char* op, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows) {
  if (N < 0 || N > 65535 || H < 1 || H > 1024 || Hq < 1 || Hq > 1024 || Hq % H || Tq < 0 || rows < 0 ||
      rows > PAGED_MAX_ROWS || (D != 32 && D != 64 && D != 128))
    return fail(1, "%s: bad sizes N=%lld Hq=%lld H=%lld Tq=%lld D=%lld rows=%lld (Hq must be a multiple of H)", op,
                (long long)N, (long long)Hq, (long long)H, (long long)Tq, (long long)D, (long long)rows);
  if (Tq > PAGED_MAX_QUERIES || N * Hq > PAGED_MAX_QUERIES || N * Hq * Tq > 16 * PAGED_MAX_QUERIES)
    return fail(1, "%s: more than 2^26 query rows, or 2^22 of one head, or 2^22 heads over all sequences", op);
  if (Tq > 0 && N * H * ((Hq / H + 15) / 16) * (rows / 128 + 1) > PAGED_MAX_UNITS)
    return fail(1, "%s: more than 2^37 cached rows over all sequences, heads and tiles of query rows", op);
  return 0;
}

}  // namespace

int64_t tabicl_paged_attn_workspace_bytes(int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows,
                                          int32_t with_weights, int32_t dtype) {
  if (dtype != TABICL_DTYPE_BF16 && dtype != TABICL_DTYPE_F32)
    return -fail(1, "paged_attn_workspace_bytes: dtype code %d not supported", dtype);
  if (int st = paged_attn_sizes("paged_attn_workspace_bytes", N, Hq, H, Tq, D, rows)) return -st;
  if (N == 0 || Tq == 0) return 0;
  return tabicl_launch_paged_attn_ws_bytes(N, Hq, H, Tq, D, rows, with_weights, dtype);
}

int tabicl_paged_attn(const void* q, const void* k_pages, const void* v_pages, int64_t pages, int64_t page_sp,
                      int64_t page_rows, const int32_t* table, int64_t table_sn, int64_t max_pages, const int32_t* lengths,
                      float* weights, int64_t weights_sn, void* out, int64_t N, int64_t Hq, int64_t H, int64_t Tq,
                      int64_t D, int64_t q_sn, int64_t q_sh, int64_t q_st, int64_t o_sn, int64_t o_sh, int64_t o_st,
                      float scale, int32_t dtype, void* ws, int64_t ws_bytes, void* stream) {
  PagedAttn a = {};
  int st = paged_pool("paged_attn", &a.pool, k_pages, v_pages, pages, page_sp, page_rows, table, table_sn, max_pages,
                      lengths, N, H, D, dtype);
  if (st) return st;
  st = paged_attn_sizes("paged_attn", N, Hq, H, Tq, D, max_pages * page_rows);
  if (st) return st;
  if (N == 0 || Tq == 0) return 0;
  if (!q || !out || !aligned16(q) || !aligned16(out)) return fail(1, "paged_attn: q and out must be 16-byte aligned");
  const int64_t s[6] = {q_sn, q_sh, q_st, o_sn, o_sh, o_st};
  for (int i = 0; i < 6; ++i)
    if (s[i] < 0 || !stride_ok(s[i], dtype))
      return fail(1, "paged_attn: strides must be non-negative multiples of 16 bytes");
  if (!(scale > -1e30f && scale < 1e30f)) return fail(1, "paged_attn: scale must be finite");
  if (weights && (((uintptr_t)weights & 3) || weights_sn < max_pages * page_rows))
    return fail(1, "paged_attn: weights needs rows of max_pages * page_rows values");
  if (weights && N * max_pages * page_rows > (1LL << 29)) return fail(1, "paged_attn: weights for more than 2^29 rows");
  const int64_t need = tabicl_launch_paged_attn_ws_bytes(N, Hq, H, Tq, D, max_pages * page_rows, weights != nullptr, dtype);
  if (need > 0 && (!ws || !aligned16(ws) || ws_bytes < need))
    return fail(1, "paged_attn: workspace of %lld bytes (16-byte aligned) required", (long long)need);
  a.q = q;
  a.q_sn = q_sn;
  a.q_sh = q_sh;
  a.q_st = q_st;
  a.out = out;
  a.o_sn = o_sn;
  a.o_sh = o_sh;
  a.o_st = o_st;
  a.weights = weights;
  a.weights_sn = weights_sn;
  a.N = (int)N;
  a.Hq = (int)Hq;
  a.Tq = (int)Tq;
  a.scale = scale;
  return launch_status(tabicl_launch_paged_attn(a, dtype, ws, (hipStream_t)stream), "paged_attn");
}

int tabicl_paged_append(void* k_pages, void* v_pages, int64_t pages, int64_t page_sp, int64_t page_rows,
                        const int32_t* table, int64_t table_sn, int64_t max_pages, const int32_t* lengths, const void* k,
                        const void* v, const int32_t* count, int64_t N, int64_t H, int64_t T, int64_t D, int64_t k_sn,
                        int64_t k_sh, int64_t k_st, int64_t v_sn, int64_t v_sh, int64_t v_st, int32_t dtype, void* stream) {
  PagedAppend a = {};
  int st = paged_pool("paged_append", &a.pool, k_pages, v_pages, pages, page_sp, page_rows, table, table_sn, max_pages,
                      lengths, N, H, D, dtype);
  if (st) return st;
  if (T < 0 || T > PAGED_MAX_ROWS) return fail(1, "paged_append: bad row count %lld", (long long)T);
  if (N == 0 || T == 0) return 0;
  if (!k || !v || !aligned16(k) || !aligned16(v)) return fail(1, "paged_append: k and v must be 16-byte aligned");
  const int64_t s[6] = {k_sn, k_sh, k_st, v_sn, v_sh, v_st};
  for (int i = 0; i < 6; ++i)
    if (s[i] < 0 || !stride_ok(s[i], dtype))
      return fail(1, "paged_append: strides must be non-negative multiples of 16 bytes");
  a.k = k;
  a.v = v;
  a.k_sn = k_sn;
  a.k_sh = k_sh;
  a.k_st = k_st;
  a.v_sn = v_sn;
  a.v_sh = v_sh;
  a.v_st = v_st;
  a.count = count;
  a.N = (int)N;
  a.T = (int)T;
  return launch_status(tabicl_launch_paged_append(a, dtype, (hipStream_t)stream), "paged_append");
}

int tabicl_paged_gather(const void* k_pages, const void* v_pages, int64_t pages, int64_t page_sp, int64_t page_rows,
                        const int32_t* table, int64_t table_sn, int64_t max_pages, const int32_t* lengths, void* k, void* v,
                        int64_t N, int64_t H, int64_t T, int64_t D, int32_t dtype, void* stream) {
  PagedGather a = {};
  int st = paged_pool("paged_gather", &a.pool, k_pages, v_pages, pages, page_sp, page_rows, table, table_sn, max_pages,
                      lengths, N, H, D, dtype);
  if (st) return st;
  if (T < 0 || T > PAGED_MAX_ROWS) return fail(1, "paged_gather: bad row count %lld", (long long)T);
  if (N == 0 || T == 0) return 0;
  if (!k || !v || !aligned16(k) || !aligned16(v)) return fail(1, "paged_gather: k and v must be 16-byte aligned");
  a.k = k;
  a.v = v;
  a.N = (int)N;
  a.T = (int)T;
  return launch_status(tabicl_launch_paged_gather(a, dtype, (hipStream_t)stream), "paged_gather");
}

int64_t tabicl_paged_evict_workspace_bytes(int64_t N, int64_t K) {
  if (N < 0 || N > 65535 || K < 0 || K > PAGED_MAX_ROWS) return -fail(1, "paged_evict_workspace_bytes: bad sizes");
  return tabicl_launch_paged_evict_ws_bytes(N, K);
}

int tabicl_paged_evict(void* k_pages, void* v_pages, int64_t blocks, int64_t block_sp, int64_t pages, int64_t page_sp,
                       int64_t page_rows, const int32_t* table, int64_t table_sn, int64_t max_pages,
                       const int32_t* lengths, const float* weights, int64_t weights_sn, const int32_t* keep_n,
                       int64_t keep_all, int64_t recent, int32_t* index, int64_t K, float* kept_weights,
                       int32_t* kept_lengths, int64_t N, int64_t H, int64_t D, int32_t dtype, void* ws, int64_t ws_bytes,
                       void* stream) {
  PagedEvict a = {};
  int st = paged_pool("paged_evict", &a.pool, k_pages, v_pages, blocks > 0 ? pages : 0, page_sp, page_rows, table, table_sn,
                      max_pages, lengths, N, H, D, dtype);
  if (st) return st;
  const int64_t cap = max_pages * page_rows;
  if (blocks < 0 || blocks > 65535 || block_sp < 0 || !stride_ok(block_sp, dtype))
    return fail(1, "paged_evict: bad block count or stride");
  if (N * (cap + 1024) > (1LL << 31) || N * ((blocks + 3) / 4 + 1) > PAGED_MAX_GRID)
    return fail(1, "paged_evict: more than 2^31 rows over all sequences, or 2^25 blocks");
  if (recent < 0 || keep_all < 0 || K < 0 || K > cap)
    return fail(1, "paged_evict: needs recent, keep >= 0 and 0 <= K <= the capacity %lld", (long long)cap);
  if (N == 0) return 0;
  if (!kept_lengths || (K > 0 && !index) || (cap > 0 && (!weights || !kept_weights)) || weights_sn < cap)
    return fail(1, "paged_evict: weights and kept_weights need rows of max_pages * page_rows values");
  if ((!ws || !aligned16(ws) || ws_bytes < tabicl_launch_paged_evict_ws_bytes(N, K)))
    return fail(1, "paged_evict: workspace of %lld bytes (16-byte aligned) required",
                (long long)tabicl_launch_paged_evict_ws_bytes(N, K));
  a.blocks = blocks;
  a.block_sp = block_sp;
  a.weights = weights;
  a.weights_sn = weights_sn;
  a.keep = keep_n;
  a.keep_all = (int)(keep_all < K ? keep_all : K);
  a.recent = (int)(recent < cap ? recent : cap);
  a.index = index;
  a.K = (int)K;
  a.kept_weights = kept_weights;
  a.kept_lengths = kept_lengths;
  a.N = (int)N;
  return launch_status(tabicl_launch_paged_evict(a, dtype, ws, (hipStream_t)stream), "paged_evict");
}

namespace {

// dtype: of queries, rows and results; code: of the pool's values.
int paged_code(const char* op, int32_t code, const void* scales, int64_t pages) {
  if (code != TABICL_CODE_E4M3 && code != TABICL_CODE_I8) return fail(1, "%s: code %d not supported (0 e4m3, 1 int8)", op, code);
  if (pages > 0 && (!scales || ((uintptr_t)scales & 7))) return fail(1, "%s: scales are required (8-byte aligned)", op);
  return 0;
}

int paged_format(const char* op, int32_t format, int32_t dtype, const void* scales, int64_t pages) {
  if (format < 0 || format > 3) return fail(1, "%s: pool format %d not supported (0 bf16, 1 fp32, 2 e4m3, 3 int8)", op, format);
  if (format < 2) return format == dtype ? 0 : fail(1, "%s: a bf16 or fp32 pool takes its own dtype", op);
  return paged_code(op, format - 2, scales, pages);
}

int64_t format_bytes(int32_t format) { return format == 0 ? 2 : format == 1 ? 4 : 1; }

int strides16(const char* op, const int64_t* s, int count, int32_t dtype) {
  for (int i = 0; i < count; ++i)
    if (s[i] < 0 || !stride_ok(s[i], dtype)) return fail(1, "%s: strides must be non-negative multiples of 16 bytes", op);
  return 0;
}

int paged_attn_fill(const char* op, PagedAttn* a, const void* q, void* out, int64_t N, int64_t Hq, int64_t Tq, int64_t q_sn,
                    int64_t q_sh, int64_t q_st, int64_t o_sn, int64_t o_sh, int64_t o_st, float scale, int32_t dtype) {
  if (!q || !out || !aligned16(q) || !aligned16(out)) return fail(1, "%s: q and out must be 16-byte aligned", op);
  const int64_t s[6] = {q_sn, q_sh, q_st, o_sn, o_sh, o_st};
  if (int st = strides16(op, s, 6, dtype)) return st;
  if (!(scale > -1e30f && scale < 1e30f)) return fail(1, "%s: scale must be finite", op);
  a->q = q;
  a->q_sn = q_sn;
  a->q_sh = q_sh;
  a->q_st = q_st;
  a->out = out;
  a->o_sn = o_sn;
  a->o_sh = o_sh;
  a->o_st = o_st;
  a->N = (int)N;
  a->Hq = (int)Hq;
  a->Tq = (int)Tq;
  a->scale = scale;
  return 0;
}

int paged_workspace(const char* op, int64_t need, const void* ws, int64_t ws_bytes) {
  if (need > 0 && (!ws || !aligned16(ws) || ws_bytes < need))
    return fail(1, "%s: workspace of %lld bytes (16-byte aligned) required", op, (long long)need);
  return 0;
}

}  // namespace

int64_t tabicl_paged_attn_q8_workspace_bytes(int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows,
                                             int32_t dtype) {
  if (dtype != TABICL_DTYPE_BF16 && dtype != TABICL_DTYPE_F32)
    return -fail(1, "paged_attn_q8_workspace_bytes: dtype code %d not supported", dtype);
  if (int st = paged_attn_sizes("paged_attn_q8_workspace_bytes", N, Hq, H, Tq, D, rows)) return -st;
  if (N == 0 || Tq == 0) return 0;
  return tabicl_launch_paged_attn_q8_ws_bytes(N, Hq, H, Tq, D, rows, dtype);
}

int tabicl_paged_attn_q8(const void* q, const void* k_pages, const void* v_pages, const float* scales, int64_t pages,
                         int64_t page_sp, int64_t page_rows, const int32_t* table, int64_t table_sn, int64_t max_pages,
                         const int32_t* lengths, void* out, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D,
                         int64_t q_sn, int64_t q_sh, int64_t q_st, int64_t o_sn, int64_t o_sh, int64_t o_st, float scale,
                         int32_t dtype, int32_t code, void* ws, int64_t ws_bytes, void* stream) {
  PagedAttn a = {};
  if (int st = paged_pool("paged_attn_q8", &a.pool, k_pages, v_pages, pages, page_sp, page_rows, table, table_sn, max_pages,
                          lengths, N, H, D, dtype, 1))
    return st;
  if (int st = paged_code("paged_attn_q8", code, scales, pages)) return st;
  if (int st = paged_attn_sizes("paged_attn_q8", N, Hq, H, Tq, D, max_pages * page_rows)) return st;
  if (N == 0 || Tq == 0) return 0;
  if (int st = paged_attn_fill("paged_attn_q8", &a, q, out, N, Hq, Tq, q_sn, q_sh, q_st, o_sn, o_sh, o_st, scale, dtype)) return st;
  if (int st = paged_workspace("paged_attn_q8",
                               tabicl_launch_paged_attn_q8_ws_bytes(N, Hq, H, Tq, D, max_pages * page_rows, dtype), ws, ws_bytes))
    return st;
  a.scales = scales;
  return launch_status(tabicl_launch_paged_attn_q8(a, dtype, code, ws, (hipStream_t)stream), "paged_attn_q8");
}

int tabicl_paged_append_q8(void* k_pages, void* v_pages, float* scales, int64_t pages, int64_t page_sp, int64_t page_rows,
                           const int32_t* table, int64_t table_sn, int64_t max_pages, const int32_t* lengths, const void* k,
                           const void* v, const int32_t* count, const int32_t* starts, int64_t N, int64_t H, int64_t T, int64_t D,
                           int64_t k_sn, int64_t k_sh, int64_t k_st, int64_t v_sn, int64_t v_sh, int64_t v_st, int32_t dtype,
                           int32_t code, void* stream) {
  PagedAppend8 a = {};
  if (int st = paged_pool("paged_append_q8", &a.rows.pool, k_pages, v_pages, pages, page_sp, page_rows, table, table_sn, max_pages,
                          lengths, N, H, D, dtype, 1))
    return st;
  if (int st = paged_code("paged_append_q8", code, scales, pages)) return st;
  if (T < 0 || T > PAGED_MAX_ROWS) return fail(1, "paged_append_q8: bad row count %lld", (long long)T);
  if (starts && !count) return fail(1, "paged_append_q8: packed rows need a count per sequence");
  if (N == 0 || T == 0 || max_pages == 0) return 0;
  if (!k || !v || !aligned16(k) || !aligned16(v)) return fail(1, "paged_append_q8: k and v must be 16-byte aligned");
  const int64_t s[6] = {k_sn, k_sh, k_st, v_sn, v_sh, v_st};
  if (int st = strides16("paged_append_q8", s, 6, dtype)) return st;
  if ((T / page_rows + 2 < max_pages ? T / page_rows + 2 : max_pages) * H > PAGED_MAX_GRID / 2)
    return fail(1, "paged_append_q8: more than 2^22 pages and heads of a sequence to look at");
  a.rows.k = k;
  a.rows.v = v;
  a.rows.k_sn = k_sn;
  a.rows.k_sh = k_sh;
  a.rows.k_st = k_st;
  a.rows.v_sn = v_sn;
  a.rows.v_sh = v_sh;
  a.rows.v_st = v_st;
  a.rows.count = count;
  a.rows.N = (int)N;
  a.rows.T = (int)T;
  a.scales = scales;
  a.starts = starts;
  return launch_status(tabicl_launch_paged_append_q8(a, dtype, code, (hipStream_t)stream), "paged_append_q8");
}

int tabicl_paged_gather_q8(const void* k_pages, const void* v_pages, const float* scales, int64_t pages, int64_t page_sp,
                           int64_t page_rows, const int32_t* table, int64_t table_sn, int64_t max_pages, const int32_t* lengths,
                           void* k, void* v, int64_t N, int64_t H, int64_t T, int64_t D, int32_t dtype, int32_t code, void* stream) {
  PagedGather a = {};
  if (int st = paged_pool("paged_gather_q8", &a.pool, k_pages, v_pages, pages, page_sp, page_rows, table, table_sn, max_pages,
                          lengths, N, H, D, dtype, 1))
    return st;
  if (int st = paged_code("paged_gather_q8", code, scales, pages)) return st;
  if (T < 0 || T > PAGED_MAX_ROWS) return fail(1, "paged_gather_q8: bad row count %lld", (long long)T);
  if (N == 0 || T == 0) return 0;
  if (!k || !v || !aligned16(k) || !aligned16(v)) return fail(1, "paged_gather_q8: k and v must be 16-byte aligned");
  a.k = k;
  a.v = v;
  a.N = (int)N;
  a.T = (int)T;
  return launch_status(tabicl_launch_paged_gather_q8(a, scales, dtype, code, (hipStream_t)stream), "paged_gather_q8");
}

int tabicl_paged_bounds(const void* k_pages, const float* scales, int64_t pages, int64_t page_sp, int64_t page_rows,
                        const int32_t* table, int64_t table_sn, int64_t max_pages, const int32_t* lengths, const int32_t* start,
                        int64_t rows, int8_t* bounds, float* bound_scales, int64_t N, int64_t H, int64_t D, int32_t format,
                        void* stream) {
  PagedBounds a = {};
  if (int st = paged_format("paged_bounds", format, format < 2 ? format : 0, scales, pages)) return st;
  if (int st = paged_pool("paged_bounds", &a.pool, k_pages, k_pages, pages, page_sp, page_rows, table, table_sn, max_pages, lengths, N,
                          H, D, format == 1 ? 1 : 0, format_bytes(format)))
    return st;
  if (rows < 0) return fail(1, "paged_bounds: rows must not be negative");
  if (pages > 0 && (!bounds || !bound_scales || !aligned16(bounds) || ((uintptr_t)bound_scales & 3)))
    return fail(1, "paged_bounds: bounds (16-byte aligned) and bound_scales are required");
  if (rows > max_pages * page_rows || !start) rows = max_pages * page_rows;
  if ((max_pages < rows / page_rows + 2 ? max_pages : rows / page_rows + 2) * H > 4 * PAGED_MAX_GRID)
    return fail(1, "paged_bounds: more than 2^25 pages and heads of a sequence to look at");
  if (N == 0 || pages == 0) return 0;
  a.scales = scales;
  a.start = start;
  a.bounds = bounds;
  a.bound_scales = bound_scales;
  a.N = (int)N;
  return launch_status(tabicl_launch_paged_bounds(a, format, rows, (hipStream_t)stream), "paged_bounds");
}

int64_t tabicl_paged_select_workspace_bytes(int64_t N, int64_t H, int64_t Tq, int64_t max_pages) {
  if (N < 0 || N > 65535 || H < 1 || H > 1024 || Tq < 0 || max_pages < 0 || max_pages > PAGED_MAX_ROWS / 16 ||
      N * H * Tq > PAGED_MAX_QUERIES / 2)
    return -fail(1, "paged_select_workspace_bytes: bad sizes N=%lld H=%lld Tq=%lld max_pages=%lld", (long long)N, (long long)H,
                 (long long)Tq, (long long)max_pages);
  return tabicl_launch_paged_select_ws_bytes(N, H, Tq, max_pages);
}

int tabicl_paged_select(const void* q, const int8_t* bounds, const float* bound_scales, int64_t pages, int64_t page_rows,
                        const int32_t* table, int64_t table_sn, int64_t max_pages, const int32_t* lengths, int32_t* index, int64_t K,
                        int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t q_sn, int64_t q_sh, int64_t q_st,
                        int32_t dtype, void* ws, int64_t ws_bytes, void* stream) {
  PagedSelect a = {};
  if (int st = paged_pool("paged_select", &a.pool, bounds, bounds, pages, H * page_rows * D, page_rows, table, table_sn, max_pages,
                          lengths, N, H, D, dtype))
    return st;
  if (int st = paged_attn_sizes("paged_select", N, Hq, H, Tq, D, max_pages * page_rows)) return st;
  if (N * H * Tq > PAGED_MAX_QUERIES / 2) return fail(1, "paged_select: more than 2^21 query rows over all sequences and K/V heads");
  if (K < 0 || K > PAGED_MAX_ROWS / page_rows) return fail(1, "paged_select: bad page count %lld", (long long)K);
  if (N == 0 || Tq == 0 || K == 0) return 0;
  if (!q || !aligned16(q) || !index || ((uintptr_t)index & 3)) return fail(1, "paged_select: q (16-byte aligned) and index are required");
  if (pages > 0 && !bound_scales) return fail(1, "paged_select: bound_scales are required");
  const int64_t s[3] = {q_sn, q_sh, q_st};
  if (int st = strides16("paged_select", s, 3, dtype)) return st;
  if (int st = paged_workspace("paged_select", tabicl_launch_paged_select_ws_bytes(N, H, Tq, max_pages), ws, ws_bytes)) return st;
  a.q = q;
  a.q_sn = q_sn;
  a.q_sh = q_sh;
  a.q_st = q_st;
  a.bounds = bounds;
  a.bound_scales = bound_scales;
  a.index = index;
  a.N = (int)N;
  a.Hq = (int)Hq;
  a.Tq = (int)Tq;
  a.K = (int)K;
  return launch_status(tabicl_launch_paged_select(a, dtype, ws, (hipStream_t)stream), "paged_select");
}

namespace {

int paged_sparse_sizes(const char* op, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows) {
  if (int st = paged_attn_sizes(op, N, Hq, H, Tq, D, rows)) return st;
  if (N * Hq * Tq > PAGED_MAX_QUERIES) return fail(1, "%s: more than 2^22 query rows over all sequences and heads", op);
  return 0;
}

}  // namespace

int64_t tabicl_paged_sparse_attn_workspace_bytes(int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows) {
  if (int st = paged_sparse_sizes("paged_sparse_attn_workspace_bytes", N, Hq, H, Tq, D, rows)) return -st;
  if (N == 0 || Tq == 0) return 0;
  return tabicl_launch_paged_sparse_ws_bytes(N, Hq, H, Tq, D, rows);
}

int tabicl_paged_sparse_attn(const void* q, const void* k_pages, const void* v_pages, const float* scales, int64_t pages,
                             int64_t page_sp, int64_t page_rows, const int32_t* table, int64_t table_sn, int64_t max_pages,
                             const int32_t* lengths, const int32_t* index, int64_t K, void* out, int64_t N, int64_t Hq, int64_t H,
                             int64_t Tq, int64_t D, int64_t q_sn, int64_t q_sh, int64_t q_st, int64_t o_sn, int64_t o_sh,
                             int64_t o_st, float scale, int32_t dtype, int32_t format, void* ws, int64_t ws_bytes, void* stream) {
  PagedAttn a = {};
  if (dtype != TABICL_DTYPE_BF16 && dtype != TABICL_DTYPE_F32) return fail(1, "paged_sparse_attn: dtype code %d not supported", dtype);
  if (int st = paged_format("paged_sparse_attn", format, dtype, scales, pages)) return st;
  if (int st = paged_pool("paged_sparse_attn", &a.pool, k_pages, v_pages, pages, page_sp, page_rows, table, table_sn, max_pages,
                          lengths, N, H, D, dtype, format_bytes(format)))
    return st;
  if (K < 0 || K > PAGED_MAX_ROWS / page_rows) return fail(1, "paged_sparse_attn: bad page count %lld", (long long)K);
  if (int st = paged_sparse_sizes("paged_sparse_attn", N, Hq, H, Tq, D, K * page_rows)) return st;
  if (N == 0 || Tq == 0) return 0;
  if (K > 0 && (!index || ((uintptr_t)index & 3))) return fail(1, "paged_sparse_attn: index is required");
  if (int st = paged_attn_fill("paged_sparse_attn", &a, q, out, N, Hq, Tq, q_sn, q_sh, q_st, o_sn, o_sh, o_st, scale, dtype)) return st;
  if (int st = paged_workspace("paged_sparse_attn", tabicl_launch_paged_sparse_ws_bytes(N, Hq, H, Tq, D, K * page_rows), ws, ws_bytes))
    return st;
  a.scales = scales;
  a.index = index;
  a.K = (int)K;
  return launch_status(tabicl_launch_paged_sparse(a, format, dtype, ws, (hipStream_t)stream), "paged_sparse_attn");
}

namespace {

int paged_books(const char* op, PagedBooks* a, int32_t* table, int64_t table_sn, int64_t max_pages, const int32_t* lengths,
                const int32_t* count, int64_t pages, int64_t page_rows, int64_t N) {
  if (page_rows < 16 || page_rows > (1 << 20) || (page_rows & (page_rows - 1)))
    return fail(1, "%s: page_rows must be a power of two from 16 to 2^20, got %lld", op, (long long)page_rows);
  if (N < 0 || N > 65535) return fail(1, "%s: needs 0 <= N <= 65535", op);
  if (pages < 0 || pages > 0x7fffffffLL || max_pages < 0 || max_pages > PAGED_MAX_ROWS / page_rows || table_sn < 0)
    return fail(1, "%s: bad page counts (pages %lld, max_pages %lld)", op, (long long)pages, (long long)max_pages);
  if (N > 0 && (!lengths || (max_pages > 0 && !table))) return fail(1, "%s: table and lengths are required", op);
  a->table = table;
  a->table_sn = table_sn;
  a->max_pages = (int)max_pages;
  a->pages = (int)pages;
  a->shift = __builtin_ctzll((unsigned long long)page_rows);
  a->N = (int)N;
  a->lengths = lengths;
  a->count = count;
  return 0;
}

}  // namespace

int64_t tabicl_paged_books_workspace_bytes(int64_t N) {
  if (N < 0 || N > 65535) return -fail(1, "paged_books_workspace_bytes: needs 0 <= N <= 65535");
  return tabicl_launch_paged_books_ws_bytes(N);
}

int tabicl_paged_reserve(int32_t* table, int64_t table_sn, int64_t max_pages, const int32_t* lengths, const int32_t* count,
                         const int32_t* free_pages, int32_t* free_count, int32_t* granted, int64_t pages, int64_t page_rows,
                         int64_t N, void* ws, int64_t ws_bytes, void* stream) {
  PagedBooks a = {};
  if (int st = paged_books("paged_reserve", &a, table, table_sn, max_pages, lengths, count, pages, page_rows, N)) return st;
  if (N > 1 && table_sn < max_pages) return fail(1, "paged_reserve: rows of the table must not overlap");
  if (N == 0) return 0;
  if (!count || !granted || !free_count || (pages > 0 && !free_pages))
    return fail(1, "paged_reserve: count, free, free_count and granted are required");
  if (int st = paged_workspace("paged_reserve", tabicl_launch_paged_books_ws_bytes(N), ws, ws_bytes)) return st;
  a.free_pages = (int32_t*)free_pages;
  a.free_count = free_count;
  a.granted = granted;
  return launch_status(tabicl_launch_paged_reserve(a, ws, (hipStream_t)stream), "paged_reserve");
}

int tabicl_paged_release(int32_t* table, int64_t table_sn, int64_t max_pages, const int32_t* lengths, int32_t* free_pages,
                         int32_t* free_count, int64_t pages, int64_t page_rows, int64_t N, void* ws, int64_t ws_bytes,
                         void* stream) {
  PagedBooks a = {};
  if (int st = paged_books("paged_release", &a, table, table_sn, max_pages, lengths, nullptr, pages, page_rows, N)) return st;
  if (N > 1 && table_sn < max_pages) return fail(1, "paged_release: rows of the table must not overlap");
  if (N == 0) return 0;
  if (!free_count || (pages > 0 && !free_pages)) return fail(1, "paged_release: free and free_count are required");
  if (int st = paged_workspace("paged_release", tabicl_launch_paged_books_ws_bytes(N), ws, ws_bytes)) return st;
  a.free_pages = free_pages;
  a.free_count = free_count;
  return launch_status(tabicl_launch_paged_release(a, ws, (hipStream_t)stream), "paged_release");
}

int tabicl_paged_slots(const int32_t* table, int64_t table_sn, int64_t max_pages, const int32_t* lengths, const int32_t* count,
                       int64_t* slots, int32_t* starts, int64_t total, int64_t pages, int64_t page_rows, int64_t N,
                       void* stream) {
  PagedBooks a = {};
  if (int st = paged_books("paged_slots", &a, (int32_t*)table, table_sn, max_pages, lengths, count, pages, page_rows, N)) return st;
  if (total < 0 || total > 0x7fffffffLL) return fail(1, "paged_slots: bad total %lld", (long long)total);
  if (!starts || (total > 0 && !slots) || (N > 0 && !count)) return fail(1, "paged_slots: count, slots and starts are required");
  return launch_status(tabicl_launch_paged_slots(a, slots, starts, total, (hipStream_t)stream), "paged_slots");
}

int tabicl_paged_append_slots(void* k_pages, void* v_pages, int64_t pages, int64_t page_sp, int64_t page_rows,
                              const int64_t* slots, const void* k, const void* v, int64_t total, int64_t H, int64_t D, int64_t k_st,
                              int64_t k_sh, int64_t v_st, int64_t v_sh, int32_t dtype, void* stream) {
  PagedAppend a = {};
  if (int st = paged_pool("paged_append_slots", &a.pool, k_pages, v_pages, pages, page_sp, page_rows, nullptr, 0, 0, nullptr, 0, H, D,
                          dtype))
    return st;
  if (total < 0 || total > 0x7fffffffLL) return fail(1, "paged_append_slots: bad total %lld", (long long)total);
  if (total == 0 || pages == 0) return 0;
  if (!k || !v || !slots || !aligned16(k) || !aligned16(v)) return fail(1, "paged_append_slots: slots, k and v (16-byte aligned) are required");
  const int64_t s[4] = {k_st, k_sh, v_st, v_sh};
  if (int st = strides16("paged_append_slots", s, 4, dtype)) return st;
  a.k = k;
  a.v = v;
  a.k_st = k_st;
  a.k_sh = k_sh;
  a.v_st = v_st;
  a.v_sh = v_sh;
  return launch_status(tabicl_launch_paged_append_slots(a, slots, total, dtype, (hipStream_t)stream), "paged_append_slots");
}
