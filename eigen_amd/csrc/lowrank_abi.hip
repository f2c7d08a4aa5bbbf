// C entries of the low-rank adapter and 8-bit checkpoint operators (declarations: include/eigen_amd_blas.h): argument checks,
// then the launches of lora.hip and ckpt8.hip.  Nothing here allocates, waits for the device or keeps anything between calls.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "../../include/eigen_amd_blas.h"
#include "lowrank.hpp"

namespace eigamd {
int abi_fail(int code, const std::string& what);  // blas_abi.hip: sets eigamd_last_error()
int abi_ensure_device();
}  // namespace eigamd
using namespace eigamd;

namespace {

// Extents the kernels' 32-bit indices and grids are good for.
constexpr int64_t kMaxFeatures = (int64_t)1 << 21, kMaxTokens = (int64_t)1 << 24, kMaxRank = 256, kMaxAdapters = 4096, kMaxStride = (int64_t)1 << 48;

int bad(const char* entry, const char* what) { return abi_fail(EIGAMD_ERR_ARG, std::string(entry) + ": " + what); }
int done(const char* entry, hipError_t e) {
  if (e == hipSuccess) return EIGAMD_OK;
  (void)hipGetLastError();
  return abi_fail(EIGAMD_ERR_DEVICE, std::string(entry) + ": " + hipGetErrorString(e));
}

bool kind_ok(int dtype) { return dtype == EIGAMD_F32 || dtype == EIGAMD_BF16 || dtype == EIGAMD_F16; }
int bytes_of(int dtype) { return dtype == EIGAMD_F32 ? 4 : 2; }
bool op_ok(int op) { return op == EIGAMD_OP_N || op == EIGAMD_OP_T; }
bool extent_ok(int64_t v, int64_t most) { return v >= 0 && v <= most; }
// a matrix of rows x cols at p: leading dimension (to 2^38, so that no offset leaves 64 bits), element alignment, and a pointer if there
// are elements
bool matrix_ok(const void* p, int64_t rows, int64_t cols, int64_t ld, int es) {
  return ld >= std::max<int64_t>(rows, 1) && ld <= (int64_t)1 << 38 && (reinterpret_cast<uintptr_t>(p) % es) == 0 && (p || rows == 0 || cols == 0);
}
bool work_ok(const void* work, int64_t have, int64_t need) {
  return need == 0 || (work && have >= need && reinterpret_cast<uintptr_t>(work) % 16 == 0);
}

}  // namespace

extern "C" {

int64_t eigamd_lora_plan_ints(int64_t n, int64_t n_adapters) {
  if (!extent_ok(n, kMaxTokens) || !extent_ok(n_adapters, kMaxAdapters)) return -1;
  return 2 * n + n_adapters + 2;
}

int eigamd_lora_plan_dev(int64_t n, int64_t n_adapters, const int32_t* d_adapter_of, int32_t* d_plan, void* stream) {
  static const char* me = "eigamd_lora_plan_dev";
  if (!extent_ok(n, kMaxTokens)) return bad(me, "number of tokens out of range");
  if (!extent_ok(n_adapters, kMaxAdapters)) return bad(me, "number of adapters out of range");
  if (!d_plan || (n > 0 && !d_adapter_of)) return bad(me, "null pointer");
  int rc = abi_ensure_device();
  if (rc != EIGAMD_OK) return rc;
  return done(me, lora_plan_device(d_adapter_of, n, n_adapters, d_plan, static_cast<hipStream_t>(stream)));
}

int64_t eigamd_lora_work_bytes(int dtype, int opw, int64_t m, int64_t n, int64_t k, const void* d_w, int64_t ldw, const void* d_x,
                               int64_t ldx) {
  if (!kind_ok(dtype) || !op_ok(opw) || !extent_ok(m, kMaxFeatures) || !extent_ok(n, kMaxTokens) || !extent_ok(k, kMaxFeatures))
    return -1;
  return lora_work_bytes(dtype, opw == EIGAMD_OP_T, m, n, k, d_w, ldw, d_x, ldx);
}

int eigamd_lora_dev(int dtype, int opw, int opa, int opb, int64_t m, int64_t n, int64_t k, int64_t rank, int64_t n_adapters,
                    const void* d_w, int64_t ldw, const void* d_x, int64_t ldx, const void* d_a, int64_t lda, int64_t stride_a,
                    const void* d_b, int64_t ldb, int64_t stride_b, const float* d_scale, const int32_t* d_plan, float* d_p,
                    int64_t ldp, void* d_y, int64_t ldy, void* d_work, int64_t work_bytes, void* stream) {
  static const char* me = "eigamd_lora_dev";
  if (!kind_ok(dtype)) return bad(me, "dtype is none of F32, BF16, F16");
  if (!op_ok(opw) || !op_ok(opa) || !op_ok(opb)) return bad(me, "an operand form is neither N nor T");
  if (!extent_ok(m, kMaxFeatures) || !extent_ok(k, kMaxFeatures) || !extent_ok(n, kMaxTokens)) return bad(me, "extent out of range");
  if (rank < 1 || rank > kMaxRank) return bad(me, "rank out of range");
  if (!extent_ok(n_adapters, kMaxAdapters)) return bad(me, "number of adapters out of range");
  const int es = bytes_of(dtype);
  const bool wt = opw == EIGAMD_OP_T, at = opa == EIGAMD_OP_T, bt = opb == EIGAMD_OP_T;
  if (!matrix_ok(d_w, wt ? k : m, wt ? m : k, ldw, es)) return bad(me, "W: pointer, alignment or leading dimension");
  if (!matrix_ok(d_x, k, n, ldx, es)) return bad(me, "X: pointer, alignment or leading dimension");
  if (!matrix_ok(d_y, m, n, ldy, es)) return bad(me, "Y: pointer, alignment or leading dimension");
  if (n_adapters > 0) {
    if (!matrix_ok(d_a, at ? k : rank, at ? rank : k, lda, es) || !extent_ok(stride_a, kMaxStride)) return bad(me, "A: pointer, alignment, leading dimension or stride");
    if (!matrix_ok(d_b, bt ? rank : m, bt ? m : rank, ldb, es) || !extent_ok(stride_b, kMaxStride)) return bad(me, "B: pointer, alignment, leading dimension or stride");
    if (!d_scale) return bad(me, "scale is null");
  }
  if ((n_adapters > 0 || d_p) && !matrix_ok(d_p, rank, n, ldp, 4)) return bad(me, "P: pointer, alignment or leading dimension");
  if (n == 0 || (m == 0 && n_adapters == 0)) return EIGAMD_OK;
  if (!d_plan) return bad(me, "plan is null");
  if (m > 0 && k > 0 && (d_y == d_x || d_y == d_w)) return bad(me, "Y overlaps an input");
  if (!work_ok(d_work, work_bytes, lora_work_bytes(dtype, wt, m, n, k, d_w, ldw, d_x, ldx))) return bad(me, "work is smaller than eigamd_lora_work_bytes or not 16-byte aligned");
  int rc = abi_ensure_device();
  if (rc != EIGAMD_OK) return rc;
  LoraArgs c;
  c.kind = dtype;
  c.w_trans = wt; c.a_trans = at; c.b_trans = bt;
  c.m = m; c.n = n; c.k = k; c.rank = rank;
  c.w = d_w; c.ldw = ldw;
  c.x = d_x; c.ldx = ldx;
  c.a = d_a; c.lda = lda; c.stride_a = stride_a;
  c.b = d_b; c.ldb = ldb; c.stride_b = stride_b;
  c.scale = d_scale;
  c.plan = lora_plan_view(d_plan, n, n_adapters);
  c.p = d_p; c.ldp = ldp;
  c.y = d_y; c.ldy = ldy;
  c.work = d_work; c.work_bytes = work_bytes;
  return done(me, lora_device(c, static_cast<hipStream_t>(stream)));
}

int64_t eigamd_lora_wgrad_work_bytes(int64_t rows, int64_t n, int64_t rank, int64_t n_adapters) {
  if (!extent_ok(rows, kMaxFeatures) || !extent_ok(n, kMaxTokens) || rank < 1 || rank > kMaxRank || !extent_ok(n_adapters, kMaxAdapters)) return -1;
  return lora_grad_work_bytes(rows, n, rank, n_adapters);
}

int eigamd_lora_wgrad_dev(int dtype, int opg, int64_t rows, int64_t n, int64_t rank, int64_t n_adapters, const void* d_u, int64_t ldu,
                          const uint8_t* d_exponents, int64_t lde, const float* d_p, int64_t ldp, const float* d_scale,
                          const int32_t* d_plan, const float* beta, float* d_g, int64_t ldg, int64_t stride_g, void* d_work,
                          int64_t work_bytes, void* stream) {
  static const char* me = "eigamd_lora_wgrad_dev";
  if (!kind_ok(dtype)) return bad(me, "dtype is none of F32, BF16, F16");
  if (!op_ok(opg)) return bad(me, "the form of G is neither N nor T");
  if (!extent_ok(rows, kMaxFeatures) || !extent_ok(n, kMaxTokens)) return bad(me, "extent out of range");
  if (rank < 1 || rank > kMaxRank) return bad(me, "rank out of range");
  if (!extent_ok(n_adapters, kMaxAdapters)) return bad(me, "number of adapters out of range");
  if (!matrix_ok(d_u, rows, n, ldu, d_exponents ? 1 : bytes_of(dtype))) return bad(me, "U: pointer, alignment or leading dimension");
  if (d_exponents && !matrix_ok(d_exponents, (rows + 31) / 32, n, lde, 1)) return bad(me, "exponents: leading dimension");
  if (!matrix_ok(d_p, rank, n, ldp, 4)) return bad(me, "P: pointer, alignment or leading dimension");
  const bool gt = opg == EIGAMD_OP_T;
  const int64_t gr = gt ? rank : rows, gc = gt ? rows : rank;
  if (n_adapters > 0 && !matrix_ok(d_g, gr, gc, ldg, 4)) return bad(me, "G: pointer, alignment or leading dimension");
  if (n_adapters > 1 && rows > 0 && (stride_g < ldg * (gc - 1) + gr || stride_g > kMaxStride)) return bad(me, "G: matrices of neighbouring adapters overlap, or a stride out of range");
  if (!beta) return bad(me, "beta is null");
  if (n_adapters == 0 || rows == 0) return EIGAMD_OK;
  if (!d_plan || !d_scale) return bad(me, "null pointer");
  if (!work_ok(d_work, work_bytes, lora_grad_work_bytes(rows, n, rank, n_adapters)))
    return bad(me, "work is smaller than eigamd_lora_wgrad_work_bytes or not 16-byte aligned");
  int rc = abi_ensure_device();
  if (rc != EIGAMD_OK) return rc;
  LoraGradArgs c;
  c.kind = dtype;
  c.trans = gt;
  c.rows = rows; c.n = n; c.rank = rank;
  c.u = d_u; c.ldu = ldu;
  c.exponents = d_exponents; c.lde = lde;
  c.p = d_p; c.ldp = ldp;
  c.scale = d_scale;
  c.plan = lora_plan_view(d_plan, n, n_adapters);
  c.beta = *beta;
  c.g = d_g; c.ldg = ldg; c.stride_g = stride_g;
  c.work = d_work; c.work_bytes = work_bytes;
  return done(me, lora_grad_device(c, static_cast<hipStream_t>(stream)));
}

static int ckpt8_check(const char* me, int dtype, int64_t k, int64_t n, const void* x, int64_t ldx, const void* q, int64_t ldq,
                       const void* e, int64_t lde) {
  if (!kind_ok(dtype)) return bad(me, "dtype is none of F32, BF16, F16");
  if (!extent_ok(k, kMaxFeatures) || !extent_ok(n, kMaxTokens)) return bad(me, "extent out of range");
  if (!matrix_ok(x, k, n, ldx, bytes_of(dtype))) return bad(me, "X: pointer, alignment or leading dimension");
  if (!matrix_ok(q, k, n, ldq, 1)) return bad(me, "Q: pointer or leading dimension");
  if (!matrix_ok(e, (k + 31) / 32, n, lde, 1)) return bad(me, "exponents: pointer or leading dimension");
  return EIGAMD_OK;
}

int eigamd_ckpt8_pack_dev(int dtype, int64_t k, int64_t n, const void* d_x, int64_t ldx, int8_t* d_q, int64_t ldq,
                          uint8_t* d_exponents, int64_t lde, void* stream) {
  static const char* me = "eigamd_ckpt8_pack_dev";
  int rc = ckpt8_check(me, dtype, k, n, d_x, ldx, d_q, ldq, d_exponents, lde);
  if (rc != EIGAMD_OK || k == 0 || n == 0) return rc;
  if ((rc = abi_ensure_device()) != EIGAMD_OK) return rc;
  return done(me, ckpt8_pack_device(dtype, k, n, d_x, ldx, d_q, ldq, d_exponents, lde, static_cast<hipStream_t>(stream)));
}

int eigamd_ckpt8_unpack_dev(int dtype, int64_t k, int64_t n, const int8_t* d_q, int64_t ldq, const uint8_t* d_exponents, int64_t lde,
                            void* d_x, int64_t ldx, void* stream) {
  static const char* me = "eigamd_ckpt8_unpack_dev";
  int rc = ckpt8_check(me, dtype, k, n, d_x, ldx, d_q, ldq, d_exponents, lde);
  if (rc != EIGAMD_OK || k == 0 || n == 0) return rc;
  if ((rc = abi_ensure_device()) != EIGAMD_OK) return rc;
  return done(me, ckpt8_unpack_device(dtype, k, n, d_q, ldq, d_exponents, lde, d_x, ldx, static_cast<hipStream_t>(stream)));
}

int64_t eigamd_ckpt8_wgrad_work_bytes(int dtype, int64_t m, int64_t n, int64_t k, const void* d_dy, int64_t lddy) {
  if (!kind_ok(dtype) || !extent_ok(m, kMaxFeatures) || !extent_ok(n, kMaxTokens) || !extent_ok(k, kMaxFeatures)) return -1;
  return ckpt8_grad_work_bytes(dtype, m, n, k, d_dy, lddy);
}

int eigamd_ckpt8_wgrad_dev(int dtype, int opw, int64_t m, int64_t n, int64_t k, const void* d_dy, int64_t lddy, const int8_t* d_q,
                           int64_t ldq, const uint8_t* d_exponents, int64_t lde, const float* beta, float* d_dw, int64_t lddw,
                           void* d_work, int64_t work_bytes, void* stream) {
  static const char* me = "eigamd_ckpt8_wgrad_dev";
  if (!op_ok(opw)) return bad(me, "the form of W is neither N nor T");
  if (!kind_ok(dtype)) return bad(me, "dtype is none of F32, BF16, F16");
  if (!extent_ok(m, kMaxFeatures) || !extent_ok(k, kMaxFeatures) || !extent_ok(n, kMaxTokens)) return bad(me, "extent out of range");
  if (!matrix_ok(d_dy, m, n, lddy, bytes_of(dtype))) return bad(me, "dY: pointer, alignment or leading dimension");
  if (!matrix_ok(d_q, k, n, ldq, 1)) return bad(me, "Q: pointer or leading dimension");
  if (!matrix_ok(d_exponents, (k + 31) / 32, n, lde, 1)) return bad(me, "exponents: pointer or leading dimension");
  const bool wt = opw == EIGAMD_OP_T;
  if (!matrix_ok(d_dw, wt ? k : m, wt ? m : k, lddw, 4)) return bad(me, "dW: pointer, alignment or leading dimension");
  if (!beta) return bad(me, "beta is null");
  if (m == 0 || k == 0) return EIGAMD_OK;
  if (!work_ok(d_work, work_bytes, ckpt8_grad_work_bytes(dtype, m, n, k, d_dy, lddy)))
    return bad(me, "work is smaller than eigamd_ckpt8_wgrad_work_bytes or not 16-byte aligned");
  int rc = abi_ensure_device();
  if (rc != EIGAMD_OK) return rc;
  Ckpt8GradArgs c;
  c.kind = dtype;
  c.trans = wt;
  c.m = m; c.n = n; c.k = k;
  c.dy = d_dy; c.lddy = lddy;
  c.q = d_q; c.ldq = ldq;
  c.e = d_exponents; c.lde = lde;
  c.beta = *beta;
  c.dw = d_dw; c.lddw = lddw;
  c.work = d_work; c.work_bytes = work_bytes;
  return done(me, ckpt8_grad_device(c, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
