// Low-rank adapters of many requests beside a shared projection, and products with activations held in 8 bits
// (lora.hip, ckpt8.hip).  Column-major matrices, one token per column.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace eigamd {

enum { BF16 = 4, F16K = 5 };   // beside F32 .. C64 (gemm_kernel.hpp)

// What a batch's adapters come to: the tokens sorted by adapter (stable; tokens without one last), where each adapter's run
// starts, and the adapter of each sorted position.  One int array: order[n], seg[n], starts[adapters + 2].
struct LoraPlan {
  const int* order;
  const int* seg;
  const int* starts;
  int n, adapters;
};
inline LoraPlan lora_plan_view(const int* d_plan, int64_t n, int64_t adapters) {
  return {d_plan, d_plan + n, d_plan + 2 * n, (int)n, (int)adapters};
}

struct LoraArgs {
  int kind;
  bool w_trans, a_trans, b_trans;
  int64_t m, n, k, rank;
  const void* w; int64_t ldw;
  const void* x; int64_t ldx;
  const void* a; int64_t lda, stride_a;
  const void* b; int64_t ldb, stride_b;
  const float* scale;
  LoraPlan plan;
  float* p; int64_t ldp;
  void* y; int64_t ldy;
  void* work; int64_t work_bytes;
};

hipError_t lora_plan_device(const int* ids, int64_t n, int64_t adapters, int* d_plan, hipStream_t s);
int64_t lora_work_bytes(int kind, bool w_trans, int64_t m, int64_t n, int64_t k, const void* w, int64_t ldw, const void* x, int64_t ldx);
hipError_t lora_device(const LoraArgs& c, hipStream_t s);

struct LoraGradArgs {
  int kind;
  bool trans;                    // G_j stored rank x rows
  int64_t rows, n, rank;
  const void* u; int64_t ldu;    // rows x n of `kind`, or 8-bit when `exponents`
  const uint8_t* exponents; int64_t lde;
  const float* p; int64_t ldp;
  const float* scale;
  LoraPlan plan;
  float beta;
  float* g; int64_t ldg, stride_g;
  void* work; int64_t work_bytes;
};
int64_t lora_grad_work_bytes(int64_t rows, int64_t n, int64_t rank, int64_t adapters);
hipError_t lora_grad_device(const LoraGradArgs& c, hipStream_t s);

hipError_t ckpt8_pack_device(int kind, int64_t k, int64_t n, const void* x, int64_t ldx, int8_t* q, int64_t ldq, uint8_t* e,
                             int64_t lde, hipStream_t s);
hipError_t ckpt8_unpack_device(int kind, int64_t k, int64_t n, const int8_t* q, int64_t ldq, const uint8_t* e, int64_t lde,
                               void* x, int64_t ldx, hipStream_t s);

struct Ckpt8GradArgs {
  int kind;
  bool trans;                    // dW stored k x m
  int64_t m, n, k;
  const void* dy; int64_t lddy;
  const int8_t* q; int64_t ldq;
  const uint8_t* e; int64_t lde;
  float beta;
  float* dw; int64_t lddw;
  void* work; int64_t work_bytes;
};
int64_t ckpt8_grad_work_bytes(int kind, int64_t m, int64_t n, int64_t k, const void* dy, int64_t lddy);
hipError_t ckpt8_grad_device(const Ckpt8GradArgs& c, hipStream_t s);

}  // namespace eigamd
