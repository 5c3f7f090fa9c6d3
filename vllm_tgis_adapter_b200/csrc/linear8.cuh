// Products with 8-bit weights (include/tgis_w8.h): arguments and launchers shared by rows8.cu, gemm8.cu and the engine.  The number format
// (scale_of, codes) is the 8-bit cache's.
#pragma once
#include "../../include/tgis_w8.h"
#include "cache8.cuh"

namespace tgis {

constexpr int W8_GROUP = TGIS_W8_GROUP;
static_assert(W8_GROUP == 128, "a k-block is 128 bytes wide, as the swizzle is, and one group; a weight tile has the rows of one block");

// ---- rows8.cu
struct Rows8Args {
  const void* x;
  int64_t ldx;
  const __nv_bfloat16* norm;     // null: none
  float eps;
  const void* residual;          // null: none; of x's type
  int64_t ldr;
  void* residual_out;
  int64_t ldro;
  uint8_t* codes;
  float* scales;
  int64_t ldc, lds;
  int T, K;
};
cudaError_t rows8_launch(const Rows8Args& a, bool f32, int num_sms, cudaStream_t stream);
cudaError_t weight8_launch(const void* w, bool f32, int64_t ldw, int N, int K, uint8_t* codes, int64_t ldc, float* scales, cudaStream_t stream);

// ---- gemm8.cu
struct Gemm8Args {
  const float* sx;               // scales of the rows [G][lds]
  int64_t lds;
  const float* sw;               // scales of the weights [N / 128][G]
  const float* sw2;              // ... of the second matrix (gated)
  int T, N, K, G;
  void* y;                       // plain: [T][ldy]
  int64_t ldy;
  uint8_t* codes;                // gated: h in 8 bits [T][ldc], scales [N / 128][ldh]
  int64_t ldc, ldh;
  float* sh;
  int32_t* status;
  int* stalled = nullptr;        // host memory: set to one where a wait ran out
  int early = 0;                 // the weights were written before the kernels in flight began: they may be read ahead of those
};
// y = x w^T (y bf16, or fp32: f32), and h of both matrices
cudaError_t gemm8_launch(const tgis_w8_rows& x, const tgis_w8_matrix& w, void* y, bool f32, int64_t ldy, int32_t* status, int* stalled, bool early,
                         int num_sms, cudaStream_t stream);
cudaError_t gemm8_gated_launch(const tgis_w8_rows& x, const tgis_w8_matrix& gate, const tgis_w8_matrix& up, const tgis_w8_rows& out, int32_t* status,
                               int* stalled, bool early, int num_sms, cudaStream_t stream);

}  // namespace tgis
