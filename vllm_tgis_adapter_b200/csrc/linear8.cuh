// Products with 8-bit weights (include/tgis_w8.h): arguments and launchers shared by rows8.cu, gemm8.cu and the engine.  The number format
// (scale_of, codes) is the 8-bit cache's.
#pragma once
#include <atomic>

#include "../../include/tgis_w8.h"
#include "cache8.cuh"
#include "ptx.cuh"

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
  int early = 0;                 // Gemm8Call
};
struct Gemm8Call {
  int32_t* status = nullptr;
  int* stalled = nullptr;
  bool early = false;            // the weights are static: they are read ahead of the end of the kernels before this one (a decode step of eight 8B layers 0.73 -> 0.68 ms)
};
// ---- what the products share
// kind::f8f6f4: C = F32, A = B = E4M3, both K-major
__host__ __device__ constexpr uint32_t idesc_f8(uint32_t m, uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((m >> 4) << 24); }

__device__ __forceinline__ void tmem_ld_x8(uint32_t at, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(at));
}
// a0 += d0 s0, a1 += d1 s1
__device__ __forceinline__ void add_scaled(float& a0, float& a1, uint32_t d0, uint32_t d1, float s0, float s1) {
  unpack2(fma2(pack2(__uint_as_float(d0), __uint_as_float(d1)), pack2(s0, s1), pack2(a0, a1)), a0, a1);
}
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t* r) {
  if constexpr (N == 8) {
    tmem_ld_x8(at, r);
  } else if constexpr (N % 32 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 32) tmem_ld_x32(at + i, r + i);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 16) tmem_ld_32x32b_x16(at + i, r + i);
  }
}

__device__ __forceinline__ void say_stalled8(const Gemm8Args& a) {
  if (a.status != nullptr) atomicOr(a.status, TGIS_W8_STALLED);
  if (a.stalled != nullptr) {
    *reinterpret_cast<volatile int*>(a.stalled) = 1;
    __threadfence_system();
  }
}
// A warp waits as a whole.  Where that runs out, the results are lost and the warp goes on with no patience left: what it reads and hands on from there is garbage
// in its own places, and its role says so at its end.  (A vote and a way out of the loop at every k-block cost prompts 9 %: 2048 x 8192 x 8192 133 us, without 122.)
__device__ __forceinline__ void await(uint64_t* bar, uint32_t parity, long long& patience) {
  if (!mbar_try_wait(bar, parity)) {
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity))
      if (clock64() - t0 > patience) {
        patience = 0;
        break;
      }
  }
  __syncwarp();
}
// ... and a CTA at its end, all of it (true: one of its roles has given up)
__device__ __forceinline__ bool say_if_stalled8(const Gemm8Args& a, const volatile int* gave_up) {
  if (!*gave_up) return false;
  for (const long long t1 = clock64(); clock64() - t1 < 2000000ll;) {}   // copies and MMAs in flight, all issued by now, are done long before this millisecond is over
  if (threadIdx.x == 0) say_stalled8(a);
  return true;
}

// silu(g) u: exp and quotient are the approximate ones, within some steps of 2^-23 of what is rounded to 2^-4 next (told in tgis_w8.h, as codes_near is)
__device__ __forceinline__ float swiglu(float g, float u) {
  float e, q;
  e = ex2(g * -1.4426950408889634f);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.f + e));   // (no denormal goes in, and what comes out as zero is below 2^-126)
  return g * q * u;
}
// codes() of sums, which are no exact numbers: their quotients are products with the scale's reciprocal (1.5 ulp; a code differs where a sum lies that near
// to the middle of two, a few in a million at most; hidden rows of 4096 / 14336 differ from those of 64 bits in 6 to 8 codes of a million, from sums in fp32 as well)
template <int N>
__device__ __forceinline__ void codes_near(const float* v, float s, uint32_t (&out)[N]) {
  const bool fine = s < INFINITY;
  const float by = __frcp_rn(s);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t w = e4m3x2(v[4 * i] * by, v[4 * i + 1] * by) | e4m3x2(v[4 * i + 2] * by, v[4 * i + 3] * by) << 16;
    out[i] = fine ? w : 0u;
  }
}

// K-major operand rows of 128 codes, `box` rows at a time
inline cudaError_t map8(CUtensorMap* out, const void* codes, int64_t rows, int64_t cols, int64_t ld, int box) {
  return make_tmap_u8_2d(out, codes, (uint64_t)rows, (uint64_t)cols, (uint64_t)ld, (uint32_t)box, W8_GROUP) == 0 ? cudaSuccess : cudaErrorInvalidValue;
}

// Clusters of a kernel that run at once, asked once a device and size: an SM's share of a GPC is not always a whole number of clusters.  0: not one does (a GPC
// may have fewer SMs, a partition of a device fewer still)
struct ClustersAtOnce {
  std::atomic<int> known[OncePerDevice::MAX][4] = {};   // (one more than the answer)
  template <class K>
  cudaError_t operator()(K kernel, int threads, int smem, int cluster, int* out) {   // cluster: 1, 2, 4 or 8
    const int at = __builtin_ctz((unsigned)cluster);
    if (cluster != 1 << at || at > 3) return cudaErrorInvalidValue;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < OncePerDevice::MAX && (*out = known[dev][at].load(std::memory_order_relaxed) - 1) >= 0) return cudaSuccess;
    if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(cluster * 1024));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(out, kernel, &cfg);
    if (e == cudaErrorInvalidClusterSize || e == cudaErrorLaunchOutOfResources) {
      cudaGetLastError();
      *out = 0;
      e = cudaSuccess;
    }
    if (e == cudaSuccess && dev < OncePerDevice::MAX) known[dev][at].store(*out + 1, std::memory_order_relaxed);
    return e;
  }
};

// How the launchers cut a product, where at_once[i] clusters of 2^i CTAs run at the same time (0: none, so such pieces are not taken; cudaErrorLaunchOutOfResources where
// nothing is left).  gemm8.cu: pieces of k of `tiles` tiles, `ctas` to an SM; gemm8_pair.cu: chunks of a half of a tile and pieces of k.
struct Plan8 { int ch, s; };
cudaError_t gemm8_plan(int tiles, int G, int ctas, const int (&at_once)[4], int* pieces);
cudaError_t gemm8_pair_plan(int N, int x_tiles, int G, bool gated, const int (&at_once)[4], Plan8* out);

// y = x w^T (y bf16, or fp32: f32), and h of both matrices
cudaError_t gemm8_launch(const tgis_w8_rows& x, const tgis_w8_matrix& w, void* y, bool f32, int64_t ldy, const Gemm8Call& call, int num_sms,
                         cudaStream_t stream);
cudaError_t gemm8_gated_launch(const tgis_w8_rows& x, const tgis_w8_matrix& gate, const tgis_w8_matrix& up, const tgis_w8_rows& out,
                               const Gemm8Call& call, int num_sms, cudaStream_t stream);

// ---- gemm8_pair.cu: prompts
bool gemm8_pair_takes(int T, int G, bool gated);
cudaError_t gemm8_pair_launch(const tgis_w8_rows& x, const tgis_w8_matrix& w, const Gemm8Args& g, bool f32, int num_sms, cudaStream_t stream);
cudaError_t gemm8_pair_gated_launch(const tgis_w8_rows& x, const tgis_w8_matrix& gate, const tgis_w8_matrix& up, const Gemm8Args& g, int num_sms,
                                    cudaStream_t stream);

}  // namespace tgis
