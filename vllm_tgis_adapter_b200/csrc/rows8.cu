// Rows of activations and weight matrices in 8 bits (include/tgis_w8.h): what products with 8-bit weights read.
//
// One pass each, bound by memory.  A half-warp has a group of 128 neighbours of a row, eight a lane: its maximum is four exchanges away and
// its codes are eight bytes a lane.  With a norm the factor 1 / rms is the same for a whole row, so the codes are those of r * norm
// and only the scales wait for the row's sum of squares: nothing is read twice or held.
#include "launch.cuh"
#include "linear8.cuh"
#include "ptx.cuh"

namespace tgis {
namespace {

constexpr int R8_WARPS = 8, R8_THREADS = R8_WARPS * 32;

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t bf_pack(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <class X>
__device__ __forceinline__ float rounded(float v) {
  if constexpr (sizeof(X) == 2) return bf16_round(v);
  else return v;
}
// Eight neighbours at k of a row of K; zeros behind it.  VEC: rows start on 16 bytes and K is a multiple of 8.
template <class X, bool VEC>
__device__ __forceinline__ void load8(const X* row, int k, int K, float (&v)[8]) {
  if constexpr (VEC) {
    if (k >= K) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    } else if constexpr (sizeof(X) == 2) {
      const uint4 u = *reinterpret_cast<const uint4*>(row + k);
      v[0] = bf_lo(u.x); v[1] = bf_hi(u.x); v[2] = bf_lo(u.y); v[3] = bf_hi(u.y); v[4] = bf_lo(u.z); v[5] = bf_hi(u.z); v[6] = bf_lo(u.w); v[7] = bf_hi(u.w);
    } else {
      const float4 a = *reinterpret_cast<const float4*>(row + k), b = *reinterpret_cast<const float4*>(row + k + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? (float)row[k + i] : 0.f;
  }
}
template <class X, bool VEC>
__device__ __forceinline__ void store8(X* row, int k, int K, const float (&v)[8]) {
  if constexpr (VEC) {
    if (k >= K) return;
    if constexpr (sizeof(X) == 2) {
      *reinterpret_cast<uint4*>(row + k) = make_uint4(bf_pack(v[0], v[1]), bf_pack(v[2], v[3]), bf_pack(v[4], v[5]), bf_pack(v[6], v[7]));
    } else {
      *reinterpret_cast<float4*>(row + k) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(row + k + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < K) row[k + i] = (X)v[i];
  }
}
__device__ __forceinline__ uint2 codes_of(const float (&v)[8], float s) {
  uint32_t c[2];
  codes(v, s, c);
  return make_uint2(c[0], c[1]);
}

// WARPS warps a row, R8_WARPS / WARPS rows a CTA.  The scales of a row wait in shared memory for its sum of squares (NORM).
template <class X, bool VEC, bool NORM, int WARPS>
__global__ void __launch_bounds__(R8_THREADS) rows8_kernel(const Rows8Args a) {
  constexpr int ROWS = R8_WARPS / WARPS;
  extern __shared__ float held[];                // NORM: [ROWS][groups]
  __shared__ float sums[R8_WARPS];
  griddep_launch();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = (int)lane_id(), half = lane >> 4, c = lane & 15;
  const int r = warp / WARPS, part = warp % WARPS, G = (a.K + W8_GROUP - 1) / W8_GROUP;
  const int64_t t = (int64_t)blockIdx.x * ROWS + r;
  float ss = 0.f;
  if (t < a.T) {
    const X* x = reinterpret_cast<const X*>(a.x) + t * a.ldx;
    const X* res = reinterpret_cast<const X*>(a.residual);
    if (res != nullptr) res += t * a.ldr;
    X* to = reinterpret_cast<X*>(a.residual_out) + (res != nullptr ? t * a.ldro : 0);
    uint8_t* code = a.codes + t * a.ldc;
#pragma unroll 2
    for (int g0 = part * 2; g0 < G; g0 += WARPS * 2) {
      const int g = g0 + half, k = g * W8_GROUP + c * 8;
      float v[8];
      load8<X, VEC>(x, k, a.K, v);
      if (res != nullptr) {
        float o[8];
        load8<X, VEC>(res, k, a.K, o);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = rounded<X>(v[i] + o[i]);
        store8<X, VEC>(to, k, a.K, v);
      }
      if constexpr (NORM) {
        float w[8];
        load8<__nv_bfloat16, VEC>(a.norm, k, a.K, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ss += v[i] * v[i];
          v[i] *= w[i];
        }
      }
      uint32_t m = largest(v, 0);
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float s = scale_of(m);
      if (g < G) {
        *reinterpret_cast<uint2*>(code + k) = codes_of(v, s);
        if (c == 0) {
          if constexpr (NORM) held[r * G + g] = s;
          else a.scales[(size_t)g * a.lds + t] = s;
        }
      }
    }
  }
  if constexpr (NORM) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (lane == 0) sums[warp] = ss;
    __syncthreads();
    // (neighbouring threads have neighbouring rows: a CTA's eight scales of a group are one sector)
    for (int i = threadIdx.x; i < G * ROWS; i += R8_THREADS) {
      const int g = i / ROWS, row = i % ROWS;
      const int64_t at = (int64_t)blockIdx.x * ROWS + row;
      float all = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) all += sums[row * WARPS + w];
      if (at < a.T) a.scales[(size_t)g * a.lds + at] = held[row * G + g] * (1.f / sqrtf(all / (float)a.K + a.eps));
    }
  }
}

// A CTA: a block of 128 x 128, eight rows a thread
template <class X, bool VEC>
__global__ void __launch_bounds__(R8_THREADS) weight8_kernel(const X* __restrict__ w, int64_t ldw, int N, int K, uint8_t* __restrict__ codes_out, int64_t ldc,
                                                             float* __restrict__ scales) {
  constexpr int EACH = W8_GROUP / (2 * R8_WARPS);
  __shared__ uint32_t most[R8_WARPS];
  griddep_launch();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = (int)lane_id(), G = (K + W8_GROUP - 1) / W8_GROUP;
  const int nb = (int)(blockIdx.x / (uint32_t)G), g = (int)(blockIdx.x % (uint32_t)G), k = g * W8_GROUP + (lane & 15) * 8;
  const int n0 = nb * W8_GROUP + warp * 2 + (lane >> 4);
  float v[EACH][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int n = n0 + i * 2 * R8_WARPS;
    if (n < N) {
      load8<X, VEC>(w + (int64_t)n * ldw, k, K, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) m = largest(v[i], m);
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) most[warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R8_WARPS; ++i) m = max(m, most[i]);
  const float s = scale_of(m);
  if (threadIdx.x == 0) scales[(size_t)nb * G + g] = s;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int n = n0 + i * 2 * R8_WARPS;
    if (n < N) *reinterpret_cast<uint2*>(codes_out + (int64_t)n * ldc + k) = codes_of(v[i], s);
  }
}

bool on16(const void* p, int64_t ld, int size) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * size % 16 == 0; }

template <class X, bool VEC, bool NORM>
cudaError_t rows8_some(const Rows8Args& a, int num_sms, cudaStream_t stream) {
  const int G = (a.K + W8_GROUP - 1) / W8_GROUP;
  // a CTA a row while that leaves no SM with more than a few, a warp a row from there
  const bool split = a.T <= 4 * num_sms;
  const int rows = split ? 1 : R8_WARPS;
  const unsigned ctas = (unsigned)(((long long)a.T + rows - 1) / rows);
  const size_t smem = NORM ? (size_t)rows * G * sizeof(float) : 0;
  return split ? launch_k(rows8_kernel<X, VEC, NORM, R8_WARPS>, dim3(ctas), dim3(R8_THREADS), smem, stream, a)
               : launch_k(rows8_kernel<X, VEC, NORM, 1>, dim3(ctas), dim3(R8_THREADS), smem, stream, a);
}
template <class X>
cudaError_t rows8_typed(const Rows8Args& a, int num_sms, cudaStream_t stream) {
  const bool vec = a.K % 8 == 0 && on16(a.x, a.ldx, sizeof(X)) && (a.norm == nullptr || on16(a.norm, 0, 2)) &&
                   (a.residual == nullptr || (on16(a.residual, a.ldr, sizeof(X)) && on16(a.residual_out, a.ldro, sizeof(X))));
  if (vec) return a.norm != nullptr ? rows8_some<X, true, true>(a, num_sms, stream) : rows8_some<X, true, false>(a, num_sms, stream);
  return a.norm != nullptr ? rows8_some<X, false, true>(a, num_sms, stream) : rows8_some<X, false, false>(a, num_sms, stream);
}

}  // namespace

cudaError_t rows8_launch(const Rows8Args& a, bool f32, int num_sms, cudaStream_t stream) {
  if (a.T <= 0) return cudaSuccess;
  return f32 ? rows8_typed<float>(a, num_sms, stream) : rows8_typed<__nv_bfloat16>(a, num_sms, stream);
}

cudaError_t weight8_launch(const void* w, bool f32, int64_t ldw, int N, int K, uint8_t* codes_out, int64_t ldc, float* scales, cudaStream_t stream) {
  const long long ctas = (long long)((N + W8_GROUP - 1) / W8_GROUP) * ((K + W8_GROUP - 1) / W8_GROUP);
  if (ctas >= 1ll << 31) return cudaErrorInvalidValue;
  const bool vec = K % 8 == 0 && on16(w, ldw, f32 ? 4 : 2);
  const dim3 grid((unsigned)ctas), block(R8_THREADS);
  if (f32) return launch_k(vec ? weight8_kernel<float, true> : weight8_kernel<float, false>, grid, block, 0, stream, (const float*)w, ldw, N, K, codes_out, ldc, scales);
  return launch_k(vec ? weight8_kernel<__nv_bfloat16, true> : weight8_kernel<__nv_bfloat16, false>, grid, block, 0, stream, (const __nv_bfloat16*)w, ldw, N, K, codes_out, ldc, scales);
}

}  // namespace tgis
