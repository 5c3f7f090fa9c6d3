// Rows of activations and weight matrices in 8 bits (include/tgis_w8.h): what products with 8-bit weights read.
//
// One pass each, bound by memory.  A half-warp has a group of 128 neighbours of a row, eight a lane: its maximum is four exchanges away and
// its codes are eight bytes a lane.  With a norm the factor 1 / rms is the same for a whole row, so the codes are those of r * norm
// and only the scales wait for the row's sum of squares: nothing is read twice or held.
//
// Measured on one B200: 2048 rows x 4096 with residual and norm 13.3 us in bf16 (4.4 TB/s; memory bound it would be 9.0), 18 to 22 in fp32 (4.9 to 5.9 TB/s); one row 2.0 us.  What bounds the
// former: two rounds of a row's loads a CTA with their latency, three waves of CTAs.  Weights 28672 x 8192 from fp32 174 us (6.7 TB/s, a
// copy's rate), from bf16 143 (4.9 TB/s).  What bounds the latter: 64 registers, so that four CTAs run on an SM, do not hold a thread's eight rows (132 bytes of them go to local memory and 264 come back: for
// 117 MB of bf16 as many bytes pass the L2 as for 235 MB of fp32), and a CTA asks for all it reads before its barrier and works after it: issue slots 55 % used, the busiest pipe (alu) 43 %, memory 45 %.  Three CTAs of 80
// registers (68 bytes to local memory) took 137.
#include "launch.cuh"
#include "linear8.cuh"
#include "ptx.cuh"

namespace tgis {
namespace {

constexpr int R8_WARPS = 8, R8_THREADS = R8_WARPS * 32;   // of a block of weights

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
// Eight neighbours at k of a row of K, as they lie in memory; zeros behind it.  VEC: rows start on 16 bytes and K is a multiple of 8.
template <class X>
struct alignas(16) Eight {
  X v[8];
};
template <>
struct alignas(16) Eight<__nv_bfloat16> {
  uint32_t v[4];
};
template <class X, bool VEC>
__device__ __forceinline__ Eight<X> load8(const X* row, int k, int K) {
  Eight<X> e = {};
  if constexpr (VEC) {
    if (k < K) {
      const uint4* p = reinterpret_cast<const uint4*>(row + k);
      *reinterpret_cast<uint4*>(e.v) = p[0];
      if constexpr (sizeof(X) == 4) *reinterpret_cast<uint4*>(e.v + 4) = p[1];
    }
  } else if constexpr (sizeof(X) == 2) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < K) e.v[i / 2] |= (uint32_t)p[k + i] << (i % 2 * 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < K) e.v[i] = row[k + i];
  }
  return e;
}
__device__ __forceinline__ void unpack(const Eight<float>& e, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = e.v[i];
}
__device__ __forceinline__ void unpack(const Eight<__nv_bfloat16>& e, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = i % 2 ? bf_hi(e.v[i / 2]) : bf_lo(e.v[i / 2]);
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

// A CTA: a row, two of its groups a warp at a time; what the next two need is on its way before these are stored (a compiler cannot know that
// outputs and inputs are apart).  The row's scales wait in shared memory for its sum of squares (NORM).
template <class X, bool VEC, bool NORM, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, sizeof(X) == 2 && WARPS == 8 ? 5 : 1) rows8_kernel(const Rows8Args a) {
  extern __shared__ float held[];                // NORM: [groups]
  __shared__ float sums[WARPS];
  griddep_launch();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = (int)lane_id(), half = lane >> 4, c = lane & 15, G = (a.K + W8_GROUP - 1) / W8_GROUP;
  const int64_t t = blockIdx.x;
  const X* x = reinterpret_cast<const X*>(a.x) + t * a.ldx;
  const X* res = a.residual != nullptr ? reinterpret_cast<const X*>(a.residual) + t * a.ldr : nullptr;
  X* to = reinterpret_cast<X*>(a.residual_out) + (res != nullptr ? t * a.ldro : 0);
  uint8_t* code = a.codes + t * a.ldc;
  float ss = 0.f;
  struct Raw {
    Eight<X> x, res;
    Eight<__nv_bfloat16> norm;
  };
  auto load = [&](int g0) {
    const int k = (g0 + half) * W8_GROUP + c * 8;
    Raw raw = {};
    raw.x = load8<X, VEC>(x, k, a.K);
    if (res != nullptr) raw.res = load8<X, VEC>(res, k, a.K);
    if constexpr (NORM) raw.norm = load8<__nv_bfloat16, VEC>(a.norm, k, a.K);
    return raw;
  };
  auto work = [&](int g0, const Raw& raw) {
    const int g = g0 + half, k = g * W8_GROUP + c * 8;
    float xv[8];
    unpack(raw.x, xv);
    if (res != nullptr) {
      float ov[8];
      unpack(raw.res, ov);
#pragma unroll
      for (int i = 0; i < 8; ++i) xv[i] = rounded<X>(xv[i] + ov[i]);
      store8<X, VEC>(to, k, a.K, xv);
    }
    float wv[8];
    if constexpr (NORM) unpack(raw.norm, wv);
    if constexpr (NORM) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ss += xv[i] * xv[i];
        xv[i] *= wv[i];
      }
    }
    uint32_t m = largest(xv, 0);
#pragma unroll
    for (int s = 1; s < 16; s <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, s));
    const float s = scale_of(m);
    if (g < G) {
      *reinterpret_cast<uint2*>(code + k) = codes_of(xv, s);
      if (c == 0) {
        if constexpr (NORM) held[g] = s;
        else a.scales[(size_t)g * a.lds + t] = s;
      }
    }
  };
  constexpr int STEP = WARPS * 2;
  for (int g0 = warp * 2; g0 < G; g0 += 2 * STEP) {
    const bool more = g0 + STEP < G;
    Raw first = load(g0), second = {};
    if (more) second = load(g0 + STEP);
    work(g0, first);
    if (more) work(g0 + STEP, second);
  }
  if constexpr (NORM) {
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, s);
    if (lane == 0) sums[warp] = ss;
    __syncthreads();
    float all = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) all += sums[i];
    const float by = 1.f / sqrtf(all / (float)a.K + a.eps);
    for (int g = threadIdx.x; g < G; g += WARPS * 32) a.scales[(size_t)g * a.lds + t] = held[g] * by;
  }
}

// A CTA: a block of 128 x 128, eight rows a thread
template <class X, bool VEC>
__global__ void __launch_bounds__(R8_THREADS, sizeof(X) == 2 ? 4 : 2) weight8_kernel(const X* __restrict__ w, int64_t ldw, int N, int K, uint8_t* __restrict__ codes_out, int64_t ldc,
                                                             float* __restrict__ scales) {
  constexpr int EACH = W8_GROUP / (2 * R8_WARPS);
  __shared__ uint32_t most[R8_WARPS];
  griddep_launch();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = (int)lane_id(), G = (K + W8_GROUP - 1) / W8_GROUP;
  const int nb = (int)(blockIdx.x / (uint32_t)G), g = (int)(blockIdx.x % (uint32_t)G), k = g * W8_GROUP + (lane & 15) * 8;
  const int n0 = nb * W8_GROUP + warp * 2 + (lane >> 4);
  Eight<X> raw[EACH];   // (as it lies in memory: half the registers of fp32)
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int n = n0 + i * 2 * R8_WARPS;
    raw[i] = n < N ? load8<X, VEC>(w + (int64_t)n * ldw, k, K) : Eight<X>{};
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    float v[8];
    unpack(raw[i], v);
    m = largest(v, m);
  }
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
    float v[8];
    unpack(raw[i], v);
    if (n < N) *reinterpret_cast<uint2*>(codes_out + (int64_t)n * ldc + k) = codes_of(v, s);
  }
}

bool on16(const void* p, int64_t ld, int size) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * size % 16 == 0; }

template <class X, bool VEC, bool NORM>
cudaError_t rows8_some(const Rows8Args& a, int num_sms, cudaStream_t stream) {
  const int G = (a.K + W8_GROUP - 1) / W8_GROUP;
  // Few rows want all of theirs asked for at once, more rows CTAs of which more run at a time.  Measured with norm and residual, 16 and 8 warps, us: 1 x 4096 2.0 / 2.1,
  // 148 x 4096 3.0 / 3.3, 200 x 4096 4.9 / 4.8, 592 x 4096 9.8 / 6.0, 2048 x 4096 30.7 / 13.3; 148 x 8192 4.1 / 5.1, 296 x 8192 7.4 / 8.3, 300 x 8192 9.1 / 8.4.
  const int warps = G <= 8 ? 4 : G <= 16 || a.T > (G <= 32 ? 1 : 2) * num_sms ? 8 : 16;
  auto go = [&](auto kernel) { return launch_k(kernel, dim3((unsigned)a.T), dim3((unsigned)warps * 32), NORM ? (size_t)G * sizeof(float) : 0, stream, a); };
  return warps == 4 ? go(rows8_kernel<X, VEC, NORM, 4>) : warps == 8 ? go(rows8_kernel<X, VEC, NORM, 8>) : go(rows8_kernel<X, VEC, NORM, 16>);
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
