// The 8-bit paged cache: rotary embedding, quantisation and scatter of a step's rows, and reading rows back (include/tgis_kv8.h;
// layout: cache8.cuh).
#include <algorithm>

#include "../../include/tgis_kv8.h"
#include "cache8.cuh"
#include "launch.cuh"
#include "ptx.cuh"

namespace tgis {
namespace {

constexpr int W8_THREADS = 256, W8_TOKENS = 16;   // a CTA: 16 tokens of one head

__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_bf(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Scale of a warp's row, four numbers a lane; odd: the row holds a number that is not finite
__device__ __forceinline__ float row_scale(const float (&x)[4], bool& odd) {
  // as whole numbers, magnitudes order as their values do, with infinities and NaN above all
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  m = __reduce_max_sync(0xffffffffu, m);
  odd = m >= 0x7f800000u;
  return odd ? __uint_as_float(0x7fc00000u) : fmaxf(__fdiv_rn(__uint_as_float(m), KV8_TOP), KV8_TINY);
}

__global__ void __launch_bounds__(W8_THREADS)
kv8_write_kernel(uint8_t* __restrict__ pages, int n_pages, int n_kv, const __nv_bfloat16* qkv, int64_t ld, int T, int n_q,
                 const int32_t* __restrict__ positions, const int32_t* __restrict__ slots, const __nv_bfloat16* __restrict__ cos_sin,
                 int n_positions, __nv_bfloat16* q_out, int64_t ldq, int first_head, int32_t* status) {
  griddep_launch();
  griddep_wait();
  const int t0 = blockIdx.x * W8_TOKENS, head = blockIdx.y + first_head;
  const int warp = threadIdx.x >> 5, lane = (int)lane_id();
  const bool is_v = head >= n_q + n_kv, is_k = !is_v && head >= n_q;
  const int kvh = is_v ? head - n_q - n_kv : head - n_q;
  uint32_t bad = 0;
  for (int i = warp; i < W8_TOKENS; i += W8_THREADS / 32) {
    const int t = t0 + i;
    if (t >= T) break;
    int slot = -1;
    if (head >= n_q) {
      slot = slots[t];
      if (slot >= n_pages * KV_BLOCK) bad |= TGIS_KV8_BAD_SLOT, slot = -1;
    }
    const __nv_bfloat16* row = qkv + (size_t)t * ld + (size_t)head * HEAD_DIM;
    uint8_t* page = pages + ((size_t)max(slot, 0) / KV_BLOCK * n_kv + max(kvh, 0)) * KV8_PAGE;
    const int at = max(slot, 0) % KV_BLOCK;
    bool odd;
    if (is_v) {
      const uint2 w = reinterpret_cast<const uint2*>(row)[lane];   // dims 4 lane ..
      const float x[4] = {lo_f(w.x), hi_f(w.x), lo_f(w.y), hi_f(w.y)};
      const float s = row_scale(x, odd);
      const uint32_t c01 = odd ? 0u : e4m3x2(__fdiv_rn(x[0], s), __fdiv_rn(x[1], s)), c23 = odd ? 0u : e4m3x2(__fdiv_rn(x[2], s), __fdiv_rn(x[3], s));
      if (slot >= 0) {
        uint8_t* v = page + KV8_CODES + v8_at(at, 4 * lane);
        v[0] = (uint8_t)c01; v[16] = (uint8_t)(c01 >> 8); v[32] = (uint8_t)c23; v[48] = (uint8_t)(c23 >> 8);
        if (lane == 0) *reinterpret_cast<float*>(page + KV8_V_SCALES + at * 4) = s;
      }
      continue;
    }
    if (!is_k && q_out == nullptr) continue;
    int pos = positions[t];
    if (pos < 0 || pos >= n_positions) bad |= TGIS_KV8_BAD_POSITION, pos = min(max(pos, 0), n_positions - 1);
    // dims 2 lane, 2 lane + 1 and their partners 64 further
    const uint32_t a = reinterpret_cast<const uint32_t*>(row)[lane], b = reinterpret_cast<const uint32_t*>(row)[32 + lane];
    const uint32_t c = reinterpret_cast<const uint32_t*>(cos_sin + (size_t)pos * HEAD_DIM)[lane];
    const uint32_t s2 = reinterpret_cast<const uint32_t*>(cos_sin + (size_t)pos * HEAD_DIM)[32 + lane];
    const float x[4] = {lo_f(a) * lo_f(c) - lo_f(b) * lo_f(s2), hi_f(a) * hi_f(c) - hi_f(b) * hi_f(s2),
                        lo_f(b) * lo_f(c) + lo_f(a) * lo_f(s2), hi_f(b) * hi_f(c) + hi_f(a) * hi_f(s2)};
    if (!is_k) {
      uint32_t* o = reinterpret_cast<uint32_t*>(q_out + (size_t)t * ldq + (size_t)head * HEAD_DIM);
      o[lane] = pack_bf(x[0], x[1]);
      o[32 + lane] = pack_bf(x[2], x[3]);
      continue;
    }
    const float s = row_scale(x, odd);
    if (slot < 0) continue;
    *reinterpret_cast<uint16_t*>(page + k8_at(at, 2 * lane)) = odd ? 0 : (uint16_t)e4m3x2(__fdiv_rn(x[0], s), __fdiv_rn(x[1], s));
    *reinterpret_cast<uint16_t*>(page + k8_at(at, 64 + 2 * lane)) = odd ? 0 : (uint16_t)e4m3x2(__fdiv_rn(x[2], s), __fdiv_rn(x[3], s));
    if (lane == 0) *reinterpret_cast<float*>(page + KV8_K_SCALES + at * 4) = s;
  }
  if (bad != 0 && lane == 0 && status != nullptr) atomicOr(status, (int)bad);
}

__global__ void __launch_bounds__(256)
kv8_read_kernel(const uint8_t* __restrict__ pages, int n_pages, int n_kv, const int32_t* __restrict__ slots, int T, __nv_bfloat16* __restrict__ k_out,
                int64_t ldk, __nv_bfloat16* __restrict__ v_out, int64_t ldv, int32_t* status) {
  griddep_launch();
  griddep_wait();
  const int lane = (int)lane_id(), i = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int t = i / n_kv, kvh = i - t * n_kv;
  if (t >= T) return;
  int slot = slots[t];
  if (slot >= n_pages * KV_BLOCK) {
    if (lane == 0 && status != nullptr) atomicOr(status, TGIS_KV8_BAD_SLOT);
    slot = -1;
  }
  uint32_t kc = 0, vc = 0;
  float ks = 0.f, vs = 0.f;
  if (slot >= 0) {
    const uint8_t* page = pages + ((size_t)(slot / KV_BLOCK) * n_kv + kvh) * KV8_PAGE;
    const int at = slot % KV_BLOCK;
    kc = *reinterpret_cast<const uint32_t*>(page + k8_at(at, 4 * lane));
    const uint8_t* v = page + KV8_CODES + v8_at(at, 4 * lane);
    vc = (uint32_t)v[0] | (uint32_t)v[16] << 8 | (uint32_t)v[32] << 16 | (uint32_t)v[48] << 24;
    ks = *reinterpret_cast<const float*>(page + KV8_K_SCALES + at * 4);
    vs = *reinterpret_cast<const float*>(page + KV8_V_SCALES + at * 4);
  }
  auto store = [&](__nv_bfloat16* to, uint32_t c, float s) {
    const float2 a = f16x2_to_f32x2(e4m3x2_to_f16x2(c & 0xffffu)), b = f16x2_to_f32x2(e4m3x2_to_f16x2(c >> 16));
    *reinterpret_cast<uint2*>(to + (size_t)kvh * HEAD_DIM + lane * 4) = make_uint2(pack_bf(a.x * s, a.y * s), pack_bf(b.x * s, b.y * s));
  };
  if (k_out != nullptr) store(k_out + (size_t)t * ldk, kc, ks);
  if (v_out != nullptr) store(v_out + (size_t)t * ldv, vc, vs);
}

}  // namespace

cudaError_t kv8_write_launch(uint8_t* pages, int n_pages, int n_kv, const __nv_bfloat16* qkv, int64_t ld, int T, int n_q, const int32_t* positions,
                             const int32_t* slots, const __nv_bfloat16* cos_sin, int n_positions, __nv_bfloat16* q_out, int64_t ldq,
                             int32_t* status, cudaStream_t stream) {
  if (T <= 0) return cudaSuccess;
  const int first = q_out != nullptr ? 0 : n_q;
  return launch_k(kv8_write_kernel, dim3((T + W8_TOKENS - 1) / W8_TOKENS, n_q + 2 * n_kv - first), dim3(W8_THREADS), 0, stream, pages, n_pages, n_kv,
                  qkv, ld, T, n_q, positions, slots, cos_sin, n_positions, q_out, ldq, first, status);
}

cudaError_t kv8_read_launch(const uint8_t* pages, int n_pages, int n_kv, const int32_t* slots, int T, __nv_bfloat16* k_out, int64_t ldk,
                            __nv_bfloat16* v_out, int64_t ldv, int32_t* status, cudaStream_t stream) {
  if (T <= 0 || (k_out == nullptr && v_out == nullptr)) return cudaSuccess;
  return launch_k(kv8_read_kernel, dim3((unsigned)(((int64_t)T * n_kv + 7) / 8)), dim3(256), 0, stream, pages, n_pages, n_kv, slots, T, k_out, ldk, v_out,
                  ldv, status);
}

}  // namespace tgis
