// The 8-bit paged cache: rotary embedding, quantisation and scatter of a step's rows, and reading rows back (include/tgis_kv8.h;
// layout: cache8.cuh).
#include <algorithm>

#include "../../include/tgis_kv8.h"
#include "cache8.cuh"
#include "launch.cuh"
#include "ptx.cuh"

namespace tgis {
namespace {

constexpr int W8_WARPS = 4, W8_THREADS = W8_WARPS * 32, W8_WINDOW = 16;   // tokens of half a page

__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_bf(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8]) {
  x[0] = lo_f(v.x); x[1] = hi_f(v.x); x[2] = lo_f(v.y); x[3] = hi_f(v.y); x[4] = lo_f(v.z); x[5] = hi_f(v.z); x[6] = lo_f(v.w); x[7] = hi_f(v.w);
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) { return make_uint4(pack_bf(x[0], x[1]), pack_bf(x[2], x[3]), pack_bf(x[4], x[5]), pack_bf(x[6], x[7])); }
// magnitudes as whole numbers order as their values do, with infinities and NaN above all
__device__ __forceinline__ uint32_t largest(const float (&x)[8], uint32_t m) {
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  return m;
}
// Scale of a row whose largest magnitude has these bits: NaN where the row holds a number that is not finite
__device__ __forceinline__ float scale_of(uint32_t m) {
  return m >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fmaxf(__fdiv_rn(__uint_as_float(m), KV8_TOP), KV8_TINY);
}
// eight codes; zeros where the scale is NaN
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float s) {
  if (!(s < INFINITY)) return make_uint2(0, 0);
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = __fdiv_rn(x[i], s);
  return make_uint2(e4m3x2(q[0], q[1]) | e4m3x2(q[2], q[3]) << 16, e4m3x2(q[4], q[5]) | e4m3x2(q[6], q[7]) << 16);
}
// bytes of four words -> words of their bytes 0, 1, 2, 3
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
  const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140), c = __byte_perm(w[0], w[1], 0x7362), d = __byte_perm(w[2], w[3], 0x7362);
  w[0] = __byte_perm(a, b, 0x5410);
  w[1] = __byte_perm(a, b, 0x7632);
  w[2] = __byte_perm(c, d, 0x5410);
  w[3] = __byte_perm(c, d, 0x7632);
}

// V lies token by token in the low address bits, so its rows are stored and read sixteen tokens at a time where those fill half a page.
// A window of sixteen tokens of the call belongs to one warp (per head); tokens with neighbouring slots in one half form a run, and the
// warp takes the runs that BEGIN in its window, whole ones by themselves and shorter ones together: batches of at most sixteen tokens.
struct Batches {
  int slot;                      // lane: of token t0 + lane, -1 where there is none (or it is not to be stored)
  uint32_t begins;               // tokens that begin a run (bits)
  int at, end;                   // the next batch's first token, behind the last one's last (less t0)
  bool bad;
  __device__ Batches(const int32_t* slots, int t0, int T, int n_pages) {
    const int lane = (int)lane_id(), t = t0 + lane;
    int s = t < T ? slots[t] : -1, before = t0 > 0 && lane == 0 ? slots[t0 - 1] : -1;
    bad = s >= n_pages * KV_BLOCK;
    slot = bad ? -1 : s;
    if (before >= n_pages * KV_BLOCK) before = -1;
    const int up = __shfl_up_sync(0xffffffffu, slot, 1);
    if (lane > 0) before = up;
    begins = __ballot_sync(0xffffffffu, slot >= 0 && before >= 0 && slot == before + 1 && (slot & 15) != 0 ? 0 : 1);   // (tokens without a slot are runs of their own)
    // a run that goes on behind the window's tokens, but no further than lane 31: sixteen at most
    at = begins & 0xffffu ? __ffs(begins & 0xffffu) - 1 : W8_WINDOW;
    const uint32_t next = begins >> W8_WINDOW;
    end = at == W8_WINDOW ? at : next ? W8_WINDOW + __ffs(next) - 1 : 2 * W8_WINDOW;
    end = min(end, T - t0);
    bad = bad && lane < end && lane >= at;   // (each token's slot is looked at by one warp a head)
  }
  // the next batch: tokens [first, first + n) less t0; whole: they fill half a page
  __device__ bool next(int& first, int& n, bool& whole) {
    if (at >= end) return false;
    auto run = [&](int a) {
      const uint32_t later = a < 31 ? begins & ~((2u << a) - 1u) : 0u;
      return min(later ? __ffs(later) - 1 : 32, end) - a;
    };
    first = at;
    n = run(at);
    whole = n == W8_WINDOW;                  // (a run of sixteen begins a half)
    while (!whole && at + n < end) {
      const int more = run(at + n);
      if (more == W8_WINDOW || n + more > W8_WINDOW) break;
      n += more;
    }
    at += n;
    return true;
  }
};

// Warps [0, qk_warps): four query or key heads of one token, eight lanes a head (a lane has dims 8 c .. 8 c + 7 and their partners 64
// further); the others: a window of tokens of one value head.
__global__ void __launch_bounds__(W8_THREADS)
kv8_write_kernel(uint8_t* __restrict__ pages, int n_pages, int n_kv, const __nv_bfloat16* qkv, int64_t ld, int T, int n_q,
                 const int32_t* __restrict__ positions, const int32_t* __restrict__ slots, const __nv_bfloat16* __restrict__ cos_sin,
                 int n_positions, __nv_bfloat16* q_out, int64_t ldq, int first_head, int quads, int qk_ctas, int32_t* status) {
  __shared__ __align__(16) uint8_t stage_s[W8_WARPS][W8_WINDOW * HEAD_DIM];
  griddep_launch();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = (int)lane_id();
  uint32_t bad = 0;
  if ((int)blockIdx.x < qk_ctas) {
    const long long w = (long long)blockIdx.x * W8_WARPS + warp;
    const int t = (int)(w / quads), head = first_head + (int)(w - (long long)t * quads) * 4 + (lane >> 3), c = lane & 7;
    if (t < T && head < n_q + n_kv) {
      int pos = positions[t], slot = head >= n_q ? slots[t] : -1;
      const __nv_bfloat16* row = qkv + (size_t)t * ld + (size_t)head * HEAD_DIM;
      const uint4 a = reinterpret_cast<const uint4*>(row)[c], b = reinterpret_cast<const uint4*>(row)[8 + c];
      if (pos < 0 || pos >= n_positions) bad |= TGIS_KV8_BAD_POSITION, pos = min(max(pos, 0), n_positions - 1);
      const uint4 co = reinterpret_cast<const uint4*>(cos_sin + (size_t)pos * HEAD_DIM)[c], si = reinterpret_cast<const uint4*>(cos_sin + (size_t)pos * HEAD_DIM)[8 + c];
      float x[8], y[8], p[8], q[8], u[8], v[8];
      unpack8(a, x);
      unpack8(b, y);
      unpack8(co, p);
      unpack8(si, q);
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = x[i] * p[i] - y[i] * q[i], v[i] = y[i] * p[i] + x[i] * q[i];
      if (head < n_q) {
        uint4* o = reinterpret_cast<uint4*>(q_out + (size_t)t * ldq + (size_t)head * HEAD_DIM);
        o[c] = pack8(u);
        o[8 + c] = pack8(v);
      } else {
        // (the eight lanes of a head are here together)
        const uint32_t group = 0xffu << (lane & 24);
        uint32_t m = largest(v, largest(u, 0));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(group, m, o));
        if (slot >= n_pages * KV_BLOCK) bad |= TGIS_KV8_BAD_SLOT, slot = -1;
        if (slot >= 0) {
          const float s = scale_of(m);
          const int at = slot % KV_BLOCK;
          uint8_t* page = pages + ((size_t)(slot / KV_BLOCK) * n_kv + (head - n_q)) * KV8_PAGE;
          *reinterpret_cast<uint2*>(page + k8_at(at, 8 * c)) = codes8(u, s);
          *reinterpret_cast<uint2*>(page + k8_at(at, 64 + 8 * c)) = codes8(v, s);
          if (c == 0) *reinterpret_cast<float*>(page + KV8_K_SCALES + at * 4) = s;
        }
      }
    }
  } else {
    const long long w = (long long)(blockIdx.x - qk_ctas) * W8_WARPS + warp;
    const int kvh = (int)(w % n_kv);
    const long long t0 = w / n_kv * W8_WINDOW;
    if (t0 >= T) return;
    uint8_t* stage = stage_s[warp];
    Batches batches(slots, (int)t0, T, n_pages);
    if (batches.bad) bad |= TGIS_KV8_BAD_SLOT;
    int first, n;
    bool whole;
    while (batches.next(first, n, whole)) {
      // sixteen lanes a row, two rows a load
      const int sub = lane >> 4, c = lane & 15;
      uint4 raw[W8_WINDOW / 2];
#pragma unroll
      for (int i = 0; i < W8_WINDOW / 2; ++i) {
        const int k = 2 * i + sub;
        if (k < n) raw[i] = reinterpret_cast<const uint4*>(qkv + (size_t)(t0 + first + k) * ld + (size_t)(n_q + n_kv + kvh) * HEAD_DIM)[c];
        else raw[i] = make_uint4(0, 0, 0, 0);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < W8_WINDOW / 2; ++i) {
        const int k = 2 * i + sub;
        float x[8];
        unpack8(raw[i], x);
        uint32_t m = largest(x, 0);
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float s = scale_of(m);
        *reinterpret_cast<uint2*>(stage + k * HEAD_DIM + c * 8) = codes8(x, s);
        const int slot = __shfl_sync(0xffffffffu, batches.slot, (first + k) & 31);
        if (c == 0 && k < n && slot >= 0)
          *reinterpret_cast<float*>(pages + ((size_t)(slot / KV_BLOCK) * n_kv + kvh) * KV8_PAGE + KV8_V_SCALES + slot % KV_BLOCK * 4) = s;
      }
      __syncwarp();
      if (whole) {
        // dims 4 lane .. 4 lane + 3: their sixteen tokens in the order of the places, 2 i, 2 i + 1, 8 + 2 i, 9 + 2 i
        const int slot = __shfl_sync(0xffffffffu, batches.slot, first);
        uint32_t word[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int k = 0; k < 4; ++k) word[i][k] = *reinterpret_cast<const uint32_t*>(stage + (2 * i + (k & 1) + (k >> 1) * 8) * HEAD_DIM + 4 * lane);
          transpose4(word[i]);
        }
        uint4* to = reinterpret_cast<uint4*>(pages + ((size_t)(slot / KV_BLOCK) * n_kv + kvh) * KV8_PAGE + KV8_CODES + v8_at(slot % KV_BLOCK & 16, 4 * lane));
#pragma unroll
        for (int d = 0; d < 4; ++d) to[d] = make_uint4(word[0][d], word[1][d], word[2][d], word[3][d]);
      } else {
        for (int k = 0; k < n; ++k) {
          const int slot = __shfl_sync(0xffffffffu, batches.slot, first + k);
          if (slot < 0) continue;
          const uint32_t x = *reinterpret_cast<const uint32_t*>(stage + k * HEAD_DIM + 4 * lane);
          uint8_t* to = pages + ((size_t)(slot / KV_BLOCK) * n_kv + kvh) * KV8_PAGE + KV8_CODES + v8_at(slot % KV_BLOCK, 4 * lane);
          to[0] = (uint8_t)x; to[16] = (uint8_t)(x >> 8); to[32] = (uint8_t)(x >> 16); to[48] = (uint8_t)(x >> 24);
        }
      }
      __syncwarp();
    }
  }
  if (bad != 0 && status != nullptr) atomicOr(status, (int)bad);
}

// A warp: a window of tokens of one head (see Batches), sixteen lanes a row
__global__ void __launch_bounds__(W8_THREADS)
kv8_read_kernel(const uint8_t* __restrict__ pages, int n_pages, int n_kv, const int32_t* __restrict__ slots, int T, __nv_bfloat16* __restrict__ k_out,
                int64_t ldk, __nv_bfloat16* __restrict__ v_out, int64_t ldv, int32_t* status) {
  __shared__ __align__(16) uint8_t stage_s[W8_WARPS][W8_WINDOW * HEAD_DIM];
  griddep_launch();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = (int)lane_id();
  const long long w = (long long)blockIdx.x * W8_WARPS + warp;
  const int kvh = (int)(w % n_kv);
  const long long t0 = w / n_kv * W8_WINDOW;
  if (t0 >= T) return;
  uint8_t* stage = stage_s[warp];
  Batches batches(slots, (int)t0, T, n_pages);
  if (batches.bad && status != nullptr) atomicOr(status, TGIS_KV8_BAD_SLOT);
  const int sub = lane >> 4, c = lane & 15;
  auto page_of = [&](int slot) { return pages + ((size_t)(slot / KV_BLOCK) * n_kv + kvh) * KV8_PAGE; };
  auto store = [&](__nv_bfloat16* out, int64_t ld, int k, uint2 codes, float s) {
    float x[8];
    const uint32_t in[2] = {codes.x, codes.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = f16x2_to_f32x2(e4m3x2_to_f16x2(in[i >> 1] >> (i & 1) * 16));
      x[2 * i] = f.x * s;
      x[2 * i + 1] = f.y * s;
    }
    reinterpret_cast<uint4*>(out + (size_t)(t0 + k) * ld + (size_t)kvh * HEAD_DIM)[c] = pack8(x);
  };
  int first, n;
  bool whole;
  while (batches.next(first, n, whole)) {
    if (v_out != nullptr) {
      __syncwarp();
      if (whole) {
        const int slot = __shfl_sync(0xffffffffu, batches.slot, first);
        const uint4* from = reinterpret_cast<const uint4*>(page_of(slot) + KV8_CODES + v8_at(slot % KV_BLOCK & 16, 4 * lane));
        uint4 x[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) x[d] = from[d];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          auto part = [&](int d) { return i == 0 ? x[d].x : i == 1 ? x[d].y : i == 2 ? x[d].z : x[d].w; };
          uint32_t word[4] = {part(0), part(1), part(2), part(3)};
          transpose4(word);
#pragma unroll
          for (int k = 0; k < 4; ++k) *reinterpret_cast<uint32_t*>(stage + (2 * i + (k & 1) + (k >> 1) * 8) * HEAD_DIM + 4 * lane) = word[k];
        }
      } else {
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
          const int slot = __shfl_sync(0xffffffffu, batches.slot, first + k);
          uint32_t x = 0;
          if (slot >= 0) {
            const uint8_t* v = page_of(slot) + KV8_CODES + v8_at(slot % KV_BLOCK, 4 * lane);
            x = (uint32_t)v[0] | (uint32_t)v[16] << 8 | (uint32_t)v[32] << 16 | (uint32_t)v[48] << 24;
          }
          *reinterpret_cast<uint32_t*>(stage + k * HEAD_DIM + 4 * lane) = x;
        }
      }
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < W8_WINDOW / 2; ++i) {
      const int k = 2 * i + sub, slot = __shfl_sync(0xffffffffu, batches.slot, (first + k) & 31);
      if (k >= n) continue;
      const uint8_t* page = page_of(max(slot, 0));
      const int at = max(slot, 0) % KV_BLOCK;
      if (k_out != nullptr)
        store(k_out, ldk, first + k, slot >= 0 ? *reinterpret_cast<const uint2*>(page + k8_at(at, 8 * c)) : make_uint2(0, 0),
              slot >= 0 ? *reinterpret_cast<const float*>(page + KV8_K_SCALES + at * 4) : 0.f);
      if (v_out != nullptr)
        store(v_out, ldv, first + k, *reinterpret_cast<const uint2*>(stage + k * HEAD_DIM + c * 8), slot >= 0 ? *reinterpret_cast<const float*>(page + KV8_V_SCALES + at * 4) : 0.f);
    }
  }
}

}  // namespace

cudaError_t kv8_write_launch(uint8_t* pages, int n_pages, int n_kv, const __nv_bfloat16* qkv, int64_t ld, int T, int n_q, const int32_t* positions,
                             const int32_t* slots, const __nv_bfloat16* cos_sin, int n_positions, __nv_bfloat16* q_out, int64_t ldq,
                             int32_t* status, cudaStream_t stream) {
  if (T <= 0) return cudaSuccess;
  const int first = q_out != nullptr ? 0 : n_q, quads = (n_q + n_kv - first + 3) / 4;
  const long long qk = ((long long)T * quads + W8_WARPS - 1) / W8_WARPS, v = ((long long)(T + W8_WINDOW - 1) / W8_WINDOW * n_kv + W8_WARPS - 1) / W8_WARPS;
  if (qk + v >= 1ll << 31) return cudaErrorInvalidValue;
  return launch_k(kv8_write_kernel, dim3((unsigned)(qk + v)), dim3(W8_THREADS), 0, stream, pages, n_pages, n_kv, qkv, ld, T, n_q, positions, slots, cos_sin,
                  n_positions, q_out, ldq, first, quads, (int)qk, status);
}

cudaError_t kv8_read_launch(const uint8_t* pages, int n_pages, int n_kv, const int32_t* slots, int T, __nv_bfloat16* k_out, int64_t ldk,
                            __nv_bfloat16* v_out, int64_t ldv, int32_t* status, cudaStream_t stream) {
  if (T <= 0 || (k_out == nullptr && v_out == nullptr)) return cudaSuccess;
  const long long ctas = ((long long)(T + W8_WINDOW - 1) / W8_WINDOW * n_kv + W8_WARPS - 1) / W8_WARPS;
  if (ctas >= 1ll << 31) return cudaErrorInvalidValue;
  return launch_k(kv8_read_kernel, dim3((unsigned)ctas), dim3(W8_THREADS), 0, stream, pages, n_pages, n_kv, slots, T, k_out, ldk, v_out, ldv, status);
}

}  // namespace tgis
