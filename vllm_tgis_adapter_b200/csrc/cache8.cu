// The 8-bit paged cache: rotary embedding, quantisation and scatter of a step's rows, and reading rows back (include/tgis_kv8.h;
// layout: cache8.cuh).
#include <algorithm>

#include "../../include/tgis_kv8.h"
#include "cache8.cuh"
#include "launch.cuh"
#include "ptx.cuh"

namespace tgis {
namespace {

constexpr int W8_WARPS = 4, W8_THREADS = W8_WARPS * 32, W8_WINDOW = 16;   // tokens of half a page: eight threads a row
static_assert(W8_THREADS == W8_WINDOW * 8 && W8_THREADS == HEAD_DIM, "a thread is an eighth of a row, and a dim");

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
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float s) {
  uint32_t c[2];
  codes(x, s, c);
  return make_uint2(c[0], c[1]);
}
// V lies token by token in the low address bits: a row alone is 128 single bytes, and the sixteen rows of half a page are 128 runs of
// sixteen.  So a window of sixteen tokens of the call belongs to one CTA (per head); tokens with neighbouring slots in one half form a run,
// and the CTA takes the runs that BEGIN in its window, whole halves by themselves and shorter runs together: batches of at most
// sixteen tokens.  Every warp works them out for itself.
struct Batches {
  int slot;                      // lane: of token t0 + lane, -1 where there is none (or it is not to be stored)
  uint32_t begins;               // tokens that begin a run (bits); those without a slot are runs of their own
  int at, end;                   // the next batch's first token, behind the last one's last (less t0)
  bool bad;
  __device__ Batches(const int32_t* slots, int t0, int T, int n_pages) {
    const int lane = (int)lane_id(), t = t0 + lane;
    const int s = t < T ? slots[t] : -1;
    int before = t0 > 0 && lane == 0 ? slots[t0 - 1] : -1;
    bad = s >= n_pages * KV_BLOCK;
    slot = bad ? -1 : s;
    if (before >= n_pages * KV_BLOCK) before = -1;
    const int up = __shfl_up_sync(0xffffffffu, slot, 1);
    if (lane > 0) before = up;
    begins = __ballot_sync(0xffffffffu, !(slot >= 0 && before >= 0 && slot == before + 1 && (slot & 15) != 0));
    // (the last run may go on behind the window: to token 30 at most, for it has sixteen at most)
    at = begins & 0xffffu ? __ffs(begins & 0xffffu) - 1 : W8_WINDOW;
    const uint32_t next = begins >> W8_WINDOW;
    end = at == W8_WINDOW ? at : min(next ? W8_WINDOW + __ffs(next) - 1 : 2 * W8_WINDOW, T - t0);
    bad = bad && lane >= at && lane < end;   // (each token is looked at by one CTA a head)
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

// CTAs [0, qk_ctas), warps: every parts-th quad of query and key heads of one token, eight lanes a head (a lane has dims 8 c .. 8 c + 7 and
// their partners 64 further).  The others: a window of tokens of one value head; SINGLE: a row a warp.  2614 tokens of 32 + 8 heads in six prompts on a B200: 14.6 us, 4.1 TB/s
// (memory bound it would be 9; the rest goes to some 190 instructions for every four heads of a token, issue slots 33 % used by a third of the warps that fit).
template <bool SINGLE>
__global__ void __launch_bounds__(W8_THREADS)
kv8_write_kernel(uint8_t* __restrict__ pages, int n_pages, int n_kv, const __nv_bfloat16* qkv, int64_t ld, int T, int n_q,
                 const int32_t* __restrict__ positions, const int32_t* __restrict__ slots, const __nv_bfloat16* __restrict__ cos_sin,
                 int n_positions, __nv_bfloat16* q_out, int64_t ldq, int first_head, int quads, int parts, int qk_ctas, int32_t* status) {
  __shared__ __align__(16) uint8_t stage[W8_WINDOW][HEAD_DIM];
  griddep_launch();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = (int)lane_id(), c = lane & 7;
  const uint32_t group = 0xffu << (lane & 24);          // the eight lanes of a row
  uint32_t bad = 0;
  if ((int)blockIdx.x < qk_ctas) {
    const uint32_t w = blockIdx.x * W8_WARPS + warp;
    const int t = (int)(w / (uint32_t)parts), part = (int)(w - (uint32_t)(t * parts)), heads = n_q + n_kv;
    if (t < T) {
      int pos = positions[t], slot = slots[t];
      const uint4* row = reinterpret_cast<const uint4*>(qkv + (size_t)t * ld) + c;
      auto head_of = [&](int quad) { return first_head + quad * 4 + (lane >> 3); };
      uint4 a = {}, b = {};
      if (head_of(part) < heads) a = row[head_of(part) * 16], b = row[head_of(part) * 16 + 8];
      if (pos < 0 || pos >= n_positions) bad |= TGIS_KV8_BAD_POSITION, pos = min(max(pos, 0), n_positions - 1);
      if (slot >= n_pages * KV_BLOCK) bad |= TGIS_KV8_BAD_SLOT, slot = -1;
      const uint4* turn = reinterpret_cast<const uint4*>(cos_sin + (size_t)pos * HEAD_DIM) + c;
      float p[8], q[8];
      unpack8(turn[0], p);
      unpack8(turn[8], q);
      for (int quad = part; quad < quads; quad += parts) {
        const int head = head_of(quad), next = head_of(quad + parts);
        float x[8], y[8], u[8], v[8];
        unpack8(a, x);
        unpack8(b, y);
        if (quad + parts < quads && next < heads) a = row[next * 16], b = row[next * 16 + 8];   // (ahead of this quad's stores)
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = x[i] * p[i] - y[i] * q[i], v[i] = y[i] * p[i] + x[i] * q[i];
        if (head < n_q) {
          uint4* o = reinterpret_cast<uint4*>(q_out + (size_t)t * ldq + (size_t)head * HEAD_DIM);
          o[c] = pack8(u);
          o[8 + c] = pack8(v);
        } else if (head < heads) {
          uint32_t m = largest(v, largest(u, 0));
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(group, m, o));
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
    }
  } else if constexpr (SINGLE) {
    const uint32_t w = (blockIdx.x - qk_ctas) * W8_WARPS + warp;
    const int t = (int)(w / (uint32_t)n_kv), kvh = (int)(w - (uint32_t)(t * n_kv));
    if (t >= T) return;
    int slot = slots[t];
    const uint2 raw = reinterpret_cast<const uint2*>(qkv + (size_t)t * ld + (size_t)(n_q + n_kv + kvh) * HEAD_DIM)[lane];
    const float x[4] = {lo_f(raw.x), hi_f(raw.x), lo_f(raw.y), hi_f(raw.y)};
    uint32_t m = 0, code[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    const float s = scale_of(__reduce_max_sync(0xffffffffu, m));
    codes(x, s, code);
    if (slot >= n_pages * KV_BLOCK) bad |= TGIS_KV8_BAD_SLOT, slot = -1;
    if (slot >= 0) {
      uint8_t* page = pages + ((size_t)(slot / KV_BLOCK) * n_kv + kvh) * KV8_PAGE;
      uint8_t* to = page + KV8_CODES + v8_at(slot % KV_BLOCK, 4 * lane);
#pragma unroll
      for (int i = 0; i < 4; ++i) to[i * 16] = (uint8_t)(code[0] >> 8 * i);
      if (lane == 0) *reinterpret_cast<float*>(page + KV8_V_SCALES + slot % KV_BLOCK * 4) = s;
    }
  } else {
    const uint32_t w = blockIdx.x - qk_ctas;
    const int t0 = (int)(w / (uint32_t)n_kv) * W8_WINDOW, kvh = (int)(w % (uint32_t)n_kv), r = threadIdx.x >> 3;
    Batches batches(slots, t0, T, n_pages);
    if (batches.bad) bad |= TGIS_KV8_BAD_SLOT;
    int first, n;
    bool whole;
    while (batches.next(first, n, whole)) {
      const int slot = __shfl_sync(0xffffffffu, batches.slot, (first + r) & 31);
      uint8_t* page = pages + ((size_t)max(slot, 0) / KV_BLOCK * n_kv + kvh) * KV8_PAGE;
      const int at = max(slot, 0) % KV_BLOCK;
      if (r < n && slot >= 0) {
        const uint4* row = reinterpret_cast<const uint4*>(qkv + (size_t)(t0 + first + r) * ld + (size_t)(n_q + n_kv + kvh) * HEAD_DIM);
        const uint4 a = row[c], b = row[8 + c];
        float x[8], y[8];
        unpack8(a, x);
        unpack8(b, y);
        uint32_t m = largest(y, largest(x, 0));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(group, m, o));
        const float s = scale_of(m);
        const uint2 u = codes8(x, s), v = codes8(y, s);
        if (c == 0) *reinterpret_cast<float*>(page + KV8_V_SCALES + at * 4) = s;
        if (whole) {
          *reinterpret_cast<uint2*>(&stage[r][8 * c]) = u;
          *reinterpret_cast<uint2*>(&stage[r][64 + 8 * c]) = v;
        } else {
          uint8_t* to = page + KV8_CODES + v8_at(at, 8 * c);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            to[i * 16] = (uint8_t)((i < 4 ? u.x : u.y) >> (i & 3) * 8);
            to[(64 + i) * 16] = (uint8_t)((i < 4 ? v.x : v.y) >> (i & 3) * 8);
          }
        }
      }
      if (whole) {
        __syncthreads();
        uint32_t word[4];                               // of this thread's dim: places 4 i .. are tokens 2 i, 2 i + 1, 8 + 2 i, 9 + 2 i
#pragma unroll
        for (int i = 0; i < 4; ++i)
          word[i] = (uint32_t)stage[2 * i][threadIdx.x] | (uint32_t)stage[2 * i + 1][threadIdx.x] << 8 | (uint32_t)stage[8 + 2 * i][threadIdx.x] << 16 |
                    (uint32_t)stage[9 + 2 * i][threadIdx.x] << 24;
        // (all rows of a whole batch have their slots in one page and half)
        *reinterpret_cast<uint4*>(page + KV8_CODES + (at >> 4) * (KV8_CODES / 2) + threadIdx.x * 16) = make_uint4(word[0], word[1], word[2], word[3]);
        __syncthreads();
      }
    }
  }
  if (bad != 0 && status != nullptr) atomicOr(status, (int)bad);
}

// A CTA: a window of tokens of one head (see Batches), eight threads a row; SINGLE: a row a warp
template <bool SINGLE>
__global__ void __launch_bounds__(W8_THREADS)
kv8_read_kernel(const uint8_t* __restrict__ pages, int n_pages, int n_kv, const int32_t* __restrict__ slots, int T, __nv_bfloat16* __restrict__ k_out,
                int64_t ldk, __nv_bfloat16* __restrict__ v_out, int64_t ldv, int32_t* status) {
  __shared__ __align__(16) uint8_t stage[W8_WINDOW][HEAD_DIM];
  griddep_launch();
  griddep_wait();
  if constexpr (SINGLE) {
    const uint32_t w = blockIdx.x * W8_WARPS + (threadIdx.x >> 5);
    const int lane = (int)lane_id(), t = (int)(w / (uint32_t)n_kv), kvh = (int)(w - (uint32_t)(t * n_kv));
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
      const uint8_t* v = page + KV8_CODES + v8_at(at, 4 * lane);
      kc = *reinterpret_cast<const uint32_t*>(page + k8_at(at, 4 * lane));
      vc = (uint32_t)v[0] | (uint32_t)v[16] << 8 | (uint32_t)v[32] << 16 | (uint32_t)v[48] << 24;
      ks = *reinterpret_cast<const float*>(page + KV8_K_SCALES + at * 4);
      vs = *reinterpret_cast<const float*>(page + KV8_V_SCALES + at * 4);
    }
    auto store = [&](__nv_bfloat16* to, uint32_t code, float s) {
      const float2 a = f16x2_to_f32x2(e4m3x2_to_f16x2(code)), b = f16x2_to_f32x2(e4m3x2_to_f16x2(code >> 16));
      reinterpret_cast<uint2*>(to + (size_t)kvh * HEAD_DIM)[lane] = make_uint2(pack_bf(a.x * s, a.y * s), pack_bf(b.x * s, b.y * s));
    };
    if (k_out != nullptr) store(k_out + (size_t)t * ldk, kc, ks);
    if (v_out != nullptr) store(v_out + (size_t)t * ldv, vc, vs);
    return;
  }
  const int c = threadIdx.x & 7, r = threadIdx.x >> 3, t0 = (int)(blockIdx.x / (uint32_t)n_kv) * W8_WINDOW, kvh = (int)(blockIdx.x % (uint32_t)n_kv);
  Batches batches(slots, t0, T, n_pages);
  if (batches.bad && status != nullptr) atomicOr(status, TGIS_KV8_BAD_SLOT);
  auto store = [&](__nv_bfloat16* out, int64_t ld, int t, uint2 lo, uint2 hi, float s) {
    const uint32_t in[4] = {lo.x, lo.y, hi.x, hi.y};
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = f16x2_to_f32x2(e4m3x2_to_f16x2(in[i >> 1] >> (i & 1) * 16));
      w[i] = pack_bf(f.x * s, f.y * s);
    }
    uint4* to = reinterpret_cast<uint4*>(out + (size_t)t * ld + (size_t)kvh * HEAD_DIM);
    to[c] = make_uint4(w[0], w[1], w[2], w[3]);
    to[8 + c] = make_uint4(w[4], w[5], w[6], w[7]);
  };
  int first, n;
  bool whole;
  while (batches.next(first, n, whole)) {
    const int slot = __shfl_sync(0xffffffffu, batches.slot, (first + r) & 31), t = t0 + first + r;
    const uint8_t* page = pages + ((size_t)max(slot, 0) / KV_BLOCK * n_kv + kvh) * KV8_PAGE;
    const int at = max(slot, 0) % KV_BLOCK;
    const bool there = r < n && slot >= 0;
    uint2 k[2] = {}, v[2] = {};
    float ks = 0.f, vs = 0.f;
    if (there) {
      k[0] = *reinterpret_cast<const uint2*>(page + k8_at(at, 8 * c));
      k[1] = *reinterpret_cast<const uint2*>(page + k8_at(at, 64 + 8 * c));
      ks = *reinterpret_cast<const float*>(page + KV8_K_SCALES + at * 4);
      vs = *reinterpret_cast<const float*>(page + KV8_V_SCALES + at * 4);
    }
    if (whole) {
      const uint4 x = *reinterpret_cast<const uint4*>(page + KV8_CODES + (at >> 4) * (KV8_CODES / 2) + threadIdx.x * 16);
      const uint32_t word[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        stage[2 * i][threadIdx.x] = (uint8_t)word[i];
        stage[2 * i + 1][threadIdx.x] = (uint8_t)(word[i] >> 8);
        stage[8 + 2 * i][threadIdx.x] = (uint8_t)(word[i] >> 16);
        stage[9 + 2 * i][threadIdx.x] = (uint8_t)(word[i] >> 24);
      }
      __syncthreads();
      v[0] = *reinterpret_cast<const uint2*>(&stage[r][8 * c]);
      v[1] = *reinterpret_cast<const uint2*>(&stage[r][64 + 8 * c]);
      __syncthreads();
    } else if (there) {
      const uint8_t* from = page + KV8_CODES + v8_at(at, 8 * c);
      uint32_t w[4] = {};
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i >> 2] |= (uint32_t)from[((i & 7) + (i >> 3) * 64) * 16] << (i & 3) * 8;
      v[0] = make_uint2(w[0], w[1]);
      v[1] = make_uint2(w[2], w[3]);
    }
    if (r < n) {
      if (k_out != nullptr) store(k_out, ldk, t, k[0], k[1], ks);
      if (v_out != nullptr) store(v_out, ldv, t, v[0], v[1], vs);
    }
  }
}

// Rows (tokens times heads) up to which a warp has one: single tokens of many sequences lie on as many pages, and a window would store or read
// its sixteen rows byte by byte in one CTA.  Microseconds of a store, a row a warp against windows, 32 + 8 heads: 96 single tokens 3.5 and
// 8.2; neighbours 16: 2.8 and 4.0, 256: 4.9 and 6.5, 512: 8.3 and 7.9, 1024: 12.5 and 8.7, 2614: 28.8 and 16.2; reading back 2614: 7.6 and 4.5.
constexpr int W8_SINGLE = 4096, W8_ALL_AT_ONCE = 4096;
long long v_ctas(int T, int n_kv, bool single) {
  return single ? ((long long)T * n_kv + W8_WARPS - 1) / W8_WARPS : (long long)(T + W8_WINDOW - 1) / W8_WINDOW * n_kv;
}

}  // namespace

cudaError_t kv8_write_launch(uint8_t* pages, int n_pages, int n_kv, const __nv_bfloat16* qkv, int64_t ld, int T, int n_q, const int32_t* positions,
                             const int32_t* slots, const __nv_bfloat16* cos_sin, int n_positions, __nv_bfloat16* q_out, int64_t ldq,
                             int32_t* status, cudaStream_t stream) {
  if (T <= 0) return cudaSuccess;
  const int first = q_out != nullptr ? 0 : n_q, quads = (n_q + n_kv - first + 3) / 4;
  // a warp a quad while there are few of them; two warps a token (whose cos and sin they then have for several heads) otherwise
  // (ten quads a token: 96 single tokens 3.0 us and 4.0; of one prompt 256 tokens 4.9 and 5.3, 384: 6.5 and 6.8, 512: 7.7 and 8.2, 768: 6.4 and 6.2, 1024: 7.8 and 6.7, 4000: 26.6 and 20.5)
  const int parts = (long long)T * quads <= W8_ALL_AT_ONCE ? quads : std::min(quads, 2);
  const bool single = (long long)T * n_kv <= W8_SINGLE;
  const long long qk = ((long long)T * parts + W8_WARPS - 1) / W8_WARPS, ctas = qk + v_ctas(T, n_kv, single);
  if (ctas >= 1ll << 29) return cudaErrorInvalidValue;
  return launch_k(single ? kv8_write_kernel<true> : kv8_write_kernel<false>, dim3((unsigned)ctas), dim3(W8_THREADS), 0, stream, pages, n_pages, n_kv, qkv, ld, T,
                  n_q, positions, slots, cos_sin, n_positions, q_out, ldq, first, quads, parts, (int)qk, status);
}

cudaError_t kv8_read_launch(const uint8_t* pages, int n_pages, int n_kv, const int32_t* slots, int T, __nv_bfloat16* k_out, int64_t ldk,
                            __nv_bfloat16* v_out, int64_t ldv, int32_t* status, cudaStream_t stream) {
  if (T <= 0 || (k_out == nullptr && v_out == nullptr)) return cudaSuccess;
  const bool single = (long long)T * n_kv <= W8_SINGLE;
  const long long ctas = v_ctas(T, n_kv, single);
  if (ctas >= 1ll << 29) return cudaErrorInvalidValue;
  return launch_k(single ? kv8_read_kernel<true> : kv8_read_kernel<false>, dim3((unsigned)ctas), dim3(W8_THREADS), 0, stream, pages, n_pages, n_kv, slots, T,
                  k_out, ldk, v_out, ldv, status);
}

}  // namespace tgis
