// Layout and number format of the 8-bit paged cache (include/tgis_kv8.h); shared by cache8.cu and attention8*.cu.
//
// A (page, kv head) is one run of 8448 bytes, fetched by one bulk copy: K codes | V codes | K scales | V scales.
//   K  [32 tok][8 chunks of 16 dims, chunk c at place c ^ (tok & 7)][16]: the 128-byte swizzled K-major operand of the tensor cores;
//      ldmatrix of 8 tokens of one chunk touches all banks once.
//   V  [2 halves of 16 tok][128 dims][16 places]: V transposed, the unswizzled K-major operand (8 dims x 16 places are a core matrix).
//      Token t of a half lies at place v8_place(t), so that the scores that a thread holds after S = Q K^T by mma.sync (columns
//      2i, 2i + 1 of neighbouring 8-token tiles) are the four consecutive k places that it needs for P V: nothing is exchanged.
#pragma once
#include <stdint.h>

#include "../../include/tgis_kv8.h"
#include "kernels.h"
#include "tc_attention.cuh"

namespace tgis {

constexpr int KV8_CODES = KV_BLOCK * HEAD_DIM;                 // bytes of a page's K (or V) codes per head
constexpr int KV8_PAGE = 2 * KV8_CODES + 2 * KV_BLOCK * 4;     // 8448
constexpr int KV8_K_SCALES = 2 * KV8_CODES, KV8_V_SCALES = KV8_K_SCALES + KV_BLOCK * 4;
constexpr float KV8_TOP = 448.f;                               // largest e4m3 number
constexpr float KV8_TINY = 1.17549435e-38f;                    // 2^-126: quotients by it stay within e4m3's range

// byte of dim d of token t (of 32) in the K codes
__host__ __device__ __forceinline__ constexpr int k8_at(int t, int d) { return t * HEAD_DIM + (((d >> 4) ^ (t & 7)) << 4) + (d & 15); }
// token bits (j, i, i, v) of a half -> place bits (i, i, j, v)
__host__ __device__ __forceinline__ constexpr int v8_place(int t) { return (t >> 1 & 3) << 2 | (t >> 3 & 1) << 1 | (t & 1); }
__host__ __device__ __forceinline__ constexpr int v8_at(int t, int d) { return (t >> 4) * (KV8_CODES / 2) + d * 16 + v8_place(t & 15); }

// low byte from lo, high byte from hi
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// the two numbers of e4m3x2, as a pair of fp16 (exact)
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t c) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)c));
  return r;
}
__device__ __forceinline__ float2 f16x2_to_f32x2(uint32_t h) {
  float2 f;
  asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.f32.f16 %0, a; cvt.f32.f16 %1, b;}" : "=f"(f.x), "=f"(f.y) : "r"(h));
  return f;
}

// bits of the largest magnitude (and of m's), those of a NaN where one is among them: as whole numbers they order as magnitudes do
__device__ __forceinline__ uint32_t largest(const float (&x)[8], uint32_t m) {
  float f = __uint_as_float(m);
#pragma unroll
  for (int i = 0; i < 8; i += 2) asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(f) : "f"(x[i]), "f"(x[i + 1]));
  return __float_as_uint(f);
}
// Scale of a row (or another group that is quantised together) whose largest magnitude has these bits: NaN where it holds a number that is not finite
__device__ __forceinline__ float scale_of(uint32_t m) {
  return m >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fmaxf(__uint_as_float(m) * (1.f / KV8_TOP), KV8_TINY);
}
// Codes of x / s; zeros where the scale is NaN.  An IEEE division is a call of some forty instructions, and numbers of bf16 lie in the middle
// of two codes often enough that no quotient that is off by a bit will do.  q = x * (1 / s) is within 1.5 ulp; x - q s is exact in a fused
// multiply-add, a first correction by it leaves less than an ulp, and after a second one q is the rounded quotient (Markstein's theorem: the
// reciprocal is the rounded one).  What lies below the least normal number is not exact: tiny groups are taken times 2^64, which no quotient sees.
template <int N>
__device__ __forceinline__ void codes(const float (&v)[N], float s, uint32_t (&out)[N / 4]) {
  const bool fine = s < INFINITY;
  uint64_t x[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) x[i] = pack2(v[2 * i], v[2 * i + 1]);
  if (s < 0x1p-60f) {
    const uint64_t up = pack2(0x1p64f, 0x1p64f);
    s *= 0x1p64f;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) x[i] = mul2(x[i], up);
  }
  const float one = __frcp_rn(s);
  const uint64_t by = pack2(one, one), minus = pack2(-s, -s);
  float q[N];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    uint64_t d = mul2(x[i], by);
    d = fma2(fma2(d, minus, x[i]), by, d);
    d = fma2(fma2(d, minus, x[i]), by, d);
    unpack2(d, q[2 * i], q[2 * i + 1]);
    q[2 * i] = copysignf(q[2 * i], v[2 * i]);   // (of a zero, the sum has lost it)
    q[2 * i + 1] = copysignf(q[2 * i + 1], v[2 * i + 1]);
  }
#pragma unroll
  for (int i = 0; i < N / 4; ++i) out[i] = fine ? e4m3x2(q[4 * i], q[4 * i + 1]) | e4m3x2(q[4 * i + 2], q[4 * i + 3]) << 16 : 0u;
}

// 2^e that brings a magnitude (the bits of a number >= 0) to [2^14, 2^15), the most that f16 has room for; no more than 2^126
__device__ __forceinline__ float power_up(uint32_t bits) {
  const int ex = min(max((int)(bits >> 23), 15), 254);
  return __uint_as_float((uint32_t)(268 - ex) << 23);   // 2^(141 - ex)
}
// of a power of two from 2^-126 to 2^126
__device__ __forceinline__ float one_over(float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); }
// power of two at or above a number > 0 (its bits)
__device__ __forceinline__ float power_above(uint32_t bits) { return __uint_as_float((bits + 0x7fffffu) & 0x7f800000u); }
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
// the smaller number, NaN where one is
__device__ __forceinline__ float min_nan(float x, float y) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
// cudaFuncSetAttribute once a device
struct OncePerDevice {
  static constexpr int MAX = 64;
  bool done[MAX] = {};
  template <class F>
  cudaError_t operator()(F&& f) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < MAX && done[dev]) return cudaSuccess;
    e = f();
    if (e == cudaSuccess && dev < MAX) done[dev] = true;   // (two threads at once: set twice, to the same value)
    return e;
  }
};

// ---- launchers (cache8.cu, attention8.cu); arguments as in include/tgis_kv8.h
cudaError_t kv8_write_launch(uint8_t* pages, int n_pages, int n_kv, const __nv_bfloat16* qkv, int64_t ld, int T, int n_q, const int32_t* positions,
                             const int32_t* slots, const __nv_bfloat16* cos_sin, int n_positions, __nv_bfloat16* q_out, int64_t ldq,
                             int32_t* status, cudaStream_t stream);
cudaError_t kv8_read_launch(const uint8_t* pages, int n_pages, int n_kv, const int32_t* slots, int T, __nv_bfloat16* k_out, int64_t ldk,
                            __nv_bfloat16* v_out, int64_t ldv, int32_t* status, cudaStream_t stream);
struct Attn8Args {
  const uint8_t* pages;
  int n_pages, n_kv;
  const __nv_bfloat16* q;
  int64_t ldq;
  int T, n_q;
  const AttnSeq* seqs;
  int n_seqs;
  const int32_t* block_table;
  int bt_rows, bt_stride;
  const uint64_t* tree;
  float scale;
  int max_q, max_kv;
  __nv_bfloat16* out;
  int64_t ldo;
  int32_t* status;
  int lo_q = -0x7fffffff - 1, hi_q = 0x7fffffff;   // sequences with fewer or more queries are another launch's
  int* stalled = nullptr;            // host memory: set to one where a wait ran out
};
// whether a record agrees with what the call said
__device__ __forceinline__ bool seq_fits(const Attn8Args& a, const AttnSeq& s) {
  return s.q_len >= 0 && s.q_len <= a.max_q && s.kv_len >= s.q_len && s.kv_len <= a.max_kv && s.q_start >= 0 && s.q_start <= a.T - s.q_len &&
         s.block_row >= 0 && s.block_row < a.bt_rows && (s.kv_len + KV_BLOCK - 1) / KV_BLOCK <= a.bt_stride && (a.tree == nullptr || s.q_len <= TGIS_KV8_MAX_TREE);
}
__device__ __forceinline__ bool seq_picked(const Attn8Args& a, const AttnSeq& s) { return s.q_len >= a.lo_q && s.q_len <= a.hi_q; }
__device__ __forceinline__ void say_stalled(const Attn8Args& a) {
  if (a.status != nullptr) atomicOr(a.status, TGIS_KV8_STALLED);
  if (a.stalled != nullptr) {
    *reinterpret_cast<volatile int*>(a.stalled) = 1;
    __threadfence_system();
  }
}
__device__ __forceinline__ AttnSeq load_seq(const Attn8Args& a, int s) {
  const int4 v = reinterpret_cast<const int4*>(a.seqs)[s];
  return AttnSeq{v.x, v.y, v.z, v.w};
}

size_t attn8_workspace(int T, int n_seqs, int n_q, int n_kv, int max_q, int max_kv);
// attention8_prompt.cu: more rows than the warps' own tensor cores take in one pass
bool attn8_prompt_takes(int T, int n_seqs, int n_q, int n_kv, int max_q, int max_kv);   // (sizes that its counters hold)
constexpr int ATTN8_MAX_SMS = 160;             // what workspaces are sized for, so that their size asks no device
size_t attn8_prompt_workspace(int num_sms);
cudaError_t attn8_prompt_launch(const Attn8Args& a, void* workspace, int num_sms, cudaStream_t stream);
// prompts: by attention8_prompt.cu whatever the bounds say (the caller has left single tokens to another launch)
cudaError_t attn8_launch(const Attn8Args& a, void* workspace, int num_sms, cudaStream_t stream, int* launches = nullptr, bool prompts = false);

}  // namespace tgis
