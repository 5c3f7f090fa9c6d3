// Attention over the 8-bit paged cache (include/tgis_kv8.h; layout and number format: cache8.cuh): single tokens, drafted trees and
// short prompts on the warps' own tensor cores.
//
//   s_t = scale sk_t (q . ck_t),  p_t = exp(s_t - m),  o = sum p_t sv_t cv_t / sum p_t     over the tokens t that the row sees
//
// Both products are mma.sync f16 x f16 -> fp32, K and V widened in registers (exact) as their fragments leave shared memory; mma.sync on
// e4m3 itself, with queries and probabilities as two e4m3 numbers each, costs the same tensor work and fifteen instructions each
// (64 tokens behind 8000, 32 / 8 heads: 211 us, against 194).  A query row (bf16) times the power of two that brings its largest number to
// [2^14, 2^15) is exact in f16 but for numbers 2^-31 of the largest and below (off by 2^-39 of it).  Scores are multiplied by their key's scale in fp32; a row's
// weight, probability times value's scale, is one f16 number of 11 bits, held times 2^7 / r.  The reference m of a row's exponentials moves
// only when a score passes it by 2^8, and r, a power of two and the row's own, only when a weight passes it by 2^8: it fits f16 (2^15 at
// most), and nothing above 2^-31 of the row's largest weight is lost, whatever tokens hold that it does not see or gives no weight.
//
// Work item = (sequence, 8 or 16 rows, kv head, split of the keys); row = token * G + head of the group.  A CTA's four warps take the
// item's blocks of 32 tokens in turn (one bulk copy each, requested RING blocks ahead across items) and join their sums in shared memory;
// a sequence of several splits leaves them in the workspace to attn8_merge_kernel.  Sequence lengths and pages are read on the device,
// so the list of items is made by every CTA for itself: a prefix sum over the sequences.
//
// What bounds it: reading the pages where they are many (64 tokens behind 8000: 201 us, 5.4 TB/s, 82% of a copy's rate); below that the
// chain of a block in a warp (copy, scores, softmax, output: about 0.5 us) and the launch: one token behind 16: 4.7 us, behind 511: 7.6,
// behind 8191: 11.9 (32 splits and their join); 32 behind 511 to 639: 12.5.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/tgis_kv8.h"
#include "cache8.cuh"
#include "launch.cuh"
#include "ptx.cuh"
#include "tc_attention.cuh"

namespace tgis {
namespace {

constexpr int R8_WARPS = 4, R8_THREADS = R8_WARPS * 32, R8_RING = 2;
constexpr int R8_CTAS(int rows) { return rows == 8 ? 3 : 2; }   // per SM
// Rows of a sequence (its queries times heads of a group) up to which this kernel reads its pages once for each 16 of them, instead of one
// unit of attention8_prompt.cu; and keys up to which it takes more rows, where all run at once.  Microseconds here and there, 32 / 8 heads:
// 8 queries behind 500: 10.4 and 15.8; 32 x 8 behind 1000: 35 and 59; 32 x 12: 52 and 60; 32 x 16: 69 and 60; a prompt of 64: 7.5 and 11.2, of
// 128: 8.1 and 12.4; 64 behind 500: 12.7 and 19.3, 128: 13.5 and 21.3; 96 behind 2000: 29 and 24; four prompts of 32 (all at once): 8.2 and
// 9.3, of 48 (not): 13.6 and 11.5.
constexpr int R8_MOST_ROWS = 48, R8_MORE_KEYS = 1024;
constexpr int R8_ONE_SPLIT = 768;                  // keys of a sequence that are not split
constexpr float R8_SLACK = 8.f;                    // exp2 domain: how far a score may exceed its row's reference
constexpr float R8_HELD = 128.f, R8_ROOM = 256.f;  // weights are held times 2^7 / r; how often r fits into the largest of them before it moves
constexpr float R8_LEAST = 0x1p-118f;              // smallest r

struct RowsArgs : Attn8Args {
  float *part_o, *part_ml;
  int max_splits, split, rows_of_seq;         // split: most tokens of one (a multiple of KV_BLOCK)
};
// a sequence's splits are of equal length but for the last
__device__ __forceinline__ int splits_of(const RowsArgs& a, const AttnSeq& s) { return (s.kv_len + a.split - 1) / a.split; }
__device__ __forceinline__ int split_blocks(const RowsArgs& a, const AttnSeq& s) {
  const int n = splits_of(a, s);
  return ((s.kv_len + KV_BLOCK - 1) / KV_BLOCK + n - 1) / max(n, 1);
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// C = A B
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
struct RowsItem {
  AttnSeq sq;
  int seq, kvh, chunk, split, tok0, n_tok;         // keys tok0 .. tok0 + n_tok - 1 of the sequence (of the split, and seen by a row of the chunk)
  __device__ int n_blk() const { return (n_tok + KV_BLOCK - 1) / KV_BLOCK; }
};

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {   // 8 x 8 f16 across the warp
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
  return d;
}

template <int ROWS>
__global__ void __launch_bounds__(R8_THREADS, R8_CTAS(ROWS)) attn8_rows_kernel(const __grid_constant__ RowsArgs a) {
  constexpr int NT = ROWS / 8;                // column tiles of the products
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full_s[R8_WARPS * R8_RING];
  __shared__ int32_t ok_s[R8_WARPS * R8_RING], wsum[R8_WARPS];
  __shared__ float2 stat_s[R8_WARPS][ROWS];
  __shared__ float4 hand_s[R8_WARPS][ROWS / 8][2][32];
  const int warp = threadIdx.x >> 5, lane = (int)lane_id();
  uint8_t* ring = smem + warp * (R8_RING * KV8_PAGE);
  int32_t* prefix = reinterpret_cast<int32_t*>(smem + R8_WARPS * R8_RING * KV8_PAGE);   // items ahead of sequence s, per kv head
  uint64_t* full = full_s + warp * R8_RING;
  volatile int32_t* page_ok = ok_s + warp * R8_RING;
  if (lane == 0) {
    for (int i = 0; i < R8_RING; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  griddep_launch();
  griddep_wait();
  const int G = a.n_q / a.n_kv;
  // ---- items of every sequence
  auto chunks_of = [&](const AttnSeq& s) { return (s.q_len * G + ROWS - 1) / ROWS; };
  int carry = 0;
  for (int base = 0; base < a.n_seqs; base += R8_THREADS) {
    const int s = base + threadIdx.x;
    int n = 0;
    if (s < a.n_seqs) {
      const AttnSeq sq = load_seq(a, s);
      if (!seq_picked(a, sq)) n = 0;
      else if (seq_fits(a, sq)) n = chunks_of(sq) * splits_of(a, sq);
      else if (blockIdx.x == 0 && a.status != nullptr) atomicOr(a.status, TGIS_KV8_BAD_SEQ);
    }
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) wsum[warp] = sum;
    __syncthreads();
    int before = carry, total = 0;
#pragma unroll
    for (int w = 0; w < R8_WARPS; ++w) {
      if (w < warp) before += wsum[w];
      total += wsum[w];
    }
    if (s < a.n_seqs) prefix[s] = before + sum - n;
    carry += total;
    __syncthreads();
  }
  const uint32_t n_flat = (uint32_t)carry * a.n_kv, n_slots = gridDim.x;   // (host: no more than 2^31)
  auto item_at = [&](uint32_t f) {
    RowsItem it;
    const int e = (int)(f / (uint32_t)a.n_kv);
    it.kvh = (int)(f - (uint32_t)(e * a.n_kv));
    int lo = 0, hi = a.n_seqs;                // last sequence whose items begin at or before e (those without items share a start)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= e) lo = mid;
      else hi = mid;
    }
    it.seq = lo;
    it.sq = load_seq(a, lo);
    const int n_splits = splits_of(a, it.sq), local = e - prefix[lo];
    it.chunk = local / n_splits;
    it.split = local - it.chunk * n_splits;
    const int len = split_blocks(a, it.sq) * KV_BLOCK;
    it.tok0 = it.split * len;
    int end = min(it.sq.kv_len, it.tok0 + len);
    if (a.tree == nullptr) end = min(end, it.sq.kv_len - it.sq.q_len + min((it.chunk + 1) * ROWS - 1, it.sq.q_len * G - 1) / G + 1);
    it.n_tok = max(end - it.tok0, 0);
    return it;
  };
  // a warp's blocks of an item: warp, warp + R8_WARPS, ...
  auto blocks_of = [&](const RowsItem& it) { return (it.n_blk() - warp + R8_WARPS - 1) / R8_WARPS; };
  auto page_of = [&](const RowsItem& it, int jb) {   // the pages of its blocks jb .. jb + 31, one a lane
    const int b = (jb + lane) * R8_WARPS + warp;
    return b < it.n_blk() ? a.block_table[(size_t)it.sq.block_row * a.bt_stride + it.tok0 / KV_BLOCK + b] : 0;
  };
  uint32_t f = blockIdx.x;
  if (f >= n_flat) return;
  // ---- issue cursor: RING blocks ahead of the consumer; the item after its own is decoded when it enters its own
  uint32_t i_f = f;
  RowsItem i_it = item_at(f), i_nxt = i_it;
  int i_pages = page_of(i_it, 0), i_pages_nxt = 0, i_jb = 0, i_st = 0;
  auto ahead = [&]() {
    if (i_f + n_slots < n_flat) {
      i_nxt = item_at(i_f + n_slots);
      i_pages_nxt = page_of(i_nxt, 0);
    }
  };
  ahead();
  bool alive = true;                          // no wait has run out; after one the warp goes on without copies, for the others wait for it
  auto issue = [&]() {
    while (i_f < n_flat && i_jb >= blocks_of(i_it)) {
      i_f += n_slots;
      if (i_f >= n_flat) return;
      i_it = i_nxt;
      i_pages = i_pages_nxt;
      i_jb = 0;
      ahead();
    }
    if (i_f >= n_flat || !alive) return;
    const int page = __shfl_sync(0xffffffffu, i_pages, i_jb & 31);
    if (lane == 0) {
      const bool ok = page >= 0 && page < a.n_pages;
      page_ok[i_st] = ok;
      if (ok) {
        mbar_arrive_expect_tx(&full[i_st], KV8_PAGE);
        bulk_load_1d(ring + i_st * KV8_PAGE, a.pages + ((size_t)page * a.n_kv + i_it.kvh) * KV8_PAGE, KV8_PAGE, &full[i_st]);
      } else {
        mbar_arrive(&full[i_st]);
        if (a.status != nullptr) atomicOr(a.status, TGIS_KV8_BAD_PAGE);
      }
    }
    i_st = i_st == R8_RING - 1 ? 0 : i_st + 1;
    if ((++i_jb & 31) == 0 && i_jb < blocks_of(i_it)) i_pages = page_of(i_it, i_jb);
  };
  for (int i = 0; i < R8_RING; ++i) issue();

  const int g = lane >> 2, t4 = lane & 3, mi = lane >> 3, ri = lane & 7;
  const uint32_t ring_base = smem_u32(ring);
  int c_st = 0;
  uint32_t c_ph = 0;
  for (; f < n_flat; f += n_slots) {
    const RowsItem it = item_at(f);
    const int n_rows = it.sq.q_len * G, prefix_len = it.sq.kv_len - it.sq.q_len;
    // ---- Q^T as B fragments: this thread has row g of each tile, of sixteen dims 4 t4 .. 4 t4 + 3
    uint32_t qb[NT][HEAD_DIM / 16][2];
    float q_mul[NT][2], m_r[NT][2], l_r[NT][2], r_r[NT][2], o[NT][HEAD_DIM / 16][4];   // of rows 2 t4, 2 t4 + 1
    int lim[NT][2];                           // causal: last token seen
    unsigned long long word[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int rr = it.chunk * ROWS + n * 8 + g, i = rr / G;
      const __nv_bfloat16* src = a.q + (size_t)(it.sq.q_start + i) * a.ldq + (size_t)(it.kvh * G + rr - i * G) * HEAD_DIM + 4 * t4;
      uint2 w[HEAD_DIM / 16];
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < HEAD_DIM / 16; ++c) {
        w[c] = rr < n_rows ? *reinterpret_cast<const uint2*>(src + c * 16) : make_uint2(0, 0);
        top = max(max(top, max(w[c].x << 16 & 0x7fff0000u, w[c].x & 0x7fff0000u)), max(w[c].y << 16 & 0x7fff0000u, w[c].y & 0x7fff0000u));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^e that brings the largest number to [2^14, 2^15); a row that is not finite: NaN, which its scores and sums then are
      const float up = power_up(top), mul = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : a.scale * 1.4426950408889634f * one_over(up);
#pragma unroll
      for (int c = 0; c < HEAD_DIM / 16; ++c) {
        qb[n][c][0] = f16x2(__uint_as_float(w[c].x << 16) * up, __uint_as_float(w[c].x & 0xffff0000u) * up);
        qb[n][c][1] = f16x2(__uint_as_float(w[c].y << 16) * up, __uint_as_float(w[c].y & 0xffff0000u) * up);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r2 = it.chunk * ROWS + n * 8 + 2 * t4 + e, i2 = r2 / G;
        q_mul[n][e] = __shfl_sync(0xffffffffu, mul, 4 * (2 * t4 + e));
        lim[n][e] = prefix_len + i2;
        word[n][e] = a.tree != nullptr && r2 < n_rows ? a.tree[it.sq.q_start + i2] : 0;
        m_r[n][e] = -INFINITY;
        l_r[n][e] = 0.f;
        r_r[n][e] = R8_LEAST;
      }
#pragma unroll
      for (int md = 0; md < HEAD_DIM / 16; ++md) o[n][md][0] = o[n][md][1] = o[n][md][2] = o[n][md][3] = 0.f;
    }
    // every row of the chunk sees the tokens below this one
    const int seen_by_all = prefix_len + (a.tree == nullptr ? it.chunk * ROWS / G + 1 : 0);
    const int n_blk = blocks_of(it);
    for (int jb = 0; jb < n_blk; ++jb) {
      alive = alive && warp_wait(&full[c_st], c_ph);
      const bool ok = alive && page_ok[c_st] != 0;
      if (ok) {
        const uint32_t k_base = ring_base + c_st * KV8_PAGE, v_base = k_base + KV8_CODES;
        const float* k_scale = reinterpret_cast<const float*>(ring + c_st * KV8_PAGE + KV8_K_SCALES) + g;
        const float* v_scale = k_scale + KV_BLOCK;
        const int tok_b = it.tok0 + (jb * R8_WARPS + warp) * KV_BLOCK;
        const bool open = tok_b + KV_BLOCK > min(seen_by_all, it.sq.kv_len);   // some row may not see some token
        // ---- S^T = K Q^T: 2 tiles of 16 tokens x 8 steps of 16 dims.  A register of codes is dims 4 t4 .. 4 t4 + 3 of a chunk: the step's
        // k places 2 t4, 2 t4 + 1 and 2 t4 + 8, 2 t4 + 9, in Q^T as in K
        float s[NT][2][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int cp = 0; cp < HEAD_DIM / 32; ++cp) {
            uint32_t k[4];                    // (tokens 0 .. 7, 8 .. 15 of the tile) x (chunk 2 cp, 2 cp + 1)
            ldsm_x4(k, k_base + (16 * mt + (mi & 1) * 8 + ri) * HEAD_DIM + (((2 * cp + (mi >> 1)) ^ ri) << 4));
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint32_t a0 = e4m3x2_to_f16x2(k[2 * c]), a1 = e4m3x2_to_f16x2(k[2 * c + 1]), a2 = e4m3x2_to_f16x2(k[2 * c] >> 16),
                             a3 = e4m3x2_to_f16x2(k[2 * c + 1] >> 16);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                if (cp + c == 0) mma_f16_first(s[n][mt], a0, a1, a2, a3, qb[n][0][0], qb[n][0][1]);
                else mma_f16(s[n][mt], a0, a1, a2, a3, qb[n][2 * cp + c][0], qb[n][2 * cp + c][1]);
              }
            }
          }
        // ---- softmax: this thread has tokens g + 8 i of its rows, score (i, e) in s[n][i / 2][2 (i % 2) + e]
        float top[NT][2];
        uint32_t hid = 0;
        bool grows = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float ks = k_scale[8 * i];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) s[n][i >> 1][2 * (i & 1) + e] *= min_nan(ks * q_mul[n][e], 0x1.fffffep127f);   // (0 * inf: a zero is one)
        }
        if (open) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int tok = tok_b + 8 * i + g, node = tok - prefix_len;
                const bool sees = tok < it.sq.kv_len && (a.tree == nullptr ? tok <= lim[n][e] : node < 0 || (word[n][e] >> node & 1) != 0);
                if (!sees) {
                  s[n][i >> 1][2 * (i & 1) + e] = -INFINITY;
                  hid |= 1u << (n * 8 + 2 * i + e);
                }
              }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = max3(fmaxf(s[n][0][e], s[n][0][2 + e]), s[n][1][e], s[n][1][2 + e]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            top[n][e] = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            grows |= top[n][e] > m_r[n][e] + R8_SLACK;
          }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const bool up = top[n][e] > m_r[n][e] + R8_SLACK;
              const float corr = up ? ex2(m_r[n][e] - top[n][e]) : 1.f;
              if (up) m_r[n][e] = top[n][e];
              l_r[n][e] *= corr;
              // (the weights so far shrink, and r with them: a power of two at or above)
              const float now = r_r[n][e] * corr, to = fmaxf(power_above(__float_as_uint(now)), R8_LEAST), f = now * one_over(to);
              r_r[n][e] = to;
#pragma unroll
              for (int md = 0; md < HEAD_DIM / 16; ++md) o[n][md][e] *= f, o[n][md][2 + e] *= f;
            }
        }
        // ---- weights: probabilities times their values' scales, none where the row does not see the token (whose scale may be NaN)
        float most[NT][2];
        bool more = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float ref = m_r[n][e] == -INFINITY ? 0.f : m_r[n][e];   // (no score above -inf: every probability is 0, not the NaN of inf - inf)
            most[n][e] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float& x = s[n][i >> 1][2 * (i & 1) + e];
              x = ex2(x - ref);
              l_r[n][e] += x;
              x *= v_scale[8 * i];
              if (open && (hid >> (n * 8 + 2 * i + e) & 1)) x = 0.f;
              most[n][e] = fmaxf(most[n][e], x);
            }
            more |= most[n][e] > r_r[n][e] * R8_ROOM;
          }
        if (__any_sync(0xffffffffu, more)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = fmaxf(most[n][e], __shfl_xor_sync(0xffffffffu, most[n][e], 4));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
              const float to = x > r_r[n][e] * R8_ROOM ? fminf(power_above(__float_as_uint(x)), 0x1p126f) : r_r[n][e], f = r_r[n][e] * one_over(to);
              r_r[n][e] = to;
#pragma unroll
              for (int md = 0; md < HEAD_DIM / 16; ++md) o[n][md][e] *= f, o[n][md][2 + e] *= f;
            }
        }
        uint32_t p[NT][4];                    // weights^T as B fragments: tokens 8 i + 2 t4, 2 t4 + 1 of row g
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float h0 = R8_HELD * one_over(r_r[n][0]), h1 = R8_HELD * one_over(r_r[n][1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) p[n][i] = movmatrix_trans(f16x2(s[n][i >> 1][2 * (i & 1)] * h0, s[n][i >> 1][2 * (i & 1) + 1] * h1));
        }
        // ---- O^T += V^T P^T: 8 tiles of 16 dims x 2 steps of 16 tokens; a register of codes is tokens 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9 of a dim
#pragma unroll
        for (int md = 0; md < HEAD_DIM / 16; ++md) {
          uint32_t v[4];                      // (dims 0 .. 7, 8 .. 15 of the tile) x (tokens 0 .. 15, 16 .. 31)
          ldsm_x4(v, v_base + (mi >> 1) * (KV8_CODES / 2) + (16 * md + (mi & 1) * 8 + ri) * 16);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t a0 = e4m3x2_to_f16x2(v[2 * h]), a1 = e4m3x2_to_f16x2(v[2 * h + 1]), a2 = e4m3x2_to_f16x2(v[2 * h] >> 16),
                           a3 = e4m3x2_to_f16x2(v[2 * h + 1] >> 16);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(o[n][md], a0, a1, a2, a3, p[n][2 * h], p[n][2 * h + 1]);
          }
        }
      }
      __syncwarp();
      issue();
      if (++c_st == R8_RING) c_st = 0, c_ph ^= 1;
    }
    // ---- the item's rows: the warps' sums joined, each warp then having two of the eight tiles of dims.  In step k a warp hands the warp
    // k places on what that one has to have
    const int n_splits = splits_of(a, it.sq);
    float m_all[NT][2], by[NT][2], l_all[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = l_r[n][e];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (g == 0) stat_s[warp][n * 8 + 2 * t4 + e] = make_float2(m_r[n][e], l);
      }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float2 ml[R8_WARPS];
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < R8_WARPS; ++w) {
          ml[w] = stat_s[w][n * 8 + 2 * t4 + e];
          m = fmaxf(m, ml[w].x);
        }
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int w = 0; w < R8_WARPS; ++w) l += ml[w].y * ex2(ml[w].x - ref);
        m_all[n][e] = m;
        l_all[n][e] = l;
        by[n][e] = ex2(m_r[n][e] - ref) * (r_r[n][e] * (1.f / R8_HELD));
      }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int md = 0; md < HEAD_DIM / 16; ++md)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][md][i] *= by[n][i & 1];
    static_assert(R8_WARPS == 4 && HEAD_DIM == 128, "a warp's share is two tiles of dims");
    float mine[NT][2][4];
    auto tiles_of = [&](int w, auto&& f2) {   // (registers are not indexed by variables)
#pragma unroll
      for (int c = 0; c < R8_WARPS; ++c)
        if (w == c) f2(c);
    };
    tiles_of(warp, [&](int c) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 8; ++x) mine[n][x >> 2][x & 3] = o[n][2 * c + (x >> 2)][x & 3];
    });
#pragma unroll
    for (int k = 1; k < R8_WARPS; ++k) {
      const int to = (warp + k) % R8_WARPS;
      tiles_of(to, [&](int c) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x) hand_s[c][n][x][lane] = make_float4(o[n][2 * c + x][0], o[n][2 * c + x][1], o[n][2 * c + x][2], o[n][2 * c + x][3]);
      });
      __syncthreads();
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float4 v = hand_s[warp][n][x][lane];
          mine[n][x][0] += v.x; mine[n][x][1] += v.y; mine[n][x][2] += v.z; mine[n][x][3] += v.w;
        }
      __syncthreads();
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int rr = it.chunk * ROWS + n * 8 + 2 * t4 + e, i = rr / G, row = it.sq.q_start + i, head = it.kvh * G + rr - i * G;
        if (rr >= n_rows) continue;
        if (n_splits == 1) {
          const float inv = l_all[n][e] == 0.f ? 0.f : 1.f / l_all[n][e];
          __nv_bfloat16* dst = a.out + (size_t)row * a.ldo + (size_t)head * HEAD_DIM + warp * 32 + g;
#pragma unroll
          for (int x = 0; x < 4; ++x) dst[x * 8] = __float2bfloat16_rn(mine[n][x >> 1][2 * (x & 1) + e] * inv);
        } else {
          const size_t at = (((size_t)it.seq * a.rows_of_seq + i) * a.n_q + head) * a.max_splits + it.split;
          float* dst = a.part_o + at * HEAD_DIM + warp * 32 + g;
#pragma unroll
          for (int x = 0; x < 4; ++x) dst[x * 8] = mine[n][x >> 1][2 * (x & 1) + e];
          if (g == 0 && warp == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m_all[n][e], l_all[n][e]);
        }
      }
  }
  if (!alive) {
    // a copy never landed: say so; those in flight are done long before this millisecond is over
    if (lane == 0) say_stalled(a);
    for (const long long t0 = clock64(); clock64() - t0 < 2000000ll;) {}
  }
}

// Splits of a row joined, PARTS warps a (query, head): each joins a stretch of them in their order, then the first joins the stretches
constexpr int M8_WARPS = 8;
template <int PARTS>
__global__ void __launch_bounds__(M8_WARPS * 32) attn8_merge_kernel(const __grid_constant__ RowsArgs a) {
  __shared__ float4 part_x[PARTS > 1 ? M8_WARPS : 1][32];
  __shared__ float2 part_ml[PARTS > 1 ? M8_WARPS : 1];
  griddep_launch();
  griddep_wait();
  const AttnSeq sq = load_seq(a, blockIdx.x);
  if (!seq_picked(a, sq) || !seq_fits(a, sq)) return;
  const int lane = (int)lane_id(), warp = threadIdx.x >> 5, n_splits = splits_of(a, sq);
  if (n_splits <= 1) return;
  const int n_rows = sq.q_len * a.n_q, step = gridDim.y * (M8_WARPS / PARTS);
  for (int base = blockIdx.y * (M8_WARPS / PARTS); base < n_rows; base += step) {
    const int i = base + warp / PARTS, part = warp % PARTS, per = (n_splits + PARTS - 1) / PARTS, s0 = part * per, s1 = min(s0 + per, n_splits);
    const int t = sq.q_start + i / a.n_q, head = i % a.n_q;
    float m = -INFINITY, l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < n_rows && s0 < s1) {
      const size_t at = (((size_t)blockIdx.x * a.rows_of_seq + i / a.n_q) * a.n_q + head) * a.max_splits;
      for (int s = s0 + lane; s < s1; s += 32) m = fmaxf(m, a.part_ml[(at + s) * 2]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll 8
      for (int s = s0; s < s1; ++s) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (at + s) * 2);
        const float4 v = reinterpret_cast<const float4*>(a.part_o + (at + s) * HEAD_DIM)[lane];
        const float f = ex2(ml.x - ref);
        l += ml.y * f;
        x.x += v.x * f; x.y += v.y * f; x.z += v.z * f; x.w += v.w * f;
      }
    }
    if constexpr (PARTS > 1) {
      part_x[warp][lane] = x;
      if (lane == 0) part_ml[warp] = make_float2(m, l);
      __syncthreads();
      if (part == 0) {
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < PARTS; ++k) top = fmaxf(top, part_ml[warp + k].x);
        const float ref = top == -INFINITY ? 0.f : top;
        l = 0.f;
        x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < PARTS; ++k) {
          const float2 ml = part_ml[warp + k];
          const float4 v = part_x[warp + k][lane];
          const float f = ex2(ml.x - ref);
          l += ml.y * f;
          x.x += v.x * f; x.y += v.y * f; x.z += v.z * f; x.w += v.w * f;
        }
      }
      __syncthreads();
      if (part != 0) continue;
    }
    if (i >= n_rows) continue;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(a.out + (size_t)t * a.ldo + (size_t)head * HEAD_DIM + lane * 4) = make_uint2(cvt2(x.x * inv, x.y * inv), cvt2(x.z * inv, x.w * inv));
  }
}

// Partial sums of a (query, head) and split; what those of a call take at most, which is what attention8_prompt.cu takes (43 MB, which stay in the L2):
// splits that would need more are fewer.  Microseconds with all of them and with those that fit, 32 / 8 heads: 256 x 8 queries behind 8100
// (4 and 1) 1408 and 1157, behind 4000 (2 and 1) 716 and 619; 64 x 12 behind 8100 (4 and 3) 540 and 515; 256 x 12 (4 and 1) 2115 and 1706.
constexpr size_t R8_PART = (HEAD_DIM + 2) * sizeof(float);
size_t parts_room() { return attn8_prompt_workspace(ATTN8_MAX_SMS); }

struct RowsPlan {
  int rows, split, max_splits;
  bool wide, prompt;                          // more than this kernel is for; attention8_prompt.cu takes them
};
RowsPlan rows_plan(int T, int n_seqs, int n_q, int n_kv, int max_q, int max_kv) {
  RowsPlan p{};
  const int rows = (int)std::min<long long>((long long)max_q * (n_q / n_kv), 1 << 30);
  p.rows = rows > 8 ? 16 : 8;
  // (a B200's SMs, whatever the device has: a workspace's size is asked for without one)
  const double items = (double)std::max(n_seqs, 1) * n_kv * ((rows + p.rows - 1) / p.rows), slots = 148. * R8_CTAS(p.rows);
  p.wide = rows > R8_MOST_ROWS && (items > slots || max_kv > R8_MORE_KEYS);
  p.prompt = p.wide && attn8_prompt_takes(T, n_seqs, n_q, n_kv, max_q, max_kv);
  // Splits (the bounds are those of the longest sequence): one for few tokens, which the second launch costs more than it saves; else as
  // many as run at once, of 256 to 4096 tokens; else one for 2048 tokens or three rounds of them, of 1024 to 2048.  Microseconds, 32 / 8 heads,
  // one single token behind 600: one split 8.5, of 256 tokens 8.3; 1024: 11.1 and 9.1; 12 behind 2048: four (all at once) 15.1, eight 18.2, one
  // 21.6; 12 behind 8192: four 43.4, eight 43.7, sixteen 51.4; 32 behind 4096: one 51.3, two 65.4, four 64.7; 64 behind 4096 (more than
  // run at once): one 115, three rounds of them 117, of 1024 tokens 123, of 2048 108, of 256 151; 64 behind 2048: one 63, two 65.
  auto length = [&](double n) { return (int)std::ceil(max_kv / std::max(n, 1.) / 128.) * 128; };
  const int at_once = std::max(length(std::floor(slots / items)), 256);
  p.split = max_kv <= R8_ONE_SPLIT ? R8_ONE_SPLIT : items <= slots && at_once <= 4096 ? at_once : max_kv <= 2048 ? 2048 : std::min(std::max(length(std::ceil(3. * slots / items)), 1024), 2048);
  const double room = std::max(1., std::floor((double)parts_room() / ((double)std::max(n_seqs, 1) * std::max(max_q, 1) * n_q * R8_PART)));
  if ((max_kv + p.split - 1) / p.split > room) p.split = length(room);
  p.max_splits = std::max(1, (max_kv + p.split - 1) / p.split);
  return p;
}

template <int ROWS>
cudaError_t rows_launch(const RowsArgs& a, int num_sms, cudaStream_t stream) {
  const int smem = R8_WARPS * R8_RING * KV8_PAGE + a.n_seqs * 4;
  static OncePerDevice once;
  cudaError_t e = once([] {
    return cudaFuncSetAttribute(attn8_rows_kernel<ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, R8_WARPS * R8_RING * KV8_PAGE + TGIS_KV8_MAX_SEQS * 4);
  });
  if (e != cudaSuccess) return e;
  const long long rows = (long long)a.max_q * (a.n_q / a.n_kv);
  const long long most = (long long)a.n_seqs * a.n_kv * a.max_splits * ((rows + ROWS - 1) / ROWS);
  if (most >= 1ll << 31) return cudaErrorInvalidValue;
  const int grid = (int)std::max<long long>(1, std::min<long long>((long long)R8_CTAS(ROWS) * num_sms, most));
  return launch_k(attn8_rows_kernel<ROWS>, dim3(grid), dim3(R8_THREADS), smem, stream, a);
}

}  // namespace

// No fewer bytes for more sequences, more of their queries or longer ones: whoever keeps one workspace asks for the largest of each.  Splits are at
// most one for 256 tokens, and at most three rounds of items and two more, or one for 2048 tokens (rows_plan); a round has 296 items of 16 rows or
// 444 of 8, so that splits times rows of all sequences are 3 * 4736 and two of each row at most.
size_t attn8_workspace(int T, int n_seqs, int n_q, int n_kv, int max_q, int max_kv) {
  const RowsPlan p = rows_plan(T, n_seqs, n_q, n_kv, max_q, max_kv);
  if (p.wide) return parts_room();
  const double rows = (double)n_seqs * n_q * max_q;
  if (max_kv <= R8_ONE_SPLIT) return 0;
  const double parts = std::min(rows * (max_kv / 256. + 1.), std::max(3. * 4736. + 2. * rows, rows * (max_kv / 2048. + 1.)));
  return std::min((size_t)std::ceil(parts) * R8_PART, parts_room());
}

cudaError_t attn8_launch(const Attn8Args& args, void* workspace, int num_sms, cudaStream_t stream, int* launches, bool prompts) {
  if (args.n_seqs <= 0 || args.T <= 0) return cudaSuccess;
  num_sms = std::min(num_sms, ATTN8_MAX_SMS);
  const RowsPlan p = rows_plan(args.T, args.n_seqs, args.n_q, args.n_kv, args.max_q, args.max_kv);
  if (launches != nullptr) *launches = 2;
  if (p.prompt || prompts) return attn8_prompt_launch(args, workspace, num_sms, stream);
  RowsArgs a;
  static_cast<Attn8Args&>(a) = args;
  a.split = p.split;
  a.max_splits = p.max_splits;
  a.rows_of_seq = a.max_q;
  a.part_o = reinterpret_cast<float*>(workspace);
  a.part_ml = a.part_o + (size_t)a.n_seqs * a.max_q * a.n_q * a.max_splits * HEAD_DIM;
  cudaError_t e = p.rows == 8 ? rows_launch<8>(a, num_sms, stream) : rows_launch<16>(a, num_sms, stream);
  if (launches != nullptr && p.max_splits == 1) *launches = 1;
  if (e != cudaSuccess || p.max_splits == 1) return e;
  // a warp a row joins four splits as fast as eight warps do (32 tokens behind 4096: 64 us both); eight splits: 69 and 62, 32 of one token behind
  // 8192: 18 and 12
  const bool wide = p.max_splits > 4;
  const int per_cta = wide ? 1 : M8_WARPS, y = (int)std::min<long long>(((long long)args.max_q * args.n_q + per_cta - 1) / per_cta, 1024);
  return wide ? launch_k(attn8_merge_kernel<M8_WARPS>, dim3(a.n_seqs, y), dim3(M8_WARPS * 32), 0, stream, a)
              : launch_k(attn8_merge_kernel<1>, dim3(a.n_seqs, y), dim3(M8_WARPS * 32), 0, stream, a);
}

}  // namespace tgis

// ------------------------------------------------------------------------------------------------------------------- C ABI
namespace {
thread_local char t_err[256];
int fail(const char* form, ...) {
  va_list v;
  va_start(v, form);
  vsnprintf(t_err, sizeof(t_err), form, v);
  va_end(v);
  return -1;
}
int done(cudaError_t e, const char* what) { return e == cudaSuccess ? 0 : fail("%s: %s", what, cudaGetErrorString(e)); }
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
constexpr int MAX_HEADS = 1024, MAX_PAGES = (1 << 26) - 1, MAX_TOKENS = 1 << 26;

// what every call says of the cache
int check_cache(const void* pages, int32_t n_pages, int32_t n_kv) {
  if (pages == nullptr || !aligned(pages, 16)) return fail("pages: a 16-byte aligned pointer is wanted");
  if (n_pages < 1 || n_pages > MAX_PAGES) return fail("n_pages %d is not in 1 .. %d", n_pages, MAX_PAGES);
  if (n_kv < 1 || n_kv > MAX_HEADS) return fail("n_kv %d is not in 1 .. %d", n_kv, MAX_HEADS);
  return 0;
}
// rows of `heads` heads, read and written 16 bytes at a time
int check_rows(const char* name, const void* p, int64_t ld, int64_t heads) {
  if (p == nullptr || !aligned(p, 16)) return fail("%s: a 16-byte aligned pointer is wanted", name);
  if (ld < heads * tgis::HEAD_DIM || ld % 8 != 0) return fail("%s: rows of %lld numbers, a multiple of 8 and no fewer than %lld, are wanted", name, (long long)ld, (long long)heads * tgis::HEAD_DIM);
  return 0;
}
int check_group(int32_t n_q, int32_t n_kv) {
  return n_q < 1 || n_q > MAX_HEADS || n_q % n_kv != 0 ? fail("n_q %d is not a multiple of n_kv %d in 1 .. %d", n_q, n_kv, MAX_HEADS) : 0;
}
int sms_of_device(int* out) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev);
  return done(e, "device");
}
}  // namespace

extern "C" {

const char* tgis_kv8_last_error(void) { return t_err; }

int tgis_kv8_write(void* pages, int32_t n_pages, int32_t n_kv, const void* qkv, int64_t ld, int32_t T, int32_t n_q, const int32_t* positions,
                   const int32_t* slots, const void* cos_sin, int32_t n_positions, void* q_out, int64_t ldq, int32_t* status, void* stream) {
  if (check_cache(pages, n_pages, n_kv) != 0) return -1;
  if (n_q < 0 || n_q > MAX_HEADS) return fail("n_q %d is not in 0 .. %d", n_q, MAX_HEADS);
  if (T < 0 || T > MAX_TOKENS) return fail("T %d is not in 0 .. %d", T, MAX_TOKENS);
  if (T == 0) return 0;
  if (check_rows("qkv", qkv, ld, (int64_t)n_q + 2 * n_kv) != 0) return -1;
  if (q_out != nullptr && n_q > 0 && check_rows("q_out", q_out, ldq, n_q) != 0) return -1;
  if (T > 1 && q_out == qkv && q_out != nullptr && ldq != ld) return fail("queries rotated in place keep their rows: ldq %lld, ld %lld", (long long)ldq, (long long)ld);
  if (positions == nullptr || slots == nullptr || !aligned(positions, 4) || !aligned(slots, 4)) return fail("positions, slots: int32 pointers are wanted");
  if (cos_sin == nullptr || !aligned(cos_sin, 16) || n_positions < 1) return fail("cos_sin: a 16-byte aligned table of at least one position is wanted");
  return done(tgis::kv8_write_launch((uint8_t*)pages, n_pages, n_kv, (const __nv_bfloat16*)qkv, ld, T, n_q, positions, slots, (const __nv_bfloat16*)cos_sin,
                                     n_positions, n_q > 0 ? (__nv_bfloat16*)q_out : nullptr, ldq, status, (cudaStream_t)stream),
              "tgis_kv8_write");
}

int tgis_kv8_read(const void* pages, int32_t n_pages, int32_t n_kv, const int32_t* slots, int32_t T, void* k_out, int64_t ldk, void* v_out,
                  int64_t ldv, int32_t* status, void* stream) {
  if (check_cache(pages, n_pages, n_kv) != 0) return -1;
  if (T < 0 || T > MAX_TOKENS) return fail("T %d is not in 0 .. %d", T, MAX_TOKENS);
  if (T == 0) return 0;
  if (slots == nullptr || !aligned(slots, 4)) return fail("slots: an int32 pointer is wanted");
  if (k_out != nullptr && check_rows("k_out", k_out, ldk, n_kv) != 0) return -1;
  if (v_out != nullptr && check_rows("v_out", v_out, ldv, n_kv) != 0) return -1;
  return done(tgis::kv8_read_launch((const uint8_t*)pages, n_pages, n_kv, slots, T, (__nv_bfloat16*)k_out, ldk, (__nv_bfloat16*)v_out, ldv, status,
                                    (cudaStream_t)stream),
              "tgis_kv8_read");
}

int64_t tgis_kv8_attention_workspace(int32_t T, int32_t n_seqs, int32_t n_q, int32_t n_kv, int32_t max_q, int32_t max_kv) {
  if (n_kv < 1 || n_kv > MAX_HEADS) return fail("n_kv %d is not in 1 .. %d", n_kv, MAX_HEADS);
  if (check_group(n_q, n_kv) != 0) return -1;
  if (T < 0 || T > MAX_TOKENS || n_seqs < 0 || n_seqs > TGIS_KV8_MAX_SEQS || max_q < 0 || max_kv < 0 || max_q > MAX_TOKENS || max_kv > MAX_TOKENS)
    return fail("T %d, n_seqs %d, max_q %d, max_kv %d: one is out of range", T, n_seqs, max_q, max_kv);
  return (int64_t)tgis::attn8_workspace(T, n_seqs, n_q, n_kv, max_q, max_kv);
}

int tgis_kv8_attention(const void* pages, int32_t n_pages, int32_t n_kv, const void* q, int64_t ldq, int32_t T, int32_t n_q, const int32_t* seqs,
                       int32_t n_seqs, const int32_t* block_table, int32_t bt_rows, int32_t bt_stride, const uint64_t* tree, float scale,
                       int32_t max_q, int32_t max_kv, void* out, int64_t ldo, void* workspace, int64_t workspace_bytes, int32_t* status,
                       void* stream) {
  if (check_cache(pages, n_pages, n_kv) != 0 || check_group(n_q, n_kv) != 0) return -1;
  const int64_t need = tgis_kv8_attention_workspace(T, n_seqs, n_q, n_kv, max_q, max_kv);
  if (need < 0) return -1;
  if (T == 0 || n_seqs == 0 || max_q == 0) return 0;
  if (check_rows("q", q, ldq, n_q) != 0 || check_rows("out", out, ldo, n_q) != 0) return -1;
  if (seqs == nullptr || !aligned(seqs, 16)) return fail("seqs: a 16-byte aligned pointer is wanted");
  if (block_table == nullptr || !aligned(block_table, 4) || bt_rows < 1 || bt_stride < 1) return fail("block_table: at least one row of one page is wanted");
  if (tree != nullptr && (!aligned(tree, 8) || max_q > TGIS_KV8_MAX_TREE)) return fail("tree: 8-byte aligned words and max_q of at most %d are wanted", TGIS_KV8_MAX_TREE);
  if (!(scale - scale == 0.f)) return fail("scale is not finite");
  if (need > 0 && (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < need))
    return fail("workspace: %lld bytes, 16-byte aligned, are wanted", (long long)need);
  int sms = 0;
  if (sms_of_device(&sms) != 0) return -1;
  const tgis::Attn8Args a{(const uint8_t*)pages, n_pages, n_kv, (const __nv_bfloat16*)q, ldq, T, n_q, (const tgis::AttnSeq*)seqs, n_seqs, block_table,
                          bt_rows, bt_stride, tree, scale, max_q, max_kv, (__nv_bfloat16*)out, ldo, status};
  return done(tgis::attn8_launch(a, workspace, sms, (cudaStream_t)stream), "tgis_kv8_attention");
}

}  // extern "C"
