// Attention over the 8-bit paged cache (include/tgis_kv8.h; layout and number format: cache8.cuh): single tokens, drafted trees and
// short portions on the warps' own tensor cores.
//
// Both products run on e4m3 operands as the cache holds them; what is not in 8 bits is written as two e4m3 numbers, x = hi + lo / 16
// with hi = e4m3(x), lo = e4m3(16 (x - hi)).  A query row (bf16: 8 significant bits) times a power of two that brings its largest
// number to [128, 256) is held exactly that way but for numbers 2^-14 of the largest and below, which lose less than 2^-22 of it.
// Probabilities times the scales of their value rows (w = p s) are brought to the same range block by block and row by row, so that
// they keep 8 bits (as bf16 would) and lose no more than 2^-22 of the largest w of their 32 tokens, whatever weight a token elsewhere
// has; a block's products start at zero and join the row's sums in fp32.  The 16 rows of mma.m16n8k32 are thus 8 rows of queries
// twice: hi in rows 0..7, lo in rows 8..15, and a thread that holds (row, row + 8) of an accumulator adds the two parts itself.
// Measured on a B200: mma.m16n8k32 e4m3 3860 multiply-adds a clock and SM (bf16 1020), sums exact to 23 bits.
//
// Work item = (sequence, 8 MT rows, kv head, split of the keys); row = token * G + head of the group.  Every warp walks its own items
// alone, its blocks of 32 tokens (one bulk copy each) requested RING blocks ahead across items; sequence lengths and pages are read
// on the device, so the list of items is made by every CTA for itself: a prefix sum over the sequences.
#include <algorithm>
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
constexpr int R8_CTAS(int mt) { return mt == 1 ? 3 : 2; }   // per SM

struct RowsArgs : Attn8Args {
  float *part_o, *part_ml;
  int max_splits, split;                      // split: tokens (a multiple of KV_BLOCK)
};

__device__ __forceinline__ void mma_e4m3(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// C = A B
__device__ __forceinline__ void mma_e4m3_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
struct RowsItem {
  AttnSeq sq;
  int kvh, chunk, split, tok0, n_tok;         // keys tok0 .. tok0 + n_tok - 1 of the sequence (of the split, and seen by a row of the chunk)
  __device__ int n_blk() const { return (n_tok + KV_BLOCK - 1) / KV_BLOCK; }
};

template <int MT>
__global__ void __launch_bounds__(R8_THREADS, R8_CTAS(MT)) attn8_rows_kernel(const __grid_constant__ RowsArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full_s[R8_WARPS * R8_RING];
  __shared__ int32_t ok_s[R8_WARPS * R8_RING], wsum[R8_WARPS];
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
  auto chunks_of = [&](const AttnSeq& s) { return (s.q_len * G + 8 * MT - 1) / (8 * MT); };
  auto splits_of = [&](const AttnSeq& s) { return (s.kv_len + a.split - 1) / a.split; };
  int carry = 0;
  for (int base = 0; base < a.n_seqs; base += R8_THREADS) {
    const int s = base + threadIdx.x;
    int n = 0;
    if (s < a.n_seqs) {
      const AttnSeq sq = load_seq(a, s);
      if (seq_fits(a, sq)) n = chunks_of(sq) * splits_of(sq);
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
  const uint32_t n_flat = (uint32_t)carry * a.n_kv, n_slots = gridDim.x * R8_WARPS;   // (host: no more than 2^31)
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
    it.sq = load_seq(a, lo);
    const int n_splits = splits_of(it.sq), local = e - prefix[lo];
    it.chunk = local / n_splits;
    it.split = local - it.chunk * n_splits;
    it.tok0 = it.split * a.split;
    int end = min(it.sq.kv_len, it.tok0 + a.split);
    if (a.tree == nullptr) end = min(end, it.sq.kv_len - it.sq.q_len + min((it.chunk + 1) * 8 * MT - 1, it.sq.q_len * G - 1) / G + 1);
    it.n_tok = max(end - it.tok0, 0);
    return it;
  };
  auto page_of = [&](const RowsItem& it, int jb) {   // this lane's page of blocks jb .. jb + 31
    const int b = jb + lane;
    return b < it.n_blk() ? a.block_table[(size_t)it.sq.block_row * a.bt_stride + it.tok0 / KV_BLOCK + b] : 0;
  };
  uint32_t f = warp * gridDim.x + blockIdx.x;   // consecutive items land on different SMs
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
  auto issue = [&]() {
    while (i_f < n_flat && i_jb >= i_it.n_blk()) {
      i_f += n_slots;
      if (i_f >= n_flat) return;
      i_it = i_nxt;
      i_pages = i_pages_nxt;
      i_jb = 0;
      ahead();
    }
    if (i_f >= n_flat) return;
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
    if ((++i_jb & 31) == 0 && i_jb < i_it.n_blk()) i_pages = page_of(i_it, i_jb);
  };
  for (int i = 0; i < R8_RING; ++i) issue();

  const int g = lane >> 2, t4 = lane & 3, mi = lane >> 3, ri = lane & 7;
  const uint32_t ring_base = smem_u32(ring);
  int c_st = 0;
  uint32_t c_ph = 0;
  bool alive = true;
  for (; alive && f < n_flat; f += n_slots) {
    const RowsItem it = item_at(f);
    const int n_rows = it.sq.q_len * G, prefix_len = it.sq.kv_len - it.sq.q_len;
    // ---- this thread's rows: fragments, scale into the exp2 domain, what they see
    uint32_t qa[MT][4][4];
    float q_mul[MT], m_r[MT], l_r[MT];
    uint64_t o[MT][16];                       // two dims each
    int row_q[MT], head[MT], lim[MT];         // lim: causal, last token seen
    unsigned long long word[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int rr = it.chunk * 8 * MT + mt * 8 + g, i = rr / G;
      row_q[mt] = rr < n_rows ? it.sq.q_start + i : -1;
      head[mt] = it.kvh * G + rr - i * G;
      lim[mt] = prefix_len + i;
      word[mt] = 0;
      if (a.tree != nullptr && row_q[mt] >= 0) word[mt] = a.tree[row_q[mt]];
      uint32_t w[4][4];                       // k-step, (dims 4 t4 .. of its first 16, of its second 16): two words each
      uint32_t top = 0;
      const __nv_bfloat16* src = a.q + (size_t)max(row_q[mt], 0) * a.ldq + (size_t)head[mt] * HEAD_DIM + 4 * t4;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint2 v = row_q[mt] >= 0 ? *reinterpret_cast<const uint2*>(src + ks * 32 + h * 16) : make_uint2(0, 0);
          w[ks][2 * h] = v.x;
          w[ks][2 * h + 1] = v.y;
          top = max(max(top, max(v.x << 16 & 0x7fff0000u, v.x & 0x7fff0000u)), max(v.y << 16 & 0x7fff0000u, v.y & 0x7fff0000u));
        }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^e that brings the largest number to [128, 256); a row that is not finite: NaN, which its scores and sums then are
      const float up = power_up(top);
      q_mul[mt] = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : a.scale * 1.4426950408889634f / up;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t x = w[ks][2 * h], y = w[ks][2 * h + 1];
          split4(__uint_as_float(x << 16) * up, __uint_as_float(x & 0xffff0000u) * up, __uint_as_float(y << 16) * up, __uint_as_float(y & 0xffff0000u) * up,
                 qa[mt][ks][2 * h], qa[mt][ks][2 * h + 1]);
        }
      m_r[mt] = -INFINITY;
      l_r[mt] = 0.f;
#pragma unroll
      for (int n = 0; n < 16; ++n) o[mt][n] = 0;
    }
    // every row of the chunk sees the tokens below this one
    const int seen_by_all = prefix_len + (a.tree == nullptr ? it.chunk * 8 * MT / G + 1 : 0);
    const int n_blk = it.n_blk();
    for (int jb = 0; jb < n_blk; ++jb) {
      if (!bounded_wait(&full[c_st], c_ph)) {
        alive = false;
        break;
      }
      const bool ok = page_ok[c_st] != 0;
      if (ok) {
        const uint32_t k_base = ring_base + c_st * KV8_PAGE, v_base = k_base + KV8_CODES;
        const float* k_scale = reinterpret_cast<const float*>(ring + c_st * KV8_PAGE + KV8_K_SCALES);
        const float* v_scale = k_scale + KV_BLOCK;
        const int tok_b = it.tok0 + jb * KV_BLOCK;
        const bool open = tok_b + KV_BLOCK > min(seen_by_all, it.sq.kv_len);   // some row may not see some token
        // ---- S = Q K^T: 4 tiles of 8 tokens x 4 steps of 32 dims
        float s[MT][4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int kp = 0; kp < 2; ++kp) {
            uint32_t kb[4];
            ldsm_x4(kb, k_base + (8 * j + ri) * HEAD_DIM + (((4 * kp + mi) ^ ri) << 4));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              if (kp == 0) mma_e4m3_first(s[mt][j], qa[mt][0], kb[0], kb[1]);
              else mma_e4m3(s[mt][j], qa[mt][2 * kp], kb[0], kb[1]);
              mma_e4m3(s[mt][j], qa[mt][2 * kp + 1], kb[2], kb[3]);
            }
          }
        // ---- softmax: this thread has tokens 8 j + 2 t4 + e of its rows
        uint32_t pa[MT][4];
        uint64_t keep2[MT], add_hi[MT], add_lo[MT];   // what the row's sums are multiplied by, and this block's products
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float x[4][2], top = -INFINITY;
          uint32_t hid = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 ks = *reinterpret_cast<const float2*>(k_scale + 8 * j + 2 * t4);
            x[j][0] = (s[mt][j][0] + s[mt][j][2] * (1.f / KV8_LO)) * (ks.x * q_mul[mt]);
            x[j][1] = (s[mt][j][1] + s[mt][j][3] * (1.f / KV8_LO)) * (ks.y * q_mul[mt]);
          }
          if (open) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int tok = tok_b + 8 * j + 2 * t4 + e, node = tok - prefix_len;
                const bool sees = tok < it.sq.kv_len && (a.tree == nullptr ? tok <= lim[mt] : node < 0 || (word[mt] >> node & 1) != 0);
                if (!sees) {
                  x[j][e] = -INFINITY;
                  hid |= 1u << (2 * j + e);
                }
              }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) top = fmaxf(top, fmaxf(x[j][0], x[j][1]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float m_new = fmaxf(m_r[mt], top);
          const float here = top == -INFINITY ? 0.f : top;   // (no score above -inf: every probability is 0, not the NaN of inf - inf)
          const float part = top == -INFINITY ? 0.f : ex2(top - m_new);
          const float keep = m_r[mt] == -INFINITY ? 0.f : ex2(m_r[mt] - m_new);
          keep2[mt] = pack2(keep, keep);
          m_r[mt] = m_new;
          float sum = 0.f, most = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 vs = *reinterpret_cast<const float2*>(v_scale + 8 * j + 2 * t4);
            x[j][0] = ex2(x[j][0] - here);
            x[j][1] = ex2(x[j][1] - here);
            sum += x[j][0] + x[j][1];
            x[j][0] *= vs.x;
            x[j][1] *= vs.y;
          }
          if (open) {                         // (a hidden row's scale may be NaN)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (hid >> (2 * j + e) & 1) x[j][e] = 0.f;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) most = fmaxf(most, fmaxf(x[j][0], x[j][1]));
          l_r[mt] = l_r[mt] * keep + sum * (sum == 0.f ? 0.f : part);
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
          const float up = power_up(__float_as_uint(most));
          const float add = part * one_over(up);
          add_hi[mt] = pack2(add, add);
          add_lo[mt] = pack2(add * (1.f / KV8_LO), add * (1.f / KV8_LO));
          split4(x[0][0] * up, x[0][1] * up, x[1][0] * up, x[1][1] * up, pa[mt][0], pa[mt][1]);
          split4(x[2][0] * up, x[2][1] * up, x[3][0] * up, x[3][1] * up, pa[mt][2], pa[mt][3]);
        }
        // ---- O += P V: 16 tiles of 8 dims, all 32 tokens in one step
#pragma unroll
        for (int n = 0; n < 16; n += 2) {
          uint32_t vb[4];
          ldsm_x4(vb, v_base + (mi & 1) * (KV8_CODES / 2) + (8 * (n + (mi >> 1)) + ri) * 16);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float c[4];
              mma_e4m3_first(c, pa[mt], vb[2 * h], vb[2 * h + 1]);
              o[mt][n + h] = fma2(pack2(c[2], c[3]), add_lo[mt], fma2(pack2(c[0], c[1]), add_hi[mt], mul2(o[mt][n + h], keep2[mt])));
            }
        }
      }
      __syncwarp();
      issue();
      if (++c_st == R8_RING) c_st = 0, c_ph ^= 1;
    }
    if (!alive) break;
    // ---- the item's rows
    const int n_splits = splits_of(it.sq);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float l = l_r[mt];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (row_q[mt] < 0) continue;
      if (n_splits == 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + (size_t)row_q[mt] * a.ldo + (size_t)head[mt] * HEAD_DIM) + t4;
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          float x, y;
          unpack2(o[mt][n], x, y);
          dst[n * 4] = cvt2(x * inv, y * inv);
        }
      } else {
        const size_t at = ((size_t)row_q[mt] * a.n_q + head[mt]) * a.max_splits + it.split;
        float2* dst = reinterpret_cast<float2*>(a.part_o + at * HEAD_DIM) + t4;
#pragma unroll
        for (int n = 0; n < 16; ++n)
          reinterpret_cast<uint64_t*>(dst)[n * 4] = o[mt][n];
        if (t4 == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m_r[mt], l);
      }
    }
  }
  if (!alive) {
    // a copy never landed: say so; those in flight are done long before this millisecond is over
    if (lane == 0 && a.status != nullptr) atomicOr(a.status, TGIS_KV8_STALLED);
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
  if (!seq_fits(a, sq)) return;
  const int lane = (int)lane_id(), warp = threadIdx.x >> 5, n_splits = (sq.kv_len + a.split - 1) / a.split;
  if (n_splits <= 1) return;
  const int n_rows = sq.q_len * a.n_q, step = gridDim.y * (M8_WARPS / PARTS);
  for (int base = blockIdx.y * (M8_WARPS / PARTS); base < n_rows; base += step) {
    const int i = base + warp / PARTS, part = warp % PARTS, per = (n_splits + PARTS - 1) / PARTS, s0 = part * per, s1 = min(s0 + per, n_splits);
    const int t = sq.q_start + i / a.n_q, head = i % a.n_q;
    float m = -INFINITY, l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < n_rows && s0 < s1) {
      const size_t at = ((size_t)t * a.n_q + head) * a.max_splits;
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

struct RowsPlan {
  int mt, split, max_splits, most_splits;     // most_splits: no call with the same rows and fewer keys has more
  bool prompt;                                // attention8_prompt.cu
};
RowsPlan rows_plan(int T, int n_seqs, int n_q, int n_kv, int max_q, int max_kv) {
  RowsPlan p{};
  const int rows = (int)std::min<long long>((long long)max_q * (n_q / n_kv), 1 << 30);
  p.prompt = rows > 16 && attn8_prompt_takes(T, n_seqs, n_q, n_kv, max_q, max_kv);
  p.mt = rows > 8 ? 2 : 1;
  // Splits: the shortest with which all items run at once; where they do not, the longest that leaves three rounds of them
  const double items = (double)std::max(n_seqs, 1) * n_kv * ((rows + 8 * p.mt - 1) / (8 * p.mt)), slots = 148. * R8_CTAS(p.mt) * R8_WARPS;
  auto rounds = [&](int split) { return items * ((max_kv + split - 1) / split) / slots; };
  p.split = 64;
  while (p.split < 512 && rounds(p.split) > 1.) p.split *= 2;
  if (rounds(p.split) > 1.)
    while (p.split > 128 && rounds(p.split) < 3.) p.split /= 2;
  if (rows > 16) p.split = 512;               // (many rows and few columns that attention8_prompt.cu does not take)
  p.max_splits = std::max(1, (max_kv + p.split - 1) / p.split);
  // (splits of 64 and more for one round; 128 and more where twice as long ones leave less than three)
  p.most_splits = std::max(p.max_splits, (int)std::min((max_kv + 63) / 64 + 0., 6. * slots / items + 2.));
  return p;
}

template <int MT>
cudaError_t rows_launch(const RowsArgs& a, int num_sms, cudaStream_t stream) {
  const int smem = R8_WARPS * R8_RING * KV8_PAGE + a.n_seqs * 4;
  static OncePerDevice once;
  cudaError_t e = once([] {
    return cudaFuncSetAttribute(attn8_rows_kernel<MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, R8_WARPS * R8_RING * KV8_PAGE + TGIS_KV8_MAX_SEQS * 4);
  });
  if (e != cudaSuccess) return e;
  const long long rows = (long long)a.max_q * (a.n_q / a.n_kv);
  const long long most = (long long)a.n_seqs * a.n_kv * a.max_splits * ((rows + 8 * MT - 1) / (8 * MT));
  if (most >= 1ll << 31) return cudaErrorInvalidValue;
  const int grid = (int)std::max<long long>(1, std::min<long long>((long long)R8_CTAS(MT) * num_sms, (most + R8_WARPS - 1) / R8_WARPS));
  return launch_k(attn8_rows_kernel<MT>, dim3(grid), dim3(R8_THREADS), smem, stream, a);
}

}  // namespace

size_t attn8_workspace(int T, int n_seqs, int n_q, int n_kv, int max_q, int max_kv) {
  const RowsPlan p = rows_plan(T, n_seqs, n_q, n_kv, max_q, max_kv);
  if (p.prompt) return attn8_prompt_workspace(ATTN8_MAX_SMS);
  return p.most_splits > 1 ? (size_t)T * n_q * p.most_splits * (HEAD_DIM + 2) * sizeof(float) : 0;
}

cudaError_t attn8_launch(const Attn8Args& args, void* workspace, int num_sms, cudaStream_t stream, int* launches) {
  if (args.n_seqs <= 0 || args.T <= 0) return cudaSuccess;
  num_sms = std::min(num_sms, ATTN8_MAX_SMS);
  const RowsPlan p = rows_plan(args.T, args.n_seqs, args.n_q, args.n_kv, args.max_q, args.max_kv);
  if (launches != nullptr) *launches = 2;
  if (p.prompt) return attn8_prompt_launch(args, workspace, num_sms, stream);
  RowsArgs a;
  static_cast<Attn8Args&>(a) = args;
  a.split = p.split;
  a.max_splits = p.max_splits;
  a.part_o = reinterpret_cast<float*>(workspace);
  a.part_ml = a.part_o + (size_t)a.T * a.n_q * a.max_splits * HEAD_DIM;
  cudaError_t e = p.mt == 1 ? rows_launch<1>(a, num_sms, stream) : rows_launch<2>(a, num_sms, stream);
  if (launches != nullptr && p.max_splits == 1) *launches = 1;
  if (e != cudaSuccess || p.max_splits == 1) return e;
  const int per_cta = p.max_splits > 16 ? 1 : M8_WARPS, y = (int)std::min<long long>(((long long)args.max_q * args.n_q + per_cta - 1) / per_cta, 1024);
  return p.max_splits > 16 ? launch_k(attn8_merge_kernel<M8_WARPS>, dim3(a.n_seqs, y), dim3(M8_WARPS * 32), 0, stream, a)
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
  if (q_out == qkv && q_out != nullptr && ldq != ld) return fail("queries rotated in place keep their rows: ldq %lld, ld %lld", (long long)ldq, (long long)ld);
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
