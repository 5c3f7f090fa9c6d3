// Attention over the 8-bit paged cache (include/tgis_kv8.h; layout and number format: cache8.cuh) of prompts, their portions and wide
// drafted trees, on tcgen05.
//
// A unit is up to 2 TM query tokens of one sequence and one kv head (row = token * G + head of the group, TM = 128 / G), half of them in each
// of two accumulators, or all in one that holds them (whose step is shorter: 16 drafts of 5 to 24 behind 200 to 1500, 34 us; halved, 39); a
// step is one tile of 128 keys of a unit.  All steps of the call lie in one row, sequence after sequence,
// and every CTA takes an equal stretch of them: a stretch that begins or ends inside a unit leaves that unit's sums (o, m, l) in
// the workspace, and attn8_join_kernel joins them in order.  So a long prompt, many short ones and a few drafts over long contexts
// all keep every SM busy to the end, and the workspace is two units a CTA whatever the lengths are.  Lengths and pages are read on
// the device.
//
// Both products are f16 x f16 -> fp32 (kind::f16).  Four warps widen K and V as they multiply them by their rows' scales (a code has 4 bits,
// so a product rounded to f16's 11 is off by 2^-11; a key's scale is applied as two f16 numbers, for an error of the whole row's
// would be one of its score); both are held relative to a power of two at or above the tile's scales.  A query row is exact in f16 but for
// numbers 2^-31 of its largest and below.  A weight (a probability times the tile's unit of V) is one f16 number of 11 bits, held times 2^7;
// a row has one reference of its exponentials and one of its weights, which move only when something passes them by 2^8, so that it
// fits f16 (2^15 at most) and nothing above 2^-31 of the row's largest is lost.  A tile whose scales lie further apart than 2^12 has no unit
// that serves a row which sees its small ones alone: its codes stay as they are, exact, and the softmax multiplies scores and probabilities by
// the scales, in fp32 and in steps.  So what a row does not see, or gives no weight, never costs it its own tokens' bits.
// (With K as the cache holds it and queries as two e4m3 numbers on kind::f8f6f4 the products cost the same and every score takes a
// multiplication by its key's scale, every probability one by its value's: as first built both took 380 us for 1859 tokens behind 6144, 32 / 8
// heads, and each later step, to 263, needed the multiplications gone.)
// Two threads share a row, half of a step's columns each; tokens of a page lie in V's columns as cache8.cuh says, so P's columns are
// written in that order.  A row with a NaN for its scale gets zeros here and a bit; who sees it gets NaN for its sum.
//
// What bounds it: the chain of a step.  Of its 4900 clocks an accumulator spends 3100 in the softmax (scores read 600, the two threads'
// maximum 300, exponentials 2000, 1024 of them the least that 16 a clock take) and 1700 in its two products, which wait for those of
// the other one; the two take turns.  Without the exponentials a step is 4500, without the widening 4550: nothing alone is the bound.  (References of
// weights, which came after that, are 150 more.)
// 1859 tokens behind 6144: 274 us, 788 TFLOP/s of the 1660 that a product of matrices reaches (the 16-bit cache's kernel: 345 us);
// prompt of 2048: 76 (61); six prompts of 90 to 593 (1679 tokens): 39 (2048 tokens in six: 30); 4 drafts of 64 behind 4000 to 8000, 64 / 8 heads: 82.
// A unit's beginning and end take as much as three and a half steps (Q copied and turned, the first pages, O): what short prompts consist of.
//
// No wait is unbounded: after about two seconds a role gives up, the call's status says so; copies and MMAs in flight land first and TMEM is
// freed on every path.
#include <algorithm>

#include "cache8.cuh"
#include "launch.cuh"
#include "ptx.cuh"
#include "tc_attention.cuh"

namespace tgis {
namespace {

constexpr int P8_THREADS = 768;                             // warps 0..7, 8..15: softmax of an accumulator; 16 walks and copies, 17 MMAs, 20..23 widen K and V
constexpr int P8_WARP_COPY = 16, P8_WARP_MMA = 17, P8_WARP_WIDEN = 20, P8_WIDEN = 4;
constexpr int P8_REGS_SOFTMAX = 88, P8_REGS_OTHER = 64;     // 512 x 88 + 256 x 64 = 768 x 80, what the launch gives every thread
constexpr int P8_KV = 128, P8_BLOCKS = P8_KV / KV_BLOCK;    // keys of a step
constexpr int P8_NOTES = 4;
constexpr int P8_TILE = P8_KV * HEAD_DIM * 2;               // bytes of a tile of K or V, of one accumulator's Q, in f16
constexpr float P8_SLACK = 8.f;                             // exp2 domain: how far a score may exceed its row's reference
constexpr float P8_HELD = 7.f, P8_HELD_TIMES = 128.f;       // exp2 domain: weights and sums are held times 2^7
constexpr float P8_LEAST = -118.f;                          // exp2 domain: smallest unit of weights
constexpr float P8_V_TOP = 64.f, P8_K_TOP = 16.f;           // largest scale that a code (448 at most) is multiplied by
constexpr int P8_V_TOP_LOG = 6;
// A tile's scales lie within this of its largest (the power of two above it), or its codes stay without them: what is held relative to
// one unit would lose the small rows' bits, and a row may see those alone.  At 2^-12 of it a key's scale as two f16 numbers is off by 2^-17 (their last
// step is 2^-24 of 16), a value's by 2^-11 like any other.  (The smallest scale of all, that of rows of zeros, does not count.)
constexpr float P8_BAND = 0x1p-12f;
// What the beginning and the end of a unit count for, in steps.  As 1, 2, 3: 2048 tokens 85, 75, 72 us; six prompts of 90 to 593 38.8, 38.6, 40.4;
// 16 drafts of 5 to 24 behind 200 to 1500 36, 33.5, 35
constexpr uint32_t P8_COST = 2;

// What the softmax has to know of a tile, beside its scores
struct TileNotes {
  uint32_t poison[P8_BLOCKS];  // tokens whose key or value row is not a number
  uint32_t special;            // bits 0..3: blocks whose page does not exist; bit 4: there are poisoned tokens; bit 5: codes without their scales
  float k_unit, v_log;         // what a number of K is in units of; log2 of what one of V is
  uint32_t pad;
};
constexpr uint32_t P8_ODD = 1u << P8_BLOCKS, P8_WIDE = 2u << P8_BLOCKS;
// Steps [tile0, tile1) of a unit: the copying warp walks the row of steps, the others take from its list
struct Task {
  int tile0, tile1;            // tile1 0: no more
  int keys, kv_len, before;    // that some row of the unit sees; of the sequence; ahead of its queries
  int first, tokens, half;     // of the unit: first token (of the sequence's queries), tokens, those of the first accumulator
  int row0, kvh, cut;          // row of the first token; bits: 1 begins behind the unit's first step, 2 ends ahead of its last
  uint32_t word_mask_lo, word_mask_hi;   // nodes of the draft
  uint32_t pad[3];
  __device__ bool two() const { return tokens > half; }
  __device__ int blocks(int j) const { return min(P8_BLOCKS, (keys + KV_BLOCK - 1) / KV_BLOCK - j * P8_BLOCKS); }
};
constexpr int P8_TASKS = 4;
struct P8Smem {
  // K-major operands under the 128-byte swizzle, p8_at
  // (two of K: a tile of it is widened while the scores of the one before wait for their probabilities)
  uint8_t q[2][P8_TILE], k[2][P8_TILE], v[P8_TILE];
  uint8_t raw_k[P8_BLOCKS][KV8_CODES], raw_v[P8_BLOCKS][KV8_CODES];   // as they come from the cache
  float scales[P8_BLOCKS][2 * KV_BLOCK];   // a block's keys', then its values'
  // scales of value rows as f16 multipliers at their places, of even and odd tiles, a copy for every warp that uses them
  __align__(16) uint16_t v_mul[P8_WIDEN][2][P8_KV];
  TileNotes notes[P8_NOTES];   // tile t's: t % P8_NOTES
  float row_scales[P8_NOTES][2][P8_KV];    // of keys, of values, where a tile's codes are without them
  Task task[P8_TASKS];
  float pair[2][2][2][128];    // what the two threads of a row tell one another: of even and odd times, accumulator, half, row
  uint64_t task_full[P8_TASKS], task_empty[P8_TASKS], raw_k_full, raw_k_empty, raw_v_full, raw_v_empty, q_full[2], note_full[P8_NOTES], pair_full[2][4],
      k_full[2], k_empty[2], v_full, v_empty, s_full[2], p_full[2], o_full[2];
  uint32_t absent;  // by the copying warp
  uint32_t tmem_base;
  int gave_up;
  uint32_t prefix[1];          // steps ahead of each sequence
};
static_assert(offsetof(P8Smem, raw_k) % 1024 == 0 && offsetof(P8Smem, scales) % 128 == 0 && offsetof(P8Smem, notes) % 16 == 0 && offsetof(P8Smem, task_full) % 8 == 0, "");

// eight numbers (16 bytes) of a row: [2 halves of 64 numbers][128 rows][8 groups, group g at place g ^ (row & 7)]
__device__ __forceinline__ int p8_at(int row, int group) { return (group >> 3) * (P8_TILE / 2) + row * 128 + (((group & 7) ^ (row & 7)) << 4); }

// What a CTA leaves of a unit that begins in its stretch and ends behind it
struct CutUnit {
  int row0, kvh, tokens, half, parts;   // parts 0: there is none; else its CTAs, this one the first
  int pad[3];
};
struct PromptArgs : Attn8Args {
  int G, TM;
  uint32_t per_g;              // row / G = row * per_g >> 16 for rows below 128
  float *frag_o, *frag_ml;     // [CTA][0: of a unit begun before it, 1: of one that ends behind it][256 rows]([128])
  CutUnit* cut;                // [CTA]
};

// ---- the row of steps
struct SeqUnits {
  AttnSeq sq;
  int n_units, tokens;         // of a unit (the last one may have fewer)
};
__device__ __forceinline__ SeqUnits units_of(const PromptArgs& a, int s) {
  SeqUnits u;
  u.sq = load_seq(a, s);
  if (!seq_picked(a, u.sq) || !seq_fits(a, u.sq)) u.sq.q_len = 0;
  u.n_units = (u.sq.q_len + 2 * a.TM - 1) / (2 * a.TM);
  u.tokens = u.n_units > 0 ? (u.sq.q_len + u.n_units - 1) / u.n_units : 0;
  return u;
}
// keys that some row of unit i sees
__device__ __forceinline__ int keys_of(const PromptArgs& a, const SeqUnits& u, int i) {
  return a.tree != nullptr ? u.sq.kv_len : u.sq.kv_len - u.sq.q_len + min((i + 1) * u.tokens, u.sq.q_len);
}
__device__ __forceinline__ int steps_of(const PromptArgs& a, const SeqUnits& u, int i) { return (keys_of(a, u, i) + P8_KV - 1) / P8_KV; }

// steps of all sequences ahead of each, by one warp; their sum
__device__ __forceinline__ uint32_t lay_out(const PromptArgs& a, uint32_t* prefix) {
  const int lane = (int)lane_id();
  uint32_t carry = 0;
  for (int base = 0; base < a.n_seqs; base += 32) {
    const int s = base + lane;
    uint32_t n = 0;
    if (s < a.n_seqs) {
      const SeqUnits u = units_of(a, s);
      for (int i = 0; i < u.n_units; ++i) n += P8_COST + (uint32_t)steps_of(a, u, i);
      n *= (uint32_t)a.n_kv;
      if (u.n_units == 0 && blockIdx.x == 0 && a.status != nullptr && seq_picked(a, load_seq(a, s)) && !seq_fits(a, load_seq(a, s))) atomicOr(a.status, TGIS_KV8_BAD_SEQ);
    }
    uint32_t sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (s < a.n_seqs) prefix[s] = carry + sum - n;
    carry += __shfl_sync(0xffffffffu, sum, 31);
  }
  __syncwarp();
  return carry;
}
__device__ __forceinline__ uint32_t stretch_begin(uint32_t total, uint32_t cta, uint32_t n) { return (uint32_t)((uint64_t)total * cta / n); }

__device__ __forceinline__ uint32_t cta_of(uint32_t total, uint32_t at, uint32_t n) { return (uint32_t)((((uint64_t)at + 1) * n - 1) / total); }

// One unit's steps [tile0, tile1) of a CTA's stretch after the other.  A unit's first P8_COST places in the row of steps stand for what its
// beginning and end take: nothing is done there.
struct Walk {
  const PromptArgs& a;
  const uint32_t* prefix;
  uint32_t at, end;
  int s = -1, i = 0, kvh = 0, steps = 0, tile0 = 0, tile1 = 0;
  SeqUnits u;
  __device__ Walk(const PromptArgs& a_, const uint32_t* p, uint32_t begin, uint32_t end_) : a(a_), prefix(p), at(begin), end(end_) {}
  __device__ uint32_t find() {     // the unit that place `at` belongs to; `at` less its first place
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= at) lo = mid;
      else hi = mid;
    }
    s = lo;
    u = units_of(a, s);
    uint32_t left = at - prefix[s];
    for (i = 0;; ++i) {
      steps = steps_of(a, u, i);
      const uint32_t all = (steps + P8_COST) * a.n_kv;
      if (left < all || i >= u.n_units - 1) break;
      left -= all;
    }
    // (the bounds hold unless sequences name rows twice, so many that the counts overflow: then results are wrong, and nothing else)
    kvh = min((int)(left / (steps + P8_COST)), a.n_kv - 1);
    return min(left - kvh * (steps + P8_COST), steps + P8_COST - 1);
  }
  __device__ bool next() {
    do {
      if (at >= end) return false;
      uint32_t place = 0;
      if (s < 0) {
        place = find();
      } else if (++kvh == a.n_kv) {   // the stretch goes on: the unit before ended
        kvh = 0;
        if (++i == u.n_units) {
          do {
            if (++s >= a.n_seqs) return false;
            u = units_of(a, s);
          } while (u.n_units == 0);
          i = 0;
        }
        steps = steps_of(a, u, i);
      }
      const uint32_t stop = min(steps + P8_COST, place + (end - at));
      at += stop - place;
      tile0 = place > P8_COST ? (int)(place - P8_COST) : 0;
      tile1 = stop > P8_COST ? (int)(stop - P8_COST) : 0;
    } while (tile1 <= tile0);
    return true;
  }
  __device__ int keys() const { return keys_of(a, u, i); }
  __device__ int tokens() const { return min(u.tokens, u.sq.q_len - i * u.tokens); }
  __device__ int half() const { return tokens() <= a.TM ? tokens() : (tokens() + 1) / 2; }   // tokens of the first accumulator; the second has the others
  __device__ int blocks(int j) const { return min(P8_BLOCKS, (keys() + KV_BLOCK - 1) / KV_BLOCK - j * P8_BLOCKS); }
};

// C fp32, A and B f16, K-major
__device__ __forceinline__ constexpr uint32_t idesc_of(uint32_t m, uint32_t n) { return 1u << 4 | (n >> 3) << 17 | (m >> 4) << 24; }
__device__ __forceinline__ uint32_t hmul2(uint32_t x, uint32_t y) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t x, uint32_t y, uint32_t z) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(y), "r"(z));
  return r;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// ---- a thread's scores in steps, 16 at a time, for tiles that need it.  Calls: in line they took 8 % of all other tiles' time, called 3 %
// (a unit that is no normal number would make scores of nothing 0 * -inf where they are hidden, or 0 * inf: NaN; scores of 2^35 units at most are
// nothing beside 2^-126 of them.  A NaN fails both comparisons and stays)
__device__ __forceinline__ float p8_normal(float x) { return x < 0x1p-126f ? 0x1p-126f : x > 0x1.fffffep127f ? 0x1.fffffep127f : x; }
// scores 16 c .. 16 c + 15, -inf where hidden; ks: scales of their keys, NULL: `times` has them
__device__ __forceinline__ void p8_scores(float (&x)[16], uint32_t s_t, int c, uint32_t vis0, uint32_t vis1, float times, const float* ks) {
  uint32_t s[16];
  tmem_ld_32x32b_x16(s_t + c * 16, s);
  const uint32_t seen = (c < 2 ? vis0 : vis1) >> (c & 1) * 16;
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = seen >> i & 1 ? __uint_as_float(s[i]) * (ks != nullptr ? p8_normal(times * ks[c * 16 + i]) : times) : -INFINITY;
}
__device__ __noinline__ float p8_top(uint32_t s_t, int nb, uint32_t vis0, uint32_t vis1, float times, const float* ks) {
  float top = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 2 * min(nb, 2); ++c) {
    float x[16];
    p8_scores(x, s_t, c, vis0, vis1, times, ks);
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, x[i]);
  }
  return top;
}
// the largest probability times its value's scale (vs NULL: 2^v_log)
__device__ __noinline__ float p8_most(uint32_t s_t, int nb, uint32_t vis0, uint32_t vis1, float times, const float* ks, float ref, const float* vs, float v_log) {
  float most = 0.f;
#pragma unroll 1
  for (int c = 0; c < 2 * min(nb, 2); ++c) {
    float x[16];
    p8_scores(x, s_t, c, vis0, vis1, times, ks);
#pragma unroll
    for (int i = 0; i < 16; ++i) most = fmaxf(most, ex2(x[i] - ref) * (vs != nullptr ? vs[c * 16 + i] : ex2(v_log)));
  }
  return most;
}
// weights to where the product reads them; the sum of the probabilities, times 2^7
__device__ __noinline__ float p8_weights(uint32_t s_t, int nb, uint32_t vis0, uint32_t vis1, float times, const float* ks, float ref, const float* vs, float v_log,
                                         float unit) {
  const float hold = ex2(P8_HELD - unit);
  float l = 0.f;
#pragma unroll 1
  for (int c = 0; c < 2 * min(nb, 2); ++c) {
    float x[16];
    uint32_t p[8];
    p8_scores(x, s_t, c, vis0, vis1, times, ks);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i] = ex2(x[i] - ref);
      l += x[i] * P8_HELD_TIMES;
      x[i] = x[i] * (vs != nullptr ? vs[c * 16 + i] : ex2(v_log)) * hold;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int col = 2 * (4 * (i & 1) + (i >> 1));   // as in the kernel
      p[i] = f16x2(x[col], x[col + 1]);
    }
    tmem_st_x8(s_t + c * 8, p);   // (over scores that have been read)
  }
  return l;
}

__global__ void __launch_bounds__(P8_THREADS, 1) attn8_prompt_kernel(const __grid_constant__ PromptArgs a) {
  extern __shared__ uint8_t smem_raw[];
  P8Smem& sm = *reinterpret_cast<P8Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = (int)lane_id();
  if (warp == P8_WARP_MMA) {
    if (elect_one()) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sm.q_full[i], 8);
        mbar_init(&sm.k_full[i], P8_WIDEN);
        mbar_init(&sm.k_empty[i], 1);
        mbar_init(&sm.s_full[i], 1);
        mbar_init(&sm.p_full[i], 8);
        for (int k = 0; k < 4; ++k) mbar_init(&sm.pair_full[i][k], 2);
        mbar_init(&sm.o_full[i], 1);
      }
      for (int i = 0; i < P8_NOTES; ++i) mbar_init(&sm.note_full[i], P8_WIDEN);
      for (int i = 0; i < P8_TASKS; ++i) {
        mbar_init(&sm.task_full[i], 1);
        mbar_init(&sm.task_empty[i], 16 + 1 + P8_WIDEN);
      }
      mbar_init(&sm.raw_k_full, 1);
      mbar_init(&sm.raw_k_empty, P8_WIDEN);
      mbar_init(&sm.raw_v_full, 1);
      mbar_init(&sm.raw_v_empty, P8_WIDEN);
      mbar_init(&sm.v_full, P8_WIDEN);
      mbar_init(&sm.v_empty, 1);
      sm.gave_up = 0;
      fence_barrier_init();
    }
    __syncwarp();
    tmem_alloc<512>(&sm.tmem_base);
  }
  griddep_launch();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = sm.tmem_base;   // [S0 | S1 | O0 | O1], 128 columns each
  griddep_wait();
  bool ok = true;
  int ti = 0;                                // list of tasks
  uint32_t tph = 0;
  // the next task, NULL: there is none (or a wait ran out)
  auto take = [&]() -> const Task* {
    ok = __all_sync(0xffffffffu, bounded_wait(&sm.task_full[ti], tph));
    return ok && sm.task[ti].tile1 != 0 ? &sm.task[ti] : nullptr;
  };
  auto done_with = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.task_empty[ti]);
    if (++ti == P8_TASKS) ti = 0, tph ^= 1;
  };
  if (warp >= P8_WARP_COPY) {
    set_regs<P8_REGS_OTHER, false>();
    if (warp == P8_WARP_COPY) {
      // ===================== walk, copies =====================
      const uint32_t total = lay_out(a, sm.prefix);
      const uint32_t n = min(gridDim.x, total), b = min(blockIdx.x, n);   // (no stretch of the first n is empty)
      Walk w(a, sm.prefix, n > 0 ? stretch_begin(total, b, n) : 0u, n > 0 ? stretch_begin(total, min(b + 1, n), n) : 0u);
      uint32_t k_ph = 1, v_ph = 1;   // the first time the buffers are empty
      tph = 1;
      CutUnit cut{};
      for (;;) {
        const bool more = w.next();
        ok = __all_sync(0xffffffffu, bounded_wait(&sm.task_empty[ti], tph));
        if (!ok) break;
        if (lane == 0) {
          Task& t = sm.task[ti];
          t.tile0 = w.tile0;
          t.tile1 = more ? w.tile1 : 0;
          if (more) {
            t.keys = w.keys();
            t.kv_len = w.u.sq.kv_len;
            t.before = w.u.sq.kv_len - w.u.sq.q_len;
            t.first = w.i * w.u.tokens;
            t.tokens = w.tokens();
            t.half = w.half();
            t.row0 = w.u.sq.q_start + t.first;
            t.kvh = w.kvh;
            t.cut = (w.tile0 > 0 ? 1 : 0) | (w.tile1 < w.steps ? 2 : 0);
            const unsigned long long nodes = ~0ull >> (TGIS_KV8_MAX_TREE - min(w.u.sq.q_len, TGIS_KV8_MAX_TREE));
            t.word_mask_lo = (uint32_t)nodes;
            t.word_mask_hi = (uint32_t)(nodes >> 32);
          }
          mbar_arrive(&sm.task_full[ti]);
        }
        __syncwarp();
        if (++ti == P8_TASKS) ti = 0, tph ^= 1;
        if (!more) break;
        if (w.tile0 == 0 && w.tile1 < w.steps)   // (the stretch ends here)
          cut = CutUnit{w.u.sq.q_start + w.i * w.u.tokens, w.kvh, w.tokens(), w.half(), (int)(cta_of(total, w.at + (w.steps - w.tile1) - 1, n) - b) + 1, {}};
        const int n_blk = (w.keys() + KV_BLOCK - 1) / KV_BLOCK;
        auto page_of = [&](int j) {   // lane: block lane & 3 of tile j
          const int b = j * P8_BLOCKS + (lane & 3);
          return b < n_blk ? a.block_table[(size_t)w.u.sq.block_row * a.bt_stride + b] : 0;
        };
        int page = page_of(w.tile0);
        const uint8_t* v_src = nullptr;
        int v_nb = 0;
        auto copy_v = [&]() {
          ok = __all_sync(0xffffffffu, bounded_wait(&sm.raw_v_empty, v_ph));
          if (!ok) return;
          v_ph ^= 1;
          if (lane == 0) mbar_arrive_expect_tx(&sm.raw_v_full, v_nb * KV8_CODES);
          __syncwarp();
          if (lane < v_nb) bulk_load_1d(sm.raw_v[lane], v_src, KV8_CODES, &sm.raw_v_full);
        };
        for (int j = w.tile0; j < w.tile1; ++j) {
          const int nb = w.blocks(j);
          const bool there = page >= 0 && page < a.n_pages;
          const uint32_t absent = __ballot_sync(0xffffffffu, !there && lane < nb);
          if (absent != 0 && lane == 0 && a.status != nullptr) atomicOr(a.status, TGIS_KV8_BAD_PAGE);
          // (an absent page's keys are not seen; some page's codes stand in for it, for they are numbers)
          const uint8_t* src = a.pages + ((size_t)(there ? page : 0) * a.n_kv + w.kvh) * KV8_PAGE;
          ok = __all_sync(0xffffffffu, bounded_wait(&sm.raw_k_empty, k_ph));
          if (!ok) break;
          k_ph ^= 1;
          if (lane == 0) {
            sm.absent = absent;
            mbar_arrive_expect_tx(&sm.raw_k_full, nb * (KV8_CODES + (int)sizeof(sm.scales[0])));
          }
          __syncwarp();
          if (lane < nb) {
            bulk_load_1d(sm.scales[lane], src + KV8_K_SCALES, sizeof(sm.scales[0]), &sm.raw_k_full);
            bulk_load_1d(sm.raw_k[lane], src, KV8_CODES, &sm.raw_k_full);
          }
          if (j + 1 < w.tile1) page = page_of(j + 1);
          // (K is widened a tile ahead of V, so its copy goes first)
          if (j > w.tile0) copy_v();
          if (!ok) break;
          v_src = src + KV8_CODES;
          v_nb = nb;
        }
        if (ok) copy_v();
        if (!ok) break;
      }
      if (lane == 0) a.cut[blockIdx.x] = cut;
    } else if (warp == P8_WARP_MMA) {
      // ===================== MMAs =====================
      uint32_t kt = 0, vph = 0, qph[2] = {0, 0}, pph[2] = {0, 0};   // kt: tile of the CTA whose K is next
      // descriptors of 16 numbers along k (their first field counts 16 bytes).  One thread issues an MMA each 64 clocks at best: nothing
      // but the issue stands between them
      const uint64_t q_desc = make_smem_desc_sw128(smem_u32(sm.q[0])), k_desc = make_smem_desc_sw128(smem_u32(sm.k[0])), v_desc = make_smem_desc_sw128(smem_u32(sm.v));
      auto along = [](int ks) { return (uint64_t)((ks >> 2) * (P8_TILE / 2 / 16) + (ks & 3) * 2); };
      auto scores = [&](int g, int nb) {
        const uint32_t idesc = idesc_of(128, nb * KV_BLOCK);
        const uint64_t q = q_desc + g * (P8_TILE / 16), k = k_desc + (kt & 1) * (P8_TILE / 16);
#pragma unroll
        for (int ks = 0; ks < HEAD_DIM / 16; ++ks) tc_mma_f16(tmem_base + g * 128, q + along(ks), k + along(ks), idesc, ks > 0);
        tc_commit(&sm.s_full[g]);
      };
      auto values = [&](int g, int nb, bool first) {
        const uint32_t idesc = idesc_of(128, HEAD_DIM), p = tmem_base + g * 128, o = p + 256;
#pragma unroll
        for (int ks = 0; ks < P8_KV / 16; ++ks)
          if (ks < 2 * nb) mma_ts(o, p + (ks >> 2) * 64 + (ks & 3) * 8, v_desc + along(ks), idesc, ks > 0 || !first);
      };
      while (const Task* tp = take()) {
        const int groups = tp->two() ? 2 : 1, tile0 = tp->tile0, tile1 = tp->tile1;
        const Task task = *tp;   // (its sizes)
        for (int g = 0; g < groups && ok; ++g) {
          ok = __all_sync(0xffffffffu, bounded_wait(&sm.q_full[g], qph[g]));
          qph[g] ^= 1;
        }
        ok = ok && __all_sync(0xffffffffu, bounded_wait(&sm.k_full[kt & 1], kt >> 1 & 1));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          for (int g = 0; g < groups; ++g) scores(g, task.blocks(tile0));
          tc_commit(&sm.k_empty[kt & 1]);
        }
        __syncwarp();
        ++kt;
        for (int j = tile0; j < tile1 && ok; ++j) {
          const bool more = j + 1 < tile1;
          ok = __all_sync(0xffffffffu, bounded_wait(&sm.v_full, vph));
          vph ^= 1;
          for (int g = 0; g < groups && ok; ++g) {
            ok = __all_sync(0xffffffffu, bounded_wait(&sm.p_full[g], pph[g]));
            if (!ok) break;
            pph[g] ^= 1;
            tc_fence_after();
            if (elect_one()) {
              values(g, task.blocks(j), j == tile0);
              if (g == groups - 1) tc_commit(&sm.v_empty);
              if (!more) tc_commit(&sm.o_full[g]);
            }
            __syncwarp();
            if (!more) continue;
            if (g == 0) {
              ok = __all_sync(0xffffffffu, bounded_wait(&sm.k_full[kt & 1], kt >> 1 & 1));
              if (!ok) break;
              tc_fence_after();
            }
            if (elect_one()) {
              scores(g, task.blocks(j + 1));
              if (g == groups - 1) tc_commit(&sm.k_empty[kt & 1]);
            }
            __syncwarp();
          }
          if (more) ++kt;
        }
        if (!ok) break;
        done_with();
      }
    } else if (warp >= P8_WARP_WIDEN) {
      // ===================== K, V to f16: thread = token, then dim =====================
      const int mine = warp - P8_WARP_WIDEN, part = mine * 32 + lane;
      const uint32_t swizzle = (uint32_t)(lane & 7) << 4, out_row = (uint32_t)part * 128 + swizzle;
      const uint32_t k_out0 = smem_u32(sm.k[0]) + out_row, v_out = smem_u32(sm.v) + out_row, v_mul = smem_u32(sm.v_mul[mine]);
      uint32_t kt = 0;                        // tile of the CTA whose K is next
      uint32_t v_full = 0;
      while (const Task* tp = take()) {
        const int tile0 = tp->tile0, tile1 = tp->tile1, kv_len = tp->kv_len;
        uint32_t hi = 0, lo = 0;              // this thread's key scale as two f16 numbers, each twice
        float row_k = 0.f, row_v = 0.f;       // its scales as they are
        TileNotes mem;                        // (poison[0]: of this warp's block)
        // Scales of tile j, which every warp looks at all of (lane = token of a block).  Done ahead of the waits for buffers, which
        // come once a step and all at once
        auto scales = [&](int j) {
          const int nb = tp->blocks(j);
          ok = __all_sync(0xffffffffu, bounded_wait(&sm.raw_k_full, kt & 1));
          if (!ok) return;
          const uint32_t absent = sm.absent;
          float vs[P8_BLOCKS], top_k = 0.f, top_v = 0.f, low_k = INFINITY, low_v = INFINITY;
          uint32_t any_odd = 0;
#pragma unroll
          for (int b = 0; b < P8_BLOCKS; ++b) {
            const float* sc = sm.scales[b];
            const bool there = b < nb && !(absent >> b & 1) && j * P8_KV + b * KV_BLOCK + lane < kv_len;
            float k = there ? sc[lane] : 0.f;
            vs[b] = there ? sc[KV_BLOCK + lane] : 0.f;
            const bool fine = k < INFINITY && vs[b] < INFINITY;
            if (!fine) k = vs[b] = 0.f;
            const uint32_t odd = __ballot_sync(0xffffffffu, !fine);
            any_odd |= odd;
            top_k = fmaxf(top_k, k);
            top_v = fmaxf(top_v, vs[b]);
            if (k > KV8_TINY) low_k = fminf(low_k, k);
            if (vs[b] > KV8_TINY) low_v = fminf(low_v, vs[b]);
            if (b == mine) row_k = k, row_v = vs[b], mem.poison[0] = odd;
          }
          auto above = [](float top) { return fmaxf(power_above(__reduce_max_sync(0xffffffffu, __float_as_uint(top))), 0x1p-118f); };
          auto least = [](float low) { return __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(low))); };
          const float k_top = above(top_k), v_top = above(top_v);
          const bool wide = least(low_k) < k_top * P8_BAND || least(low_v) < v_top * P8_BAND;
          const float v_to = P8_V_TOP * one_over(v_top), k = row_k * (P8_K_TOP * one_over(k_top));
          hi = wide ? f16x2(1.f, 1.f) : f16x2(k, k);
          lo = wide ? 0u : f16x2(k - f16x2_to_f32x2(hi).x, k - f16x2_to_f32x2(hi).x);
#pragma unroll
          for (int b = 0; b < P8_BLOCKS; ++b)
            sm.v_mul[mine][kt & 1][b * KV_BLOCK + (lane & 16) + v8_place(lane & 15)] = (uint16_t)f16x2(wide ? 1.f : vs[b] * v_to, 0.f);
          mem.special = absent | (any_odd != 0 ? P8_ODD : 0u) | (wide ? P8_WIDE : 0u);
          mem.k_unit = k_top * (1.f / P8_K_TOP);
          mem.v_log = wide ? 0.f : (float)((int)(__float_as_uint(v_top) >> 23) - 127 - P8_V_TOP_LOG);
        };
        // K: sixteen dims at a time -> two groups of eight numbers.  (A block that a last tile does not have is not read.)
        auto widen_k = [&](int j) {
          ok = __all_sync(0xffffffffu, bounded_wait(&sm.k_empty[kt & 1], (kt >> 1 & 1) ^ 1));
          if (!ok) return;
          // (the scores of the tile before the last are done, so who reads the notes of the one before that has finished)
          TileNotes& t = sm.notes[kt % P8_NOTES];
          const uint32_t k_out = k_out0 + (kt & 1) * P8_TILE;
          if (lane == 0) {
            t.poison[mine] = mem.poison[0];
            if (mine == 0) t.special = mem.special, t.k_unit = mem.k_unit, t.v_log = mem.v_log;
          }
          if (mem.special & P8_WIDE) {
            sm.row_scales[kt % P8_NOTES][0][part] = row_k;
            sm.row_scales[kt % P8_NOTES][1][part] = row_v;
          }
          auto wide = [&](uint32_t two) {
            const uint32_t h = e4m3x2_to_f16x2(two);
            return hfma2(h, hi, hmul2(h, lo));
          };
          if (mine < tp->blocks(j)) {
            const uint32_t from = smem_u32(sm.raw_k[mine]) + (uint32_t)lane * HEAD_DIM + swizzle;
#pragma unroll 1
            for (int d0 = 0; d0 < HEAD_DIM / 16; d0 += 2) {
              uint4 x[2];
#pragma unroll
              for (int d = 0; d < 2; ++d) x[d] = lds128(from ^ ((d0 + d) << 4));
#pragma unroll
              for (int d = 0; d < 2; ++d) {
                const uint32_t to = (k_out ^ ((2 * (d0 + d) & 7) << 4)) + (d0 >> 2) * (P8_TILE / 2);
                sts128(to, wide(x[d].x), wide(x[d].x >> 16), wide(x[d].y), wide(x[d].y >> 16));
                sts128(to ^ 16, wide(x[d].z), wide(x[d].z >> 16), wide(x[d].w), wide(x[d].w >> 16));
              }
            }
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&sm.note_full[kt % P8_NOTES]);
            mbar_arrive(&sm.k_full[kt & 1]);
            mbar_arrive(&sm.raw_k_empty);
          }
          ++kt;
        };
        // V: sixteen tokens at a time
        auto widen_v = [&](int j, int odd) {
          ok = __all_sync(0xffffffffu, bounded_wait(&sm.raw_v_full, v_full) && bounded_wait(&sm.v_empty, v_full ^ 1));
          if (!ok) return;
          v_full ^= 1;
          const int nh = 2 * tp->blocks(j);
          const uint32_t from = smem_u32(sm.raw_v[0]) + (uint32_t)part * 16, mul = v_mul + odd * (P8_KV * 2);
#pragma unroll 1
          for (int h0 = 0; h0 < nh; h0 += 2) {
            uint4 x[2], m[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              x[h] = lds128(from + (h0 >> 1) * KV8_CODES + h * (KV8_CODES / 2));
              m[2 * h] = lds128(mul + (h0 + h) * 32);
              m[2 * h + 1] = lds128(mul + (h0 + h) * 32 + 16);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t to = (v_out ^ ((2 * (h0 + h) & 7) << 4)) + (h0 >> 2) * (P8_TILE / 2);
              sts128(to, hmul2(e4m3x2_to_f16x2(x[h].x), m[2 * h].x), hmul2(e4m3x2_to_f16x2(x[h].x >> 16), m[2 * h].y), hmul2(e4m3x2_to_f16x2(x[h].y), m[2 * h].z),
                     hmul2(e4m3x2_to_f16x2(x[h].y >> 16), m[2 * h].w));
              sts128(to ^ 16, hmul2(e4m3x2_to_f16x2(x[h].z), m[2 * h + 1].x), hmul2(e4m3x2_to_f16x2(x[h].z >> 16), m[2 * h + 1].y),
                     hmul2(e4m3x2_to_f16x2(x[h].w), m[2 * h + 1].z), hmul2(e4m3x2_to_f16x2(x[h].w >> 16), m[2 * h + 1].w));
            }
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&sm.v_full);
            mbar_arrive(&sm.raw_v_empty);
          }
        };
        scales(tile0);
        if (ok) widen_k(tile0);
        for (int j = tile0; j < tile1 && ok; ++j) {
          const int odd = (int)(kt - 1) & 1;
          if (j + 1 < tile1) {
            scales(j + 1);
            if (ok) widen_k(j + 1);
          }
          if (ok) widen_v(j, odd);
        }
        if (!ok) break;
        done_with();
      }
    }
  } else {
    // ===================== softmax: two threads a row, 64 columns (and dims) each =====================
    set_regs<P8_REGS_SOFTMAX, true>();
    const int g = warp >> 3, h = warp >> 2 & 1, quarter = warp & 3;
    const int r = quarter * 32 + lane, tok = (int)(r * a.per_g >> 16);
    const uint32_t s_t = tmem_base + g * 128 + ((uint32_t)(quarter * 32) << 16) + h * 64, o_t = s_t + 256;
    uint32_t sph = 0, oph = 0, tile = 0, met = 0;   // tile: of the CTA; met: times that the row's threads have told one another something
    // this thread's number said, the other one's heard
    auto meet = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.pair_full[g][quarter]);
      ok = __all_sync(0xffffffffu, bounded_wait(&sm.pair_full[g][quarter], met & 1));
      ++met;
    };
    auto pair_up = [&](float mine) {
      float(*to)[128] = sm.pair[met & 1][g];
      to[h][r] = mine;
      meet();
      return to[h ^ 1][r];
    };
    while (const Task* tp = take()) {
      const Task& t = *tp;
      if (g == 1 && !t.two()) {
        tile += (uint32_t)(t.tile1 - t.tile0);
        done_with();
        continue;
      }
      const int in_unit = g * t.half + tok;
      const bool mine = tok < t.half && in_unit < t.tokens;
      int lim = t.before + t.first + in_unit;               // causal: last key seen
      unsigned long long word = 0;
      if (!mine) lim = 0x7fffffff;
      else if (a.tree != nullptr) lim = t.before - 1, word = a.tree[t.row0 + in_unit] & ((unsigned long long)t.word_mask_hi << 32 | t.word_mask_lo);
      // ---- Q, every row's largest number at 2^14 to 2^15.  The half rows of this warp come as they are to the place of its part of the operand
      // (eight lanes copy 128 bytes of one); then a thread turns its own into f16 there.  (Loops, for code that runs once a unit is
      // fetched as it runs: unrolled this took six thousand clocks.)
      const int sub = lane >> 3, at = lane & 7;
      // (where a row of 32 lies is its thread's to say: numbers ahead of it in q or out, -1: there is none)
      auto row_at = [&](int64_t ld) { return mine ? (long long)(t.row0 + in_unit) * ld + (t.kvh * a.G + r - tok * a.G) * HEAD_DIM : -1ll; };
      const long long q_at = row_at(a.ldq);
      __syncwarp();                                             // the last unit's rows have been read there
#pragma unroll 1
      for (int i = 0; i < 32; i += 4) {
        const long long from = __shfl_sync(0xffffffffu, q_at, i + sub);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(sm.q[g] + p8_at(quarter * 32 + i + sub, h * 8 + at))),
                     "l"(a.q + (from < 0 ? 0 : from + h * 64 + at * 8)), "r"(from < 0 ? 0 : 16)
                     : "memory");
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
      uint32_t q_top = 0;
#pragma unroll 2
      for (int c = 0; c < 8; ++c) {
        const uint4 x = *reinterpret_cast<const uint4*>(sm.q[g] + p8_at(r, h * 8 + c));
        q_top = max(q_top, max(max(max(x.x << 16 & 0x7fff0000u, x.x & 0x7fff0000u), max(x.y << 16 & 0x7fff0000u, x.y & 0x7fff0000u)),
                               max(max(x.z << 16 & 0x7fff0000u, x.z & 0x7fff0000u), max(x.w << 16 & 0x7fff0000u, x.w & 0x7fff0000u))));
      }
      q_top = max(q_top, __float_as_uint(pair_up(__uint_as_float(q_top))));
      if (!ok) break;
      // (hidden scores are -inf before they are scaled; a row that is not finite: NaN, which its scores and sums then are)
      const float qm = q_top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fmaxf(fabsf(a.scale), 1e-30f) * 1.4426950408889634f * one_over(power_up(q_top));
      {
        const float up = a.scale < 0.f ? -power_up(q_top) : power_up(q_top);
#pragma unroll 2
        for (int c = 0; c < 8; ++c) {
          uint4* at_c = reinterpret_cast<uint4*>(sm.q[g] + p8_at(r, h * 8 + c));
          const uint4 x = *at_c;
          auto turn = [&](uint32_t w) { return f16x2(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up); };
          *at_c = make_uint4(turn(x.x), turn(x.y), turn(x.z), turn(x.w));
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full[g]);
      float m = 0.f, l = 0.f, unit = 0.f;                       // unit: log2 of what O is in units of, 2^m apart
      float most_unit = 0.f;                                    // no row's is larger
      bool large = false;                                       // some row's m is far from 0
      const int tile0 = t.tile0, tile1 = t.tile1;
      for (int j = tile0; j < tile1; ++j) {
        const int nb = t.blocks(j) - 2 * h;                 // of this thread's half
        // (in this order: with its scores there, a tile's notes are, and the next tile's in their place are not)
        ok = __all_sync(0xffffffffu, bounded_wait(&sm.s_full[g], sph) && bounded_wait(&sm.note_full[tile % P8_NOTES], tile / P8_NOTES & 1));
        if (!ok) break;
        sph ^= 1;
        tc_fence_after();
        const int at_note = tile % P8_NOTES;
        const TileNotes& sc = sm.notes[at_note];
        ++tile;
        const int seen = lim - j * P8_KV - h * 64;          // last column seen (of the keys before a draft)
        const uint32_t special = sc.special;
        const bool wide = (special & P8_WIDE) != 0, mask = __any_sync(0xffffffffu, seen < nb * KV_BLOCK - 1 || (special & ~P8_WIDE) != 0);
        uint32_t vis[2] = {0xffffffffu, 0xffffffffu};       // columns that the row sees
        if (mask) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            vis[c] = seen >= c * 32 + 31 ? 0xffffffffu : seen < c * 32 ? 0u : (2u << (seen - c * 32)) - 1u;
            if (a.tree != nullptr && mine) {
              const int d = c * 32 - (seen + 1);            // node of the block's first column
              if (d > -32 && d < 64) vis[c] |= d >= 0 ? (uint32_t)(word >> d) : (uint32_t)word << -d;
            }
            if (special >> (2 * h + c) & 1) vis[c] = 0;
            if (c < nb && (sc.poison[2 * h + c] & vis[c]) != 0) l = __uint_as_float(0x7fc00000u);
          }
        }
        auto hide = [&](uint32_t (&s)[32], uint32_t seen_of_it) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(seen_of_it >> i & 1)) s[i] = __float_as_uint(-INFINITY);
        };
        const float qk = p8_normal(qm * sc.k_unit);
        auto k_scales = [&]() { return wide ? sm.row_scales[at_note][0] + h * 64 : nullptr; };
        auto v_scales = [&]() { return wide ? sm.row_scales[at_note][1] + h * 64 : nullptr; };
        // The scores are read twice, 32 at a time: once for their maximum, once for the probabilities (all at once spill).  The loops are not
        // unrolled: the instruction cache does not hold the roles' code if they are
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (__builtin_expect(!wide, 1)) {
#pragma unroll 1
          for (int c = 0; c < min(nb, 2); ++c) {
            uint32_t s[32];
            tmem_ld_x32(s_t + c * 32, s);
            tmem_ld_wait();
            if (mask) hide(s, c == 0 ? vis[0] : vis[1]);
#pragma unroll
            for (int i = 0; i < 32; i += 2) mx[i >> 1 & 3] = max3(mx[i >> 1 & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
          }
        } else {
          mx[0] = p8_top(s_t, nb, vis[0], vis[1], qm, k_scales());
        }
        float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        top = fmaxf(top, pair_up(top));
        if (!wide) top *= qk;
        else if (!(qm < INFINITY)) top = qm;                 // (the maximum of NaN and -inf)
        if (!ok) break;
        // A row's weights, probabilities times what their values are in units of, have a reference of their own, 2^(m + unit): the row's largest one
        // may belong to another token than its largest probability.  Both move only when something passes them by 2^8
        const float v_log = sc.v_log;
        float f = 1.f;                                       // what O is multiplied by
        bool moved = false;                                  // some row's is not 1
        auto reference = [&]() { return m == -INFINITY ? 0.f : m; };   // (no score above -inf so far: every probability is 0, not the NaN of inf - inf)
        if (j == tile0) {
          m = top;
          unit = most_unit = v_log;
          large = __any_sync(0xffffffffu, fabsf(reference()) > 0x1p20f);
        } else if (__any_sync(0xffffffffu, top > m + P8_SLACK || (!wide && top - m + v_log > unit + P8_SLACK))) {
          const bool up = top > m + P8_SLACK;
          const float by = up ? m - top : 0.f;
          if (up) m = top;
          // (a row without a score above -inf so far has nothing in O, whatever its unit is)
          const float to = fmaxf(ceilf(unit + by), wide ? P8_LEAST : v_log + ceilf(top - reference()));
          l *= ex2(by);
          f = ex2(by + unit - to);
          unit = to;
          most_unit = fmaxf(most_unit, v_log + P8_SLACK);
          moved = true;
          large = __any_sync(0xffffffffu, fabsf(reference()) > 0x1p20f);
        }
        const float ref = reference();
        // One product and one addition make an exponent, and a row's sum is that of its weights, unless its scales differ, its values are so much
        // smaller than earlier ones that the sum would lose what they do, or its scores are so large that an exact product less a rounded one
        // may be far from zero: then in steps, which costs such a tile five to seven times its time (2048 tokens 381 us, not 76)
        const bool in_steps = wide || large || (most_unit - v_log > 64.f && __any_sync(0xffffffffu, unit - v_log > 64.f));
        if (__builtin_expect(in_steps, 0)) {
          float most = p8_most(s_t, nb, vis[0], vis[1], wide ? qm : qk, k_scales(), ref, v_scales(), v_log);
          most = fmaxf(most, pair_up(most));
          if (!ok) break;
          // exponent of the power of two at or above it; 2^127 has room for the largest
          float to = fminf(fmaxf((float)((int)(__float_as_uint(power_above(__float_as_uint(most))) >> 23) - 127), P8_LEAST), 127.f);
          if (j != tile0) {
            to = fmaxf(to, unit);
            f *= ex2(unit - to);
            moved = true;
          }
          unit = to;
          most_unit = INFINITY;
        }
        if (moved) {
          // the products that wrote O retired before these scores did
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(o_t + c * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st_x16(o_t + c * 16, o);
          }
        }
        uint64_t sum0 = 0, sum1 = 0;
        if (__builtin_expect(!in_steps, 1)) {
          const float add = P8_HELD + (v_log - unit) - ref;
          const uint64_t qm2 = pack2(qk, qk), neg_m = pack2(add, add);
#pragma unroll 1
          for (int c = 0; c < min(nb, 2); ++c) {
            uint32_t s[32];
            tmem_ld_x32(s_t + c * 32, s);
            tmem_ld_wait();
            if (mask) hide(s, c == 0 ? vis[0] : vis[1]);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              uint32_t p[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int col = k * 16 + 2 * (4 * (i & 1) + (i >> 1));   // places 2 i, 2 i + 1 of half a block (cache8.cuh v8_place)
                float x, y;
                unpack2(fma2(pack2(__uint_as_float(s[col]), __uint_as_float(s[col + 1])), qm2, neg_m), x, y);
                x = ex2(x);
                y = ex2(y);
                if (i & 1) sum1 = add2(sum1, pack2(x, y));
                else sum0 = add2(sum0, pack2(x, y));
                p[i] = f16x2(x, y);
              }
              tmem_st_x8(s_t + c * 16 + k * 8, p);   // (over scores that have been read)
            }
          }
        } else {
          l += p8_weights(s_t, nb, vis[0], vis[1], wide ? qm : qk, k_scales(), ref, v_scales(), v_log, unit);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[g]);
        float x, y;
        unpack2(add2(sum0, sum1), x, y);
        if (!in_steps) l += (x + y) * ex2(unit - v_log);
      }
      if (!ok) break;
      ok = __all_sync(0xffffffffu, bounded_wait(&sm.o_full[g], oph));
      if (!ok) break;
      oph ^= 1;
      tc_fence_after();
      l += pair_up(l);
      if (!ok) break;
      // the rows leave through shared memory, where this warp's part of Q was (the last scores are done): eight lanes then write 128 bytes of one
      auto put = [&](int c, uint32_t x, uint32_t y, uint32_t z, uint32_t w) { *reinterpret_cast<uint4*>(sm.q[g] + p8_at(r, h * 8 + c)) = make_uint4(x, y, z, w); };
      auto send = [&](auto&& to) {   // to(row, what its thread says of it): where its 16 bytes go, NULL: nowhere
        __syncwarp();
        const long long o_at = row_at(a.ldo);
#pragma unroll 1
        for (int i = 0; i < 32; i += 4) {
          uint4* dst = to(quarter * 32 + i + sub, __shfl_sync(0xffffffffu, o_at, i + sub));
          if (dst != nullptr) *dst = *reinterpret_cast<const uint4*>(sm.q[g] + p8_at(quarter * 32 + i + sub, h * 8 + at));
        }
        __syncwarp();
      };
      // (in two steps, for values next to fp32's largest)
      const float by = t.cut != 0 ? ex2(unit) : l == 0.f ? 0.f : ex2(unit - 8.f) / (l * 0x1p-8f);
      const size_t slot = ((size_t)blockIdx.x * 2 + ((t.cut & 1) == 0)) * 256 + g * 128;
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        uint32_t o[32];
        tmem_ld_x32(o_t + c * 32, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
        if (t.cut == 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = cvt2(__uint_as_float(o[i * 8 + 2 * k]), __uint_as_float(o[i * 8 + 2 * k + 1]));
            put(c * 4 + i, v[0], v[1], v[2], v[3]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) put(i, o[i * 4], o[i * 4 + 1], o[i * 4 + 2], o[i * 4 + 3]);
          send([&](int rr, long long o) { return o < 0 ? nullptr : reinterpret_cast<uint4*>(a.frag_o + (slot + rr) * HEAD_DIM + h * 64 + c * 32) + at; });
        }
      }
      if (t.cut == 0) send([&](int, long long o) { return o < 0 ? nullptr : reinterpret_cast<uint4*>(a.out + o + h * 64) + at; });
      else if (mine && h == 0) *reinterpret_cast<float2*>(a.frag_ml + (slot + r) * 2) = make_float2(m, l);
      tc_fence_before();
      done_with();
    }
  }
  if (!ok && lane == 0) sm.gave_up = 1;
  tc_fence_before();
  __syncthreads();
  // after a wait that ran out copies and MMAs of the other roles may be in flight; they are done long before this millisecond is over
  if (*reinterpret_cast<volatile int*>(&sm.gave_up)) {
    if (threadIdx.x == 0) say_stalled(a);
    for (const long long t0 = clock64(); clock64() - t0 < 2000000ll;) {}
  }
  __syncthreads();
  if (warp == P8_WARP_MMA) {
    tc_fence_after();
    tmem_dealloc<512>(tmem_base);
  }
}

// A unit that begins in CTA blockIdx.x's stretch and ends behind it: its parts joined in the order of the keys, a warp a row
constexpr int J8_WARPS = 8;
__global__ void __launch_bounds__(J8_WARPS * 32) attn8_join_kernel(const __grid_constant__ PromptArgs a) {
  griddep_launch();
  griddep_wait();
  const CutUnit u = a.cut[blockIdx.x];
  const int lane = (int)lane_id(), r = blockIdx.y * J8_WARPS + (threadIdx.x >> 5);
  const int tok = (r & 127) / a.G, head = (r & 127) - tok * a.G, in_unit = (r >> 7) * u.half + tok;
  if (u.parts == 0 || tok >= u.half || in_unit >= u.tokens) return;
  // part k: of CTA blockIdx.x + k; its first is that of a unit begun there
  auto slot = [&](int k) { return ((size_t)(blockIdx.x + k) * 2 + (k == 0)) * 256 + r; };
  float m = -INFINITY;
  for (int k = lane; k < u.parts; k += 32) m = fmaxf(m, a.frag_ml[slot(k) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int k = 0; k < u.parts; ++k) {
    const float2 ml = *reinterpret_cast<const float2*>(a.frag_ml + slot(k) * 2);
    const float4 v = reinterpret_cast<const float4*>(a.frag_o + slot(k) * HEAD_DIM)[lane];
    const float f = ex2(ml.x - ref);
    l += ml.y * f;
    x[0] += v.x * f; x[1] += v.y * f; x[2] += v.z * f; x[3] += v.w * f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(a.out + (size_t)(u.row0 + in_unit) * a.ldo + (size_t)(u.kvh * a.G + head) * HEAD_DIM + lane * 4) =
      make_uint2(cvt2(x[0] * inv, x[1] * inv), cvt2(x[2] * inv, x[3] * inv));
}

}  // namespace

bool attn8_prompt_takes(int T, int n_seqs, int n_q, int n_kv, int max_q, int max_kv) {
  const int G = n_q / n_kv, TM = 128 / std::max(G, 1);
  if (TM < 1) return false;
  const double steps = ((double)T / TM + n_seqs) * ((double)max_kv / P8_KV + 1 + P8_COST) * n_kv;
  return steps < 2e9;
}

size_t attn8_prompt_workspace(int num_sms) { return (size_t)num_sms * (2 * 256 * (HEAD_DIM + 2) * sizeof(float) + sizeof(CutUnit)); }

cudaError_t attn8_prompt_launch(const Attn8Args& args, void* workspace, int num_sms, cudaStream_t stream) {
  PromptArgs a;
  static_cast<Attn8Args&>(a) = args;
  a.G = a.n_q / a.n_kv;
  a.TM = 128 / a.G;
  a.per_g = (65536 + a.G - 1) / a.G;
  const size_t smem = sizeof(P8Smem) + 1024 + (size_t)a.n_seqs * 4;
  static OncePerDevice once;
  cudaError_t e = once([] {
    return cudaFuncSetAttribute(attn8_prompt_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(sizeof(P8Smem) + 1024 + TGIS_KV8_MAX_SEQS * 4));
  });
  if (e != cudaSuccess) return e;
  const long long units = (long long)a.n_seqs * ((a.max_q + 2 * a.TM - 1) / (2 * a.TM)) * a.n_kv;
  const int grid = (int)std::max<long long>(1, std::min<long long>(num_sms, units * ((a.max_kv + P8_KV - 1) / P8_KV)));
  a.frag_o = reinterpret_cast<float*>(workspace);
  a.frag_ml = a.frag_o + (size_t)num_sms * 2 * 256 * HEAD_DIM;
  a.cut = reinterpret_cast<CutUnit*>(a.frag_ml + (size_t)num_sms * 2 * 256 * 2);
  e = launch_k(attn8_prompt_kernel, dim3(grid), dim3(P8_THREADS), smem, stream, a);
  if (e != cudaSuccess || grid == 1 || a.max_kv <= P8_KV) return e;   // (units of one step are never cut)
  return launch_k(attn8_join_kernel, dim3(grid, 256 / J8_WARPS), dim3(J8_WARPS * 32), 0, stream, a);
}

}  // namespace tgis
