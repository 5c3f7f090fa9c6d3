// The products of gemm8.cu for more tokens (gemm8_pair_takes), on CTA pairs (tcgen05 cta_group::2, kind::f8f6f4).
//
// Two neighbouring SMs work on one tile of 256 tokens x up to 256 weight rows.  Here tokens are the MMA's A operand (a CTA has 128 of them, a lane
// each) and weights its B operand (a CTA holds half of them and the tensor cores read both halves): a thread of the epilogue has one token, whose
// scale is one number a k-block, and its columns lie in at most two blocks of weights, so scaling costs a group's sums nothing but the multiply-add
// that adds them up.  A k-block is one group of 128.  Each half of the columns is an MMA, an accumulator and a set of four warps of its own, so that one
// half's sums are taken while the tensor cores make the other's, and accumulators go round through all of TMEM.
//
// Measured on one B200, T x N x K: 2048 x 8192 x 8192 118 us (2330 TFLOP/s), 2048 x 6144 x 4096 47 (2170), 512 x 8192 x 8192 32.5 (2110), 256 x 4096 x 4096 12.5; gated 2048 x 14336 x
// 4096 208 (2310).  What bounds it: a k-block of 256 x 256 takes some 740 clocks where the tensor cores need 512 and their operands' way through shared memory (A is read for
// each half) 640: the epilogue's chain of barrier, TMEM loads and 64 multiply-adds of pairs a thread (305 clocks of the SM's fp32 lanes).  Back to back for a second it is the
// power limit.  What mattered for the first: arrivals that wait for no memory (mbar_arrive_tmem: 311 -> 172 us), 32 columns a load instead of 16 (-> 146), a chunk on
// its way while one is added (-> 141), results through shared memory (-> 130), waits without a vote (-> 122), scales four k-blocks ahead by pointers that move (-> 118).
//
// Roles per CTA: warps 0..7 epilogue (two a lane quarter, half of the columns each), warp 8 TMA producer, warp 9 MMA issuer (leader CTA only) and
// TMEM owner.  The leader's `full` barrier counts both CTAs' bytes; tcgen05.commit releases a ring slot in both.  Waits on barriers in shared
// memory end after about two seconds.
#include <algorithm>

#include "launch.cuh"
#include "linear8.cuh"

namespace tgis {
namespace {

constexpr int P8_EPI = 8, P8_LOAD = 8, P8_MMA = 9, P8_THREADS = 384;
// registers of a thread: 168 at launch, of which the third warpgroup (load, MMA) gives up what the epilogue's two take
constexpr int P8_REGS = 168, P8_REGS_EPI = 232, P8_REGS_REST = 40;
static_assert(2 * P8_REGS_EPI + P8_REGS_REST <= 3 * P8_REGS, "a split may not be more than the block was launched with");
constexpr int P8_HALF = 128 * W8_GROUP;          // one CTA's share of a k-block of either operand
constexpr int P8_STAGES = 6;                   // k-blocks in flight
constexpr int P8_RING = P8_STAGES * 2 * P8_HALF;
constexpr int P8_BARS = 256, P8_MOST = 2 * 256 * 4, P8_OUT = 2048;   // barriers; maxima of a gated tile [parity][256]; a warp's way out: 32 rows of 64 bytes
constexpr int P8_SMEM = P8_RING + P8_BARS + P8_MOST + P8_EPI * P8_OUT + 1024;
static_assert(P8_SMEM <= 227 * 1024 && 2 * P8_SMEM > 228 * 1024, "one CTA an SM: it has all of tensor memory");

__device__ __forceinline__ void mma_pair_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

struct Pair8Args {
  Gemm8Args g;
  int n_tiles, x_tiles;
};

// A thread's row of 64 bytes (v: four 16-byte words) of rows that lie `pitch` bytes apart: the warp's 32 of them leave in runs of 64 bytes, eight
// rows an instruction (a row a lane takes 32 lines an instruction: 5600 clocks a tile of 128 x 256 where this takes 1500).
__device__ __forceinline__ void leave64(uint8_t* way, int lane, const uint32_t (&v)[16], uint8_t* first_row, int64_t pitch, int rows) {
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4*>(way + lane * 64 + ((c ^ (lane >> 1 & 3)) << 4)) = make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
  __syncwarp();
  const int c = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2);
    const uint4 o = *reinterpret_cast<const uint4*>(way + r * 64 + ((c ^ (r >> 1 & 3)) << 4));
    if (r < rows) *reinterpret_cast<uint4*>(first_row + r * pitch + c * 16) = o;
  }
}

// One token's sums of N neighbouring columns from n0 on -> y.  GATED: N / 2 gates, then their ups -> h in 8 bits; the maxima of the token's group meet
// in most[part of `parts`][256 / parts] by way of a barrier of `threads`.
template <int N, bool GATED, class OT>
__device__ __forceinline__ void finish(const Gemm8Args& a, float (&acc)[N], int t, int n0, int n_tile, int part, int place, uint32_t* most, int parts, uint8_t* way, int lane,
                                       int bar, int threads) {
  const int t_first = t - lane, rows = min(32, a.T - t_first);
  if constexpr (GATED) {
    constexpr int F = N / 2;
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < F; ++j) {
      acc[j] = n0 + j < a.N ? swiglu(acc[j], acc[F + j]) : 0.f;
      m = max(m, __float_as_uint(acc[j]) & 0x7fffffffu);
    }
    const int each = 256 / parts;
    most[part * each + place] = m;
    asm volatile("bar.sync %0, %1;\n" ::"r"(bar), "r"(threads) : "memory");
    for (int i = 0; i < parts; ++i) m = max(m, most[i * each + place]);
    const float s = scale_of(m);
    if (part == 0 && t < a.T) a.sh[(size_t)n_tile * a.ldh + t] = s;
    uint32_t w[F / 4];
    codes_near(acc, s, w);
    uint8_t* to = a.codes + (size_t)t_first * a.ldc + n0;
    if constexpr (F == 64) {
      leave64(way, lane, w, to, a.ldc, rows);
    } else if (t < a.T) {
      uint4* row = reinterpret_cast<uint4*>(to + (size_t)lane * a.ldc);
#pragma unroll
      for (int j = 0; j < F / 16; ++j) row[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    }
  } else {
    constexpr int EACH = 64 / (int)sizeof(OT);   // numbers of 64 bytes
    static_assert(N % EACH == 0, "");
    OT* y = reinterpret_cast<OT*>(a.y) + (size_t)t_first * a.ldy + n0;
    const bool wide = ((reinterpret_cast<uintptr_t>(y) | (uintptr_t)(a.ldy * sizeof(OT))) & 15) == 0;
    const int valid = a.N - n0;
#pragma unroll
    for (int j = 0; j < N; j += EACH) {
      if (j >= valid) break;
      if (wide && j + EACH <= valid) {
        uint32_t o[16];
#pragma unroll
        for (int l = 0; l < 16; ++l) {
          if constexpr (sizeof(OT) == 4) {
            o[l] = __float_as_uint(acc[j + l]);
          } else {
            const __nv_bfloat162 v = __floats2bfloat162_rn(acc[j + 2 * l], acc[j + 2 * l + 1]);
            o[l] = *reinterpret_cast<const uint32_t*>(&v);
          }
        }
        leave64(way, lane, o, reinterpret_cast<uint8_t*>(y + j), a.ldy * (int64_t)sizeof(OT), rows);
      } else if (t < a.T) {
#pragma unroll
        for (int l = 0; l < EACH; ++l)
          if (j + l < valid) y[(size_t)lane * a.ldy + j + l] = (OT)acc[j + l];
      }
    }
  }
}

// CH: chunks of 32 columns that a half of a tile has.  A tile has 64 CH weight rows; gated (CH = 4) 128 of either matrix, a half has 64 gates and
// then their 64 ups, the first from the leader's share of the weights, the others from its peer's.
//
// S > 1: few tiles, so the pairs of a cluster have a piece of k each and meet in distributed shared memory: each CTA leaves its sums in place of its ring
// and takes 128 / S of its tokens from all S, in the order of k.
template <int CH, int S, bool GATED, class OT>
__global__ void __launch_bounds__(P8_THREADS, 1)
gemm8_pair_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap wmap2, const __grid_constant__ CUtensorMap xmap,
                  const __grid_constant__ Pair8Args pa) {
  constexpr int NH = 32 * CH, N_TILE = GATED ? 128 : 2 * NH;   // columns of a half; weight rows (features) of a tile
  constexpr int AHEAD = GATED ? 2 : 4;   // k-blocks whose scales are asked for at once (registers; 2048 x 8192 x 8192 121.2 us by two, 118.9 by four, gated 2048 x 14336 x 4096 206 and 212)
  constexpr int BUFS = 512 / NH;   // accumulators of a half in TMEM, the halves in turn: 4, 5 or 8
  static_assert(!GATED || CH == 4, "");
  extern __shared__ uint8_t smem_raw[];
  const Gemm8Args& a = pa.g;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + P8_RING);
  uint64_t* empty = full + P8_STAGES;
  uint64_t* tmem_full = empty + P8_STAGES;
  uint64_t* tmem_empty = tmem_full + BUFS;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(tmem_empty + BUFS);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_at + 1);
  uint32_t* most = reinterpret_cast<uint32_t*>(smem + P8_RING + P8_BARS);

  const int warp = threadIdx.x >> 5, lane = (int)lane_id();
  const int rank = (int)cluster_ctarank() & 1, leader = (int)cluster_ctarank() & ~1, piece = (int)cluster_ctarank() >> 1;
  const int pair = blockIdx.x / (2 * S), pairs = gridDim.x / (2 * S), tiles = pa.n_tiles * pa.x_tiles;   // (of a cluster's pairs the tile is the same)
  const int kb0 = S == 1 ? 0 : (int)((long long)piece * a.G / S), KB = S == 1 ? a.G : (int)((long long)(piece + 1) * a.G / S) - kb0;

  if (warp == P8_LOAD && elect_one()) {
    tma_prefetch_desc(&wmap);
    if (GATED) tma_prefetch_desc(&wmap2);
    tma_prefetch_desc(&xmap);
  }
  if (warp == P8_MMA) {
    if (elect_one()) {
      for (int i = 0; i < P8_STAGES; ++i) {
        mbar_init(&full[i], 1);    // the leader's expect_tx (both CTAs' bytes)
        mbar_init(&empty[i], 1);   // commit_pair
      }
      for (int i = 0; i < BUFS; ++i) {
        mbar_init(&tmem_full[i], 1);         // commit_pair
        mbar_init(&tmem_empty[i], P8_EPI);   // a half's epilogue warps of both CTAs (leader's barrier)
      }
      *gave_up = 0;
      fence_barrier_init();
    }
    __syncwarp();
    tmem_alloc_pair<512>(tmem_at);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // the peer's barriers exist
  tc_fence_after();
  const uint32_t tmem = *tmem_at;
  griddep_launch();

  // how all warps end (in either branch: what follows the two has the registers of the poorer one)
  auto meet = [&] {
    __syncwarp();
    tc_fence_before();
    asm volatile("bar.sync 0;\n" ::: "memory");
    say_if_stalled8(a, gave_up);
    cluster_sync_all();   // nobody leaves while the peer may still read its shared memory or signal its barriers
  };
  if (warp >= P8_EPI) {
    set_regs<P8_REGS_REST, false>();
    if (warp == P8_LOAD && elect_one()) {
      // ===================== TMA producer (both CTAs) =====================
      const uint32_t full0 = dsmem_addr(smem_u32(full), leader);   // the leader's barriers
      constexpr uint32_t bytes = 2u * (uint32_t)(P8_HALF + (GATED ? 128 : NH) * W8_GROUP);
      auto load_w = [&](int s, int tile, int kb) {
        if (rank == 0) mbar_arrive_expect_tx(&full[s], bytes);
        uint8_t* to = smem + s * 2 * P8_HALF + P8_HALF;
        const int row = tile / pa.x_tiles * N_TILE;
        if (GATED) {
          tma_load_pair(rank == 0 ? &wmap : &wmap2, full0 + s * 8, to, (kb0 + kb) * W8_GROUP, row);
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) tma_load_pair(&wmap, full0 + s * 8, to + h * (NH / 2) * W8_GROUP, (kb0 + kb) * W8_GROUP, row + h * NH + rank * (NH / 2));
        }
      };
      auto load_x = [&](int s, int tile, int kb) {
        tma_load_pair(&xmap, full0 + s * 8, smem + s * 2 * P8_HALF, (kb0 + kb) * W8_GROUP, tile % pa.x_tiles * 256 + rank * 128);
      };
      const int pre = pair < tiles ? min(KB, P8_STAGES) : 0;
      if (!a.early) griddep_wait();
      for (int kb = 0; kb < pre; ++kb) load_w(kb, pair, kb);
      if (a.early) griddep_wait();
      for (int kb = 0; kb < pre; ++kb) load_x(kb, pair, kb);
      int s = pre % P8_STAGES;
      uint32_t phase = pre == P8_STAGES ? 1 : 0;
      bool ok = true;
      for (int tile = pair, first = pre; tile < tiles && ok; tile += pairs, first = 0) {
        for (int kb = first; kb < KB; ++kb) {
          if (!(ok = bounded_wait(&empty[s], phase ^ 1))) break;
          load_w(s, tile, kb);
          load_x(s, tile, kb);
          if (++s == P8_STAGES) s = 0, phase ^= 1;
        }
      }
      if (!ok) *gave_up = 1;
    }
    if (warp == P8_MMA && rank == 0 && elect_one()) {
      // ===================== MMA issuer (leader) =====================
      griddep_wait();   // (rows and scales come after the grids before this one, which may take longer than a wait has patience)
      constexpr uint32_t idesc = idesc_f8(256, NH);
      const uint32_t ring = smem_u32(smem);
      int s = 0, b = 0;
      uint32_t phase = 0, phase_b = 0;
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs) {
        for (int kb = 0; kb < KB && ok; ++kb) {
          if (!(ok = bounded_wait(&full[s], phase))) break;
          tc_fence_after();
          const uint32_t at = ring + s * 2 * P8_HALF;
          const uint64_t x = make_smem_desc_sw128(at);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!(ok = ok && bounded_wait(&tmem_empty[b], phase_b ^ 1))) break;
            tc_fence_after();
            const uint64_t w = make_smem_desc_sw128(at + P8_HALF + h * (NH / 2) * W8_GROUP);
#pragma unroll
            for (int k = 0; k < W8_GROUP / 32; ++k) mma_pair_f8(tmem + b * NH, x + (uint64_t)(k * 2), w + (uint64_t)(k * 2), idesc, k > 0);
            commit_pair(&tmem_full[b], leader);
            if (++b == BUFS) b = 0, phase_b ^= 1;
          }
          if (!ok) break;
          commit_pair(&empty[s], leader);
          if (++s == P8_STAGES) s = 0, phase ^= 1;
        }
      }
      if (!ok) *gave_up = 1;
    }
    meet();
    if (warp == P8_MMA) {
      tc_fence_after();
      tmem_dealloc_pair<512>(tmem);
    }
    if constexpr (S > 1) cluster_sync_all();
  } else {
    // ===================== epilogue (both CTAs): lane = token, column = weight row =====================
    set_regs<P8_REGS_EPI, true>();
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t free0 = dsmem_addr(smem_u32(tmem_empty), leader);
    uint8_t* way = smem + P8_RING + P8_BARS + P8_MOST + warp * P8_OUT;
    griddep_wait();   // the scales of the rows; y may still be in use by the previous kernels
    int b = half;   // this half's next accumulator
    uint32_t phase = 0;
    long long patience = WAIT_LIMIT;
    for (int tile = pair, turn = 0; tile < tiles; tile += pairs, turn ^= 1) {
      const int n_tile = tile / pa.x_tiles, t = tile % pa.x_tiles * 256 + rank * 128 + quarter * 32 + lane;
      const int n0 = n_tile * N_TILE + half * (N_TILE / 2);   // first column (gated: feature)
      // columns [0, cut) have the scales sw, those behind them sw2
      const int nb = n0 / 128, cut = GATED ? 64 : 128 - n0 % 128;
      const float* sw = a.sw + (size_t)min(nb, (a.N - 1) / 128) * a.G;
      const float* sw2 = GATED ? a.sw2 + (size_t)nb * a.G : a.sw + (size_t)min(nb + 1, (a.N - 1) / 128) * a.G;
      const float* sx = a.sx + min(t, a.T - 1);
      float acc[NH];
#pragma unroll
      for (int j = 0; j < NH; ++j) acc[j] = 0.f;
      float x[AHEAD] = {}, w[AHEAD] = {}, w2[AHEAD] = {};
      const float *px = sx + (size_t)kb0 * a.lds, *pw = sw + kb0, *pw2 = sw2 + kb0;
      auto load = [&](int kb) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
          if (kb + u < KB) {
            x[u] = *px;
            w[u] = *pw++;
            w2[u] = *pw2++;
            px += a.lds;
          }
      };
      load(0);
      // One chunk of columns is added while the next one is on its way out of TMEM, across k-blocks too.
      uint32_t r[2][32];
      await(&tmem_full[b], phase, patience);
      tc_fence_after();
      tmem_ld<32>(from + b * NH, r[0]);
      for (int at = 0; at < KB; at += AHEAD) {
        float f[AHEAD], f2[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          f[u] = x[u] * w[u];
          f2[u] = x[u] * w2[u];
        }
        if (at + AHEAD < KB) load(at + AHEAD);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          if (at + u >= KB) break;
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            uint32_t* now = r[(u * CH + c) & 1];
            uint32_t* next = r[(u * CH + c + 1) & 1];
            tmem_ld_wait();
            if (c + 1 < CH) {
              tmem_ld<32>(from + b * NH + (c + 1) * 32, next);
            } else {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive_tmem(free0 + b * 8);
              b += 2;
              if (b >= BUFS) b -= BUFS, phase ^= 1;
              if (at + u + 1 < KB) {
                await(&tmem_full[b], phase, patience);
                tc_fence_after();
                tmem_ld<32>(from + b * NH, next);
              }
            }
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float s = c * 32 < cut ? f[u] : f2[u];   // (n0 and 64 are multiples of 32)
              add_scaled(acc[c * 32 + j], acc[c * 32 + j + 1], now[j], now[j + 1], s, s);
            }
          }
        }
      }
      static_assert(AHEAD * CH % 2 == 0, "r[0] is the first chunk's in every turn");
      if constexpr (S == 1) {
        finish<NH, GATED, OT>(a, acc, t, n0, n_tile, half, quarter * 32 + lane, most + turn * 256, 2, way, lane, 1 + quarter, 64);
      } else {
        // (one tile a cluster) [four columns][128 tokens][4]; the ring is done with once both halves have their last sums
        asm volatile("bar.sync 1, 256;\n" ::: "memory");
        float4* sums = reinterpret_cast<float4*>(smem) + (half * NH / 4) * 128 + quarter * 32 + lane;
#pragma unroll
        for (int j = 0; j < NH; j += 4) sums[j / 4 * 128] = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
      }
    }
    if (patience == 0) *gave_up = 1;
    meet();
    if constexpr (S > 1) {
      // a warp: 32 of the CTA's 128 / S tokens and a 2 S-th of the columns
      constexpr int GROUPS = 2 * S, EACH = NH / S;   // (gated: half of EACH features, their gates and their ups)
      const int tokens = piece * (128 / S) + warp / GROUPS * 32 + lane, group = warp % GROUPS;
      const int n_tile = pair / pa.x_tiles, t = pair % pa.x_tiles * 256 + rank * 128 + tokens;
      float acc[EACH];
#pragma unroll
      for (int j = 0; j < EACH; ++j) acc[j] = 0.f;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const uint32_t from = dsmem_addr(smem_u32(smem), s * 2 + rank) + tokens * 16;
#pragma unroll
        for (int j = 0; j < EACH; j += 4) {
          // gated: feature f's gate is column f / 64 * 128 + f % 64, its up 64 further
          const int f = group * (EACH / 2) + j % (EACH / 2), col = GATED ? f / 64 * 128 + f % 64 + j / (EACH / 2) * 64 : group * EACH + j;
          const float4 v = ld_dsmem_f4(from + (uint32_t)(col / 4) * 2048);
          acc[j] += v.x; acc[j + 1] += v.y; acc[j + 2] += v.z; acc[j + 3] += v.w;
        }
      }
      uint8_t* way = smem + P8_RING + P8_BARS + P8_MOST + warp * P8_OUT;
      finish<EACH, GATED, OT>(a, acc, t, n_tile * N_TILE + group * (GATED ? EACH / 2 : EACH), n_tile, group, warp / GROUPS * 32 + lane, most, GROUPS, way, lane,
                              1, 256);
      cluster_sync_all();   // nobody leaves while its sums are read
    }
  }
}

template <int CH, int S, bool GATED, class OT>
cudaError_t launch_pair8(const CUtensorMap& w, const CUtensorMap& w2, const CUtensorMap& x, const Pair8Args& a, int num_sms, cudaStream_t stream) {
  static OncePerDevice once;
  cudaError_t e = once([] { return cudaFuncSetAttribute(gemm8_pair_kernel<CH, S, GATED, OT>, cudaFuncAttributeMaxDynamicSharedMemorySize, P8_SMEM); });
  if (e != cudaSuccess) return e;
  const long long tiles = (long long)a.n_tiles * a.x_tiles;
  if (tiles >= 1ll << 28) return cudaErrorInvalidValue;
  const int pairs = std::max(num_sms / 2, 1);
  return launch_k_cluster(gemm8_pair_kernel<CH, S, GATED, OT>, dim3(2 * S * (unsigned)(S > 1 ? tiles : std::min<long long>(tiles, pairs))), dim3(P8_THREADS), P8_SMEM,
                          stream, 2 * S, w, w2, x, a);
}

template <class OT>
cudaError_t plan(int N, int x_tiles, int G, bool gated, Plan8* out) {
  static ClustersAtOnce at_once;
  int n[4] = {};
  for (int i = 1; i < 4 && G >= 1 << (i - 1); ++i) {
    const cudaError_t e = at_once(gemm8_pair_kernel<4, 1, false, OT>, P8_THREADS, P8_SMEM, 1 << i, &n[i]);
    if (e != cudaSuccess) return e;
  }
  return gemm8_pair_plan(N, x_tiles, G, gated, n, out);
}

template <class OT>
cudaError_t launch_plain(const Plan8& p, const CUtensorMap& w, const CUtensorMap& x, const Pair8Args& a, int num_sms, cudaStream_t stream) {
  if (p.s == 4) return launch_pair8<4, 4, false, OT>(w, w, x, a, num_sms, stream);
  if (p.s == 2) return p.ch == 4 ? launch_pair8<4, 2, false, OT>(w, w, x, a, num_sms, stream) : launch_pair8<2, 2, false, OT>(w, w, x, a, num_sms, stream);
  return p.ch == 4 ? launch_pair8<4, 1, false, OT>(w, w, x, a, num_sms, stream) : p.ch == 3 ? launch_pair8<3, 1, false, OT>(w, w, x, a, num_sms, stream)
                                                                                            : launch_pair8<2, 1, false, OT>(w, w, x, a, num_sms, stream);
}
template <class OT>
cudaError_t product_pair8(const tgis_w8_rows& x, const tgis_w8_matrix& w, const Gemm8Args& g, int num_sms, cudaStream_t stream) {
  Pair8Args a{g, 0, (g.T + 255) / 256};
  Plan8 p{4, 1};
  cudaError_t e = plan<OT>(g.N, a.x_tiles, g.G, false, &p);
  if (e != cudaSuccess) return e;
  a.n_tiles = (g.N + 64 * p.ch - 1) / (64 * p.ch);
  CUtensorMap wm, xm;
  e = map8(&wm, w.codes, w.n, w.k, w.ld, 16 * p.ch);
  if (e == cudaSuccess) e = map8(&xm, x.codes, x.t, x.k, x.ld, 128);
  return e != cudaSuccess ? e : launch_plain<OT>(p, wm, xm, a, num_sms, stream);
}

}  // namespace

// Chunks of a half and pieces of k: those whose waves take least, in hundredths of a microsecond.  A k-block of 256 x 64 CH takes P8_BLOCK[CH] while it is the
// epilogue's chain that bounds it, a launch's beginning and end P8_ENDS[S] and P8_WIDE[S] more for every chunk above two; pieces are for one wave.  Measured (us; taken first):
// 256 x 4096 x 4096 CH 2, S 2: 12.6; CH 2, S 1: 13.6; CH 4, S 2: 14.6; CH 4, S 1: 16.6.  512 x 6144 x 4096 CH 3: 17.0, CH 4: 18.3, CH 2: 24.4.  301 x 2128 x 11264 CH 4, S 2: 25.5, CH 2, S 1: 30.2,
// CH 4, S 1: 35.3.  1024 x 512 x 8192 CH 4, S 4: 15.5, CH 2, S 2: 15.2, S 1: 22.2.  203 x 512 x 1536 CH 2, S 1: 6.8, S 2: 7.0, CH 4, S 4: 8.9.  2048 x 8192 x 8192 CH 4: 118, CH 3: 131, CH 2: 154.
constexpr int P8_BLOCK[5] = {0, 0, 30, 33, 36}, P8_ENDS[5] = {0, 400, 600, 0, 700}, P8_WIDE[5] = {0, 50, 100, 0, 100};
cudaError_t gemm8_pair_plan(int N, int x_tiles, int G, bool gated, const int (&at_once)[4], Plan8* out) {
  long long least = -1;
  for (int i = 1, s = 1; i < 4 && s <= G; ++i, s *= 2) {
    const int n = at_once[i];
    if (n < 1) continue;
    for (int c = 4; c >= 2; --c) {
      if (gated ? c < 4 : (s == 2 && c == 3) || (s == 4 && c < 4)) continue;   // (a thread's share of what pieces leave: whole runs of 64 bytes)
      const int rows = gated ? 128 : 64 * c;
      const long long tiles = (long long)((N + rows - 1) / rows) * x_tiles, waves = (tiles + n - 1) / n;
      if (s > 1 && waves > 1) continue;
      const long long cost = waves * ((long long)P8_BLOCK[c] * ((G + s - 1) / s)) + P8_ENDS[s] + P8_WIDE[s] * (c - 2);
      if (least < 0 || cost < least) *out = Plan8{c, s}, least = cost;
    }
  }
  return least < 0 ? cudaErrorLaunchOutOfResources : cudaSuccess;
}

// More than 128 tokens; from 65 on gated ones (us, gemm8.cu and here: 65 tokens, 4096 / 14336 38.5 and 33.5, 512 / 1536 9.4 and 6.0; 64 tokens 26.5 and 33) and those of few
// k-blocks, whose end is what counts (65 x 512 x 512 6.4 and 4.1, but 65 x 2128 x 2048 7.8 and 9.2, 128 x 4096 x 14336 20.3 and 24.4; 200: 32.0 and 25.6).
bool gemm8_pair_takes(int T, int G, bool gated) { return T > 128 || (T > 64 && (gated || G <= 8)); }

cudaError_t gemm8_pair_launch(const tgis_w8_rows& x, const tgis_w8_matrix& w, const Gemm8Args& g, bool f32, int num_sms, cudaStream_t stream) {
  return f32 ? product_pair8<float>(x, w, g, num_sms, stream) : product_pair8<__nv_bfloat16>(x, w, g, num_sms, stream);
}

cudaError_t gemm8_pair_gated_launch(const tgis_w8_rows& x, const tgis_w8_matrix& gate, const tgis_w8_matrix& up, const Gemm8Args& g, int num_sms,
                                    cudaStream_t stream) {
  Pair8Args a{g, (g.N + 127) / 128, (g.T + 255) / 256};
  CUtensorMap wm, wm2, xm;
  cudaError_t e = map8(&wm, gate.codes, gate.n, gate.k, gate.ld, 128);
  if (e == cudaSuccess) e = map8(&wm2, up.codes, up.n, up.k, up.ld, 128);
  if (e == cudaSuccess) e = map8(&xm, x.codes, x.t, x.k, x.ld, 128);
  if (e != cudaSuccess) return e;
  Plan8 p{4, 1};
  if ((e = plan<__nv_bfloat16>(g.N, a.x_tiles, g.G, true, &p)) != cudaSuccess) return e;
  return p.s == 4 ? launch_pair8<4, 4, true, __nv_bfloat16>(wm, wm2, xm, a, num_sms, stream)
       : p.s == 2 ? launch_pair8<4, 2, true, __nv_bfloat16>(wm, wm2, xm, a, num_sms, stream) : launch_pair8<4, 1, true, __nv_bfloat16>(wm, wm2, xm, a, num_sms, stream);
}

}  // namespace tgis
