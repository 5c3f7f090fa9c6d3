// y[t, n] = sum_g sx[t, g] sw[n / 128, g] sum_{k in g} cx[t, k] cw[n, k]: 8-bit weights (include/tgis_w8.h) times rows in 8 bits, and the gated
// form h = silu(x gate^T) * (x up^T), which leaves as rows in 8 bits.
//
// Up to 128 tokens, gated up to 64 (gemm8_pair.cu has more, and those above 64 of few k-blocks).  A CTA has a block of 128 weight rows (the MMA's A operand, a lane a row) and all tokens (B, a column
// each): such a product is bound by its weight bytes, which are read once.  The tensor cores (tcgen05 kind::f8f6f4) sum one group of 128 k, that is
// one k-block, in an accumulator; the epilogue's threads take it over, times both scales, into fp32 registers while the next one is summed in the
// other half of the CTA's TMEM.  A tile's weights have one scale a k-block and a column has one, so a warp of its own puts their product where the
// epilogue reads it.  K is cut into pieces for the CTAs of a cluster, which push their sums into the shared memory of the CTA that a token belongs to:
// added there in the order of k, so that a result is the same in every call, without a workspace.
//
// Measured on one B200, us (weight bytes a second), T x N x K, launches one behind the other with cold weights: 1 x 4096 x 4096 6.4 (2.6 TB/s), 1 x 8192 x 8192 13.6
// (4.9), 32 x 4096 x 14336 14.0 (4.3), 64 x 8192 x 8192 16.7 (4.1), 128 x 4096 x 14336 20 (3.0); gated 1 x 14336 x 4096 22.6 (5.2), 48: 25.3.  What bounds it: of
// 4096 x 4096 a launch's beginning (0.6 us), the first bytes' way (2.5, of which the bytes themselves are most) and the cluster's end (two
// barriers and the sums, 2 to 3); large ones the memory, short of a copy's 6.5 TB/s by those 4 us.
//
// Roles: warps 0..7 epilogue, warp 8 TMA producer, warp 9 MMA issuer and TMEM owner, warp 10 scales.  Waits on barriers in shared memory end
// after about two seconds.
#include <stdarg.h>

#include <algorithm>
#include <cmath>

#include "launch.cuh"
#include "linear8.cuh"
#include "ptx.cuh"

namespace tgis {
namespace {

constexpr int G8_EPI = 8, G8_WARPS = 11, G8_THREADS = G8_WARPS * 32;   // epilogue: warps 0 .. 7
constexpr int G8_LOAD = 8, G8_MMA = 9, G8_SCALE = 10;
constexpr int G8_W_BYTES = 128 * W8_GROUP;                   // a k-block of a weight tile
constexpr int G8_SLOTS = 4;                                  // k-blocks whose scales are there
constexpr int G8_ENDS = 6;                                    // what a wave's beginning and end take, in k-blocks

// D[tmem] (+)= A[smem] B[smem], e4m3, fp32 sums
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Tokens of a tile, and what follows from them.  Two CTAs share an SM while their accumulators (TMEM has 512 columns) and registers allow: 64 x 8192 x 8192 in 256
// CTAs 16.7 us, in the 128 of one an SM 22.
template <int NT, bool GATED>
struct Form {
  static constexpr int HALVES = GATED ? 2 : 1;                       // matrices
  static constexpr int NC = GATED ? NT : NT / 2;                     // columns of an epilogue warp: two warps a lane quarter
  static constexpr int COLS = NT * HALVES;                           // TMEM columns of a k-block's sums
  static constexpr int TMEM = 2 * COLS < 32 ? 32 : 2 * COLS;
  static constexpr int X_BYTES = NT * W8_GROUP;
  static constexpr int STAGE = G8_W_BYTES * HALVES + X_BYTES;
  static constexpr int CTAS = TMEM <= 256 && NC <= 32 ? 2 : 1;
  static constexpr int SCALES = G8_SLOTS * HALVES * NT * 4, BARS = 320;
  static constexpr int ROOM = (CTAS == 2 ? 112 : 226) * 1024 - 1024 - SCALES - BARS;
  static constexpr int STAGES = ROOM / STAGE < 12 ? ROOM / STAGE : 12;
  static constexpr int SUMS = HALVES * NT * 128 * 4;                 // a cluster's sums, in place of the ring
  static constexpr int RING = STAGES * STAGE > SUMS ? STAGES * STAGE : SUMS;
  static constexpr int SMEM = RING + SCALES + BARS + 1024;
  static_assert(STAGES >= 2 && TMEM <= 512 && SMEM <= 227 * 1024, "");
  // (a second CTA that waited for tensor memory of a first one could wait for its cluster's other CTAs in turn: shared memory keeps it out)
  static_assert(CTAS == 2 || 2 * SMEM > 228 * 1024, "");
};

template <int NT, bool GATED, class OT>
__global__ void __launch_bounds__(G8_THREADS, (Form<NT, GATED>::CTAS))
gemm8_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap wmap2, const __grid_constant__ CUtensorMap xmap,
             const __grid_constant__ Gemm8Args a, int x_box) {
  using F = Form<NT, GATED>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* scale = reinterpret_cast<float*>(smem + F::RING);            // [G8_SLOTS][HALVES][NT]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + F::RING + F::SCALES);
  uint64_t* empty = full + F::STAGES;
  uint64_t* tmem_full = empty + F::STAGES;
  uint64_t* tmem_empty = tmem_full + 2;
  uint64_t* scale_full = tmem_empty + 2;
  uint64_t* scale_empty = scale_full + G8_SLOTS;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(scale_empty + G8_SLOTS);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_at + 1);

  const int warp = threadIdx.x >> 5, lane = (int)lane_id();
  const int rank = (int)cluster_ctarank(), S = (int)gridDim.z, log_s = __ffs(S) - 1;   // cluster: the CTAs of blockIdx.z, one, two, four or eight
  const int nb = (int)blockIdx.x;
  const int kb0 = (int)((long long)rank * a.G / S), kb1 = (int)((long long)(rank + 1) * a.G / S);

  if (warp == G8_LOAD && elect_one()) {
    tma_prefetch_desc(&wmap);
    if (GATED) tma_prefetch_desc(&wmap2);
    tma_prefetch_desc(&xmap);
  }
  if (warp == G8_MMA) {
    if (elect_one()) {
      for (int i = 0; i < F::STAGES; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&tmem_full[i], 1);
        mbar_init(&tmem_empty[i], G8_EPI);
      }
      for (int i = 0; i < G8_SLOTS; ++i) {
        mbar_init(&scale_full[i], 1);
        mbar_init(&scale_empty[i], G8_EPI);
      }
      *gave_up = 0;
      fence_barrier_init();
    }
    __syncwarp();
    tmem_alloc<F::TMEM>(tmem_at);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_at;
  griddep_launch();

  if (warp == G8_LOAD) {
    // ===================== TMA producer =====================
    if (elect_one()) {
      const uint64_t once = policy_evict_first();
      const uint32_t bytes = (uint32_t)(G8_W_BYTES * F::HALVES + x_box * W8_GROUP);
      auto load_w = [&](int s, int kb) {
        mbar_arrive_expect_tx(&full[s], bytes);
        tma_load_2d_hint(&wmap, &full[s], smem + s * F::STAGE, kb * W8_GROUP, nb * 128, once);
        if (GATED) tma_load_2d_hint(&wmap2, &full[s], smem + s * F::STAGE + G8_W_BYTES, kb * W8_GROUP, nb * 128, once);
      };
      auto load_x = [&](int s, int kb) { tma_load_2d(&xmap, &full[s], smem + s * F::STAGE + G8_W_BYTES * F::HALVES, kb * W8_GROUP, 0); };
      const int pre = min(kb1 - kb0, F::STAGES);
      if (!a.early) griddep_wait();
      for (int i = 0; i < pre; ++i) load_w(i, kb0 + i);
      if (a.early) griddep_wait();
      for (int i = 0; i < pre; ++i) load_x(i, kb0 + i);
      int s = pre % F::STAGES;
      uint32_t phase = pre == F::STAGES ? 1 : 0;
      for (int kb = kb0 + pre; kb < kb1; ++kb) {
        if (!bounded_wait(&empty[s], phase ^ 1)) {
          *gave_up = 1;
          break;
        }
        load_w(s, kb);
        load_x(s, kb);
        if (++s == F::STAGES) s = 0, phase ^= 1;
      }
    }
  } else if (warp == G8_MMA) {
    // ===================== MMA issuer =====================
    if (elect_one()) {
      griddep_wait();   // (rows and scales come after the grids before this one, which may take longer than a wait has patience)
      constexpr uint32_t idesc = idesc_f8(128, NT);
      const uint32_t ring = smem_u32(smem);
      int s = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int i = kb - kb0, buf = i & 1;
        if (!bounded_wait(&tmem_empty[buf], (uint32_t)(i >> 1 & 1) ^ 1) || !bounded_wait(&full[s], phase)) {
          *gave_up = 1;
          break;
        }
        tc_fence_after();
        const uint32_t at = ring + s * F::STAGE;
        const uint64_t x = make_smem_desc_sw128(at + G8_W_BYTES * F::HALVES);
#pragma unroll
        for (int h = 0; h < F::HALVES; ++h) {
          const uint64_t w = make_smem_desc_sw128(at + h * G8_W_BYTES);
#pragma unroll
          for (int k = 0; k < W8_GROUP / 32; ++k) mma_f8(tmem + buf * F::COLS + h * NT, w + (uint64_t)(k * 2), x + (uint64_t)(k * 2), idesc, k > 0);
        }
        tc_commit(&empty[s]);
        tc_commit(&tmem_full[buf]);
        if (++s == F::STAGES) s = 0, phase ^= 1;
      }
    }
  } else if (warp == G8_SCALE) {
    // ===================== scales: sx[t] sw of the k-blocks to come =====================
    griddep_wait();
    const float* sw = a.sw + (size_t)nb * a.G;
    const float* sw2 = GATED ? a.sw2 + (size_t)nb * a.G : nullptr;
    // (AHEAD k-blocks at a time, asked for while those before them are handed out: one at a time took the L2's latency for each)
    constexpr int EACH = (NT + 31) / 32, AHEAD = 8;
    float x[AHEAD][EACH], w[AHEAD], w2[AHEAD];
    auto load = [&](int from) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int kb = min(from + u, kb1 - 1);
        w[u] = sw[kb];
        w2[u] = GATED ? sw2[kb] : 0.f;
#pragma unroll
        for (int j = 0; j < EACH; ++j) x[u][j] = j * 32 + lane < NT && j * 32 + lane < a.T ? a.sx[(size_t)kb * a.lds + j * 32 + lane] : 0.f;
      }
    };
    load(kb0);
    long long patience = WAIT_LIMIT;
    for (int at = kb0; at < kb1; at += AHEAD) {
      float f[AHEAD][F::HALVES][EACH];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
          f[u][0][j] = x[u][j] * w[u];
          if (GATED) f[u][F::HALVES - 1][j] = x[u][j] * w2[u];
        }
      if (at + AHEAD < kb1) load(at + AHEAD);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (at + u >= kb1) break;
        const int i = at + u - kb0, slot = i % G8_SLOTS;
        await(&scale_empty[slot], (uint32_t)(i / G8_SLOTS & 1) ^ 1, patience);
        float* to = scale + slot * F::HALVES * NT;
#pragma unroll
        for (int h = 0; h < F::HALVES; ++h)
#pragma unroll
          for (int j = 0; j < EACH; ++j)
            if (j * 32 + lane < NT) to[h * NT + j * 32 + lane] = f[u][h][j];
        __syncwarp();
        if (lane == 0) mbar_arrive(&scale_full[slot]);
      }
    }
    if (patience == 0) *gave_up = 1;
  } else {
    // ===================== epilogue: lane = weight row, column = token =====================
    griddep_wait();   // (as the issuer)
    const int quarter = warp & 3, half = warp >> 2, col0 = half * F::NC;   // gated: the other half is the other matrix
    float acc[F::NC];
#pragma unroll
    for (int j = 0; j < F::NC; ++j) acc[j] = 0.f;
    long long patience = WAIT_LIMIT;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int i = kb - kb0, buf = i & 1, slot = i % G8_SLOTS;
      await(&scale_full[slot], (uint32_t)(i / G8_SLOTS & 1), patience);
      await(&tmem_full[buf], (uint32_t)(i >> 1 & 1), patience);
      tc_fence_after();
      const uint32_t at = tmem + buf * F::COLS + col0 + ((uint32_t)(quarter * 32) << 16);
      const float4* sc = reinterpret_cast<const float4*>(scale + slot * F::HALVES * NT + col0);
      constexpr int STEP = F::NC < 16 ? F::NC : 16;
      uint32_t r[2][STEP];
      tmem_ld<STEP>(at, r[0]);
#pragma unroll
      for (int c = 0; c < F::NC; c += STEP) {
        tmem_ld_wait();
        if (c + STEP < F::NC) {   // (on its way while this one is added)
          tmem_ld<STEP>(at + c + STEP, r[(c / STEP + 1) & 1]);
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&tmem_empty[buf]);
        }
        const uint32_t* now = r[(c / STEP) & 1];
#pragma unroll
        for (int j = 0; j < STEP; j += 4) {
          const float4 f = sc[(c + j) / 4];
          add_scaled(acc[c + j], acc[c + j + 1], now[j], now[j + 1], f.x, f.y);
          add_scaled(acc[c + j + 2], acc[c + j + 3], now[j + 2], now[j + 3], f.z, f.w);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&scale_empty[slot]);
    }
    if (patience == 0) *gave_up = 1;
    if (S > 1) cluster_sync_all();   // every CTA's ring is done with: the sums take its place
    // Token t is the CTA's of rank t mod S: sums [CTA that they come from][matrix][token / S][weight row].  (Stores that nobody waits for: with sums kept here
    // and read from there, 64 tokens' latency was 1400 to 3900 clocks.)
    const uint32_t mine = smem_u32(smem) + (uint32_t)(((rank * F::HALVES + (GATED ? half : 0)) * (NT >> log_s)) * 512 + (quarter * 32 + lane) * 4);
#pragma unroll
    for (int j = 0; j < F::NC; ++j) {
      const int t = (GATED ? 0 : col0) + j;
      if (t < a.T) st_dsmem_f32(dsmem_addr(mine + (uint32_t)(t >> log_s) * 512, t & (S - 1)), acc[j]);
    }
  }
  __syncwarp();
  if (warp >= G8_EPI && S > 1) cluster_sync_all();   // (the epilogue's first)
  tc_fence_before();
  if (S > 1) cluster_sync_all();
  else __syncthreads();
  if (say_if_stalled8(a, gave_up)) __syncthreads();
  if (warp == G8_MMA) {
    tc_fence_after();
    tmem_dealloc<F::TMEM>(tmem);
  }
  // ===================== the cluster's sums -> y or h: a warp a token, four weight rows a lane =====================
  griddep_wait();   // (the issuer's and the producer's other lanes; y may still be in use by the kernels before)
  for (int i = warp, t; t = (i << log_s) + rank, t < NT && t < a.T; i += G8_WARPS) {
    float v[F::HALVES][4] = {};
    for (int r = 0; r < S; ++r)
#pragma unroll
      for (int h = 0; h < F::HALVES; ++h) {
        const float4 p = *reinterpret_cast<const float4*>(smem + (size_t)((r * F::HALVES + h) * (NT >> log_s) + i) * 512 + lane * 16);
        v[h][0] += p.x; v[h][1] += p.y; v[h][2] += p.z; v[h][3] += p.w;
      }
    const int n = nb * 128 + lane * 4;
    if constexpr (GATED) {
      float h[4];
      uint32_t m = 0, c[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        h[i] = n + i < a.N ? swiglu(v[0][i], v[1][i]) : 0.f;
        m = max(m, __float_as_uint(h[i]) & 0x7fffffffu);
      }
      const float s = scale_of(__reduce_max_sync(0xffffffffu, m));
      codes_near(h, s, c);
      *reinterpret_cast<uint32_t*>(a.codes + (size_t)t * a.ldc + n) = c[0];
      if (lane == 0) a.sh[(size_t)nb * a.ldh + t] = s;
    } else {
      OT* y = reinterpret_cast<OT*>(a.y) + (size_t)t * a.ldy + n;
      constexpr int ALIGN = 4 * (int)sizeof(OT);
      if (n + 4 <= a.N && (reinterpret_cast<uintptr_t>(y) & (ALIGN - 1)) == 0) {
        if constexpr (sizeof(OT) == 4) {
          *reinterpret_cast<float4*>(y) = make_float4(v[0][0], v[0][1], v[0][2], v[0][3]);
        } else {
          const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0][0], v[0][1]), hi = __floats2bfloat162_rn(v[0][2], v[0][3]);
          *reinterpret_cast<uint2*>(y) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < a.N) y[i] = (OT)v[0][i];
      }
    }
  }
}

template <int NT, bool GATED, class OT>
cudaError_t launch8(const CUtensorMap& w, const CUtensorMap& w2, const CUtensorMap& x, const Gemm8Args& a, int box, cudaStream_t stream) {
  using F = Form<NT, GATED>;
  static OncePerDevice once;
  cudaError_t e = once([] { return cudaFuncSetAttribute(gemm8_kernel<NT, GATED, OT>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM); });
  if (e != cudaSuccess) return e;
  const int tiles = (a.N + 127) / 128;
  static ClustersAtOnce at_once;
  int n[4] = {}, S = 1;
  for (int i = 0; i < 4 && (i == 0 || a.G >= 2 << i); ++i)
    if ((e = at_once(gemm8_kernel<NT, GATED, OT>, G8_THREADS, F::SMEM, 1 << i, &n[i])) != cudaSuccess) return e;
  if ((e = gemm8_plan(tiles, a.G, F::CTAS, n, &S)) != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)tiles, 1, (unsigned)S);
  cfg.blockDim = dim3(G8_THREADS);
  cfg.dynamicSmemBytes = F::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = (unsigned)S;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, gemm8_kernel<NT, GATED, OT>, w, w2, x, a, box);
}

template <bool GATED, class OT>
cudaError_t launch_tokens(const CUtensorMap& w, const CUtensorMap& w2, const tgis_w8_rows& x, const Gemm8Args& a, cudaStream_t stream) {
  const int nt = a.T <= 16 ? 16 : a.T <= 32 ? 32 : a.T <= 64 ? 64 : 128;
  const int box = std::min(nt, a.T);
  CUtensorMap xm;
  cudaError_t e = map8(&xm, x.codes, x.t, x.k, x.ld, box);
  if (e != cudaSuccess) return e;
  switch (nt) {
    case 16: return launch8<16, GATED, OT>(w, w2, xm, a, box, stream);
    case 32: return launch8<32, GATED, OT>(w, w2, xm, a, box, stream);
    case 64: return launch8<64, GATED, OT>(w, w2, xm, a, box, stream);
    default:
      if constexpr (GATED) return cudaErrorInvalidValue;   // (gemm8_pair_takes)
      else return launch8<128, GATED, OT>(w, w2, xm, a, box, stream);
  }
}

}  // namespace

// The pieces of k whose waves take the fewest k-blocks: a wave's beginning and end take about G8_ENDS of them.  (A tenth of a wave too many costs less than
// a wave, for the memory is what all wait for: 32 x 4096 x 14336 in 32 clusters of eight where 30 run at once 14.4 us, of four 15.5, of two 20.7)
cudaError_t gemm8_plan(int tiles, int G, int ctas, const int (&at_once)[4], int* pieces) {
  float least = -1.f;
  for (int i = 0; i < 4 && (i == 0 || G >= 2 << i); ++i) {
    if (at_once[i] < 1) continue;
    const float waves = (float)tiles / (float)(at_once[i] * ctas);   // (the answer is for one CTA an SM)
    const float cost = std::max(std::ceil(waves - 0.1f), 1.f) * (float)((G + (1 << i) - 1) / (1 << i) + G8_ENDS);
    if (least < 0.f || cost < least) *pieces = 1 << i, least = cost;
  }
  return least < 0.f ? cudaErrorLaunchOutOfResources : cudaSuccess;
}

cudaError_t gemm8_launch(const tgis_w8_rows& x, const tgis_w8_matrix& w, void* y, bool f32, int64_t ldy, const Gemm8Call& call, int num_sms,
                         cudaStream_t stream) {
  if (x.t <= 0 || w.n <= 0) return cudaSuccess;
  Gemm8Args a{};
  a.sx = x.scales; a.lds = x.lds; a.sw = w.scales;
  a.T = x.t; a.N = w.n; a.K = x.k; a.G = (x.k + W8_GROUP - 1) / W8_GROUP;
  a.y = y; a.ldy = ldy; a.status = call.status; a.stalled = call.stalled; a.early = call.early;
  if (gemm8_pair_takes(a.T, a.G, false)) return gemm8_pair_launch(x, w, a, f32, num_sms, stream);
  CUtensorMap wm;
  cudaError_t e = map8(&wm, w.codes, w.n, w.k, w.ld, 128);
  if (e != cudaSuccess) return e;
  return f32 ? launch_tokens<false, float>(wm, wm, x, a, stream) : launch_tokens<false, __nv_bfloat16>(wm, wm, x, a, stream);
}

cudaError_t gemm8_gated_launch(const tgis_w8_rows& x, const tgis_w8_matrix& gate, const tgis_w8_matrix& up, const tgis_w8_rows& out,
                               const Gemm8Call& call, int num_sms, cudaStream_t stream) {
  if (x.t <= 0 || gate.n <= 0) return cudaSuccess;
  Gemm8Args a{};
  a.sx = x.scales; a.lds = x.lds; a.sw = gate.scales; a.sw2 = up.scales;
  a.T = x.t; a.N = gate.n; a.K = x.k; a.G = (x.k + W8_GROUP - 1) / W8_GROUP;
  a.codes = (uint8_t*)out.codes; a.ldc = out.ld; a.sh = out.scales; a.ldh = out.lds;
  a.status = call.status; a.stalled = call.stalled; a.early = call.early;
  if (gemm8_pair_takes(a.T, a.G, true)) return gemm8_pair_gated_launch(x, gate, up, a, num_sms, stream);
  CUtensorMap wm, wm2;
  cudaError_t e = map8(&wm, gate.codes, gate.n, gate.k, gate.ld, 128);
  if (e == cudaSuccess) e = map8(&wm2, up.codes, up.n, up.k, up.ld, 128);
  if (e != cudaSuccess) return e;
  return launch_tokens<true, __nv_bfloat16>(wm, wm2, x, a, stream);
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
constexpr int MAX_ROWS = 1 << 22;

int check_size(const char* name, int64_t rows, int64_t k) {
  if (rows < 0 || rows > MAX_ROWS) return fail("%s: %lld rows are not in 0 .. %d", name, (long long)rows, MAX_ROWS);
  if (k < 1 || k > TGIS_W8_MAX_K) return fail("%s: rows of %lld numbers are not in 1 .. %d", name, (long long)k, TGIS_W8_MAX_K);
  return 0;
}
int check_codes(const char* name, const void* codes, const float* scales, int64_t ld, int64_t k) {
  if (codes == nullptr || !aligned(codes, 16) || ld < k || ld % 16 != 0 || ld >= 1ll << 39)
    return fail("%s: 16-byte aligned codes and rows of %lld bytes, a multiple of 16, are wanted", name, (long long)k);
  if (scales == nullptr || !aligned(scales, 4)) return fail("%s: fp32 scales are wanted", name);
  return 0;
}
int check_matrix(const char* name, const tgis_w8_matrix* w, bool made) {
  if (w == nullptr) return fail("%s: a record is wanted", name);
  if (check_size(name, w->n, w->k) != 0) return -1;
  if (w->n < 1) return fail("%s: no rows", name);
  return check_codes(name, w->codes, w->scales, w->ld, made ? (w->k + 127ll) / 128 * 128 : w->k);
}
int check_rows(const char* name, const tgis_w8_rows* x, bool made) {
  if (x == nullptr) return fail("%s: a record is wanted", name);
  if (check_size(name, x->t, x->k) != 0) return -1;
  if (x->t == 0) return 0;
  if (x->lds < x->t) return fail("%s: scales of %lld rows where %d are", name, (long long)x->lds, x->t);
  return check_codes(name, x->codes, x->scales, x->ld, made ? (x->k + 127ll) / 128 * 128 : x->k);
}
// (a CTA's features are written while others still read all of x)
int check_apart(const char* name, const tgis_w8_rows& x, const tgis_w8_rows& out) {
  return x.codes == out.codes || x.scales == out.scales ? fail("%s: x itself is not wanted", name) : 0;
}
int check_gated(const tgis_w8_rows* x, const tgis_w8_matrix* gate, const tgis_w8_matrix* up, const tgis_w8_rows* out) {
  if (check_rows("x", x, false) != 0 || check_matrix("gate", gate, false) != 0 || check_matrix("up", up, false) != 0 || check_rows("out", out, true) != 0) return -1;
  if (x->k != gate->k || x->k != up->k || gate->n != up->n) return fail("x has rows of %d numbers, gate is %d x %d, up %d x %d", x->k, gate->n, gate->k, up->n, up->k);
  if (out->t != x->t || out->k != gate->n) return fail("out: %d x %d is wanted, not %d x %d", x->t, gate->n, out->t, out->k);
  return 0;
}
int check_type(int32_t type) { return type == TGIS_W8_BF16 || type == TGIS_W8_F32 ? 0 : fail("type %d is not TGIS_W8_BF16 or TGIS_W8_F32", type); }
int check_plain(const char* name, const void* p, int32_t type, int64_t ld, int64_t k) {
  if (p == nullptr || !aligned(p, type == TGIS_W8_F32 ? 4 : 2) || ld < k) return fail("%s: rows of %lld numbers of the type are wanted", name, (long long)k);
  return 0;
}
int sms_of_device(int* out) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev);
  return done(e, "device");
}
}  // namespace

extern "C" {

const char* tgis_w8_last_error(void) { return t_err; }

int tgis_w8_quantise_rows(const void* x, int32_t type, int64_t ldx, const void* norm, float eps, const void* residual, int64_t ldr,
                          void* residual_out, int64_t ldro, const tgis_w8_rows* out, void* stream) {
  if (check_type(type) != 0 || check_rows("out", out, true) != 0) return -1;
  if (norm != nullptr && !(eps > 0.f && eps - eps == 0.f)) return fail("eps: a finite number above zero is wanted");
  if (norm != nullptr && !aligned(norm, 2)) return fail("norm: a bf16 pointer is wanted");
  if (out->t == 0) return 0;
  if (check_plain("x", x, type, ldx, out->k) != 0) return -1;
  if (residual != nullptr && (check_plain("residual", residual, type, ldr, out->k) != 0 || check_plain("residual_out", residual_out, type, ldro, out->k) != 0)) return -1;
  if (residual != nullptr && out->t > 1 && ((residual_out == residual && ldro != ldr) || (residual_out == x && ldro != ldx)))
    return fail("residual_out: a residual that is updated in place keeps its rows");
  int sms = 0;
  if (sms_of_device(&sms) != 0) return -1;
  const tgis::Rows8Args a{x, ldx, (const __nv_bfloat16*)norm, eps, residual, ldr, residual_out, ldro, (uint8_t*)out->codes, out->scales, out->ld, out->lds, out->t, out->k};
  return done(tgis::rows8_launch(a, type == TGIS_W8_F32, sms, (cudaStream_t)stream), "tgis_w8_quantise_rows");
}

int tgis_w8_quantise_weight(const void* w, int32_t type, int64_t ldw, const tgis_w8_matrix* out, void* stream) {
  if (check_type(type) != 0 || check_matrix("out", out, true) != 0 || check_plain("w", w, type, ldw, out->k) != 0) return -1;
  return done(tgis::weight8_launch(w, type == TGIS_W8_F32, ldw, out->n, out->k, (uint8_t*)out->codes, out->ld, out->scales, (cudaStream_t)stream), "tgis_w8_quantise_weight");
}

int tgis_w8_product(const tgis_w8_rows* x, const tgis_w8_matrix* w, void* y, int32_t type, int64_t ldy, int32_t* status, void* stream) {
  if (check_type(type) != 0 || check_rows("x", x, false) != 0 || check_matrix("w", w, false) != 0) return -1;
  if (x->k != w->k) return fail("x has rows of %d numbers, w of %d", x->k, w->k);
  if (x->t == 0) return 0;
  if (check_plain("y", y, type, ldy, w->n) != 0) return -1;
  int sms = 0;
  if (sms_of_device(&sms) != 0) return -1;
  return done(tgis::gemm8_launch(*x, *w, y, type == TGIS_W8_F32, ldy, tgis::Gemm8Call{status}, sms, (cudaStream_t)stream), "tgis_w8_product");
}

int tgis_w8_gated(const tgis_w8_rows* x, const tgis_w8_matrix* gate, const tgis_w8_matrix* up, const tgis_w8_rows* out, int32_t* status, void* stream) {
  if (check_gated(x, gate, up, out) != 0) return -1;
  if (x->t == 0) return 0;
  if (check_apart("out", *x, *out) != 0) return -1;
  int sms = 0;
  if (sms_of_device(&sms) != 0) return -1;
  return done(tgis::gemm8_gated_launch(*x, *gate, *up, *out, tgis::Gemm8Call{status}, sms, (cudaStream_t)stream), "tgis_w8_gated");
}

int tgis_w8_feed_forward(const tgis_w8_rows* x, const tgis_w8_matrix* gate, const tgis_w8_matrix* up, const tgis_w8_matrix* down,
                         const tgis_w8_rows* hidden, void* y, int32_t type, int64_t ldy, int32_t* status, void* stream) {
  if (check_type(type) != 0 || check_gated(x, gate, up, hidden) != 0 || check_matrix("down", down, false) != 0) return -1;
  if (hidden->k != down->k) return fail("hidden has rows of %d numbers, down of %d", hidden->k, down->k);
  if (x->t == 0) return 0;
  if (check_plain("y", y, type, ldy, down->n) != 0 || check_apart("hidden", *x, *hidden) != 0) return -1;
  int sms = 0;
  if (sms_of_device(&sms) != 0) return -1;
  const int rc = done(tgis::gemm8_gated_launch(*x, *gate, *up, *hidden, tgis::Gemm8Call{status}, sms, (cudaStream_t)stream), "tgis_w8_feed_forward");
  return rc != 0 ? rc : done(tgis::gemm8_launch(*hidden, *down, y, type == TGIS_W8_F32, ldy, tgis::Gemm8Call{status}, sms, (cudaStream_t)stream), "tgis_w8_feed_forward");
}

}  // extern "C"
