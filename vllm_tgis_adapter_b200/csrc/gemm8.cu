// y[t, n] = sum_g sx[t, g] sw[n / 128, g] sum_{k in g} cx[t, k] cw[n, k]: 8-bit weights (include/tgis_w8.h) times rows in 8 bits, and the gated
// form h = silu(x gate^T) * (x up^T), which leaves as rows in 8 bits.
//
// A CTA has a block of 128 weight rows (the MMA's A operand, a lane a row) and up to 256 rows of activations (B, a column each): with few tokens
// such a product is bound by its weight bytes, which are then read once.  The tensor cores (tcgen05 kind::f8f6f4) sum one group of 128 k, that
// is one k-block, in an accumulator; the epilogue's threads take it over, times both scales, into fp32 registers while the next one is summed
// in the other half of TMEM.  A tile's weights have one scale a k-block and a column has one, so a warp of its own puts their product where
// the epilogue reads it.  K is split over the CTAs of a cluster, whose sums meet in distributed shared memory in the order of k.
//
// Roles: warp 0 TMA producer, warp 1 MMA issuer and TMEM owner, warp 2 scales, warps 4..11 epilogue.  No wait is unbounded.
#include <stdarg.h>

#include <algorithm>

#include "launch.cuh"
#include "linear8.cuh"
#include "ptx.cuh"

namespace tgis {
namespace {

constexpr int G8_THREADS = 384, G8_WARPS = 12, G8_EPI = 4;   // epilogue: warps 4 .. 11
constexpr int G8_W_BYTES = 128 * W8_GROUP;                   // a k-block of a weight tile
constexpr int G8_SLOTS = 4;                                  // k-blocks whose scales are there

// D[tmem] (+)= A[smem] B[smem], e4m3, fp32 sums
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// kind::f8f6f4: C = F32, A = B = E4M3, both K-major
__host__ __device__ constexpr uint32_t idesc_f8(uint32_t m, uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((m >> 4) << 24); }

__device__ __forceinline__ void tmem_ld_x8(uint32_t at, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(at));
}
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t* r) {
  if constexpr (N == 8) {
    tmem_ld_x8(at, r);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 16) tmem_ld_32x32b_x16(at + i, r + i);
  }
}

__device__ __forceinline__ void say_stalled8(const Gemm8Args& a) {
  if (a.status != nullptr) atomicOr(a.status, TGIS_W8_STALLED);
  if (a.stalled != nullptr) {
    *reinterpret_cast<volatile int*>(a.stalled) = 1;
    __threadfence_system();
  }
}
__device__ __forceinline__ bool wait8(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (clock64() - t0 > 4000000000ll) return false;   // about two seconds: no wait of a working pipeline is that long
  }
  return true;
}

__device__ __forceinline__ float swiglu(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// Tokens of a tile, and what follows from them.  Two CTAs share an SM while their accumulators (TMEM has 512 columns) and registers allow.
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
  const int rank = (int)cluster_ctarank(), S = (int)gridDim.z;        // cluster: the CTAs of blockIdx.z
  const int nb = (int)blockIdx.x, t0 = (int)blockIdx.y * NT;
  const int kb0 = (int)((long long)rank * a.G / S), kb1 = (int)((long long)(rank + 1) * a.G / S);

  if (warp == 0 && elect_one()) {
    tma_prefetch_desc(&wmap);
    if (GATED) tma_prefetch_desc(&wmap2);
    tma_prefetch_desc(&xmap);
  }
  if (warp == 1) {
    if (elect_one()) {
      for (int i = 0; i < F::STAGES; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&tmem_full[i], 1);
        mbar_init(&tmem_empty[i], G8_WARPS - G8_EPI);
      }
      for (int i = 0; i < G8_SLOTS; ++i) {
        mbar_init(&scale_full[i], 1);
        mbar_init(&scale_empty[i], G8_WARPS - G8_EPI);
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

  if (warp == 0) {
    // ===================== TMA producer =====================
    if (elect_one()) {
      const uint64_t once = policy_evict_first();
      const uint32_t bytes = (uint32_t)(G8_W_BYTES * F::HALVES + x_box * W8_GROUP);
      auto load_w = [&](int s, int kb) {
        mbar_arrive_expect_tx(&full[s], bytes);
        tma_load_2d_hint(&wmap, &full[s], smem + s * F::STAGE, kb * W8_GROUP, nb * 128, once);
        if (GATED) tma_load_2d_hint(&wmap2, &full[s], smem + s * F::STAGE + G8_W_BYTES, kb * W8_GROUP, nb * 128, once);
      };
      auto load_x = [&](int s, int kb) { tma_load_2d(&xmap, &full[s], smem + s * F::STAGE + G8_W_BYTES * F::HALVES, kb * W8_GROUP, t0); };
      const int pre = min(kb1 - kb0, F::STAGES);
      if (!a.early) griddep_wait();
      for (int i = 0; i < pre; ++i) load_w(i, kb0 + i);
      if (a.early) griddep_wait();
      for (int i = 0; i < pre; ++i) load_x(i, kb0 + i);
      int s = pre % F::STAGES;
      uint32_t phase = pre == F::STAGES ? 1 : 0;
      for (int kb = kb0 + pre; kb < kb1; ++kb) {
        if (!wait8(&empty[s], phase ^ 1)) {
          *gave_up = 1;
          break;
        }
        load_w(s, kb);
        load_x(s, kb);
        if (++s == F::STAGES) s = 0, phase ^= 1;
      }
    }
  } else if (warp == 1) {
    // ===================== MMA issuer =====================
    if (elect_one()) {
      constexpr uint32_t idesc = idesc_f8(128, NT);
      const uint32_t ring = smem_u32(smem);
      int s = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int i = kb - kb0, buf = i & 1;
        if (!wait8(&tmem_empty[buf], (uint32_t)(i >> 1 & 1) ^ 1) || !wait8(&full[s], phase)) {
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
  } else if (warp == 2) {
    // ===================== scales: sx[t] sw of the k-blocks to come =====================
    griddep_wait();
    const float* sw = a.sw + (size_t)nb * a.G;
    const float* sw2 = GATED ? a.sw2 + (size_t)nb * a.G : nullptr;
    constexpr int EACH = (NT + 31) / 32;
    float x[EACH], w = 0.f, w2 = 0.f;
    auto load = [&](int kb) {
      w = sw[kb];
      if (GATED) w2 = sw2[kb];
#pragma unroll
      for (int i = 0; i < EACH; ++i) x[i] = i * 32 + lane < NT && t0 + i * 32 + lane < a.T ? a.sx[(size_t)kb * a.lds + t0 + i * 32 + lane] : 0.f;
    };
    load(kb0);
    for (int kb = kb0; kb < kb1; ++kb) {
      const int i = kb - kb0, slot = i % G8_SLOTS;
      if (!__all_sync(0xffffffffu, wait8(&scale_empty[slot], (uint32_t)(i / G8_SLOTS & 1) ^ 1))) {
        if (lane == 0) *gave_up = 1;
        break;
      }
      float* to = scale + slot * F::HALVES * NT;
#pragma unroll
      for (int j = 0; j < EACH; ++j)
        if (j * 32 + lane < NT) {
          to[j * 32 + lane] = x[j] * w;
          if (GATED) to[NT + j * 32 + lane] = x[j] * w2;
        }
      __syncwarp();
      if (lane == 0) mbar_arrive(&scale_full[slot]);
      if (kb + 1 < kb1) load(kb + 1);
    }
  } else if (warp >= G8_EPI) {
    // ===================== epilogue: lane = weight row, column = token =====================
    const int quarter = warp & 3, half = (warp - G8_EPI) >> 2, col0 = half * F::NC;   // gated: the other half is the other matrix
    float acc[F::NC];
#pragma unroll
    for (int j = 0; j < F::NC; ++j) acc[j] = 0.f;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int i = kb - kb0, buf = i & 1, slot = i % G8_SLOTS;
      ok = wait8(&scale_full[slot], (uint32_t)(i / G8_SLOTS & 1)) && wait8(&tmem_full[buf], (uint32_t)(i >> 1 & 1));
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0) *gave_up = 1;
        break;
      }
      tc_fence_after();
      const uint32_t at = tmem + buf * F::COLS + col0 + ((uint32_t)(quarter * 32) << 16);
      const float4* sc = reinterpret_cast<const float4*>(scale + slot * F::HALVES * NT + col0);
      constexpr int STEP = F::NC < 32 ? F::NC : 32;
#pragma unroll
      for (int c = 0; c < F::NC; c += STEP) {
        uint32_t r[STEP];
        tmem_ld<STEP>(at + c, r);
        tmem_ld_wait();
        if (c + STEP == F::NC) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&tmem_empty[buf]);
        }
#pragma unroll
        for (int j = 0; j < STEP; j += 4) {
          const float4 f = sc[(c + j) / 4];
          acc[c + j] += __uint_as_float(r[j]) * f.x;
          acc[c + j + 1] += __uint_as_float(r[j + 1]) * f.y;
          acc[c + j + 2] += __uint_as_float(r[j + 2]) * f.z;
          acc[c + j + 3] += __uint_as_float(r[j + 3]) * f.w;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&scale_empty[slot]);
    }
    // the ring is done with once the last accumulator is there: the sums take its place, [matrix][token][weight row]
    if (!*gave_up) {
      float* to = reinterpret_cast<float*>(smem) + (size_t)col0 * 128 + quarter * 32 + lane;
#pragma unroll
      for (int j = 0; j < F::NC; ++j) to[j * 128] = acc[j];
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*gave_up) {   // copies and MMAs in flight, all issued by now, are done long before this millisecond is over
    for (const long long t1 = clock64(); clock64() - t1 < 2000000ll;) {}
    if (threadIdx.x == 0) say_stalled8(a);
  }
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<F::TMEM>(tmem);
  }
  // ===================== the cluster's sums -> y or h: a warp a token, four weight rows a lane =====================
  griddep_wait();
  const uint32_t mine = smem_u32(smem) + lane * 16;
  for (int t = rank * G8_WARPS + warp; t < NT && t0 + t < a.T; t += S * G8_WARPS) {
    float v[F::HALVES][4] = {};
    for (int r = 0; r < S; ++r) {
      const uint32_t from = dsmem_addr(mine, r);
#pragma unroll
      for (int h = 0; h < F::HALVES; ++h) {
        const float4 p = ld_dsmem_f4(from + (uint32_t)(h * NT + t) * 512);
        v[h][0] += p.x; v[h][1] += p.y; v[h][2] += p.z; v[h][3] += p.w;
      }
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
      codes(h, s, c);
      *reinterpret_cast<uint32_t*>(a.codes + (size_t)(t0 + t) * a.ldc + n) = c[0];
      if (lane == 0) a.sh[(size_t)nb * a.ldh + t0 + t] = s;
    } else {
      OT* y = reinterpret_cast<OT*>(a.y) + (size_t)(t0 + t) * a.ldy + n;
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
  cluster_sync_all();   // nobody leaves while its sums are read
}

// K-major operand rows of 128 codes a box
cudaError_t map8(CUtensorMap* out, const void* codes, int64_t rows, int64_t cols, int64_t ld, int box) {
  return make_tmap_u8_2d(out, codes, (uint64_t)rows, (uint64_t)cols, (uint64_t)ld, (uint32_t)box, W8_GROUP) == 0 ? cudaSuccess : cudaErrorInvalidValue;
}

template <int NT, bool GATED, class OT>
cudaError_t launch8(const CUtensorMap& w, const CUtensorMap& w2, const CUtensorMap& x, const Gemm8Args& a, int box, int num_sms, cudaStream_t stream) {
  using F = Form<NT, GATED>;
  static OncePerDevice once;
  cudaError_t e = once([] { return cudaFuncSetAttribute(gemm8_kernel<NT, GATED, OT>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM); });
  if (e != cudaSuccess) return e;
  const int tiles = (a.N + 127) / 128, x_tiles = (a.T + NT - 1) / NT;
  if (x_tiles > 65535) return cudaErrorInvalidValue;
  // as many CTAs as run at once, and two k-blocks for each at least
  int S = 1;
  while (S < 8 && (long long)tiles * x_tiles * S * 2 <= (long long)num_sms * F::CTAS && a.G >= S * 4) S *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)tiles, (unsigned)x_tiles, (unsigned)S);
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
cudaError_t launch_tokens(const CUtensorMap& w, const CUtensorMap& w2, const tgis_w8_rows& x, const Gemm8Args& a, int num_sms, cudaStream_t stream) {
  const int nt = a.T <= 16 ? 16 : a.T <= 32 ? 32 : a.T <= 64 ? 64 : a.T <= 128 || GATED ? 128 : 256;
  const int box = std::min(nt, a.T);
  CUtensorMap xm;
  cudaError_t e = map8(&xm, x.codes, x.t, x.k, x.ld, box);
  if (e != cudaSuccess) return e;
  switch (nt) {
    case 16: return launch8<16, GATED, OT>(w, w2, xm, a, box, num_sms, stream);
    case 32: return launch8<32, GATED, OT>(w, w2, xm, a, box, num_sms, stream);
    case 64: return launch8<64, GATED, OT>(w, w2, xm, a, box, num_sms, stream);
    case 128: return launch8<128, GATED, OT>(w, w2, xm, a, box, num_sms, stream);
    default:
      if constexpr (GATED) return cudaErrorInvalidValue;
      else return launch8<256, GATED, OT>(w, w2, xm, a, box, num_sms, stream);
  }
}

}  // namespace

cudaError_t gemm8_launch(const tgis_w8_rows& x, const tgis_w8_matrix& w, void* y, bool f32, int64_t ldy, int32_t* status, int* stalled, bool early,
                         int num_sms, cudaStream_t stream) {
  if (x.t <= 0 || w.n <= 0) return cudaSuccess;
  Gemm8Args a{};
  a.sx = x.scales; a.lds = x.lds; a.sw = w.scales;
  a.T = x.t; a.N = w.n; a.K = x.k; a.G = (x.k + W8_GROUP - 1) / W8_GROUP;
  a.y = y; a.ldy = ldy; a.status = status; a.stalled = stalled; a.early = early;
  CUtensorMap wm;
  cudaError_t e = map8(&wm, w.codes, w.n, w.k, w.ld, 128);
  if (e != cudaSuccess) return e;
  return f32 ? launch_tokens<false, float>(wm, wm, x, a, num_sms, stream) : launch_tokens<false, __nv_bfloat16>(wm, wm, x, a, num_sms, stream);
}

cudaError_t gemm8_gated_launch(const tgis_w8_rows& x, const tgis_w8_matrix& gate, const tgis_w8_matrix& up, const tgis_w8_rows& out, int32_t* status,
                               int* stalled, bool early, int num_sms, cudaStream_t stream) {
  if (x.t <= 0 || gate.n <= 0) return cudaSuccess;
  Gemm8Args a{};
  a.sx = x.scales; a.lds = x.lds; a.sw = gate.scales; a.sw2 = up.scales;
  a.T = x.t; a.N = gate.n; a.K = x.k; a.G = (x.k + W8_GROUP - 1) / W8_GROUP;
  a.codes = (uint8_t*)out.codes; a.ldc = out.ld; a.sh = out.scales; a.ldh = out.lds;
  a.status = status; a.stalled = stalled; a.early = early;
  CUtensorMap wm, wm2;
  cudaError_t e = map8(&wm, gate.codes, gate.n, gate.k, gate.ld, 128);
  if (e == cudaSuccess) e = map8(&wm2, up.codes, up.n, up.k, up.ld, 128);
  if (e != cudaSuccess) return e;
  return launch_tokens<true, __nv_bfloat16>(wm, wm2, x, a, num_sms, stream);
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
constexpr int MAX_ROWS = 1 << 22;   // (65535 tiles of a gated product's 128)

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
  return done(tgis::gemm8_launch(*x, *w, y, type == TGIS_W8_F32, ldy, status, nullptr, false, sms, (cudaStream_t)stream), "tgis_w8_product");
}

int tgis_w8_gated(const tgis_w8_rows* x, const tgis_w8_matrix* gate, const tgis_w8_matrix* up, const tgis_w8_rows* out, int32_t* status, void* stream) {
  if (check_rows("x", x, false) != 0 || check_matrix("gate", gate, false) != 0 || check_matrix("up", up, false) != 0 || check_rows("out", out, true) != 0) return -1;
  if (x->k != gate->k || x->k != up->k || gate->n != up->n) return fail("x has rows of %d numbers, gate is %d x %d, up %d x %d", x->k, gate->n, gate->k, up->n, up->k);
  if (out->t != x->t || out->k != gate->n) return fail("out: %d x %d is wanted, not %d x %d", x->t, gate->n, out->t, out->k);
  if (x->t == 0) return 0;
  int sms = 0;
  if (sms_of_device(&sms) != 0) return -1;
  return done(tgis::gemm8_gated_launch(*x, *gate, *up, *out, status, nullptr, false, sms, (cudaStream_t)stream), "tgis_w8_gated");
}

int tgis_w8_feed_forward(const tgis_w8_rows* x, const tgis_w8_matrix* gate, const tgis_w8_matrix* up, const tgis_w8_matrix* down,
                         const tgis_w8_rows* hidden, void* y, int32_t type, int64_t ldy, int32_t* status, void* stream) {
  // (all of it is checked before the first launch)
  if (check_type(type) != 0 || check_matrix("down", down, false) != 0 || check_rows("hidden", hidden, true) != 0) return -1;
  if (hidden->k != down->k) return fail("hidden has rows of %d numbers, down of %d", hidden->k, down->k);
  if (hidden->t > 0 && check_plain("y", y, type, ldy, down->n) != 0) return -1;
  if (tgis_w8_gated(x, gate, up, hidden, status, stream) != 0) return -1;
  return tgis_w8_product(hidden, down, y, type, ldy, status, stream);
}

}  // extern "C"
