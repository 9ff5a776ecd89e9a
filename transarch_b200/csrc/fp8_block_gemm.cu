// Products of 8-bit matrices with block scales, and the quantisers that make their operands.
//
//   y[m, n] = sum_g  sa[m, g] * sw[n / 128, g] * sum_{k in block g} a[m, k] * w[n, k]
//
// a: activations, e4m3 [M, K], one fp32 scale for 128 values of a row; w: weights, e4m3 [N, K], one fp32 scale for
// a block of 128 x 128.  Blocks at the right and lower edge may be partial.  The scales are arbitrary fp32 numbers, so
// a block's product has to leave the tensor pipe before it is scaled: the inner sum of every 128-deep block is one
// accumulator in TMEM (4 MMAs of K = 32), and fp32 registers hold the outer sum.
//
// Orientation: 128 weight rows are the UMMA M dimension (one TMEM lane and one epilogue thread for an output column n),
// NT tokens are N.  A decode batch is then a narrow tile that still streams whole weight tiles, the weight scale is
// one number for a tile and block, and the token scales are shared by all threads of the tile (read from shared memory
// four at a time).  NT is 16 .. 256 by M.
//
// Few tiles (decode, narrow projections) split the blocks of K over the 2 - 8 CTAs of a cluster: each CTA keeps its
// partial sums in its own shared memory and adds up its share of the tokens over the cluster in rank order, so the
// result does not depend on timing and no workspace exists.
//
// Roles (352 threads): warp 0 TMA loads, warp 1 MMA, warp 2 scales, warps 3-10 accumulate (two warps per TMEM lane
// quadrant, half of the token columns each).  Every wait is bounded.
#include <stdio.h>

#include "latent_cache.cuh"

namespace b200dsa {

void set_last_error(const char* msg);

// ---------------------------------------------------------------------------------------- products
constexpr int kGemmThreads = 352;
constexpr int kGemmScaleSlots = 8;

struct GemmParams {
  const float* a_scale;        // sa[m, g] at m * sa_m + g * sa_g
  int64_t sa_m, sa_g;
  const float* w_scale;        // sw[r, g] at r * sw_r + g * sw_g
  int64_t sw_r, sw_g;
  void* out;                   // [M, N], rows ldo elements apart
  int64_t ldo;
  int out_f32, out_pair;       // out_pair: bf16 rows start on 4-byte boundaries
  int m, n, blocks;            // blocks of K
  int m_tiles, n_tiles, splits;
  int32_t* status;
};

template <int NT>
struct GemmShape {
  static constexpr int kWBytes = 128 * 128, kABytes = NT * 128, kStageBytes = kWBytes + kABytes;
  static constexpr int kStages = NT == 256 ? 4 : NT == 128 ? 6 : 8;
  static constexpr int kAccBufs = NT == 256 ? 2 : 4;
  static constexpr uint32_t kTmemCols = NT * kAccBufs < 32 ? 32 : NT * kAccBufs;
  static constexpr int kCols = NT / 2;                        // token columns of one accumulating warp
  static constexpr int kScaleOff = kStages * kStageBytes;
  static constexpr int kBarOff = kScaleOff + kGemmScaleSlots * NT * 4;
  static constexpr int kSmem = kBarOff + 256 + 1024;
  // partial sums of a split tile live where the operand ring was: NT tokens x 128 columns fp32
  static_assert(NT > 128 || NT * 128 * 4 <= kStages * kStageBytes, "partial sums must fit the operand ring");
};

__device__ __forceinline__ uint32_t gemm_cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void gemm_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float gemm_ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t r;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r) : "memory");
  return v;
}
__device__ __forceinline__ void tmem_ld_32x8(uint32_t taddr, uint32_t (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(taddr)
               : "memory");
}

// One output value pair for tokens t and t + 1 of thread column n: neighbouring lanes swap one value, so that each
// lane stores two neighbouring columns of one token.
__device__ __forceinline__ void store_bf16_pair(const GemmParams& p, float v0, float v1, int tok, int n, int lane) {
  const bool odd = lane & 1;
  const float other = __shfl_xor_sync(0xffffffffu, odd ? v0 : v1, 1);
  const int t = odd ? tok + 1 : tok;
  const int c = odd ? n - 1 : n;
  const float x = odd ? other : v0, y = odd ? v1 : other;
  if (t >= p.m || c >= p.n) return;
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + static_cast<int64_t>(t) * p.ldo + c;
  if (p.out_pair && c + 1 < p.n) {
    *reinterpret_cast<__nv_bfloat162*>(o) = __floats2bfloat162_rn(x, y);
  } else {
    o[0] = __float2bfloat16_rn(x);
    if (c + 1 < p.n) o[1] = __float2bfloat16_rn(y);
  }
}

template <int NT>
__global__ void __launch_bounds__(kGemmThreads, 1)
fp8_block_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_a,
                      const GemmParams p) {
  using S = GemmShape<NT>;
  pdl_launch_dependents();
  extern __shared__ uint8_t smem_dyn[];
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;
  const uint32_t smem_base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
  uint8_t* smem_al = smem_dyn + (smem_base - smem_u32(smem_dyn));
  float* s_scale = reinterpret_cast<float*>(smem_al + S::kScaleOff);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_al + S::kBarOff);
  uint64_t* full = bars;                          // [stages] bytes of an operand pair
  uint64_t* empty = full + S::kStages;            // [stages] MMAs of the stage retired
  uint64_t* acc_full = empty + S::kStages;        // [bufs]   block product complete
  uint64_t* acc_empty = acc_full + S::kAccBufs;   // [bufs]   eight warps have read it
  uint64_t* sc_full = acc_empty + S::kAccBufs;    // [slots]  32 lanes have stored a block's scales
  uint64_t* sc_empty = sc_full + kGemmScaleSlots; // [slots]  eight warps are done with them
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &s_abort;
  if (tid == 0) {
    s_abort = 0;
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < S::kAccBufs; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], 8);
    }
    for (int s = 0; s < kGemmScaleSlots; ++s) {
      mbar_init(&sc_full[s], 32);
      mbar_init(&sc_empty[s], 8);
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(&s_tmem_base, S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = s_tmem_base;
  pdl_wait_prior();      // nothing above touches global memory: as a dependent launch it overlaps the previous kernel

  // tiles: neighbouring CTAs share a token tile's neighbours in N, i.e. the same activations
  const int n_work = p.m_tiles * p.n_tiles;
  const int rank = p.splits > 1 ? static_cast<int>(gemm_cluster_rank()) : 0;
  const int first = blockIdx.x / p.splits, stride = gridDim.x / p.splits;
  const int b_lo = static_cast<int>(static_cast<int64_t>(p.blocks) * rank / p.splits);
  const int b_hi = static_cast<int>(static_cast<int64_t>(p.blocks) * (rank + 1) / p.splits);

  if (warp == 0) {
    // ------------------------------------------------------------------ loads
    int it = 0;
    bool ok = true;
    for (int w = first; ok && w < n_work; w += stride) {
      const int n0 = (w % p.n_tiles) * 128, m0 = (w / p.n_tiles) * NT;
      for (int b = b_lo; b < b_hi; ++b, ++it) {
        const int s = it % S::kStages;
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], ((it / S::kStages) & 1) ^ 1, abort_flag));
        if (!ok) break;
        if (elect_one()) {
          uint8_t* dst = smem_al + s * S::kStageBytes;
          mbar_arrive_expect_tx(&full[s], S::kStageBytes);
          tma_load_2d(dst, &tmap_w, &full[s], b * 128, n0);
          tma_load_2d(dst + S::kWBytes, &tmap_a, &full[s], b * 128, m0);
        }
        __syncwarp();
      }
    }
    // whatever ended the loop, the copies in flight land before the shared memory is given up
    for (int j = it > S::kStages ? it - S::kStages : 0; j < it; ++j) {
      const long long t0 = clock64();
      while (!mbar_test(&full[j % S::kStages], (j / S::kStages) & 1) && clock64() - t0 < kWaitLimitCycles) {
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA
    constexpr uint32_t idesc = make_idesc(kFmtE4M3, kFmtE4M3, 128, NT);
    int it = 0;
    bool ok = true;
    for (int w = first; ok && w < n_work; w += stride) {
      for (int b = b_lo; b < b_hi; ++b, ++it) {
        const int s = it % S::kStages, buf = it % S::kAccBufs;
        ok = __all_sync(0xffffffffu, mbar_wait(&acc_empty[buf], ((it / S::kAccBufs) & 1) ^ 1, abort_flag) &&
                                         mbar_wait(&full[s], (it / S::kStages) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t wd = make_desc_k_sw128(smem_base + s * S::kStageBytes);
          const uint64_t ad = make_desc_k_sw128(smem_base + s * S::kStageBytes + S::kWBytes);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f8f6f4_ss(tmem_base + buf * NT, wd + 2 * kk, ad + 2 * kk, idesc, kk != 0);
          tc_commit(&empty[s]);
          tc_commit(&acc_full[buf]);
        }
        __syncwarp();
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ scales, four blocks of loads in flight
    constexpr int kPer = NT <= 32 ? 1 : NT / 32;
    constexpr int kAhead = 4;
    int it = 0;
    bool ok = true;
    for (int w = first; ok && w < n_work; w += stride) {
      const int nb = w % p.n_tiles, m0 = (w / p.n_tiles) * NT;
      for (int b0 = b_lo; ok && b0 < b_hi; b0 += kAhead) {
        float v[kAhead][kPer];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int b = b0 + u;
          const float ws = b < b_hi ? __ldg(p.w_scale + nb * p.sw_r + b * p.sw_g) : 0.f;
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            const int t = m0 + lane + 32 * j;
            v[u][j] = b < b_hi && t < p.m && lane + 32 * j < NT ? ws * __ldg(p.a_scale + t * p.sa_m + b * p.sa_g) : 0.f;
          }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (b0 + u >= b_hi) break;
          const int sl = it % kGemmScaleSlots;
          ok = __all_sync(0xffffffffu, mbar_wait(&sc_empty[sl], ((it / kGemmScaleSlots) & 1) ^ 1, abort_flag));
          if (!ok) break;
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if (lane + 32 * j < NT) s_scale[sl * NT + lane + 32 * j] = v[u][j];
          mbar_arrive(&sc_full[sl]);
          ++it;
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ accumulation and output
    const int wq = warp & 3, half = (warp - 3) >> 2;       // warps 3..6: first half of the tokens, 7..10: second
    const uint32_t lane_addr = static_cast<uint32_t>(wq * 32) << 16;
    const int row = wq * 32 + lane, col0 = half * S::kCols;
    constexpr int kChunk = S::kCols < 16 ? 8 : 16;
    int it = 0;
    bool ok = true;
    for (int w = first; ok && w < n_work; w += stride) {
      float acc[S::kCols];
#pragma unroll
      for (int j = 0; j < S::kCols; ++j) acc[j] = 0.f;
      for (int b = b_lo; b < b_hi; ++b, ++it) {
        const int buf = it % S::kAccBufs, sl = it % kGemmScaleSlots;
        ok = __all_sync(0xffffffffu, mbar_wait(&sc_full[sl], (it / kGemmScaleSlots) & 1, abort_flag) &&
                                         mbar_wait(&acc_full[buf], (it / S::kAccBufs) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const float4* sc = reinterpret_cast<const float4*>(s_scale + sl * NT + col0);
#pragma unroll
        for (int c = 0; c < S::kCols; c += kChunk) {
          uint32_t v[kChunk];
          if constexpr (kChunk == 8) tmem_ld_32x8(tmem_base + lane_addr + buf * NT + col0 + c, v);
          else tmem_ld_32x16(tmem_base + lane_addr + buf * NT + col0 + c, v);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < kChunk; j += 4) {
            const float4 f = sc[(c + j) >> 2];
            acc[c + j] = fmaf(__uint_as_float(v[j]), f.x, acc[c + j]);
            acc[c + j + 1] = fmaf(__uint_as_float(v[j + 1]), f.y, acc[c + j + 1]);
            acc[c + j + 2] = fmaf(__uint_as_float(v[j + 2]), f.z, acc[c + j + 2]);
            acc[c + j + 3] = fmaf(__uint_as_float(v[j + 3]), f.w, acc[c + j + 3]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&acc_empty[buf]);
          mbar_arrive(&sc_empty[sl]);
        }
      }
      if (!ok) break;
      const int n = (w % p.n_tiles) * 128 + row, m0 = (w / p.n_tiles) * NT + col0;
      if (p.splits > 1) {
        // every MMA of this CTA has read its operands: the ring holds the partial sums now, [token][128]
        float* part = reinterpret_cast<float*>(smem_al);
#pragma unroll
        for (int j = 0; j < S::kCols; ++j) part[(col0 + j) * 128 + row] = acc[j];
      } else if (p.out_f32) {
#pragma unroll
        for (int j = 0; j < S::kCols; ++j)
          if (n < p.n && m0 + j < p.m) static_cast<float*>(p.out)[static_cast<int64_t>(m0 + j) * p.ldo + n] = acc[j];
      } else {
#pragma unroll
        for (int j = 0; j < S::kCols; j += 2) store_bf16_pair(p, acc[j], acc[j + 1], m0 + j, n, lane);
      }
    }
  }

  __syncwarp();
  if (p.splits > 1) {
    // one tile per cluster: add the partial sums of this CTA's share of the tokens in rank order
    gemm_cluster_sync();
    if (warp >= 3) {
      const int t = tid - 96, row = t & 127, pair = t >> 7;           // 256 threads: two token pairs at a time
      const int n0 = (first % p.n_tiles) * 128, m0 = (first / p.n_tiles) * NT;
      const int per = (NT / 2 + p.splits - 1) / p.splits;             // token pairs of a CTA
      const uint32_t base = smem_base + row * 4;
      for (int q = rank * per + pair; q < min((rank + 1) * per, NT / 2); q += 2) {
        if (m0 + 2 * q >= p.m) break;
        float v0 = 0.f, v1 = 0.f;
        for (int r = 0; r < p.splits; ++r) {
          v0 += gemm_ld_cluster(base + (2 * q) * 512, r);
          v1 += gemm_ld_cluster(base + (2 * q + 1) * 512, r);
        }
        if (p.out_f32) {
          float* o = static_cast<float*>(p.out) + static_cast<int64_t>(m0 + 2 * q) * p.ldo + n0 + row;
          if (n0 + row < p.n) {
            o[0] = v0;
            if (m0 + 2 * q + 1 < p.m) o[p.ldo] = v1;
          }
        } else {
          store_bf16_pair(p, v0, v1, m0 + 2 * q, n0 + row, lane);
        }
      }
    }
    gemm_cluster_sync();               // nobody leaves while a peer reads its shared memory
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, S::kTmemCols);
  if (tid == 0 && s_abort) atomicMax(p.status, kDevWaitTimeout);
}

template <int NT>
static cudaError_t gemm_launch(const CUtensorMap& mw, const CUtensorMap& ma, const GemmParams& p, const DeviceInfo& dev,
                               bool dependent, cudaStream_t stream) {
  using S = GemmShape<NT>;
  static OncePerDevice once;
  cudaError_t e = once.run(dev.index, [] {
    return cudaFuncSetAttribute(fp8_block_gemm_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  });
  if (e != cudaSuccess) return e;
  const int sms = dev.sms;
  const int tiles = p.m_tiles * p.n_tiles;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.splits > 1 ? tiles * p.splits : (tiles < sms ? tiles : sms));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (p.splits > 1) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = p.splits;
    attr[na].val.clusterDim.y = 1;
    attr[na].val.clusterDim.z = 1;
    ++na;
  }
  if (dependent || pdl_enabled()) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na].val.programmaticStreamSerializationAllowed = 1;
    ++na;
  }
  cfg.attrs = attr;
  cfg.numAttrs = na;
  e = cudaLaunchKernelEx(&cfg, fp8_block_gemm_kernel<NT>, mw, ma, p);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

// ---------------------------------------------------------------------------------------- quantisers
// Rows: a warp takes two groups of 128 values at a time (lane = 8 values, 16 lanes a group) of one row; the eight warps
// of a CTA are eight neighbouring rows, whose scales are neighbours in the column-major scale matrix.
constexpr int kQuantPairs = 4;         // group pairs of a warp, loads of all of them in flight

struct QuantRowsParams {
  const void* in;
  int in_f32, in_vec;
  int64_t in_stride, m;
  int k;
  uint8_t* q;                  // [m, k]
  float* scale;                // [m, g] at g * ld + m
  int64_t ld;
  int use_ue8m0;
};

__device__ __forceinline__ void quant_load8(const QuantRowsParams& p, int64_t i, float (&x)[8]) {
  if (p.in_f32) {
    const float* q = static_cast<const float*>(p.in) + i;
    if (p.in_vec) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(q)), b = __ldg(reinterpret_cast<const float4*>(q) + 1);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __ldg(q + j);
    }
  } else {
    const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.in) + i;
    if (p.in_vec) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(q));
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = __uint_as_float(w[j] << 16);
        x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __bfloat162float(q[j]);
    }
  }
}

__global__ void __launch_bounds__(256) fp8_quantise_rows_kernel(const QuantRowsParams p) {
  pdl_launch_dependents();
  pdl_wait_prior();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= p.m) return;
  const int lane = threadIdx.x & 31;
  const int k0 = blockIdx.y * (kQuantPairs * 256) + lane * 8;
  float x[kQuantPairs][8];
#pragma unroll
  for (int u = 0; u < kQuantPairs; ++u) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[u][j] = 0.f;
    if (k0 + 256 * u < p.k) quant_load8(p, row * p.in_stride + k0 + 256 * u, x[u]);   // K is a multiple of 16
  }
#pragma unroll
  for (int u = 0; u < kQuantPairs; ++u) {
    const int k = k0 + 256 * u;
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[u][j]));
    for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    float scale = __fdiv_rn(fmaxf(amax, 1e-10f), 448.0f);
    if (p.use_ue8m0) scale = pow2_at_least(scale);
    if (k >= p.k) continue;
    uint2 codes;
    codes.x = quant_e4m3x4(x[u][0], x[u][1], x[u][2], x[u][3], scale);
    codes.y = quant_e4m3x4(x[u][4], x[u][5], x[u][6], x[u][7], scale);
    *reinterpret_cast<uint2*>(p.q + row * p.k + k) = codes;
    if ((lane & 15) == 0) p.scale[(k >> 7) * p.ld + row] = scale;
  }
}

// Blocks of 128 x 128 (weights): one CTA a block, 64 values a thread, partial blocks at the edges.
__global__ void __launch_bounds__(256) fp8_quantise_blocks_kernel(const void* in, int in_f32, int64_t in_stride, int n,
                                                                  int k, int use_ue8m0, uint8_t* __restrict__ q,
                                                                  float* __restrict__ scale, int groups) {
  pdl_launch_dependents();
  pdl_wait_prior();
  __shared__ float s_max[8];
  const int r0 = blockIdx.y * 128 + (threadIdx.x >> 5) * 16, c0 = blockIdx.x * 128 + (threadIdx.x & 31) * 4;
  float x[16][4];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float v = 0.f;
      if (r0 + i < n && c0 + j < k) {
        const int64_t at = (r0 + i) * in_stride + c0 + j;
        v = in_f32 ? __ldg(static_cast<const float*>(in) + at)
                   : __bfloat162float(static_cast<const __nv_bfloat16*>(in)[at]);
      }
      x[i][j] = v;
      amax = fmaxf(amax, fabsf(v));
    }
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, s_max[i]);
  float sc = __fdiv_rn(fmaxf(amax, 1e-10f), 448.0f);
  if (use_ue8m0) sc = pow2_at_least(sc);
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (r0 + i < n && c0 < k)                            // K is a multiple of 16: four codes are in or out together
      *reinterpret_cast<uint32_t*>(q + static_cast<int64_t>(r0 + i) * k + c0) =
          quant_e4m3x4(x[i][0], x[i][1], x[i][2], x[i][3], sc);
  if (threadIdx.x == 0) scale[static_cast<int64_t>(blockIdx.y) * groups + blockIdx.x] = sc;
}

static int gemm_rc(cudaError_t e) {
  if (e == cudaSuccess) return B200DSA_OK;
  set_last_error(cudaGetErrorString(e));
  return B200DSA_ECUDA;
}

// Tokens of a tile and CTAs of a cluster for a product of m x n over `blocks` blocks of 128.
static void gemm_plan(int m, int n, int blocks, int sms, int* nt_out, int* splits_out) {
  const int n_tiles = (n + 127) / 128;
  int best_nt = 16, best_s = 1;
  double best = 0;
  for (int nt = 16; nt <= 256; nt *= 2) {
    if (nt < 256 && nt < m && nt < 128) continue;        // one token tile as long as 128 tokens hold the batch
    if (nt > 16 && nt / 2 >= m) break;
    const int64_t tiles = static_cast<int64_t>(n_tiles) * ((m + nt - 1) / nt);
    for (int s = 1; s <= 8; s *= 2) {
      if (s > 1 && (nt > 128 || tiles * s > sms || blocks < 2 * s)) break;
      // clocks of a block: the MMAs (2 NT) or the operands from L2 (about 48 bytes a clock and SM); a split costs a
      // cluster barrier pair and the exchange of the partial sums
      const double block = nt * 2.0 > (128 + nt) * 128 / 48.0 ? nt * 2.0 : (128 + nt) * 128 / 48.0;
      const int64_t waves = (tiles * s + sms - 1) / sms;
      const double cost = waves * ((blocks + s - 1) / s * block + 600.0) + (s > 1 ? 1000.0 + 12.0 * nt : 0.0);
      if (best == 0 || cost < best) {
        best = cost;
        best_nt = nt;
        best_s = s;
      }
    }
  }
  *nt_out = best_nt;
  *splits_out = best_s;
}

}  // namespace b200dsa

using namespace b200dsa;

extern "C" int b200dsa_fp8_quantise_rows(const void* x, int32_t in_f32, int64_t in_stride, int64_t m, int32_t k,
                                         int32_t use_ue8m0, void* q_e4m3, float* scale, int64_t scale_ld, void* stream) {
  if (m == 0) return B200DSA_OK;
  if (!x || !q_e4m3 || !scale || m < 0 || m > (1ll << 31) || k < 16 || (k & 15) || in_stride < k || scale_ld < m) {
    set_last_error("b200dsa_fp8_quantise_rows: bad argument (K a multiple of 16, scale_ld >= rows)");
    return B200DSA_EINVAL;
  }
  const uintptr_t elem = in_f32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(q_e4m3) & 15) || (reinterpret_cast<uintptr_t>(x) % elem)) {
    set_last_error("b200dsa_fp8_quantise_rows: q must be 16-byte aligned");
    return B200DSA_EALIGN;
  }
  QuantRowsParams p{};
  p.in = x;
  p.in_f32 = in_f32 != 0;
  p.in_vec = !(reinterpret_cast<uintptr_t>(x) & 15) && !((in_stride * static_cast<int64_t>(elem)) & 15);
  p.in_stride = in_stride;
  p.m = m;
  p.k = k;
  p.q = static_cast<uint8_t*>(q_e4m3);
  p.scale = scale;
  p.ld = scale_ld;
  p.use_ue8m0 = use_ue8m0 != 0;
  const dim3 grid(static_cast<unsigned>((m + 7) / 8), (k + kQuantPairs * 256 - 1) / (kQuantPairs * 256));
  cudaError_t e = launch_chained(fp8_quantise_rows_kernel, grid, dim3(256), 0, static_cast<cudaStream_t>(stream), p);
  return gemm_rc(e == cudaSuccess ? cudaGetLastError() : e);
}

extern "C" int b200dsa_fp8_quantise_blocks(const void* w, int32_t in_f32, int64_t in_stride, int32_t n, int32_t k,
                                           int32_t use_ue8m0, void* q_e4m3, float* scale, void* stream) {
  if (n == 0) return B200DSA_OK;
  if (!w || !q_e4m3 || !scale || n < 0 || k < 16 || (k & 15) || in_stride < k || n > 65535 * 128) {
    set_last_error("b200dsa_fp8_quantise_blocks: bad argument (K a multiple of 16)");
    return B200DSA_EINVAL;
  }
  if (reinterpret_cast<uintptr_t>(q_e4m3) & 15) {
    set_last_error("b200dsa_fp8_quantise_blocks: q must be 16-byte aligned");
    return B200DSA_EALIGN;
  }
  const int groups = (k + 127) / 128;
  cudaError_t e = launch_chained(fp8_quantise_blocks_kernel, dim3(groups, (n + 127) / 128), dim3(256), 0,
                                 static_cast<cudaStream_t>(stream), w, static_cast<int>(in_f32 != 0), in_stride,
                                 static_cast<int>(n), static_cast<int>(k), static_cast<int>(use_ue8m0 != 0),
                                 static_cast<uint8_t*>(q_e4m3), scale, groups);
  return gemm_rc(e == cudaSuccess ? cudaGetLastError() : e);
}

static int check_matmul(const void* a_e4m3, int64_t a_stride, const float* a_scale, const void* w_e4m3, int64_t w_stride,
                        const float* w_scale, int32_t m, int32_t n, int32_t k, const void* out, int32_t out_f32,
                        int64_t out_stride, const int32_t* status) {
  if (!a_e4m3 || !a_scale || !w_e4m3 || !w_scale || !out || !status || m < 0 || n < 0 || k < 16 || (k & 15) ||
      a_stride < k || w_stride < k || out_stride < n) {
    set_last_error("b200dsa_fp8_block_matmul: bad argument (K a multiple of 16, strides at least the row lengths)");
    return B200DSA_EINVAL;
  }
  if ((reinterpret_cast<uintptr_t>(a_e4m3) & 15) || (reinterpret_cast<uintptr_t>(w_e4m3) & 15) || (a_stride & 15) ||
      (w_stride & 15) || (reinterpret_cast<uintptr_t>(out) & (out_f32 ? 3 : 1))) {
    set_last_error("b200dsa_fp8_block_matmul: operands and their row strides must be multiples of 16 bytes");
    return B200DSA_EALIGN;
  }
  return B200DSA_OK;
}

// dependent: the launch may start while the previous kernel of the stream drains (its results are waited for inside)
static int block_matmul(const void* a_e4m3, int64_t a_stride, const float* a_scale, int64_t sa_m, int64_t sa_g,
                        const void* w_e4m3, int64_t w_stride, const float* w_scale, int64_t sw_r, int64_t sw_g, int32_t m,
                        int32_t n, int32_t k, void* out, int32_t out_f32, int64_t out_stride, int32_t* status,
                        bool dependent, void* stream) {
  if (m == 0 || n == 0) return B200DSA_OK;
  if (int rc = check_matmul(a_e4m3, a_stride, a_scale, w_e4m3, w_stride, w_scale, m, n, k, out, out_f32, out_stride, status)) return rc;
  PFN_encodeTiled enc = get_encode_tiled();
  if (!enc) return B200DSA_ECUDA;
  DeviceInfo dev;
  if (cudaError_t e = current_device_info(&dev)) return gemm_rc(e);
  int nt = 0, splits = 1;
  const int blocks = (k + 127) / 128;
  gemm_plan(m, n, blocks, dev.sms, &nt, &splits);
  CUtensorMap mw, ma;
  cuuint32_t es[2] = {1, 1};
  cuuint64_t dw[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(n)}, sw[1] = {static_cast<cuuint64_t>(w_stride)};
  cuuint64_t da[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(m)}, sa[1] = {static_cast<cuuint64_t>(a_stride)};
  cuuint32_t bw[2] = {128, 128}, ba[2] = {128, static_cast<cuuint32_t>(nt)};
  // out-of-range rows and the tail of the last block arrive as zeros
  if (enc(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(w_e4m3), dw, sw, bw, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS ||
      enc(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(a_e4m3), da, sa, ba, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
    set_last_error("b200dsa_fp8_block_matmul: cuTensorMapEncodeTiled rejected an operand");
    return B200DSA_ECUDA;
  }
  GemmParams p{};
  p.a_scale = a_scale;
  p.sa_m = sa_m;
  p.sa_g = sa_g;
  p.w_scale = w_scale;
  p.sw_r = sw_r;
  p.sw_g = sw_g;
  p.out = out;
  p.ldo = out_stride;
  p.out_f32 = out_f32 != 0;
  p.out_pair = !(reinterpret_cast<uintptr_t>(out) & 3) && !(out_stride & 1);
  p.m = m;
  p.n = n;
  p.blocks = blocks;
  p.m_tiles = (m + nt - 1) / nt;
  p.n_tiles = (n + 127) / 128;
  p.splits = splits;
  p.status = status;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (nt) {
    case 16: return gemm_rc(gemm_launch<16>(mw, ma, p, dev, dependent, st));
    case 32: return gemm_rc(gemm_launch<32>(mw, ma, p, dev, dependent, st));
    case 64: return gemm_rc(gemm_launch<64>(mw, ma, p, dev, dependent, st));
    case 128: return gemm_rc(gemm_launch<128>(mw, ma, p, dev, dependent, st));
    default: return gemm_rc(gemm_launch<256>(mw, ma, p, dev, dependent, st));
  }
}

extern "C" int b200dsa_fp8_block_matmul(const void* a_e4m3, int64_t a_stride, const float* a_scale, int64_t sa_m,
                                        int64_t sa_g, const void* w_e4m3, int64_t w_stride, const float* w_scale,
                                        int64_t sw_r, int64_t sw_g, int32_t m, int32_t n, int32_t k, void* out,
                                        int32_t out_f32, int64_t out_stride, int32_t* status, void* stream) {
  return block_matmul(a_e4m3, a_stride, a_scale, sa_m, sa_g, w_e4m3, w_stride, w_scale, sw_r, sw_g, m, n, k, out, out_f32,
                      out_stride, status, false, stream);
}

extern "C" int b200dsa_fp8_block_linear(const void* x, int32_t in_f32, int64_t in_stride, int32_t use_ue8m0,
                                        const void* w_e4m3, int64_t w_stride, const float* w_scale, int64_t sw_r,
                                        int64_t sw_g, int32_t m, int32_t n, int32_t k, void* out, int32_t out_f32,
                                        int64_t out_stride, void* workspace, int64_t workspace_bytes, int32_t* status,
                                        void* stream) {
  if (m == 0 || n == 0) return B200DSA_OK;
  const int64_t codes = static_cast<int64_t>(m) * k, groups = (static_cast<int64_t>(k) + 127) / 128;
  if (m < 0 || k < 16 || (k & 15) || !workspace || workspace_bytes < codes + 4 * groups * m) {
    set_last_error("b200dsa_fp8_block_linear: bad argument (K a multiple of 16, workspace of m * (k + 4 * ceil(k / 128)) bytes)");
    return B200DSA_EINVAL;
  }
  if (reinterpret_cast<uintptr_t>(workspace) & 15) {
    set_last_error("b200dsa_fp8_block_linear: the workspace must be 16-byte aligned");
    return B200DSA_EALIGN;
  }
  float* scale = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + codes);
  // the product's arguments are checked before anything is launched
  if (int rc = check_matmul(workspace, k, scale, w_e4m3, w_stride, w_scale, m, n, k, out, out_f32, out_stride, status)) return rc;
  if (int rc = b200dsa_fp8_quantise_rows(x, in_f32, in_stride, m, k, use_ue8m0, workspace, scale, m, stream)) return rc;
  return block_matmul(workspace, k, scale, 1, m, w_e4m3, w_stride, w_scale, sw_r, sw_g, m, n, k, out, out_f32, out_stride,
                      status, true, stream);
}
