// Products of 8-bit matrices with block scales, and the quantisers that make their operands.
//
//   y[m, n] = sum_g  sa[m, g] * sw[n / 128, g] * sum_{k in block g} a[m, k] * w[n, k]
//
// a: activations, e4m3 [M, K], one fp32 scale for 128 values of a row; w: weights, e4m3 [N, K], one fp32 scale for
// a block of 128 x 128.  Blocks at the right and lower edge may be partial.  The scales are arbitrary fp32 numbers, so
// a block's product has to leave the tensor pipe before it is scaled: the inner sum of every 128-deep block is one
// accumulator in TMEM (4 MMAs of K = 32), and fp32 registers hold the outer sum.
//
// Two kernels.  Few tokens (up to 128): 128 weight rows are the UMMA M dimension (one TMEM lane and one accumulating
// thread for an output column n) and 16 .. 128 tokens are N, so that a decode batch is a narrow tile that still streams
// whole weight tiles.  Few tiles split the blocks of K over the 2 - 8 CTAs of a cluster: each CTA keeps its partial
// sums in its own shared memory and adds up its share of the tokens over the cluster in rank order, so the result does
// not depend on timing and no workspace exists.
// Many tokens: 128 tokens are M and 256 weight rows N.  A thread owns one token, so that the scale of a block is one
// register and the shared-memory port carries nothing but the operands (48 KB in by TMA and 48 KB out to the MMAs a block).
//
// Measured: 4096 x 7168 x 7168 in 189 - 226 us by box (1.9 - 2.2 PFLOP/s; 920 clocks a block where its MMAs take 512: the tensor pipe
// waits for the accumulating warps); 16 x 18944 x 7168 in 27 us (5.1 TB/s of weights);
// 64 x 8192 x 1536 in 8 us, of which the blocks are 3.
//
// Narrow kernel, 352 threads: warp 0 TMA loads, warp 1 MMAs, warp 2 scales, warps 3-10 accumulate (two a TMEM lane
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
  int out_vec;                 // rows of the result start on 16-byte boundaries
  int m, n, blocks;            // blocks of K
  int m_tiles, n_tiles, splits;
  int work0, work;             // tiles work0 .. work - 1 are this launch's
  int32_t* status;
};

template <int NT>
struct GemmShape {
  static constexpr int kWBytes = 128 * 128, kABytes = NT * 128, kStageBytes = kWBytes + kABytes;
  static constexpr int kStages = NT == 128 ? 6 : 8;
  static constexpr int kAccBufs = 4;
  static constexpr uint32_t kTmemCols = NT * kAccBufs < 32 ? 32 : NT * kAccBufs;
  static constexpr int kCols = NT / 2;                        // token columns of one accumulating warp
  static constexpr int kScaleOff = kStages * kStageBytes;
  static constexpr int kBarOff = kScaleOff + kGemmScaleSlots * NT * 4;
  static constexpr int kSmem = kBarOff + 256 + 1024;
  // partial sums of a split tile live where the operand ring was: NT tokens x 128 columns fp32
  static_assert(NT <= 128 && NT * 128 * 4 <= kStages * kStageBytes, "partial sums must fit the operand ring");
};

__device__ __forceinline__ uint32_t gemm_cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void gemm_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 gemm_ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t r;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(r));
  return v;
}
__device__ __forceinline__ void tmem_ld_32x8(uint32_t taddr, uint32_t (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(taddr)
               : "memory");
}

template <int N>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&v)[N]) {
  static_assert(N == 8 || N == 16 || N == 32, "columns of one load");
  if constexpr (N == 8) tmem_ld_32x8(taddr, v);
  else if constexpr (N == 16) tmem_ld_32x16(taddr, v);
  else tmem_ld_32x32(taddr, v);
}

// Two fp32 sums in one 64-bit register pair: a += (x0, x1) * s, one packed instruction.
__device__ __forceinline__ void fma_pair(uint64_t& a, uint32_t x0, uint32_t x1, uint64_t s) {
  asm("{\n\t.reg .b64 x;\n\t"
      "mov.b64 x, {%1, %2};\n\t"
      "fma.rn.f32x2 %0, x, %3, %0;\n\t}"
      : "+l"(a)
      : "r"(x0), "r"(x1), "l"(s));
}
__device__ __forceinline__ void fma_pairs(uint64_t& a, uint64_t x, uint64_t s) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(x), "l"(s));
}
__device__ __forceinline__ uint64_t pair_of(float v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
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

// Sum of the cluster's partial sums of columns n .. n + 3 of a token, in rank order; `at`: where they lie in every CTA.
__device__ __forceinline__ void add_partials(const GemmParams& p, uint32_t at, int tok, int n) {
  float4 v[8];
#pragma unroll
  for (int r = 0; r < 8; ++r)
    if (r < p.splits) v[r] = gemm_ld_cluster(at, r);
  float4 sum = v[0];
#pragma unroll
  for (int r = 1; r < 8; ++r)
    if (r < p.splits) {
      sum.x += v[r].x; sum.y += v[r].y; sum.z += v[r].z; sum.w += v[r].w;
    }
  const int64_t o = static_cast<int64_t>(tok) * p.ldo + n;
  const float x[4] = {sum.x, sum.y, sum.z, sum.w};
  if (p.out_vec && n + 4 <= p.n) {
    if (p.out_f32) {
      *reinterpret_cast<float4*>(static_cast<float*>(p.out) + o) = sum;
    } else {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x, sum.y), hi = __floats2bfloat162_rn(sum.z, sum.w);
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + o) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < p.n) {
        if (p.out_f32) static_cast<float*>(p.out)[o + j] = x[j];
        else static_cast<__nv_bfloat16*>(p.out)[o + j] = __float2bfloat16_rn(x[j]);
      }
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
  const int n_work = p.work;
  const int rank = p.splits > 1 ? static_cast<int>(gemm_cluster_rank()) : 0;
  const int first = p.work0 + blockIdx.x / p.splits, stride = gridDim.x / p.splits;
  const int b_lo = static_cast<int>(static_cast<int64_t>(p.blocks) * rank / p.splits);
  const int b_hi = static_cast<int>(static_cast<int64_t>(p.blocks) * (rank + 1) / p.splits);

  if (warp == 0) {
    // ------------------------------------------------------------------ loads
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int w = first; ok && w < n_work; w += stride) {
        const int n0 = (w % p.n_tiles) * 128, m0 = (w / p.n_tiles) * NT;
        for (int b = b_lo; b < b_hi; ++b, ++it) {
          const int s = it % S::kStages;
          ok = mbar_wait(&empty[s], ((it / S::kStages) & 1) ^ 1, abort_flag);
          if (!ok) break;
          uint8_t* dst = smem_al + s * S::kStageBytes;
          mbar_arrive_expect_tx(&full[s], S::kStageBytes);
          tma_load_2d(dst, &tmap_w, &full[s], b * 128, n0);
          tma_load_2d(dst + S::kWBytes, &tmap_a, &full[s], b * 128, m0);
        }
      }
      // whatever ended the loop, the copies in flight land before the shared memory is given up
      for (int j = it > S::kStages ? it - S::kStages : 0; j < it; ++j) {
        const long long t0 = clock64();
        while (!mbar_test(&full[j % S::kStages], (j / S::kStages) & 1) && clock64() - t0 < kWaitLimitCycles) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA
    // The whole warp waits, one elected lane issues: in a loop of a single thread the descriptors are not in uniform
    // registers and every MMA takes longer to issue.
    constexpr uint32_t idesc = make_idesc(kFmtE4M3, kFmtE4M3, 128, NT);
    int it = 0;
    bool ok = true;
    for (int w = first; ok && w < n_work; w += stride) {
      for (int b = b_lo; b < b_hi; ++b, ++it) {
        const int s = it % S::kStages, buf = it % S::kAccBufs, sl = it % kGemmScaleSlots;
        // the block's scales are waited for here, so that the accumulating warps have one barrier to look at
        ok = __all_sync(0xffffffffu, mbar_wait(&sc_full[sl], (it / kGemmScaleSlots) & 1, abort_flag) &&
                                         mbar_wait(&acc_empty[buf], ((it / S::kAccBufs) & 1) ^ 1, abort_flag) &&
                                         mbar_wait(&full[s], (it / S::kStages) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t wd = make_desc_k_sw128(smem_base + s * S::kStageBytes);
          const uint64_t ad = make_desc_k_sw128(smem_base + s * S::kStageBytes + S::kWBytes);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f8f6f4_ss(tmem_base + buf * NT, wd + 2 * kk, ad + 2 * kk, idesc, kk != 0);
          tc_commit(&acc_full[buf]);
          tc_commit(&empty[s]);
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
        // every load is issued before the first is used: addresses are clamped, what lies outside becomes zero below
        float v[kAhead][kPer], ws[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int b = min(b0 + u, b_hi - 1);
          ws[u] = __ldg(p.w_scale + nb * p.sw_r + b * p.sw_g);
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            v[u][j] = __ldg(p.a_scale + min(m0 + lane + 32 * j, p.m - 1) * p.sa_m + b * p.sa_g);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (b0 + u >= b_hi) break;
          const int sl = it % kGemmScaleSlots;
          ok = __all_sync(0xffffffffu, mbar_wait(&sc_empty[sl], ((it / kGemmScaleSlots) & 1) ^ 1, abort_flag));
          if (!ok) break;
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if (lane + 32 * j < NT)
              s_scale[sl * NT + lane + 32 * j] = m0 + lane + 32 * j < p.m ? ws[u] * v[u][j] : 0.f;
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
    constexpr int kChunk = S::kCols < 32 ? S::kCols : 32, kChunks = S::kCols / kChunk;
    int it = 0;
    bool ok = true;
    for (int w = first; ok && w < n_work; w += stride) {
      uint64_t acc[S::kCols / 2];
#pragma unroll
      for (int j = 0; j < S::kCols / 2; ++j) acc[j] = 0;
      uint32_t v[2][kChunk];
      auto first_columns = [&](int i) -> bool {            // wait for block product i, start on its columns
        const bool there = __all_sync(0xffffffffu, mbar_wait(&acc_full[i % S::kAccBufs], (i / S::kAccBufs) & 1, abort_flag));
        tc_fence_after();
        tmem_ld_cols<kChunk>(tmem_base + lane_addr + (i % S::kAccBufs) * NT + col0, v[0]);
        return there;
      };
      ok = first_columns(it);
      if (!ok) break;
#pragma unroll 1
      for (int b = b_lo; b < b_hi; ++b, ++it) {
        const int buf = it % S::kAccBufs, sl = it % kGemmScaleSlots;
        const ulonglong2* sc = reinterpret_cast<const ulonglong2*>(s_scale + sl * NT + col0);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {      // the next columns are under way while these are added
          tc_wait_ld();
          uint64_t x[kChunk / 2];
#pragma unroll
          for (int j = 0; j < kChunk / 2; ++j)
            asm("mov.b64 %0, {%1, %2};" : "=l"(x[j]) : "r"(v[c & 1][2 * j]), "r"(v[c & 1][2 * j + 1]));
          if (c + 1 < kChunks) {
            tmem_ld_cols<kChunk>(tmem_base + lane_addr + buf * NT + col0 + (c + 1) * kChunk, v[(c + 1) & 1]);
          } else {
            tc_fence_before();                   // everything is in registers: the buffer may be written
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[buf]);
            if (kChunks > 1 && b + 1 < b_hi) ok = first_columns(it + 1);
          }
#pragma unroll
          for (int j = 0; j < kChunk / 2; j += 2) {
            const ulonglong2 f = sc[(c * kChunk + 2 * j) >> 2];
            fma_pairs(acc[c * kChunk / 2 + j], x[j], f.x);
            fma_pairs(acc[c * kChunk / 2 + j + 1], x[j + 1], f.y);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sc_empty[sl]);
        if (kChunks == 1 && b + 1 < b_hi) ok = first_columns(it + 1);
        if (!ok) break;
      }
      if (!ok) break;
      const int n = (w % p.n_tiles) * 128 + row, m0 = (w / p.n_tiles) * NT + col0;
      if (p.splits > 1) {
        // every MMA of this CTA has read its operands: the ring holds the partial sums now, [token][128]
        float* part = reinterpret_cast<float*>(smem_al);
#pragma unroll
        for (int j = 0; j < S::kCols; j += 2) {
          const float2 f = unpair(acc[j / 2]);
          part[(col0 + j) * 128 + row] = f.x;
          part[(col0 + j + 1) * 128 + row] = f.y;
        }
      } else if (p.out_f32) {
#pragma unroll
        for (int j = 0; j < S::kCols; ++j) {
          const float2 f = unpair(acc[j / 2]);
          if (n < p.n && m0 + j < p.m) static_cast<float*>(p.out)[static_cast<int64_t>(m0 + j) * p.ldo + n] = j & 1 ? f.y : f.x;
        }
      } else {
#pragma unroll
        for (int j = 0; j < S::kCols; j += 2) {
          const float2 f = unpair(acc[j / 2]);
          store_bf16_pair(p, f.x, f.y, m0 + j, n, lane);
        }
      }
    }
  }

  __syncwarp();
  if (p.splits > 1) {
    // one tile per cluster: add the partial sums of this CTA's share of the tokens in rank order
    gemm_cluster_sync();
    if (warp >= 3) {
      const int n0 = (first % p.n_tiles) * 128, m0 = (first / p.n_tiles) * NT;
      const int per = NT / p.splits;                                  // tokens of a CTA
      for (int i = tid - 96; i < per * 32; i += 256) {                // a thread: four neighbouring columns of a token
        const int tok = rank * per + (i >> 5), n = n0 + (i & 31) * 4;
        if (m0 + tok >= p.m || n >= p.n) continue;
        add_partials(p, smem_base + tok * 512 + (i & 31) * 16, m0 + tok, n);
      }
      __syncwarp();
    }
    gemm_cluster_sync();               // nobody leaves while a peer reads its shared memory
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, S::kTmemCols);
  if (tid == 0 && s_abort) atomicMax(p.status, kDevWaitTimeout);
}

// Persistent CTAs over the tiles, or one cluster of p.splits CTAs a tile.
static cudaError_t gemm_launch_config(void (*kernel)(CUtensorMap, CUtensorMap, GemmParams), int threads, int smem,
                                      const CUtensorMap& mw, const CUtensorMap& ma, const GemmParams& p, int sms,
                                      bool dependent, cudaStream_t stream) {
  const int tiles = p.work - p.work0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.splits > 1 ? tiles * p.splits : (tiles < sms ? tiles : sms));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, mw, ma, p);
  return e == cudaSuccess ? cudaGetLastError() : e;
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
  return gemm_launch_config(fp8_block_gemm_kernel<NT>, kGemmThreads, S::kSmem, mw, ma, p, dev.sms, dependent, stream);
}

// ---------------------------------------------------------------------------------------- many tokens
// 384 threads: warp 0 TMA loads, warp 1 MMA (warps 2 and 3 fill their warpgroup), warps 4-11 accumulate, two a TMEM lane
// quadrant, 128 columns (one block of weight rows, one weight scale) each.  A thread holds 128 fp32 sums: the register
// split gives the accumulating warps 232 registers and the others 40, or 224 and 56 in the split form, whose issuing
// threads hold more (128 * 40 + 256 * 232 = 128 * 56 + 256 * 224 = 384 * 168).  A spill in either costs 15 - 50 %.
constexpr int kWideThreads = 384;
constexpr int kWideStages = 4;
constexpr int kWideABytes = 128 * 128, kWideWBytes = 256 * 128, kWideStageBytes = kWideABytes + kWideWBytes;
constexpr int kWideOutOff = kWideStages * kWideStageBytes;          // 8 warps x 32 rows x 128 bytes
constexpr int kWideBarOff = kWideOutOff + 8 * 32 * 128;
constexpr int kWideSmem = kWideBarOff + 256 + 1024;

// The warp's staged 32 rows of 128 bytes to the result: a store instruction covers 128 bytes of four rows.  kElem: bytes
// of a value.
template <int kElem>
__device__ __forceinline__ void wide_store(const GemmParams& p, uint32_t stage, int m0, int n0, int lane) {
  constexpr int kPer = 16 / kElem;                  // values of a piece
  const int n = n0 + (lane & 7) * kPer;
  if (n >= p.n) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + (lane >> 3);
    if (m0 + r >= p.m) break;
    uint32_t v[4];
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4)));
    uint8_t* o = static_cast<uint8_t*>(p.out) + (static_cast<int64_t>(m0 + r) * p.ldo + n) * kElem;
    if (p.out_vec && n + kPer <= p.n) {
      *reinterpret_cast<uint4*>(o) = make_uint4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (n + j < p.n) {
          if constexpr (kElem == 4) reinterpret_cast<uint32_t*>(o)[j] = v[j];
          else reinterpret_cast<uint16_t*>(o)[j] = static_cast<uint16_t>(v[j >> 1] >> (16 * (j & 1)));
        }
    }
  }
}

template <bool kSplit>      // K cut over a cluster; a kernel of its own, because its exchange costs the other one registers
__global__ void __launch_bounds__(kWideThreads, 1)
fp8_block_gemm_wide_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_a,
                           const GemmParams p) {
  pdl_launch_dependents();
  extern __shared__ uint8_t smem_dyn[];
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;
  const uint32_t smem_base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
  uint8_t* smem_al = smem_dyn + (smem_base - smem_u32(smem_dyn));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem_al + kWideBarOff);   // [stages] bytes of an operand pair
  uint64_t* empty = full + kWideStages;                                  // [stages] MMAs of the stage retired
  uint64_t* acc_full = empty + kWideStages;                              // [2] block product complete
  uint64_t* acc_empty = acc_full + 2;                                    // [2] eight warps have read it
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &s_abort;
  if (tid == 0) {
    s_abort = 0;
    for (int s = 0; s < kWideStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], 8);
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(&s_tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = s_tmem_base;
  pdl_wait_prior();
  const int n_work = p.work;
  const int rank = kSplit ? static_cast<int>(gemm_cluster_rank()) : 0;
  const int first = kSplit ? p.work0 + blockIdx.x / p.splits : blockIdx.x, stride = kSplit ? gridDim.x / p.splits : gridDim.x;
  const int b_lo = kSplit ? static_cast<int>(static_cast<int64_t>(p.blocks) * rank / p.splits) : 0;
  const int b_hi = kSplit ? static_cast<int>(static_cast<int64_t>(p.blocks) * (rank + 1) / p.splits) : p.blocks;

  if (warp < 4) {
    if (kSplit) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0 && lane == 0) {
      int it = 0;
      bool ok = true;
      for (int w = first; ok && w < n_work; w += stride) {
        const int n0 = (w % p.n_tiles) * 256, m0 = (w / p.n_tiles) * 128;
        for (int b = b_lo; b < b_hi; ++b, ++it) {
          const int s = it % kWideStages;
          ok = mbar_wait(&empty[s], ((it / kWideStages) & 1) ^ 1, abort_flag);
          if (!ok) break;
          uint8_t* dst = smem_al + s * kWideStageBytes;
          mbar_arrive_expect_tx(&full[s], kWideStageBytes);
          tma_load_2d(dst, &tmap_a, &full[s], b * 128, m0);
          tma_load_2d(dst + kWideABytes, &tmap_w, &full[s], b * 128, n0);
        }
      }
      // whatever ended the loop, the copies in flight land before the shared memory is given up
      for (int j = it > kWideStages ? it - kWideStages : 0; j < it; ++j) {
        const long long t0 = clock64();
        while (!mbar_test(&full[j % kWideStages], (j / kWideStages) & 1) && clock64() - t0 < kWaitLimitCycles) {
        }
      }
    } else if (warp == 1) {
      constexpr uint32_t idesc = make_idesc(kFmtE4M3, kFmtE4M3, 128, 256);
      int it = 0;
      bool ok = true;
      for (int w = first; ok && w < n_work; w += stride) {
        for (int b = b_lo; b < b_hi; ++b, ++it) {
          const int s = it % kWideStages, buf = it & 1;
          ok = __all_sync(0xffffffffu, mbar_wait(&acc_empty[buf], ((it >> 1) & 1) ^ 1, abort_flag) &&
                                           mbar_wait(&full[s], (it / kWideStages) & 1, abort_flag));
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t ad = make_desc_k_sw128(smem_base + s * kWideStageBytes);
            const uint64_t wd = make_desc_k_sw128(smem_base + s * kWideStageBytes + kWideABytes);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_f8f6f4_ss(tmem_base + buf * 256, ad + 2 * kk, wd + 2 * kk, idesc, kk != 0);
            tc_commit(&acc_full[buf]);
            tc_commit(&empty[s]);
          }
          __syncwarp();
        }
      }
    }
    __syncwarp();
  } else {
    if (kSplit) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int wq = warp & 3, half = (warp - 4) >> 2;
    const uint32_t src0 = tmem_base + (static_cast<uint32_t>(wq * 32) << 16) + half * 128;
    const uint32_t stage = smem_base + kWideOutOff + (warp - 4) * 4096;
    int it = 0;
    bool ok = true;
    for (int w = first; ok && w < n_work; w += stride) {
      const int n0 = (w % p.n_tiles) * 256 + half * 128, m0 = (w / p.n_tiles) * 128 + wq * 32;
      const bool live = m0 + lane < p.m && n0 < p.n;
      const float* sa = p.a_scale + static_cast<int64_t>(m0 + lane) * p.sa_m + b_lo * p.sa_g;
      const float* sw = p.w_scale + static_cast<int64_t>(n0 >> 7) * p.sw_r + b_lo * p.sw_g;
      // scales of the next two blocks are under way
      float sn[2], wn[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bool in = live && b_lo + u < b_hi;
        sn[u] = in ? __ldg(sa + u * p.sa_g) : 0.f;
        wn[u] = in ? __ldg(sw + u * p.sw_g) : 0.f;
      }
      sa += 2 * p.sa_g;
      sw += 2 * p.sw_g;
      uint64_t acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = 0;
      constexpr int kCols = 32;                            // columns of a load
      uint32_t v[2][kCols];
      auto first_columns = [&](int i) -> bool {            // wait for block product i, start on its columns
        const bool there = __all_sync(0xffffffffu, mbar_wait(&acc_full[i & 1], (i >> 1) & 1, abort_flag));
        tc_fence_after();
        tmem_ld_cols<kCols>(src0 + (i & 1) * 256, v[0]);
        return there;
      };
      ok = first_columns(it);
      if (!ok) break;
#pragma unroll 2
      for (int b = b_lo; b < b_hi; ++b, ++it) {
        const uint64_t s = pair_of(sn[0] * wn[0]);
        sn[0] = sn[1];
        wn[0] = wn[1];
        const bool in = live && b + 2 < b_hi;
        sn[1] = in ? __ldg(sa) : 0.f;
        wn[1] = in ? __ldg(sw) : 0.f;
        sa += p.sa_g;
        sw += p.sw_g;
        const int buf = it & 1;
#pragma unroll
        for (int c = 0; c < 128 / kCols; ++c) {
          tc_wait_ld();
          if (c + 1 < 128 / kCols) {
            tmem_ld_cols<kCols>(src0 + buf * 256 + (c + 1) * kCols, v[(c + 1) & 1]);
          } else {
            tc_fence_before();                             // everything is in registers: the buffer may be written
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[buf]);
            if (b + 1 < b_hi) ok = first_columns(it + 1);   // of the next block, under the additions below
          }
#pragma unroll
          for (int j = 0; j < kCols; j += 2) fma_pair(acc[(c * kCols + j) / 2], v[c & 1][j], v[c & 1][j + 1], s);
        }
        if (!ok) break;
      }
      if (!ok) break;
      if (kSplit) {
        // every MMA of this CTA has read its operands: the ring holds the partial sums now, [token][256], 16-byte pieces
        // swizzled by token
        const uint32_t part = smem_base + (wq * 32 + lane) * 1024;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          asm volatile("st.shared.v2.b64 [%0], {%1, %2};" ::"r"(part + (((half * 32 + j) ^ (lane & 7)) << 4)),
                       "l"(acc[2 * j]), "l"(acc[2 * j + 1]) : "memory");
        continue;
      }
      if (n0 >= p.n) continue;
      if (p.out_f32) {
        // 32 columns at a time: a lane writes its row's 128 bytes into the warp's 4 KB, 16-byte pieces swizzled by row,
        // and reads back pieces of four rows that lie side by side
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            asm volatile("st.shared.v2.b64 [%0], {%1, %2};" ::"r"(stage + lane * 128 + ((j ^ (lane & 7)) << 4)),
                         "l"(acc[c * 16 + j * 2]), "l"(acc[c * 16 + j * 2 + 1]) : "memory");
          __syncwarp();
          wide_store<4>(p, stage, m0, n0 + c * 32, lane);
          __syncwarp();
        }
      } else {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint32_t o[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float2 f = unpair(acc[c * 32 + j * 4 + q]);
              const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
              o[q] = *reinterpret_cast<const uint32_t*>(&h);
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + ((j ^ (lane & 7)) << 4)),
                         "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
          }
          __syncwarp();
          wide_store<2>(p, stage, m0, n0 + c * 64, lane);
          __syncwarp();
        }
      }
    }
  }
  __syncwarp();
  if (kSplit) {
    // one tile per cluster: add the partial sums of this CTA's share of the tokens in rank order
    gemm_cluster_sync();
    if (warp >= 4) {
      const int n0 = (first % p.n_tiles) * 256, m0 = (first / p.n_tiles) * 128, per = 128 / p.splits;
      for (int i = tid - 128; i < per * 64; i += 256) {               // a thread: four neighbouring columns of a token
        const int tok = rank * per + (i >> 6), n = n0 + (i & 63) * 4;
        if (m0 + tok < p.m && n < p.n)
          add_partials(p, smem_base + tok * 1024 + (((i & 63) ^ (tok & 7)) << 4), m0 + tok, n);
      }
    }
    __syncwarp();
    gemm_cluster_sync();               // nobody leaves while a peer reads its shared memory
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, 512);
  if (tid == 0 && s_abort) atomicMax(p.status, kDevWaitTimeout);
}

template <bool kSplit>
static cudaError_t wide_launch(const CUtensorMap& mw, const CUtensorMap& ma, const GemmParams& p, const DeviceInfo& dev,
                               bool dependent, cudaStream_t stream) {
  static OncePerDevice once;
  cudaError_t e = once.run(dev.index, [] {
    return cudaFuncSetAttribute(fp8_block_gemm_wide_kernel<kSplit>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWideSmem);
  });
  if (e != cudaSuccess) return e;
  return gemm_launch_config(fp8_block_gemm_wide_kernel<kSplit>, kWideThreads, kWideSmem, mw, ma, p, dev.sms, dependent, stream);
}

// ---------------------------------------------------------------------------------------- quantisers
// Rows: a warp takes two groups of 128 values at a time (lane = 8 values, 16 lanes a group) of one row; the eight warps
// of a CTA are eight neighbouring rows, whose scales are neighbours in the column-major scale matrix.
constexpr int kQuantPairs = 4;         // group pairs of a warp, loads of all of them in flight

struct QuantRowsParams {
  const void* in;
  int in_vec;                  // rows start on 16-byte boundaries
  int64_t in_stride, m;
  int k;
  uint8_t* q;                  // [m, k]
  float* scale;                // [m, g] at g * ld + m
  int64_t ld;
};

// Eight values as they lie in memory (bf16 packed: half the registers of a batch of loads), widened when they are used.
template <bool kF32>
struct Raw8 {
  uint32_t w[kF32 ? 8 : 4];
  __device__ __forceinline__ void load(const void* in, int64_t i, int vec) {
    if (kF32) {
      const uint32_t* q = static_cast<const uint32_t*>(in) + i;
      if (vec) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(q)), b = __ldg(reinterpret_cast<const uint4*>(q) + 1);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        w[4 % (kF32 ? 8 : 4)] = b.x; w[5 % (kF32 ? 8 : 4)] = b.y; w[6 % (kF32 ? 8 : 4)] = b.z; w[7 % (kF32 ? 8 : 4)] = b.w;
      } else {
#pragma unroll
        for (int j = 0; j < (kF32 ? 8 : 4); ++j) w[j] = __ldg(q + j);
      }
    } else {
      const uint16_t* q = static_cast<const uint16_t*>(in) + i;
      if (vec) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(q));
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __ldg(q + 2 * j) | static_cast<uint32_t>(__ldg(q + 2 * j + 1)) << 16;
      }
    }
  }
  // values 2j and 2j + 1 in one 64-bit register pair
  __device__ __forceinline__ uint64_t pair(int j) const {
    uint64_t r;
    const uint32_t lo = kF32 ? w[2 * j % (kF32 ? 8 : 4)] : w[j] << 16, hi = kF32 ? w[(2 * j + 1) % (kF32 ? 8 : 4)] : w[j] & 0xffff0000u;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
  }
  // largest magnitude of the half warp's values (without NaN); a lane that is not `in` has none
  __device__ __forceinline__ float group_amax(bool in) const {
    if (kF32) {
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(__uint_as_float(w[j % (kF32 ? 8 : 4)])));
      if (!in) m = 0.f;
      for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      return m;
    }
    uint32_t m = 0;                         // two bf16 maxima at a time
    auto grow = [&m](uint32_t v) { asm("max.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(v)); };
#pragma unroll
    for (int j = 0; j < 4; ++j) grow(w[j] & 0x7fff7fffu);
    if (!in) m = 0;
    for (int o = 8; o > 0; o >>= 1) grow(__shfl_xor_sync(0xffffffffu, m, o));
    return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
};

// Two values over a scale as e4m3 codes: quant_e4m3x4's arithmetic (div_by) in packed instructions, two values at a time.
template <bool kPow2>
__device__ __forceinline__ uint32_t quant_pair(uint64_t x, uint64_t rcp, uint64_t minus_scale) {
  uint64_t q;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(q) : "l"(x), "l"(rcp));
  if (!kPow2) {
    uint64_t rest = x;
    fma_pairs(rest, q, minus_scale);
    fma_pairs(q, rest, rcp);
  }
  return __nv_cvt_float2_to_fp8x2(unpair(q), __NV_SATFINITE, __NV_E4M3);
}

template <bool kF32, bool kPow2>
__global__ void __launch_bounds__(256) fp8_quantise_rows_kernel(const QuantRowsParams p) {
  pdl_launch_dependents();
  pdl_wait_prior();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= p.m) return;
  const int lane = threadIdx.x & 31;
  const int k0 = blockIdx.y * (kQuantPairs * 256) + lane * 8;
  Raw8<kF32> x[kQuantPairs];
#pragma unroll
  for (int u = 0; u < kQuantPairs; ++u)       // K is a multiple of 16; a lane behind it reads its first values again
    x[u].load(p.in, row * p.in_stride + (k0 + 256 * u < p.k ? k0 + 256 * u : 0), p.in_vec);
  float amax[kQuantPairs];
#pragma unroll
  for (int u = 0; u < kQuantPairs; ++u) {
    amax[u] = x[u].group_amax(k0 + 256 * u < p.k);
    amax[u] = fmaxf(amax[u], 1e-10f);
  }
  // A division and a reciprocal take more instructions than the codes of eight values: lane u of every half warp does
  // them for pair u, all at once.  (Quantising 4096 x 7168 was bound by issue slots: 19 us before this, 17 with it, 15.7 with the
  // packed maxima and divisions; 16384 x 7168 65 us, 5.4 TB/s.)
  GroupScale mine;
  if (!kPow2) mine = group_scale(lane & 2 ? (lane & 1 ? amax[3] : amax[2]) : (lane & 1 ? amax[1] : amax[0]));
#pragma unroll
  for (int u = 0; u < kQuantPairs; ++u) {
    const int k = k0 + 256 * u;
    GroupScale g;
    if (kPow2) {
      g = group_scale_pow2(amax[u]);
    } else {
      g.scale = __shfl_sync(0xffffffffu, mine.scale, (lane & 16) | u);
      g.rcp = __shfl_sync(0xffffffffu, mine.rcp, (lane & 16) | u);
    }
    if (k < p.k) {
      uint2 codes;
      const uint64_t rcp = pair_of(g.rcp), minus = pair_of(-g.scale);
      codes.x = quant_pair<kPow2>(x[u].pair(0), rcp, minus) | quant_pair<kPow2>(x[u].pair(1), rcp, minus) << 16;
      codes.y = quant_pair<kPow2>(x[u].pair(2), rcp, minus) | quant_pair<kPow2>(x[u].pair(3), rcp, minus) << 16;
      *reinterpret_cast<uint2*>(p.q + row * p.k + k) = codes;
      if ((lane & 15) == 0) p.scale[(k >> 7) * p.ld + row] = g.scale;
    }
  }
}
static_assert(kQuantPairs == 4, "lanes 0 .. 3 of a half warp stand for the pairs");

// Blocks of 128 x 128 (weights): one CTA a block, 64 values a thread, partial blocks at the edges.
template <bool kPow2>
__global__ void __launch_bounds__(256) fp8_quantise_blocks_kernel(const void* in, int in_f32, int64_t in_stride, int n,
                                                                  int k, uint8_t* __restrict__ q,
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
  amax = fmaxf(amax, 1e-10f);
  const GroupScale g = kPow2 ? group_scale_pow2(amax) : group_scale(amax);
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (r0 + i < n && c0 < k)                            // K is a multiple of 16: four codes are in or out together
      *reinterpret_cast<uint32_t*>(q + static_cast<int64_t>(r0 + i) * k + c0) =
          quant_e4m3x4<kPow2>(x[i][0], x[i][1], x[i][2], x[i][3], g);
  if (threadIdx.x == 0) scale[static_cast<int64_t>(blockIdx.y) * groups + blockIdx.x] = g.scale;
}

static int gemm_rc(cudaError_t e) {
  if (e == cudaSuccess) return B200DSA_OK;
  set_last_error(cudaGetErrorString(e));
  return B200DSA_ECUDA;
}

// Kernel, tokens of a tile and CTAs of a cluster for a product of m x n over `blocks` blocks of 128: the least
// estimated time.  Measured clocks of a block: narrow 830 (16 tokens) .. 1000 (128), bound by the weights from HBM or
// by the accumulating warps; wide 930.  A wave costs 600 more, a split its barriers and the exchange of the partial sums.
// Tiles that would start one more, mostly empty wave can be a launch of their own, their K split over clusters:
// without and with it on one box 256 x 19200 x 7168 73 -> 58 us, 2048 x 4736 x 7168 92 -> 76 - 81, 16 x 19200 x 7168 46 -> 33.5,
// 64 x 24576 x 7168 47 -> 44 (faster boxes: 46, 70 and 33 us for the first three, with it).  An estimated gain below 7 % was none:
// 8192 x 7168 x 7168 370 -> 377, 64 x 19200 x 1536 13.4 -> 14.0 (after many full waves the tensor pipes are at the power limit, and an idle last wave is paid back in clocks).
struct GemmPlan {
  int nt;             // tokens of a tile; 0 = the kernel for many tokens
  int splits;
  int rest_splits;    // above 1: the tiles behind the last full wave are a second launch with so many splits
};
constexpr double gemm_cost(int64_t tiles, int splits, int blocks, int sms, double block_clocks, double exchange) {
  return static_cast<double>((tiles * splits + sms - 1) / sms) * ((blocks + splits - 1) / splits * block_clocks + 600.0) +
         (splits > 1 ? 1000.0 + exchange : 0.0);
}
static GemmPlan gemm_plan(int m, int n, int blocks, int sms) {
  GemmPlan plan{};
  double best = 0;
  for (int nt = 16; nt <= 256; nt *= 2) {                // 256 stands for the wide kernel: 128 tokens x 256 columns
    if (nt < 128 && nt < m) continue;                    // one token tile as long as 128 tokens hold the batch
    if (nt > 16 && (nt == 256 ? m <= 128 : nt / 2 >= m)) break;
    const bool wide = nt == 256;
    const int64_t tiles = wide ? static_cast<int64_t>((n + 255) / 256) * ((m + 127) / 128)
                               : static_cast<int64_t>((n + 127) / 128) * ((m + nt - 1) / nt);
    const double block_clocks = wide ? 930.0 : 800.0 + 1.5 * nt, exchange = wide ? 3000.0 : 12.0 * nt;
    const double second_launch = wide ? 16000.0 : 6000.0;
    auto consider = [&](double cost, int splits, int rest_splits) {
      if (best == 0 || cost < best) {
        best = cost;
        plan = GemmPlan{wide ? 0 : nt, splits, rest_splits};
      }
    };
    const int64_t rest = tiles % sms;
    for (int s = 1; s <= 8; s *= 2) {
      if (s == 1 || (tiles * s <= sms && blocks >= 2 * s)) consider(gemm_cost(tiles, s, blocks, sms, block_clocks, exchange), s, 1);
      if (s > 1 && tiles > sms && rest > 0 && rest * s <= sms && blocks >= 2 * s)
        consider(1.07 * (gemm_cost(tiles - rest, 1, blocks, sms, block_clocks, exchange) +
                         gemm_cost(rest, s, blocks, sms, block_clocks, exchange) + second_launch), 1, s);
    }
  }
  return plan;
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
  p.in_vec = !(reinterpret_cast<uintptr_t>(x) & 15) && !((in_stride * static_cast<int64_t>(elem)) & 15);
  p.in_stride = in_stride;
  p.m = m;
  p.k = k;
  p.q = static_cast<uint8_t*>(q_e4m3);
  p.scale = scale;
  p.ld = scale_ld;
  const dim3 grid(static_cast<unsigned>((m + 7) / 8), (k + kQuantPairs * 256 - 1) / (kQuantPairs * 256));
  void (*kernel)(QuantRowsParams) = in_f32 ? (use_ue8m0 ? fp8_quantise_rows_kernel<true, true> : fp8_quantise_rows_kernel<true, false>)
                                           : (use_ue8m0 ? fp8_quantise_rows_kernel<false, true> : fp8_quantise_rows_kernel<false, false>);
  cudaError_t e = launch_chained(kernel, grid, dim3(256), 0, static_cast<cudaStream_t>(stream), p);
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
  cudaError_t e = launch_chained(use_ue8m0 ? fp8_quantise_blocks_kernel<true> : fp8_quantise_blocks_kernel<false>, dim3(groups, (n + 127) / 128), dim3(256), 0,
                                 static_cast<cudaStream_t>(stream), w, static_cast<int>(in_f32 != 0), in_stride,
                                 static_cast<int>(n), static_cast<int>(k), static_cast<uint8_t*>(q_e4m3), scale, groups);
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
  const int blocks = (k + 127) / 128;
  const GemmPlan plan = gemm_plan(m, n, blocks, dev.sms);
  const int nt = plan.nt;
  CUtensorMap mw, ma;
  cuuint32_t es[2] = {1, 1};
  cuuint64_t dw[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(n)}, sw[1] = {static_cast<cuuint64_t>(w_stride)};
  cuuint64_t da[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(m)}, sa[1] = {static_cast<cuuint64_t>(a_stride)};
  cuuint32_t bw[2] = {128, nt ? 128u : 256u}, ba[2] = {128, nt ? static_cast<cuuint32_t>(nt) : 128u};
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
  p.out_vec = !(reinterpret_cast<uintptr_t>(out) & 15) && !((out_stride * (out_f32 ? 4 : 2)) & 15);
  p.out_pair = !(reinterpret_cast<uintptr_t>(out) & 3) && !(out_stride & 1);
  p.m = m;
  p.n = n;
  p.blocks = blocks;
  p.m_tiles = nt ? (m + nt - 1) / nt : (m + 127) / 128;
  p.n_tiles = nt ? (n + 127) / 128 : (n + 255) / 256;
  p.status = status;
  const int tiles = p.m_tiles * p.n_tiles, rest = plan.rest_splits > 1 ? tiles % dev.sms : 0;
  auto launch = [&](int work0, int work, int splits, bool dep) -> cudaError_t {
    p.work0 = work0;
    p.work = work;
    p.splits = splits;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (nt) {
      case 16: return gemm_launch<16>(mw, ma, p, dev, dep, st);
      case 32: return gemm_launch<32>(mw, ma, p, dev, dep, st);
      case 64: return gemm_launch<64>(mw, ma, p, dev, dep, st);
      case 128: return gemm_launch<128>(mw, ma, p, dev, dep, st);
      default: return splits > 1 ? wide_launch<true>(mw, ma, p, dev, dep, st) : wide_launch<false>(mw, ma, p, dev, dep, st);
    }
  };
  cudaError_t e = launch(0, tiles - rest, plan.splits, dependent);
  // its CTAs start as those of the full waves leave
  if (e == cudaSuccess && rest > 0) e = launch(tiles - rest, tiles, plan.rest_splits, true);
  return gemm_rc(e);
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
