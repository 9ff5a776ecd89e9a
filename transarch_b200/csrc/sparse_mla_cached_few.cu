// Sparse MLA attention over the quantised latent cache for up to 16 heads (a tensor-parallel share of a model's heads, or
// a draft model): the codes go into the tensor cores as they are.
//
// With 64 heads a CTA (sparse_mla_cached.cu) the 64 x 64 tiles of a 16-head item would be three quarters empty, and the
// time of a tile is set by widening 64 rows to bf16.  Here the keys are the UMMA M dimension and the heads are N:
//
//   S^T_g [128 keys x 32]  = K_g [128 x 128 dims, e4m3] * (Q_hi | Q_lo)_g      for each group g of 128 dims
//   R^T   [128 keys x 16]  = K_pe [128 x 64, bf16] * Q_pe
//   s[key, h] = q_scale[h] * sum_g scale_g[key] * (S_hi + S_lo / 16) + R       one thread a key: its scales are its own
//   p = 2^(s - m[h]),   P_g = 2^10 p * scale_g / 2^(u_g[h] - m[h]) in three terms       the scales of V differ by group
//   O^T_g [128 dims x 48] += V_g^T [128 dims x 128 keys, the same bytes read MN-major] * (P_0 | P_1 | P_2)_g
//
// q over a power of two that brings a row's largest latent value to 224 .. 448 is hi = e4m3(q) and lo = e4m3(16 (q - hi)):
// eight bits, as bf16 has, and off by at most 2^-14 (half of e4m3's smallest step, 2^-10, over 16), 2^-21 of the largest value.  (A rest
// is at most 16, so that 16 of it fit; unlifted, one large dim took the other dims' lower bits.)  Probabilities need more range: thousands of keys
// that hold 2^-17 of the largest one's each are a share of the result.  P is t0 + t1 / 16 + t2 / 256 in e5m2,
//   t0 = e5m2(P),  t1 = e5m2(16 (P - t0)),  t2 = e5m2(16 (16 (P - t0) - t1)),
// each rounding off by 2^-3 of what it rounds: three leave 2^-9 of P, half of a bf16 rounding's 2^-8, as long as t2 is a normal
// number, and never more than 2^-25 (half of e5m2's smallest step, 2^-17, over 256).  P stays below 2^15, so that a rest, at
// most 2^11, times 16 does too.  (Two e4m3 terms of one unit lost everything below 2^-14 of the largest probability.)  The terms stand
// side by side in N and are added in fp32.  The position dims stay bf16.  A tile of 128 keys takes 36 MMAs of at
// most 48 columns, where two tiles of the other kernel take 88 and 128 widened rows.
//
// Each head has a running maximum m[h] of the scores, each head and group one u_g[h] of s + log2(scale_g): what a key adds
// to the group's values, so that a key of large scales but no weight does not push the others out of the terms' range.  Both
// are whole numbers (rescaling is exact) and common to the CTA; they are renewed, and O and the sums rescaled, when a score exceeds
// m by 4.5 (base 2) or a P_g 2^15.
//
// Work split: CTA = (item, split), as in the other kernel.  Roles (512 threads): warps 0-3 rows (TMA gathers of four rows
// x 128 bytes straight into the operand layout, the scales by 16-byte asynchronous copies), warp 4 keys, warps 5 and 6 MMAs,
// warps 8-15 softmax (thread = key, eight heads).  All waits are bounded.  148 items x 16 heads x 2048 keys, every item a
// request of its own: 53 - 54 us (76 us for 17 heads in the other kernel); 592 items of 148 requests: 196 us.  A tile takes 2.1 us: of
// the 7.6 k clocks of its chain (rows 2.5, scores 1.3, softmax 2.2, values 1.4) two stages overlap two, and a third does not fit
// beside P and Q.  (With probabilities of two e4m3 terms and one reference, which were wrong, 49.4 and 174 us.)  A
// gather takes its issuing lane about 50 clocks: two issuing warps take 2 - 4 % longer, one 14 - 20 %, and a copy of each lane of
// a warp 90 clocks.  The key warp prefetches no rows: two tiles of copies in flight cover the latency, and its 896 lines a tile take
// longer than the tile (148 items of as many requests 59.9 us with prefetches, 53.7 without; 64 items x 3 73.1 and 67.7).
#include "sparse_mla_cached.cuh"

namespace b200dsa {

constexpr int kFewThreads = 512;
constexpr int kFewTile = 128;
constexpr int kFewHeads = kMlcFewHeads;
constexpr int kFewStages = 2;
constexpr int kFewKeyTiles = 4;
constexpr int kFewRowWarps = 4;
constexpr int kFewGroupBytes = kFewTile * 128;                      // 128 keys x 128 codes
constexpr int kFewPeOff = 4 * kFewGroupBytes;                       // 128 keys x 64 bf16
constexpr int kFewScaleOff = kFewPeOff + kFewTile * 128;            // 128 keys x 4 fp32
constexpr int kFewStageBytes = kFewScaleOff + kFewTile * 16;
static_assert(kFewStageBytes % 1024 == 0, "stages start on swizzle atoms");
constexpr int kFewTerms = 3;                                        // e5m2 terms of a probability
constexpr int kFewPOctet = kFewTerms * 128;                         // 8 keys x 16 heads a term
constexpr int kFewPGroup = kFewTile / 8 * kFewPOctet;
constexpr int kFewPOff = kFewStages * kFewStageBytes;               // 4 groups x 16 octets of keys
constexpr int kFewQOff = kFewPOff + 4 * kFewPGroup;                 // 4 groups x 32 rows (hi, lo) x 128 dims
constexpr int kFewQpeOff = kFewQOff + 4 * 32 * 128;                 // 16 rows x 64 bf16
constexpr int kFewBarOff = kFewQpeOff + 16 * 128;
constexpr int kFewSmem = kFewBarOff + 256 + 1024;
constexpr uint32_t kFewOCols = kFewTerms * 16;                      // O of a group
constexpr uint32_t kFewTmemS = 4 * kFewOCols;                       // two score buffers of 144 columns behind O
constexpr uint32_t kFewSCols = 144;                                 // 4 groups x (16 hi + 16 lo), 16 position products
static_assert(kFewTmemS + 2 * kFewSCols <= 512, "O and two score buffers");
constexpr float kFewLift = 10.0f;                                   // log2 of the largest P after a renewal
constexpr float kFewMaxP = 32768.0f;                                // and P before the next one
constexpr float kFewHeadroom = 4.5f;
constexpr float kFewMinScale = -100.0f;                             // u_g - m: groups of scales below 2^-100 lose range

__device__ __align__(16) uint8_t g_few_zero[16];

// 128 bytes from byte x of the rows r.x .. r.w, zeros for a row that does not exist (-1).
__device__ __forceinline__ void few_gather4(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int x, int4 r) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
      "%6}], [%7];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w),
      "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void few_ld8(uint32_t taddr, float (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void few_st8(uint32_t taddr, const float (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "f"(v[0]),
               "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
// a and b as e4m3 codes (hi a, hi b) and, of 16 times what those leave, (lo a, lo b)
__device__ __forceinline__ void split_e4m3x2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(hi), __NV_E4M3);
  const float2 f = __half22float2(__half2(h));
  lo = __nv_cvt_float2_to_fp8x2(make_float2((a - f.x) * 16.0f, (b - f.y) * 16.0f), __NV_SATFINITE, __NV_E4M3);
}
// The next e5m2 term of a and b; they become 16 times what it leaves.
__device__ __forceinline__ uint32_t term_e5m2x2(float& a, float& b) {
  const uint32_t t = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E5M2);
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(t), __NV_E5M2);
  const float2 f = __half22float2(__half2(h));
  a = (a - f.x) * 16.0f;
  b = (b - f.y) * 16.0f;
  return t;
}

// 2^n for a whole n up to 127; zero below the normal numbers.
__device__ __forceinline__ float pow2_of(float n) {
  return n < -126.f ? 0.f : __int_as_float((static_cast<int>(n) + 127) << 23);
}

// The largest of each of N values over the warp: lane L ends up with that of value L / (32 / N) in v[0].
template <int N>
__device__ __forceinline__ void warp_max_spread(float (&v)[N]) {
#pragma unroll
  for (int o = 16, n = N; o > 0; o >>= 1) {
    const bool up = threadIdx.x & o;
    if (n > 1) {
      n /= 2;
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
        if (i < n) {
          const float keep = up ? v[i + n] : v[i], give = up ? v[i] : v[i + n];
          v[i] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, give, o));
        }
    } else {
      v[0] = fmaxf(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
    }
  }
}

__global__ void __launch_bounds__(kFewThreads, 1)
sparse_mla_cached_few_kernel(const MlaCachedParams p, const __grid_constant__ CUtensorMap tmap_rows) {
  pdl_launch_dependents();
  pdl_wait_prior();
  extern __shared__ uint8_t smem_dyn[];
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;
  __shared__ __align__(16) int s_slot[kFewKeyTiles][kFewTile];
  __shared__ uint32_t s_mask[kFewStages][4];      // validity bit per key of the stage
  __shared__ int s_renew[3];                      // somebody's key exceeds the references (tile % 3)
  __shared__ uint32_t s_top[kFewHeads];           // largest score so far, in the order of unsigned numbers
  __shared__ uint32_t s_vtop[4][kFewHeads];       // largest s + log2(scale_g) so far, likewise
  __shared__ float s_m[kFewHeads];                // m[h] and, of every group, u_g[h], 2^(10 + m - u_g) and the factor that a
  __shared__ float s_u[4][kFewHeads];             // renewal, or the output, applies to O
  __shared__ __align__(16) float s_lift[4][kFewHeads];
  __shared__ __align__(16) float s_shrink[4][kFewHeads];
  __shared__ float s_sum[4][kFewHeads];
  __shared__ float s_qscale[kFewHeads];

  const int split = blockIdx.x % p.splits;
  const int item = blockIdx.x / p.splits;
  const uint32_t smem_base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
  uint8_t* smem_al = smem_dyn + (smem_base - smem_u32(smem_dyn));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_al + kFewBarOff);
  uint64_t* kv_full = bars;                       // [stages] the row warps' threads, their issuing lanes and bytes
  uint64_t* kv_empty = bars + kFewStages;         // [stages] value MMAs retired
  uint64_t* s_full = bars + 2 * kFewStages;       // [2] score MMAs retired
  uint64_t* s_empty = s_full + 2;                 // [2] 256 softmax threads have read the scores
  uint64_t* p_full = s_empty + 2;                 // [1] 256 softmax threads: P written
  uint64_t* pv_done = p_full + 1;                 // [1] value MMAs retired (P free, O stable)
  uint64_t* q_full = pv_done + 1;                 // [1] 256 softmax threads: Q written
  uint64_t* meet = q_full + 1;                    // [1] rendezvous of the eight softmax warps
  uint64_t* key_full = meet + 1;                  // [kFewKeyTiles]
  uint64_t* key_empty = key_full + kFewKeyTiles;  // [kFewKeyTiles] the row warps

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n_idx = p.n_idx_item ? max(0, min(p.n_idx, p.n_idx_item[item])) : p.n_idx;
  const int all_tiles = (n_idx + kFewTile - 1) / kFewTile + (p.tree_mask ? 1 : 0);
  const int tile0 = static_cast<int>(static_cast<int64_t>(all_tiles) * split / p.splits);
  const int n_tiles = static_cast<int>(static_cast<int64_t>(all_tiles) * (split + 1) / p.splits) - tile0;
  volatile int* abort_flag = &s_abort;

  if (tid < 4 * kFewHeads) {
    if (tid < kFewHeads) s_top[tid] = float_to_ordered(-INFINITY);
    s_vtop[tid / kFewHeads][tid % kFewHeads] = float_to_ordered(-INFINITY);
    s_u[tid / kFewHeads][tid % kFewHeads] = -INFINITY;
    s_m[tid % kFewHeads] = -INFINITY;
    s_lift[tid / kFewHeads][tid % kFewHeads] = 0.f;
  }
  if (tid == 0) {
    s_abort = 0;
    s_renew[0] = s_renew[1] = s_renew[2] = 0;
    for (int s = 0; s < kFewStages; ++s) {
      mbar_init(&kv_full[s], 33 * kFewRowWarps);
      mbar_init(&kv_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_empty[s], 256);
    }
    mbar_init(p_full, 256);
    mbar_init(pv_done, 1);
    mbar_init(q_full, 256);
    mbar_init(meet, 8);
    for (int s = 0; s < kFewKeyTiles; ++s) {
      mbar_init(&key_full[s], 1);
      mbar_init(&key_empty[s], kFewRowWarps);
    }
    mbar_fence_init();
  }
  if (warp == 5) {
    tmem_alloc(&s_tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = s_tmem_base;

  if (warp < kFewRowWarps) {
    // ------------------------------------------------------------------ rows: warp w the rows w * kPer ... of a tile
    constexpr int kPer = kFewTile / kFewRowWarps;
    int started = 0;
    for (int t = 0; t < n_tiles; ++t) {
      const int s = t % kFewStages, ring = t % kFewKeyTiles;
      const bool ok = mbar_wait(&key_full[ring], (t / kFewKeyTiles) & 1, abort_flag) &&
                      mbar_wait(&kv_empty[s], ((t / kFewStages) & 1) ^ 1, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) break;
      const uint32_t stage = smem_base + s * kFewStageBytes;
#pragma unroll
      for (int u = 0; u < kPer / 32; ++u) {
        const int row = warp * kPer + u * 32 + lane, slot = s_slot[ring][row];
        const unsigned valid = __ballot_sync(0xffffffffu, slot >= 0);
        if (lane == 0) s_mask[s][row >> 5] = valid;
        const uint8_t* src = slot >= 0 ? p.cache + static_cast<int64_t>(slot) * kLatentRowBytes + 512 : g_few_zero;
        cp_async_16(stage + kFewScaleOff + row * 16, src, slot >= 0);
      }
      __syncwarp();
      if (elect_one()) {
        mbar_arrive_expect_tx(&kv_full[s], kPer * 640);
        const int4* quads = reinterpret_cast<const int4*>(&s_slot[ring][warp * kPer]);
#pragma unroll 4
        for (int q = 0; q < kPer / 4; ++q) {
          const int4 rows = quads[q];
#pragma unroll
          for (int g = 0; g < 5; ++g)
            few_gather4(stage + g * kFewGroupBytes + (warp * (kPer / 4) + q) * 512, &tmap_rows, &kv_full[s],
                        g < 4 ? g * 128 : 528, rows);
        }
        mbar_arrive(&key_empty[ring]);
      }
      __syncwarp();
      cp_async_mbar_arrive(&kv_full[s]);       // this thread's arrival once its copies above have landed
      started = t + 1;
    }
    cp_async_wait_all();
    // whatever ended the loop, the copies in flight land before the shared memory is given up
    for (int t = max(0, started - kFewStages); t < started; ++t) {
      const long long t0 = clock64();
      while (!mbar_test(&kv_full[t % kFewStages], (t / kFewStages) & 1) && clock64() - t0 < kWaitLimitCycles) {
      }
    }
  } else if (warp == 4) {
    mlc_key_warp<kFewTile, kFewKeyTiles, false>(p, item, tile0, n_tiles, n_idx, &s_slot[0][0], key_full, key_empty, abort_flag);
  } else if (warp == 5) {
    // ------------------------------------------------------------------ score MMAs
    constexpr uint32_t idesc_s = make_idesc(kFmtE4M3, kFmtE4M3, 128, 32);
    constexpr uint32_t idesc_r = make_idesc(kFmtBF16, kFmtBF16, 128, 16);
    bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0, abort_flag));
    for (int t = 0; ok && t < n_tiles; ++t) {
      const int s = t % kFewStages, sb = t & 1;
      ok = __all_sync(0xffffffffu, mbar_wait(&kv_full[s], (t / kFewStages) & 1, abort_flag) &&
                                       mbar_wait(&s_empty[sb], ((t >> 1) & 1) ^ 1, abort_flag));
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t d = tmem_base + kFewTmemS + sb * kFewSCols;
        const uint64_t k0 = make_desc_k_sw128(smem_base + s * kFewStageBytes);
        const uint64_t q0 = make_desc_k_sw128(smem_base + kFewQOff);
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f8f6f4_ss(d + g * 32, k0 + ((g * kFewGroupBytes + kk * 32) >> 4), q0 + ((g * 4096 + kk * 32) >> 4), idesc_s,
                          kk != 0);
        const uint64_t r0 = make_desc_k_sw128(smem_base + s * kFewStageBytes + kFewPeOff);
        const uint64_t qr = make_desc_k_sw128(smem_base + kFewQpeOff);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) mma_f16_ss(d + 128, r0 + 2 * kk, qr + 2 * kk, idesc_r, kk != 0);
        tc_commit(&s_full[sb]);
      }
      __syncwarp();
    }
  } else if (warp == 6) {
    // ------------------------------------------------------------------ value MMAs.  A warp of their own: behind S(t+1) in
    // one warp's order they would wait for the rows of tile t+1, which wait for the stage that these MMAs free.
    constexpr uint32_t idesc_pv = make_idesc(kFmtE4M3, kFmtE5M2, 128, kFewOCols, 1, 1);   // both read MN-major: dims x keys x heads
    bool ok = true;
    for (int t = 0; ok && t < n_tiles; ++t) {
      const int s = t % kFewStages;
      ok = __all_sync(0xffffffffu, mbar_wait(&kv_full[s], (t / kFewStages) & 1, abort_flag) &&
                                       mbar_wait(p_full, t & 1, abort_flag));
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        // 32 keys an MMA: four atoms of 8 keys x 128 dims, 1024 bytes apart
        const uint64_t v0 = make_desc_mn_sw128(smem_base + s * kFewStageBytes, kFewGroupBytes, 1024);
        // P without swizzle: 128 bytes between core matrices along the heads and terms, kFewPOctet along the keys
        const uint64_t p0 = make_desc_k_noswz(smem_base + kFewPOff, kFewPOctet, 128);
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f8f6f4_ss(tmem_base + g * kFewOCols, v0 + ((g * kFewGroupBytes + kk * 4096) >> 4),
                          p0 + ((g * kFewPGroup + kk * 4 * kFewPOctet) >> 4), idesc_pv, (t | kk) != 0);
        tc_commit(&kv_empty[s]);
        tc_commit(pv_done);
      }
      __syncwarp();
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------------------ softmax: thread = key, heads hb .. hb + 7
    const int wq = warp & 3, hb = ((warp >> 2) & 1) * 8;
    const int key = wq * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(wq * 32) << 16;
    bool ok = true;
    uint32_t meets = 0;
    // rendezvous of the softmax warps, bounded like every wait (a warp that gave up does not come)
    auto rendezvous = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(meet);
      return __all_sync(0xffffffffu, mbar_wait(meet, meets++ & 1, abort_flag));
    };
    {
      // Q: warps 8-15 two heads each.  q over a power of two that brings the row's largest value below 448, as hi and lo
#pragma unroll 1
      for (int u = 0; u < 2; ++u) {
        const int h = (warp - 8) * 2 + u;
        const __nv_bfloat16* row = p.q + (static_cast<int64_t>(item) * p.n_heads + h) * kMlaD;
        const bool have = h < p.n_heads;
        float x[16];                                      // dims 8 l + j of either half
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (have) v = __ldg(reinterpret_cast<const uint4*>(row + 256 * half) + lane);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[half * 8 + 2 * j] = __uint_as_float(w[j] << 16);
            x[half * 8 + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
          }
        }
        uint32_t pe = 0;
        if (have) pe = __ldg(reinterpret_cast<const uint32_t*>(row + 512) + lane);
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) top = max_nan(top, fabsf(x[j]));
        for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float sc = pow2_at_least(__fdiv_rn(max_nan(top, 1e-30f), 448.0f));
        const float inv = 1.0f / sc;
        if (lane == 0) s_qscale[h] = sc;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            split_e4m3x2(x[half * 8 + 2 * j] * inv, x[half * 8 + 2 * j + 1] * inv, hi[j], lo[j]);
          // dims 256 half + 8 lane: group 2 half + lane / 16, bytes 8 (lane % 16) of its 128
          const uint32_t at = smem_base + kFewQOff + (2 * half + (lane >> 4)) * 4096 + ((lane & 1) << 3);
          const uint32_t piece = (lane & 15) >> 1;
          asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at + h * 128 + ((piece ^ (h & 7)) << 4)),
                       "r"(hi[0] | hi[1] << 16), "r"(hi[2] | hi[3] << 16) : "memory");
          const int l = 16 + h;
          asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at + l * 128 + ((piece ^ (l & 7)) << 4)),
                       "r"(lo[0] | lo[1] << 16), "r"(lo[2] | lo[3] << 16) : "memory");
        }
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(smem_base + kFewQpeOff + h * 128 + (((lane >> 2) ^ (h & 7)) << 4) + (lane & 3) * 4),
                     "r"(pe) : "memory");
      }
      fence_proxy_async();
      mbar_arrive(q_full);
      ok = rendezvous();                                   // s_qscale
    }
    float qs[8], m[8], l[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      qs[j] = s_qscale[hb + j] * p.scale_log2;
      m[j] = -INFINITY;
      l[j] = 0.f;
    }
    for (int t = 0; ok && t < n_tiles; ++t) {
      const int sb = t & 1, st = t % kFewStages;
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[sb], (t >> 1) & 1, abort_flag) &&
                                       mbar_wait(&kv_full[st], (t / kFewStages) & 1, abort_flag));   // scales, mask
      if (!ok) break;
      {
        tc_fence_after();
        const uint32_t src = tmem_base + lane_addr + kFewTmemS + sb * kFewSCols + hb;
        const bool valid = (s_mask[st][wq] >> lane) & 1;
        float sc[4];
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(sc[0]), "=f"(sc[1]), "=f"(sc[2]), "=f"(sc[3])
                     : "r"(smem_base + st * kFewStageBytes + kFewScaleOff + key * 16));
        float r[8], hi[4][8], lo[4][8];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          few_ld8(src + g * 32, hi[g]);
          few_ld8(src + g * 32 + 16, lo[g]);
        }
        few_ld8(src + 128, r);
        tc_wait_ld();
        float s[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float a = 0.f;
#pragma unroll
          for (int g = 0; g < 4; ++g) a = fmaf(sc[g], fmaf(lo[g][j], 1.0f / 16, hi[g][j]), a);
          s[j] = valid ? fmaf(a, qs[j], r[j] * p.scale_log2) : -INFINITY;
        }
        tc_fence_before();
        mbar_arrive(&s_empty[sb]);
        float e[8], x[4][8];
        auto probabilities = [&]() {                        // and P of every group; a missing key has p = 0 and scales of 0
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = fast_exp2(s[j] - (m[j] == -INFINITY ? 0.f : m[j]));
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float4 a = *reinterpret_cast<const float4*>(&s_lift[g][hb]), b = *reinterpret_cast<const float4*>(&s_lift[g][hb + 4]);
            const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) x[g][j] = e[j] * sc[g] * f[j];
          }
        };
        probabilities();
        float big = 0.f;                                    // a NaN needs no other reference
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(x[g][j]));
        bool over = big > kFewMaxP;
#pragma unroll
        for (int j = 0; j < 8; ++j) over = over || s[j] > m[j] + kFewHeadroom;
        if (__any_sync(0xffffffffu, over) && lane == 0) *reinterpret_cast<volatile int*>(&s_renew[t % 3]) = 1;
        ok = rendezvous();
        if (!ok) break;
        if (tid == 256) s_renew[(t + 2) % 3] = 0;           // read by everyone before this barrier, set after the next
        if (*reinterpret_cast<volatile int*>(&s_renew[t % 3])) {
          // New references from the tile's 128 keys: lane 8 g + j of a warp ends up with the largest value of group g and head j.
          float top[32];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float size = log2f(fabsf(sc[g]));
#pragma unroll
            for (int j = 0; j < 8; ++j) top[g * 8 + j] = s[j] + size;
          }
          warp_max_spread(top);
          atomicMax(&s_vtop[lane >> 3][hb + (lane & 7)], float_to_ordered(top[0]));
          float best[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) best[j] = s[j];
          warp_max_spread(best);
          if ((lane & 3) == 0) atomicMax(&s_top[hb + (lane >> 2)], float_to_ordered(best[0]));
          ok = rendezvous();
          if (!ok) break;
          if (tid < 256 + 4 * kFewHeads) {
            const int h = tid % kFewHeads, g = (tid - 256) / kFewHeads;
            const float nm = ceilf(ordered_to_float(s_top[h]));
            const float nu = fmaxf(ceilf(ordered_to_float(s_vtop[g][h])), nm + kFewMinScale), u = s_u[g][h];
            s_shrink[g][h] = pow2_of(u - nu);
            s_lift[g][h] = nm == -INFINITY ? 0.f : pow2_of(nm - nu + kFewLift);
            s_u[g][h] = nu;
            if (g == 0) s_m[h] = nm;
          }
          ok = rendezvous();
          if (!ok) break;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float n = s_m[hb + j];
            l[j] *= pow2_of(m[j] - n);
            m[j] = n;
          }
          probabilities();
          if (t > 0) {
            ok = __all_sync(0xffffffffu, mbar_wait(pv_done, (t - 1) & 1, abort_flag));
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 4 * kFewTerms; ++c) {       // the terms of every group
              float o[8];
              const uint32_t at = tmem_base + lane_addr + c * 16 + hb;
              const float* f = &s_shrink[c / kFewTerms][hb];
              few_ld8(at, o);
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 8; ++j) o[j] *= f[j];
              few_st8(at, o);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
          }
        } else if (t > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(pv_done, (t - 1) & 1, abort_flag));    // P is free
        }
        // P of group g, MN-major: core matrices of 8 keys x 16 bytes, the terms of the 16 heads side by side.  (Stored
        // K-major, one byte a store, it took 64 stores a thread.)
#pragma unroll
        for (int j = 0; j < 8; ++j) l[j] += e[j];
        const uint32_t row = smem_base + kFewPOff + (key >> 3) * kFewPOctet + (key & 7) * 16 + hb;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
#pragma unroll
          for (int c = 0; c < kFewTerms; ++c) {
            uint32_t t2[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) t2[j] = term_e5m2x2(x[g][2 * j], x[g][2 * j + 1]);
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(row + g * kFewPGroup + c * 128), "r"(t2[0] | t2[1] << 16),
                         "r"(t2[2] | t2[3] << 16) : "memory");
          }
        }
        fence_proxy_async();
        mbar_arrive(p_full);
      }
    }
    // ---- output: sums over the keys, then thread = dim
    if (ok && n_tiles > 0) ok = __all_sync(0xffffffffu, mbar_wait(pv_done, (n_tiles - 1) & 1, abort_flag));
    tc_fence_after();
    for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) l[j] += __shfl_xor_sync(0xffffffffu, l[j], o);
    }
    if (lane == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s_sum[wq][hb + j] = l[j];
    }
    const int64_t parts = static_cast<int64_t>(p.n_items) * p.n_heads, row0 = static_cast<int64_t>(item) * p.n_heads;
    if (ok) ok = rendezvous();
    if (ok && tid < 256 + 4 * kFewHeads) {
      // the factor of a head's O: what its P was multiplied by is taken out, and the sum
      const int h = tid % kFewHeads, g = (tid - 256) / kFewHeads;
      const float sum = s_sum[0][h] + s_sum[1][h] + s_sum[2][h] + s_sum[3][h];
      const bool any = n_tiles > 0 && sum != 0.f;           // a NaN sum stays NaN in the result
      s_shrink[g][h] = any ? pow2_of(s_u[g][h] - s_m[h] - kFewLift) / sum : 0.f;
      if (g == 0 && h < p.n_heads) {
        float* lse = p.splits == 1 ? p.lse + row0 + h : p.part + p.splits * parts * kMlaDv + split * parts + row0 + h;
        *lse = any ? (s_m[h] + log2f(sum)) * 0.6931471805599453f : -INFINITY;
      }
    }
    if (ok) ok = rendezvous();
    if (ok) {
#pragma unroll 1
      for (int g = 0; g < 4; ++g) {
        float a[8], b[8], c[8];
        if (n_tiles > 0) {
          few_ld8(tmem_base + lane_addr + g * kFewOCols + hb, a);
          few_ld8(tmem_base + lane_addr + g * kFewOCols + 16 + hb, b);
          few_ld8(tmem_base + lane_addr + g * kFewOCols + 32 + hb, c);
          tc_wait_ld();
        }
        const int dim = g * 128 + key;                      // the lane is a dim of the group here
        float unit[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) unit[j] = s_shrink[g][hb + j];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (hb + j >= p.n_heads) continue;
          const float v = unit[j] != 0.f ? fmaf(fmaf(c[j], 1.0f / 16, b[j]), 1.0f / 16, a[j]) * unit[j] : 0.f;
          if (p.splits > 1) p.part[(split * parts + row0 + hb + j) * kMlaDv + dim] = v;
          else if (p.ctx_bf16) static_cast<__nv_bfloat16*>(p.ctx)[(row0 + hb + j) * kMlaDv + dim] = __float2bfloat16_rn(v);
          else static_cast<float*>(p.ctx)[(row0 + hb + j) * kMlaDv + dim] = v;
        }
        __syncwarp();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tmem_base, 512);
  if (tid == 0 && s_abort) atomicMax(p.status, kDevWaitTimeout);
}

cudaError_t mla_cached_few_launch(const MlaCachedParams& p, int device, cudaStream_t stream) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (!enc) return cudaErrorNotSupported;
  // the rows of all slots, in pieces of 128 bytes and the operands' swizzle
  CUtensorMap rows;
  const cuuint64_t dims[2] = {kLatentRowBytes, static_cast<cuuint64_t>(p.n_slots)}, pitch[1] = {kLatentRowBytes};
  const cuuint32_t box[2] = {128, 1}, step[2] = {1, 1};
  if (enc(&rows, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(p.cache), dims, pitch, box, step,
          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cudaErrorInvalidValue;
  static OncePerDevice once;
  const cudaError_t e = once.run(device, [] {
    return cudaFuncSetAttribute(sparse_mla_cached_few_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem);
  });
  if (e != cudaSuccess) return e;
  return launch_chained(sparse_mla_cached_few_kernel, dim3(p.n_items * p.splits), dim3(kFewThreads), kFewSmem, stream, p, rows);
}

}  // namespace b200dsa
