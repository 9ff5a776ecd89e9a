// Sparse MLA attention over the quantised, paged latent cache (rows of 656 bytes, latent_cache.cuh), with the drafted
// tokens of a speculative step as a tree.
//
//   keys of an item:  the selected positions idx_j with  0 <= idx_j <= q_pos + q_pos_bias  (and idx_j < tree_base)
//                     and, for a drafted token, the positions tree_base + i for every bit i of its ancestor mask
//   s[h, j] = sm_scale * <q[h, 0:576], row_j>,  p = softmax_j(s),  ctx[h, :] = sum_j p[h, j] row_j[0:512],  lse[h]
//
// The tensor work is that of the bf16 kernel (sparse_mla_decode.cu: 64 heads a CTA as UMMA M, 64 keys a tile, O and two
// score buffers and Q in TMEM, the row bytes read K-major by the scores and MN-major by the values).  What differs is
// the way of a row into shared memory: 656 bytes come from HBM into registers, are widened to bf16 (exactly, when the
// scales are powers of two) and stored in the 128-byte-swizzled layout of the MMA operands.  Eight warps do that, eight
// rows of a tile each; the loads of tile t+1 are issued row by row as the registers of tile t are stored.  (Staging the
// codes in shared memory by cp.async would add 84 KB of shared-memory traffic a tile to the 220 KB that the MMAs and
// the widened rows take, and that port is already the second busiest unit.)
//
// A tree is one more tile: its 64 keys are the drafted positions in order, its validity bits are the mask itself.
//
// Work split: CTA = (item, 64-head half, split).  Small batches cut an item's tiles into `splits` runs whose partial
// contexts (normalised, fp32) and log-sum-exps are merged by mla_merge_kernel; large ones have splits = 1 and no merge,
// or (splits < 0) cut only the items behind the last full wave, in a second launch: 80 x 128 x 2048 134 -> 99 us, 192 x 16 x 2048
// 90 - 94 -> 76 - 81, 170 x 64 x 2048 139 -> 111.
//
// Roles (448 threads): warps 0-7 rows, warps 8-11 softmax, warp 12 MMAs, warp 13 keys: it turns positions into slots, up
// to four tiles ahead of the rows, and has their bytes brought into L2 meanwhile.  (The row warps did that themselves at
// first: 16 of 79 us at 64 x 128 x 2048.)  All waits are bounded.
#include "sparse_mla_cached.cuh"

namespace b200dsa {

void set_last_error(const char* msg);

constexpr int kMlcThreads = 448;
constexpr int kMlcRowWarps = 8;
constexpr int kMlcMaxSplits = 32;
constexpr int kMlcKeyTiles = 4;      // tiles whose slots are held in shared memory

__device__ __align__(16) uint8_t g_zero_row[kLatentRowBytes];   // what a missing key reads

__device__ __forceinline__ void st_shared_v4(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w));
}

template <bool kPrefetch>
__global__ void __launch_bounds__(kMlcThreads, 1)
sparse_mla_cached_kernel(const MlaCachedParams p) {
  pdl_launch_dependents();
  pdl_wait_prior();
  extern __shared__ uint8_t smem_dyn[];
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;
  __shared__ uint32_t s_mask[kMlaStages][2];  // validity bit per key of the stage
  __shared__ int s_slot[kMlcKeyTiles][kMlaTile];
  __shared__ float s_inv[kMlaHeadsTile];      // 1 / sum of the probabilities of a head row, 0 without a key

  const int split = blockIdx.x % p.splits;
  const int hh = (blockIdx.x / p.splits) % p.halves;
  const int item = blockIdx.x / (p.splits * p.halves);

  const uint32_t smem_base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
  uint8_t* smem_al = smem_dyn + (smem_base - smem_u32(smem_dyn));
  const uint32_t kv_addr = smem_base;
  const uint32_t p_addr = kv_addr + kMlaStages * kMlaStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_al + kMlaStages * kMlaStageBytes + kMlaPBytes);
  uint64_t* q_full = bars;                       // [1] Q sits in TMEM
  uint64_t* s_full = bars + 1;                   // [2] score MMA retired
  uint64_t* s_empty = bars + 3;                  // [2] 128 softmax threads have read the scores
  uint64_t* p_full = bars + 5;                   // [1] 128 softmax threads: P written
  uint64_t* pv_done = bars + 6;                  // [1] value MMA retired (P buffer free, O stable)
  uint64_t* kv_full = bars + 7;                  // [stages] eight row warps
  uint64_t* kv_empty = bars + 7 + kMlaStages;    // [stages] value MMA retired
  uint64_t* key_full = bars + 8 + 2 * kMlaStages;  // [kMlcKeyTiles] slots of a tile written
  uint64_t* key_empty = key_full + kMlcKeyTiles;   // [kMlcKeyTiles] eight row warps have read them
  uint64_t* q_land = bars + 7 + 2 * kMlaStages;  // [1] 256 row-warp threads: their copies of Q have landed

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const int n_idx = p.n_idx_item ? max(0, min(p.n_idx, p.n_idx_item[item])) : p.n_idx;
  const int sel_tiles = (n_idx + kMlaTile - 1) / kMlaTile;
  const int all_tiles = sel_tiles + (p.tree_mask ? 1 : 0);
  // this CTA's run of tiles; below, t counts from its first one
  const int tile0 = static_cast<int>(static_cast<int64_t>(all_tiles) * split / p.splits);
  const int n_tiles = static_cast<int>(static_cast<int64_t>(all_tiles) * (split + 1) / p.splits) - tile0;
  volatile int* abort_flag = &s_abort;

  if (tid == 0) {
    s_abort = 0;
    mbar_init(q_full, 128);
    for (int s = 0; s < kMlaStages; ++s) {
      mbar_init(&kv_full[s], kMlcRowWarps);
      mbar_init(&kv_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_empty[s], 128);
    }
    mbar_init(p_full, 128);
    mbar_init(pv_done, 1);
    mbar_init(q_land, 32 * kMlcRowWarps);
    for (int s = 0; s < kMlcKeyTiles; ++s) {
      mbar_init(&key_full[s], 1);
      mbar_init(&key_empty[s], kMlcRowWarps);
    }
    mbar_fence_init();
  }
  if (warp == 12) {
    tmem_alloc(&s_tmem_base, kMlaTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = s_tmem_base;

  if (warp < kMlcRowWarps) {
    // ------------------------------------------------------------------ rows
    // Q first: 64 rows of 72 16-byte pieces into the tail of the key ring, which the rows do not reach before q_full
    // (rows padded by 16 bytes against bank conflicts; the last one spills into the P tile, unused so far).  The softmax
    // warps move it to TMEM.  One bulk copy a row instead took 8 k clocks to issue.
    {
      const int have = min(kMlaHeadsTile, p.n_heads - hh * kMlaHeadsTile);
      const uint8_t* q0 = reinterpret_cast<const uint8_t*>(
          p.q + (static_cast<int64_t>(item) * p.n_heads + hh * kMlaHeadsTile) * kMlaD);
#pragma unroll
      for (int u = 0; u < kMlaHeadsTile * 72 / (32 * kMlcRowWarps); ++u) {
        const int c = tid + u * 32 * kMlcRowWarps, r = c / 72;
        cp_async_16(smem_base + kMlaQStageOff + r * kMlaQRowBytes + (c - 72 * r) * 16, q0 + (r < have ? c * 16 : 0),
                    r < have);
      }
      cp_async_mbar_arrive(q_land);
    }
    const int r0 = warp * 8;
    // A row's registers: lane l holds codes 16l..16l+15 and their scale, and of two rows (lane / 8 + 4 j) the 16-byte
    // chunk lane % 8 of the position dims.  A missing key reads a row of zeros: whatever lies in the cache, its products
    // with a probability of zero are zero.
    uint4 code[8];
    float scale[8];
    uint4 pe[2];
    auto row_ptr = [&](int s) { return s >= 0 ? p.cache + static_cast<int64_t>(s) * kLatentRowBytes : g_zero_row; };
    auto load_row = [&](int slot, int i) {
      const uint8_t* src = row_ptr(__shfl_sync(0xffffffffu, slot, i));
      code[i] = __ldg(reinterpret_cast<const uint4*>(src) + lane);
      scale[i] = __ldg(reinterpret_cast<const float*>(src + 512) + (lane >> 3));
    };
    auto load_pe = [&](int slot, int j) {
      const uint8_t* src = row_ptr(__shfl_sync(0xffffffffu, slot, (lane >> 3) + 4 * j));
      pe[j] = __ldg(reinterpret_cast<const uint4*>(src + 528) + (lane & 7));
    };
    // this lane's slot of tile t (lanes 0..7: the warp's rows), -1 = none; false when the wait gave up
    auto key_slot = [&](int t, int& slot) -> bool {
      slot = -1;
      if (t >= n_tiles) return true;
      const int ring = t % kMlcKeyTiles;
      const bool ok = __all_sync(0xffffffffu, mbar_wait(&key_full[ring], (t / kMlcKeyTiles) & 1, abort_flag));
      if (lane < 8) slot = s_slot[ring][r0 + lane];
      __syncwarp();
      if (lane == 0) mbar_arrive(&key_empty[ring]);
      return ok;
    };
    int slot, next;
    bool ok = key_slot(0, slot);
#pragma unroll
    for (int i = 0; i < 8; ++i) load_row(slot, i);
    load_pe(slot, 0);
    load_pe(slot, 1);
    // Lane l stores 16-byte chunks 2 (l % 4) and 2 (l % 4) + 1 of the 128-byte chunk l / 4 of a row; lanes 4..7 of every
    // eight take them in the other order, so that eight neighbouring lanes write eight different bank groups.
    const bool flip = (lane >> 2) & 1;
    constexpr int kBatch = 2;
    auto store_rows = [&](uint32_t stage_addr, int next) {
      const uint32_t dst0 = stage_addr + (lane >> 2) * kMlaChunkBytesK + r0 * 128;
      const int c0 = (lane & 3) * 2 + flip;
#pragma unroll
      for (int i0 = 0; i0 < 8; i0 += kBatch) {
        uint4 w0[kBatch], w1[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int i = i0 + u;
          const uint4 c = code[i];
          const float sc = scale[i];
          dequant_e4m3x4(flip ? c.z : c.x, sc, w0[u].x, w0[u].y);
          dequant_e4m3x4(flip ? c.w : c.y, sc, w0[u].z, w0[u].w);
          dequant_e4m3x4(flip ? c.x : c.z, sc, w1[u].x, w1[u].y);
          dequant_e4m3x4(flip ? c.y : c.w, sc, w1[u].z, w1[u].w);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) load_row(next, i0 + u);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int i = i0 + u;
          const uint32_t dst = dst0 + i * 128;
          st_shared_v4(dst + ((c0 ^ i) << 4), w0[u]);
          st_shared_v4(dst + ((c0 ^ 1 ^ i) << 4), w1[u]);
        }
      }
    };
    for (int t = 0; ok && t < n_tiles; ++t) {
      const int s = t % kMlaStages;
      const unsigned vmask = __ballot_sync(0xffffffffu, lane < 8 && slot >= 0);
      ok = key_slot(t + 1, next) && mbar_wait(&kv_empty[s], ((t / kMlaStages) & 1) ^ 1, abort_flag);
      // the tail of the ring holds the Q rows until the softmax threads have moved them to TMEM
      if (t < kMlaStages && (t + 1) * kMlaStageBytes > kMlaQStageOff) ok = ok && mbar_wait(q_full, 0, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint32_t stage_addr = kv_addr + s * kMlaStageBytes;
      store_rows(stage_addr, next);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = (lane >> 3) + 4 * j;
        const uint32_t dst = stage_addr + 8 * kMlaChunkBytesK + (r0 + i) * 128 + (((lane & 7) ^ i) << 4);
        st_shared_v4(dst, pe[j]);
        load_pe(next, j);
      }
      if (lane == 0) reinterpret_cast<volatile uint8_t*>(&s_mask[s][0])[warp] = static_cast<uint8_t>(vmask);
      // The rows were written through the generic proxy; the MMAs read them.  (No thread fence here: it would wait for
      // the loads of the next tile, 1200 clocks a tile; the arrival releases the mask.)
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&kv_full[s]);
      slot = next;
    }
    cp_async_wait_all();     // Q, should everything have been given up early
  } else if (warp < 12) {
    // ------------------------------------------------------------------ softmax
    // lanes 16..31: score row `row`; lanes 0..15: the same row of O (partner lane = lane ^ 16)
    const int wq = warp & 3;
    const int row = wq * 16 + (lane & 15);          // head row inside this CTA's 64
    const bool is_s = lane >= 16;
    const uint32_t lane_addr = static_cast<uint32_t>(wq * 32) << 16;  // sub-partition base lane
    float m_ref = -INFINITY, l = 0.f;
    bool aborted = false;
    {
      // Q -> TMEM once: lane 16+i stores head row 16*wq+i into the upper half-lanes (two bf16 per cell, 288 cells per
      // row).  The lower half-lanes of these columns belong to O, not written yet.
      const bool okq = mbar_wait(q_land, 0, abort_flag);
      aborted = !__all_sync(0xffffffffu, okq);
      const uint32_t qrow = smem_base + kMlaQStageOff + row * kMlaQRowBytes;
#pragma unroll 1
      for (int c = 0; c < kMlaD / 64 && !aborted; ++c) {
        uint32_t qv[32];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(qv[4 * j]), "=r"(qv[4 * j + 1]), "=r"(qv[4 * j + 2]), "=r"(qv[4 * j + 3])
                       : "r"(qrow + c * 128 + j * 16));
        tmem_st_32x32(tmem_base + lane_addr + 128 + c * 32, qv);
      }
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(q_full);
    }
    for (int t = 0; t < n_tiles && !aborted; ++t) {
      const int sb = t & 1;
      bool ok = mbar_wait(&s_full[sb], (t >> 1) & 1, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) { aborted = true; break; }
      tc_fence_after();
      const int ks = t % kMlaStages;
      constexpr int kNV = kMlaTile / 32;   // 32-column groups per tile
      uint32_t v[kNV][32];
#pragma unroll
      for (int h = 0; h < kNV; ++h)
        tmem_ld_32x32(tmem_base + lane_addr + sb * kMlaTile + 32 * h, v[h]);   // lanes 16-31: score rows
      tc_wait_ld();
      float mt = -INFINITY;   // tile maximum of the raw scores, scaled once below (the scale is positive)
#pragma unroll
      for (int h = 0; h < kNV; ++h) {
        const uint32_t mk = s_mask[ks][h];
        if (mk == 0xffffffffu) {   // common case: all 32 keys of the group are valid
#pragma unroll
          for (int j = 0; j < 32; ++j) mt = fmaxf(mt, __uint_as_float(v[h][j]));
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float a = ((mk >> j) & 1u) ? __uint_as_float(v[h][j]) : -INFINITY;
            v[h][j] = __float_as_uint(a);
            mt = fmaxf(mt, a);
          }
        }
      }
      mt *= p.scale_log2;
      if (!is_s) mt = -INFINITY;
      bool waited_pv = false;
      // lazy rescale: only when the running maximum grows by more than 2^8
      const bool grow = is_s && (mt > m_ref + 8.0f);
      if (__any_sync(0xffffffffu, grow) && t > 0) {
        ok = mbar_wait(pv_done, (t - 1) & 1, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) { aborted = true; break; }
        waited_pv = true;
        if (t + 1 < n_tiles) {
          // the write-back below also touches the upper half-lanes of columns 0..127, where the
          // next tile's scores may still be landing: let that MMA finish first
          ok = mbar_wait(&s_full[(t + 1) & 1], ((t + 1) >> 1) & 1, abort_flag);
          if (!__all_sync(0xffffffffu, ok)) { aborted = true; break; }
        }
        tc_fence_after();
        float f = grow ? ((m_ref == -INFINITY) ? 0.f : exp2f(m_ref - mt)) : 1.0f;
        if (is_s) l *= f;
        f = __shfl_xor_sync(0xffffffffu, f, 16);   // O-row lanes take the factor of their partner
#pragma unroll 1
        for (int c = 0; c < kMlaDv / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32(tmem_base + lane_addr + kMlaTmemO + c * 32, o);
          tc_wait_ld();
          if (!is_s) {
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
          }
          // upper lanes write back what they read (score buffers and unused cells)
          tmem_st_32x32(tmem_base + lane_addr + kMlaTmemO + c * 32, o);
        }
        tc_wait_st();
        tc_fence_before();
      }
      // Only now may the score issuer overwrite this buffer (two tiles ahead): the write-back of a
      // rescale above also touches the score cells.
      tc_fence_before();
      mbar_arrive(&s_empty[sb]);
      if (grow) m_ref = mt;
      uint32_t pk[kMlaTile / 2];
      float lsum = 0.f;
      // p = 2^(s*scale - m_ref) as one FMA and one ex2; masked scores are -inf and give exactly 0
      const float neg_m = (m_ref == -INFINITY) ? 0.f : -m_ref;
#pragma unroll
      for (int h = 0; h < kNV; ++h) {
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float p0 = fast_exp2(fmaf(__uint_as_float(v[h][j]), p.scale_log2, neg_m));
          const float p1 = fast_exp2(fmaf(__uint_as_float(v[h][j + 1]), p.scale_log2, neg_m));
          lsum += p0 + p1;
          __nv_bfloat162 h01 = __floats2bfloat162_rn(p0, p1);
          pk[16 * h + (j >> 1)] = *reinterpret_cast<uint32_t*>(&h01);
        }
      }
      if (is_s) l += lsum;
      if (t > 0 && !waited_pv) {
        ok = mbar_wait(pv_done, (t - 1) & 1, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) { aborted = true; break; }
      }
      if (is_s) {
        // P row (tile bf16) as core-matrix rows of 16 bytes: (row/8)*(tile/8*128) + c*128 + (row%8)*16
        const uint32_t prow = p_addr + (row >> 3) * (kMlaTile / 8 * 128) + (row & 7) * 16;
#pragma unroll
        for (int c = 0; c < kMlaTile / 8; ++c) {
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(prow + c * 128), "r"(pk[4 * c]),
                       "r"(pk[4 * c + 1]), "r"(pk[4 * c + 2]), "r"(pk[4 * c + 3])
                       : "memory");
        }
      }
      fence_proxy_async();
      mbar_arrive(p_full);
    }
    // 1 / sum and the log-sum-exp of every row; the rows leave below, by all warps
    bool ok = !aborted;
    if (ok && n_tiles > 0) ok = __all_sync(0xffffffffu, mbar_wait(pv_done, (n_tiles - 1) & 1, abort_flag));
    if (ok && is_s) {
      const bool any = n_tiles > 0 && l != 0.f;          // a NaN sum stays NaN in the result
      s_inv[row] = any ? 1.0f / l : 0.f;
      const int head = hh * kMlaHeadsTile + row;
      const int64_t out_row = static_cast<int64_t>(item) * p.n_heads + head, parts = static_cast<int64_t>(p.n_items) * p.n_heads;
      float* lse_out = p.splits == 1 ? p.lse + out_row : p.part + p.splits * parts * kMlaDv + split * parts + out_row;
      if (head < p.n_heads) *lse_out = any ? (m_ref + log2f(l)) * 0.6931471805599453f : -INFINITY;
    }
    tc_fence_before();
  } else if (warp == 13) {
    // ------------------------------------------------------------------ keys
    mlc_key_warp<kMlaTile, kMlcKeyTiles, kPrefetch>(p, item, tile0, n_tiles, n_idx, &s_slot[0][0], key_full, key_empty, abort_flag);
  } else {
    // ------------------------------------------------------------------ MMA issuer (warp 12)
    // One warp issues everything, in the order S(0), S(1), PV(0), S(2), PV(1), ...: the tensor pipe runs its instructions
    // in issue order, so S(t+1) keeps it busy while the softmax of tile t runs, and the ring stage that PV(t-1) frees is
    // not needed before S(t+2), a whole tile of tensor work later.  The rows and P were made visible to the MMAs by the
    // threads that wrote them (fence, then arrival), so no fence is needed here.  The whole warp waits and one elected
    // lane issues: a loop of a single thread is slower by a fifth (its descriptors are not in uniform registers).
    constexpr uint32_t idesc_s = make_idesc(kFmtBF16, kFmtBF16, kMlaHeadsTile, kMlaTile);
    constexpr uint32_t idesc_pv = make_idesc(kFmtBF16, kFmtBF16, kMlaHeadsTile, 256, 0, 1);
    auto issue_scores = [&](int t) -> bool {
      const int s = t % kMlaStages, sb = t & 1;
      const bool w = mbar_wait(&kv_full[s], (t / kMlaStages) & 1, abort_flag) &&
                     mbar_wait(&s_empty[sb], ((t >> 1) & 1) ^ 1, abort_flag);
      if (!__all_sync(0xffffffffu, w)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t d = tmem_base + kMlaTmemS + sb * kMlaTile;
        // descriptors differ only in the 16-byte-granular start address: one add per operand
        const uint64_t b0 = make_desc_k_sw128(kv_addr + s * kMlaStageBytes);
#pragma unroll
        for (int c = 0; c < kMlaChunks; ++c) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f16_ts(d, tmem_base + kMlaTmemQ + c * 32 + kk * 8, b0 + ((c * kMlaChunkBytesK + kk * 32) >> 4), idesc_s,
                       (c | kk) != 0);
        }
        tc_commit(&s_full[sb]);
      }
      __syncwarp();
      return true;
    };
    bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0, abort_flag));
    if (ok && n_tiles > 0) ok = issue_scores(0);
    for (int t = 0; ok && t < n_tiles; ++t) {
      if (t + 1 < n_tiles && !issue_scores(t + 1)) break;
      const int s = t % kMlaStages;
      if (!__all_sync(0xffffffffu, mbar_wait(p_full, t & 1, abort_flag))) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t pa0 = make_desc_k_noswz(p_addr, 128, kMlaTile / 8 * 128);
        const uint64_t vb0 = make_desc_mn_sw128(kv_addr + s * kMlaStageBytes, kMlaChunkBytesK, 1024);
#pragma unroll
        for (int j = 0; j < kMlaTile / 16; ++j) {  // 16 keys per MMA
#pragma unroll
          for (int nh = 0; nh < 2; ++nh)           // value dims [256*nh, 256*nh+256)
            mma_f16_ss(tmem_base + kMlaTmemO + nh * 256, pa0 + ((j * 256) >> 4),
                       vb0 + (((4 * nh) * kMlaChunkBytesK + j * 2048) >> 4), idesc_pv, (t | j) != 0);
        }
        tc_commit(&kv_empty[s]);
        tc_commit(pv_done);
      }
      __syncwarp();
    }
  }

  // ------------------------------------------------------------------------ output
  // Three warps a TMEM lane quadrant bring O (lanes 0..15 of the quadrant) into the ring, which is free now, 32 columns at
  // a time, and whole rows leave from there with every store instruction one run of 512 bytes.  (Stores straight from
  // the softmax threads, 16 bytes at a row's pitch, took 11 k clocks a CTA; a bulk store a row 8 k.)
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const bool write = *abort_flag == 0;
  const bool to_bf16 = p.splits == 1 && p.ctx_bf16;        // a split writes its normalised fp32 part
  const uint32_t pitch = to_bf16 ? kMlaDv * 2 + 16 : kMlaDv * 4 + 16;
  if (write && warp < 12 && n_tiles > 0) {
    const int wq = warp & 3, row = wq * 16 + (lane & 15);
    const float inv = s_inv[row];
    const uint32_t stage = smem_base + row * pitch;
#pragma unroll 2
    for (int c = warp >> 2; c < kMlaDv / 32; c += 3) {
      uint32_t o[32];
      tmem_ld_32x32(tmem_base + (static_cast<uint32_t>(wq * 32) << 16) + kMlaTmemO + c * 32, o);
      tc_wait_ld();
      // a row without a single key holds zeros, or nothing yet: zero times its stale cells would keep a NaN
#pragma unroll
      for (int j = 0; j < 32; ++j) o[j] = inv != 0.f ? __float_as_uint(__uint_as_float(o[j]) * inv) : 0u;
      if (lane < 16 && to_bf16) {
#pragma unroll
        for (int j = 0; j < 32; j += 8)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + c * 64 + j * 2),
                       "r"(pack_bf16x2(__uint_as_float(o[j]), __uint_as_float(o[j + 1]))),
                       "r"(pack_bf16x2(__uint_as_float(o[j + 2]), __uint_as_float(o[j + 3]))),
                       "r"(pack_bf16x2(__uint_as_float(o[j + 4]), __uint_as_float(o[j + 5]))),
                       "r"(pack_bf16x2(__uint_as_float(o[j + 6]), __uint_as_float(o[j + 7])))
                       : "memory");
      } else if (lane < 16) {
#pragma unroll
        for (int j = 0; j < 32; j += 4)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + c * 128 + j * 4), "r"(o[j]),
                       "r"(o[j + 1]), "r"(o[j + 2]), "r"(o[j + 3])
                       : "memory");
      }
      __syncwarp();
    }
    tc_fence_before();
  }
  __syncthreads();
  if (write) {
    const int heads = min(kMlaHeadsTile, p.n_heads - hh * kMlaHeadsTile), pieces = to_bf16 ? 2 : 4;
    const int64_t first = (static_cast<int64_t>(p.splits > 1 ? split : 0) * p.n_items + item) * p.n_heads + hh * kMlaHeadsTile;
    uint8_t* out = static_cast<uint8_t*>(p.splits > 1 ? static_cast<void*>(p.part) : p.ctx) + first * (pitch - 16);
    for (int i = warp; i < heads * pieces; i += kMlcThreads / 32) {
      const int r = i / pieces, at = (i - r * pieces) * 512 + lane * 16;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (n_tiles > 0)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(smem_base + r * pitch + at));
      *reinterpret_cast<uint4*>(out + static_cast<int64_t>(r) * (pitch - 16) + at) = v;
    }
  }
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem_base, kMlaTmemCols);
  if (tid == 0 && s_abort) atomicMax(p.status, kDevWaitTimeout);
}

// Merge of the splits of a (item, head) row: weights exp(lse_s - max), parts without a key left out.  One CTA a row,
// four dims a thread.
__global__ void __launch_bounds__(128) mla_merge_kernel(const float* __restrict__ part, int n_rows, int splits,
                                                        void* __restrict__ ctx, int ctx_bf16, float* __restrict__ lse) {
  pdl_launch_dependents();
  pdl_wait_prior();
  const int row = blockIdx.x;
  const float* part_lse = part + static_cast<int64_t>(splits) * n_rows * kMlaDv;
  float top = -INFINITY;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, __ldg(part_lse + static_cast<int64_t>(s) * n_rows + row));
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float den = 0.f;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) {
    const float l = __ldg(part_lse + static_cast<int64_t>(s) * n_rows + row);
    const float4 v = __ldg(reinterpret_cast<const float4*>(part + (static_cast<int64_t>(s) * n_rows + row) * kMlaDv) + threadIdx.x);
    if (l != -INFINITY) {
      const float w = expf(l - top);
      den += w;
      acc.x = fmaf(w, v.x, acc.x); acc.y = fmaf(w, v.y, acc.y);
      acc.z = fmaf(w, v.z, acc.z); acc.w = fmaf(w, v.w, acc.w);
    }
  }
  const float inv = den != 0.f ? 1.0f / den : 0.f;   // a NaN denominator stays one
  acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
  const int64_t at = static_cast<int64_t>(row) * kMlaDv + threadIdx.x * 4;
  if (ctx_bf16) {
    uint2 o;
    o.x = pack_bf16x2(acc.x, acc.y);
    o.y = pack_bf16x2(acc.z, acc.w);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(ctx) + at) = o;
  } else {
    *reinterpret_cast<float4*>(static_cast<float*>(ctx) + at) = acc;
  }
  if (threadIdx.x == 0) lse[row] = den != 0.f ? top + logf(den) : -INFINITY;
}

template <bool kPrefetch>
static cudaError_t mlc_launch(const MlaCachedParams& p, int device, cudaStream_t stream) {
  static OncePerDevice once;
  const cudaError_t e = once.run(device, [] {
    return cudaFuncSetAttribute(sparse_mla_cached_kernel<kPrefetch>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMlaSmemBytes);
  });
  if (e != cudaSuccess) return e;
  return launch_chained(sparse_mla_cached_kernel<kPrefetch>, dim3(p.n_items * p.halves * p.splits), dim3(kMlcThreads),
                        kMlaSmemBytes, stream, p);
}

// Items whose CTAs fill whole waves of the multiprocessors.
static int whole_wave_items(int n_items, int n_heads, int sms) {
  const int halves = n_heads > kMlaHeadsTile ? 2 : 1;
  return static_cast<int>(static_cast<int64_t>(n_items) * halves / sms * sms / halves);
}

static cudaError_t mlc_run(const MlaCachedParams& p, bool prefetch, int device, cudaStream_t stream) {
  if (p.n_items == 0) return cudaSuccess;
  // Up to 16 heads the codes are multiplied as they are: 148 items x 2048 keys take 54 us for 16 heads, and 76 us for 17,
  // which the kernel for 64 heads does (it takes the same time for 1 head as for 64).
  cudaError_t e;
  if (p.n_heads <= kMlcFewHeads) e = mla_cached_few_launch(p, device, stream);
  else e = prefetch ? mlc_launch<true>(p, device, stream) : mlc_launch<false>(p, device, stream);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess || p.splits == 1) return e;
  // the merge becomes resident while the attention drains (it waits for it inside)
  const int rows = p.n_items * p.n_heads;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, mla_merge_kernel, static_cast<const float*>(p.part), rows, p.splits, p.ctx, p.ctx_bf16, p.lse);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

static int mlc_rc(cudaError_t e) {
  if (e == cudaSuccess) return B200DSA_OK;
  set_last_error(cudaGetErrorString(e));
  return B200DSA_ECUDA;
}

}  // namespace b200dsa

using namespace b200dsa;

extern "C" int b200dsa_sparse_mla_decode_cached_splits(int32_t n_items, int32_t n_heads, int32_t n_idx, int32_t tree) {
  if (n_items < 1 || n_heads < 1 || n_idx < 0) return 1;
  DeviceInfo dev;
  if (current_device_info(&dev) != cudaSuccess) return 1;
  // The least estimated time, in clocks: waves of CTAs over the SMs, so much a tile (64 keys; 128 in the kernel for few
  // heads) and 23000 around them (start of the CTA, first positions, pages and rows, Q, output), and for the merge 6000 and
  // the traffic of the parts (2 KB a row written and read, 2 KB a clock).  Measured at 1 .. 592 items: the choice is
  // within 5 % of the best.
  const bool few = n_heads <= kMlcFewHeads;
  const int64_t ctas = static_cast<int64_t>(n_items) * (n_heads > kMlaHeadsTile ? 2 : 1);
  const int keys = few ? 2 * kMlaTile : kMlaTile;
  const int tiles = (n_idx + keys - 1) / keys + (tree ? 1 : 0);
  const double tile_clocks = few ? 3900.0 : 3700.0;
  int best = 1;
  double least = 0;
  for (int s = 1; s <= kMlcMaxSplits && (s == 1 || s <= tiles); ++s) {
    const double waves = static_cast<double>((ctas * s + dev.sms - 1) / dev.sms);
    const double cost = waves * ((tiles + s - 1) / s * tile_clocks + 23000.0) +
                        (s > 1 ? 6000.0 + 2.0 * s * n_items * n_heads : 0.0);
    if (s == 1 || cost < least) {
      least = cost;
      best = s;
    }
  }
  // Items that would start one more, mostly empty wave can be a launch of their own, cut into runs, while those of the full
  // waves stay whole (192 items x 16 heads on 148 SMs: 148 whole, 44 in three runs).
  const int rest = n_items - whole_wave_items(n_items, n_heads, dev.sms);
  for (int s = 2; rest > 0 && rest < n_items && s <= kMlcMaxSplits && s <= tiles; ++s) {
    const int64_t rest_ctas = static_cast<int64_t>(rest) * (n_heads > kMlaHeadsTile ? 2 : 1);
    const double cost = static_cast<double>(ctas / dev.sms) * (tiles * tile_clocks + 23000.0) +
                        static_cast<double>((rest_ctas * s + dev.sms - 1) / dev.sms) * ((tiles + s - 1) / s * tile_clocks + 23000.0) +
                        6000.0 + 2.0 * s * rest * n_heads + 4000.0;
    if (cost * 1.03 < least) {
      least = cost * 1.03;
      best = -s;
    }
  }
  return best;
}

extern "C" int b200dsa_sparse_mla_decode_cached(const void* q_bf16, const void* cache, int64_t n_slots, int32_t page_size,
                                                const int32_t* block_table, int64_t table_stride, int32_t table_cols,
                                                int32_t n_requests, const int32_t* row_request, const int32_t* indices,
                                                int64_t idx_stride, int32_t n_idx, const int32_t* n_idx_item,
                                                const int32_t* q_pos, int32_t q_pos_bias, const int64_t* tree_mask,
                                                const int32_t* tree_base, int32_t n_items, int32_t n_heads,
                                                float sm_scale, void* ctx, int32_t ctx_bf16, float* lse, int32_t splits,
                                                void* workspace, int64_t workspace_bytes, int32_t* status,
                                                void* stream) {
  if (n_items == 0) return B200DSA_OK;
  if (!q_bf16 || !cache || !block_table || (!indices && n_idx > 0) || !ctx || !lse || !status || n_items < 0 ||
      n_heads < 1 || n_heads > kMlaMaxHeads || n_idx < 0 || n_idx > (1 << 30) || idx_stride < n_idx || n_slots < 1 ||
      n_slots > 0x7fffffffll || page_size < 1 || table_cols < 1 || table_stride < table_cols || n_requests < 1 ||
      (!row_request && n_requests < n_items) || !(sm_scale > 0.f) || (tree_mask && !tree_base) || splits < -kMlcMaxSplits ||
      splits == 0 || splits == -1 || splits > kMlcMaxSplits || static_cast<int64_t>(n_items) * 2 * kMlcMaxSplits > 0x7fffffffll) {
    set_last_error("b200dsa_sparse_mla_decode_cached: bad argument (1 <= n_heads <= 128, 1 <= splits <= 32 or -32 <= splits <= -2, "
                   "idx_stride >= n_idx, sm_scale > 0, a request for every item)");
    return B200DSA_EINVAL;
  }
  DeviceInfo dev{};
  cudaError_t e = cudaSuccess;
  if (splits < 0 && (e = current_device_info(&dev)) != cudaSuccess) return mlc_rc(e);
  // splits < 0: the items of full waves whole, the others in -splits runs
  const int whole = splits == 1 ? n_items : splits < 0 ? whole_wave_items(n_items, n_heads, dev.sms) : 0;
  const int runs = splits < 0 ? -splits : splits;
  const int64_t rows = static_cast<int64_t>(n_items - whole) * n_heads;
  if (rows > 0 && (!workspace || workspace_bytes < rows * runs * (kMlaDv + 1) * 4)) {
    set_last_error("b200dsa_sparse_mla_decode_cached: the workspace is smaller than 513 floats for every run of every head");
    return B200DSA_EINVAL;
  }
  if ((reinterpret_cast<uintptr_t>(q_bf16) & 15) || (reinterpret_cast<uintptr_t>(cache) & 15) ||
      (reinterpret_cast<uintptr_t>(ctx) & 15) || (rows > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15))) {
    set_last_error("b200dsa_sparse_mla_decode_cached: q, cache, ctx and workspace must be 16-byte aligned");
    return B200DSA_EALIGN;
  }
  if (splits > 0 && (e = current_device_info(&dev)) != cudaSuccess) return mlc_rc(e);
  MlaCachedParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q_bf16);
  p.cache = static_cast<const uint8_t*>(cache);
  p.n_slots = n_slots;
  p.table = block_table;
  p.table_stride = table_stride;
  p.table_cols = table_cols;
  p.page_size = page_size;
  p.n_requests = n_requests;
  p.row_request = row_request;
  p.indices = indices;
  p.idx_stride = idx_stride;
  p.n_idx = n_idx;
  p.n_idx_item = n_idx_item;
  p.q_pos = q_pos;
  p.q_pos_bias = q_pos_bias;
  p.tree_mask = tree_mask;
  p.tree_base = tree_base;
  p.n_items = n_items;
  p.n_heads = n_heads;
  p.halves = n_heads > kMlaHeadsTile ? 2 : 1;
  p.splits = runs;
  p.ahead = dev.sms;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.ctx = ctx;
  p.ctx_bf16 = ctx_bf16 != 0;
  p.lse = lse;
  p.part = static_cast<float*>(workspace);
  p.status = status;
  // Rows that several items of a request select are in L2 after the first of them; prefetches then only take load slots (2048
  // items of one request 1788 us with, 1748 without; one item a request 71.7 with, 78.7 without).  The rows of the block table stand for
  // the requests, which with row_request only the device knows: a table much larger than the call's requests keeps the prefetches.
  // (The kernel for few heads has none.)
  const bool prefetch = n_items < 4ll * n_requests;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  MlaCachedParams first = p;
  first.n_items = whole;
  first.splits = 1;
  e = mlc_run(first, prefetch, dev.index, st);
  if (e != cudaSuccess) return mlc_rc(e);
  p.n_items -= whole;
  p.q += static_cast<int64_t>(whole) * n_heads * kMlaD;
  if (p.indices) p.indices += whole * idx_stride;
  if (p.n_idx_item) p.n_idx_item += whole;
  if (p.q_pos) p.q_pos += whole;
  if (p.tree_mask) p.tree_mask += whole;
  if (p.row_request) {
    p.row_request += whole;
  } else {                     // item i is request i
    p.table += whole * table_stride;
    p.n_requests -= whole;
    if (p.tree_base) p.tree_base += whole;
  }
  p.ctx = static_cast<uint8_t*>(ctx) + static_cast<int64_t>(whole) * n_heads * kMlaDv * (ctx_bf16 ? 2 : 4);
  p.lse += static_cast<int64_t>(whole) * n_heads;
  e = mlc_run(p, prefetch, dev.index, st);
  return mlc_rc(e);
}
