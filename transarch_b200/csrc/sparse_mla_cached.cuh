// Parameters and the key warp of the attention kernels over the quantised latent cache.
#pragma once

#include "latent_cache.cuh"
#include "sparse_mla.cuh"

namespace b200dsa {

struct MlaCachedParams {
  const __nv_bfloat16* q;        // [n_items, n_heads, 576]
  const uint8_t* cache;
  int64_t n_slots;
  const int32_t* table;          // [n_requests, table_stride] pages
  int64_t table_stride;
  int table_cols, page_size, n_requests;
  const int32_t* row_request;    // nullable [n_items]
  const int32_t* indices;        // [n_items, idx_stride]
  int64_t idx_stride;
  int n_idx;
  const int32_t* n_idx_item;     // nullable [n_items]
  const int32_t* q_pos;          // nullable [n_items]
  int q_pos_bias;
  const int64_t* tree_mask;      // nullable [n_items]
  const int32_t* tree_base;      // [n_requests] with tree_mask
  int n_items, n_heads, halves, splits;
  int ahead;                     // CTAs that run at a time
  float scale_log2;
  void* ctx;
  int ctx_bf16;
  float* lse;
  float* part;                   // splits > 1: [splits, n_items, n_heads, 512] then [splits, n_items, n_heads]
  int32_t* status;
};


// One warp turns the positions of an item's keys into slots of the cache, kTile keys at a time, up to kRing tiles ahead of
// the warps that fetch the rows, and with kPrefetch has the rows brought into L2 meanwhile.  Tiles tile0 .. tile0 + n_tiles - 1 of the
// item: its selected positions, then (with a tree mask) one tile of drafted tokens.
template <int kTile, int kRing, bool kPrefetch>
__device__ __forceinline__ void mlc_key_warp(const MlaCachedParams& p, int item, int tile0, int n_tiles, int n_idx,
                                             int* s_slot, uint64_t* key_full, uint64_t* key_empty,
                                             volatile int* abort_flag) {
  constexpr int kPer = kTile / 32;
  const int lane = threadIdx.x & 31;
  const int sel_tiles = (n_idx + kTile - 1) / kTile;
  const int32_t* idx_row = p.indices + static_cast<int64_t>(item) * p.idx_stride;
  int req = p.row_request ? __ldg(p.row_request + item) : item;
  bool known = req >= 0 && req < p.n_requests;
  if (!known) {
    if (lane == 0) atomicMax(p.status, kDevBadIndex);
    req = 0;
  }
  const int32_t* table = p.table + static_cast<int64_t>(req) * p.table_stride;
  const unsigned long long mask = p.tree_mask ? static_cast<unsigned long long>(__ldg(p.tree_mask + item)) : 0ull;
  const int base = p.tree_mask ? __ldg(p.tree_base + req) : 0x7fffffff;
  int64_t last = static_cast<int64_t>(base) - 1;    // the last position that may be attended by selection
  if (p.q_pos) last = min(last, static_cast<int64_t>(__ldg(p.q_pos + item)) + p.q_pos_bias);
  struct Key {
    int page, off;       // page -1: outside the table; off -1: no key
  };
  // Positions of keys lane, lane + 32, ... of tile t, -1 = none.  Positions are fetched two tiles ahead of the pages'
  // entries, those one ahead of the slots, so that no step waits for the load of the one before it.
  auto positions = [&](int t, int (&pos)[kPer]) {
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
      const int tt = tile0 + t, i = lane + 32 * h;
      pos[h] = -1;
      if (t >= n_tiles || !known) continue;
      if (tt < sel_tiles) {
        const int j = tt * kTile + i;
        if (j < n_idx) pos[h] = __ldg(idx_row + j);
      } else {
        const int64_t v = static_cast<int64_t>(base) + i;
        if (i < 64 && ((mask >> i) & 1) && base >= 0 && v <= 0x7fffffff) pos[h] = static_cast<int>(v);
      }
    }
  };
  auto pages = [&](int t, const int (&pos)[kPer], Key (&key)[kPer]) {
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
      const int v = pos[h];
      key[h].page = key[h].off = -1;
      if (v < 0 || (v > last && tile0 + t < sel_tiles)) continue;
      const int col = v / p.page_size;
      key[h].off = v - col * p.page_size;
      if (col < p.table_cols) key[h].page = __ldg(table + col);
    }
  };
  auto slot_of = [&](const Key& k) -> int {         // -1 = none; a page that does not exist is reported
    if (k.off < 0) return -1;
    const int64_t slot = static_cast<int64_t>(k.page) * p.page_size + k.off;
    if (k.page < 0 || slot >= p.n_slots) {
      atomicMax(p.status, kDevBadIndex);
      return -1;
    }
    return static_cast<int>(slot);
  };
  int pos[2][kPer];
  Key key[kPer];
  positions(0, pos[0]);
  pages(0, pos[0], key);
  positions(1, pos[1]);
  positions(2, pos[0]);
  bool ok = true;
#pragma unroll 2
  for (int t = 0; ok && t < n_tiles; ++t) {
    const int ring = t % kRing;
    int slot[kPer];
#pragma unroll
    for (int h = 0; h < kPer; ++h) slot[h] = slot_of(key[h]);
    pages(t + 1, pos[(t + 1) & 1], key);
    positions(t + 3, pos[(t + 1) & 1]);
    ok = __all_sync(0xffffffffu, mbar_wait(&key_empty[ring], ((t / kRing) & 1) ^ 1, abort_flag));
    if (!ok) break;
#pragma unroll
    for (int h = 0; h < kPer; ++h) s_slot[ring * kTile + lane + 32 * h] = slot[h];
    __syncwarp();
    if (lane == 0) mbar_arrive(&key_full[ring]);
    // 656 bytes lie in at most seven lines of 128; the first tiles are loaded at once
    for (int i = 0; kPrefetch && t >= 2 && i < kTile / 4; ++i) {
      const int r = 4 * i + (lane >> 3), s = s_slot[ring * kTile + r];
      if (s >= 0 && (lane & 7) < 7)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p.cache + static_cast<int64_t>(s) * kLatentRowBytes +
                                                     min((lane & 7) * 128, kLatentRowBytes - 1)));
    }
  }
  // With many items: the positions and queries of the CTA that takes this one's place, into L2 (2048 x 128 x 2048: 1750 ->
  // 1721 us)
  const int next = blockIdx.x + p.ahead;
  if (!kPrefetch && next < gridDim.x) {
    const int it = next / (p.splits * p.halves), h0 = next / p.splits % p.halves * kMlaHeadsTile;
    const char* idx = reinterpret_cast<const char*>(p.indices + static_cast<int64_t>(it) * p.idx_stride);
    for (int64_t b = lane * 128; b < static_cast<int64_t>(p.n_idx) * 4; b += 32 * 128)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(idx + b));
    const char* q = reinterpret_cast<const char*>(p.q + (static_cast<int64_t>(it) * p.n_heads + h0) * kMlaD);
    const int bytes = min(kMlaHeadsTile, p.n_heads - h0) * kMlaD * 2;
    for (int b = lane * 128; b < bytes; b += 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + b));
  }
}

// Up to kMlcFewHeads heads: the kernel that multiplies the codes as they are (sparse_mla_cached_few.cu).
constexpr int kMlcFewHeads = 16;
cudaError_t mla_cached_few_launch(const MlaCachedParams& p, int device, cudaStream_t stream);

}  // namespace b200dsa
