// The quantised latent cache of MLA: rows of 656 bytes, token slot s at byte 656 * s,
//   [0, 512)    e4m3 codes of the 512 latent dims
//   [512, 528)  four fp32 scales, one for every 128 dims:  value = code * scale
//   [528, 656)  the 64 position dims in bf16
//
// Write (one pass from the projection's output to the cache):
//   n = c * rsqrt(mean(c^2) + eps) * gain          over the 512 latent dims (optional)
//   r = rotation of the 64 position dims           (optional; half form or interleaved pairs)
//   scale_g = max(amax_g |n|, 1e-4) / 448, rounded up to a power of two for the "ue8m0" format
//   code = e4m3(n / scale_g), nearest even; r is rounded to bf16 once.  All arithmetic in fp32.
//   A group with a NaN or an infinity gets scale NaN and reads as NaN throughout.
// A power-of-two scale makes every later use exact: code * scale has four significant bits and fits bf16, so the
// attention over the cache and the rows read back see the same numbers.
//
// One warp per row.  Lane l holds dims 8l..8l+7 of either half of the latent dims (group = half * 2 + l / 16) and the
// rotation pair l, so that every load and store of the warp is one contiguous run of 256 or 512 bytes.  Reading 72 384 rows
// takes 24.6 us (5.3 TB/s of bytes read and written; what it writes stays in L2, issue slots are 59 % busy), a million rows run at
// 6.1 TB/s, near the memory's rate.  Writing 4096 tokens and reading them back takes 6.1 us, two launches; writing 65 536 takes 50 us
// (3.0 TB/s): a row's loads wait for that of its slot.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "latent_cache.cuh"

namespace b200dsa {

void set_last_error(const char* msg);

struct LatentWriteParams {
  const void* in;              // [n_tokens] rows of 576 values, in_stride elements apart
  int in_f32, in_vec;          // in_vec: rows start on 16-byte boundaries
  int64_t in_stride, n_tokens;
  const void* gain;            // nullable [512]
  int gain_f32;
  float eps;
  const float* cos;            // nullable [n_tokens, 64]
  const float* sin;
  int interleaved;
  const int64_t* slot_mapping;
  uint8_t* cache;
  int64_t n_slots;
  int32_t* status;
};

constexpr int kRowWarps = 4;   // warps (rows) per CTA: a decode batch spreads over more SMs than with eight

__device__ __forceinline__ float latent_load1(const void* p, int64_t i, int f32) {
  return f32 ? __ldg(static_cast<const float*>(p) + i) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
// eight consecutive values
__device__ __forceinline__ void latent_load8(const void* p, int64_t i, int f32, int vec, float (&x)[8]) {
  if (!vec) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = latent_load1(p, i + j, f32);
  } else if (f32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 a = __ldg(q), b = __ldg(q + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + i));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __uint_as_float(w[j] << 16);
      x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  }
}

template <bool kPow2>
__global__ void __launch_bounds__(32 * kRowWarps) latent_write_kernel(const LatentWriteParams p) {
  pdl_launch_dependents();
  pdl_wait_prior();
  const int64_t tok = static_cast<int64_t>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5);
  if (tok >= p.n_tokens) return;
  const int lane = threadIdx.x & 31;
  const int64_t slot = __ldg(p.slot_mapping + tok);
  if (slot < 0) return;                       // padding token
  if (slot >= p.n_slots) {
    if (lane == 0) atomicMax(p.status, kDevBadIndex);
    return;
  }
  const int64_t base = tok * p.in_stride;
  float x[2][8];
  latent_load8(p.in, base + 8 * lane, p.in_f32, p.in_vec, x[0]);
  latent_load8(p.in, base + 256 + 8 * lane, p.in_f32, p.in_vec, x[1]);
  const int ia = p.interleaved ? 2 * lane : lane, ib = p.interleaved ? 2 * lane + 1 : lane + 32;
  float ra = latent_load1(p.in, base + 512 + ia, p.in_f32), rb = latent_load1(p.in, base + 512 + ib, p.in_f32);
  float ca = 1.f, cb = 1.f, sa = 0.f, sb = 0.f;
  if (p.cos) {
    const float* c = p.cos + tok * 64;
    const float* s = p.sin + tok * 64;
    ca = __ldg(c + lane); sa = __ldg(s + lane);
    cb = p.interleaved ? ca : __ldg(c + lane + 32);
    sb = p.interleaved ? sa : __ldg(s + lane + 32);
  }
  if (p.gain) {
    float sq = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = fmaf(x[h][j], x[h][j], sq);
    for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    const float rstd = rsqrtf(sq * (1.0f / 512.0f) + p.eps);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float g[8];
      latent_load8(p.gain, 256 * h + 8 * lane, p.gain_f32, 1, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[h][j] = x[h][j] * rstd * g[j];
    }
  }
  uint8_t* row = p.cache + slot * kLatentRowBytes;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(x[h][j]));
    for (int o = 8; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    GroupScale g = kPow2 ? group_scale_pow2(max_nan(amax, 1e-4f)) : group_scale(max_nan(amax, 1e-4f));
    if (!(amax < INFINITY)) g.scale = __int_as_float(0x7fffffff);   // not finite: the whole group reads as NaN
    const float scale = g.scale;
    uint2 codes;
    codes.x = quant_e4m3x4<kPow2>(x[h][0], x[h][1], x[h][2], x[h][3], g);
    codes.y = quant_e4m3x4<kPow2>(x[h][4], x[h][5], x[h][6], x[h][7], g);
    *reinterpret_cast<uint2*>(row + 256 * h + 8 * lane) = codes;
    if ((lane & 15) == 0) *reinterpret_cast<float*>(row + 512 + 4 * (2 * h + (lane >> 4))) = scale;
  }
  const float oa = ra * ca - rb * sa, ob = rb * cb + ra * sb;
  __nv_bfloat16* pe = reinterpret_cast<__nv_bfloat16*>(row + 528);
  if (p.interleaved) {
    reinterpret_cast<__nv_bfloat162*>(pe)[lane] = __floats2bfloat162_rn(oa, ob);
  } else {
    pe[lane] = __float2bfloat16_rn(oa);
    pe[lane + 32] = __float2bfloat16_rn(ob);
  }
}

struct LatentReadParams {
  const uint8_t* cache;
  int64_t n_slots;
  const int64_t* slots;        // by slot: [n_rows], negative = a row of zeros
  const int32_t* table;        // by request: [n_requests, table_stride] pages
  int64_t table_stride;
  int table_cols, page_size;
  const int32_t* cu;           // [n_requests + 1] first row of every request
  int n_requests;
  int64_t n_rows;
  __nv_bfloat16* out;          // [n_rows, 576]
  int32_t* status;
};

__global__ void __launch_bounds__(32 * kRowWarps) latent_read_kernel(const LatentReadParams p) {
  pdl_launch_dependents();
  pdl_wait_prior();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5);
  if (row >= p.n_rows) return;
  const int lane = threadIdx.x & 31;
  int64_t slot = -1;
  if (p.slots) {
    slot = __ldg(p.slots + row);
    if (slot >= p.n_slots) {
      if (lane == 0) atomicMax(p.status, kDevBadIndex);
      slot = -1;
    }
  } else {
    // request of the row: how many requests end at or before it (the lanes look at 32 ends at a time)
    int r = 0;
    for (int r0 = 0; r0 < p.n_requests; r0 += 32) {
      const bool ends = r0 + lane < p.n_requests && __ldg(p.cu + r0 + lane + 1) <= row;
      const unsigned m = __ballot_sync(0xffffffffu, ends);
      r += __popc(m);
      if (m != 0xffffffffu) break;
    }
    if (r >= p.n_requests) return;            // behind the last request: left as it was
    const int64_t pos = row - __ldg(p.cu + r);
    const int64_t col = pos / p.page_size;
    const int page = pos >= 0 && col < p.table_cols ? __ldg(p.table + r * p.table_stride + col) : -1;
    slot = static_cast<int64_t>(page) * p.page_size + (pos - col * p.page_size);
    if (page < 0 || slot >= p.n_slots) {
      if (lane == 0) atomicMax(p.status, kDevBadIndex);
      slot = -1;
    }
  }
  __nv_bfloat16* out = p.out + row * 576;
  uint32_t pe = 0;
  uint4 o[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (slot >= 0) {
    const uint8_t* in = p.cache + slot * kLatentRowBytes;
    const uint2 c0 = __ldg(reinterpret_cast<const uint2*>(in + 8 * lane));
    const uint2 c1 = __ldg(reinterpret_cast<const uint2*>(in + 256 + 8 * lane));
    const float s0 = __ldg(reinterpret_cast<const float*>(in + 512) + (lane >> 4));
    const float s1 = __ldg(reinterpret_cast<const float*>(in + 512) + 2 + (lane >> 4));
    pe = __ldg(reinterpret_cast<const uint32_t*>(in + 528) + lane);
    dequant_e4m3x4(c0.x, s0, o[0].x, o[0].y);
    dequant_e4m3x4(c0.y, s0, o[0].z, o[0].w);
    dequant_e4m3x4(c1.x, s1, o[1].x, o[1].y);
    dequant_e4m3x4(c1.y, s1, o[1].z, o[1].w);
  }
  *reinterpret_cast<uint4*>(out + 8 * lane) = o[0];
  *reinterpret_cast<uint4*>(out + 256 + 8 * lane) = o[1];
  reinterpret_cast<uint32_t*>(out + 512)[lane] = pe;
}

// Ancestor masks of trees of drafted tokens: bit i of mask[r, j] = node i lies on the path from node j to its root
// (j itself included).  A parent comes before its children, so a walk takes at most 64 steps.
__global__ void __launch_bounds__(64) draft_tree_masks_kernel(const int32_t* __restrict__ parents, int n_nodes,
                                                              int64_t* __restrict__ masks, int32_t* status) {
  pdl_launch_dependents();
  pdl_wait_prior();
  __shared__ int32_t s_parent[64];
  const int64_t base = static_cast<int64_t>(blockIdx.x) * n_nodes;
  const int j = threadIdx.x;
  if (j < n_nodes) s_parent[j] = parents[base + j];
  __syncthreads();
  if (j >= n_nodes) return;
  unsigned long long m = 0;
  int at = j;
  while (at >= 0) {
    m |= 1ull << at;
    const int up = s_parent[at];
    if (up >= at) {                           // not a tree in order: the path ends here
      atomicMax(status, kDevBadIndex);
      break;
    }
    at = up;
  }
  masks[base + j] = static_cast<int64_t>(m);
}

static int cuda_rc(cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e == cudaSuccess) return B200DSA_OK;
  set_last_error(cudaGetErrorString(e));
  return B200DSA_ECUDA;
}

}  // namespace b200dsa

using namespace b200dsa;

extern "C" int b200dsa_latent_quant_and_cache(const void* kv, int32_t in_f32, int64_t in_stride, int64_t n_tokens,
                                              const void* gain, int32_t gain_f32, float eps, const float* cos,
                                              const float* sin, int32_t interleaved, const int64_t* slot_mapping,
                                              void* cache, int64_t n_slots, int32_t use_ue8m0, int32_t* status,
                                              void* stream) {
  if (n_tokens == 0) return B200DSA_OK;
  if (!kv || !slot_mapping || !cache || !status || n_tokens < 0 || n_tokens > (1ll << 31) || n_slots < 1 ||
      in_stride < 576 || ((cos == nullptr) != (sin == nullptr))) {
    set_last_error("b200dsa_latent_quant_and_cache: bad argument (rows of 576 values, cos and sin together)");
    return B200DSA_EINVAL;
  }
  const uintptr_t elem = in_f32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(cache) & 15) || (gain && (reinterpret_cast<uintptr_t>(gain) & 15)) ||
      (reinterpret_cast<uintptr_t>(kv) % elem)) {
    set_last_error("b200dsa_latent_quant_and_cache: cache and gain must be 16-byte aligned");
    return B200DSA_EALIGN;
  }
  LatentWriteParams p{};
  p.in = kv;
  p.in_f32 = in_f32 != 0;
  p.in_vec = !(reinterpret_cast<uintptr_t>(kv) & 15) && !((in_stride * static_cast<int64_t>(elem)) & 15);
  p.in_stride = in_stride;
  p.n_tokens = n_tokens;
  p.gain = gain;
  p.gain_f32 = gain_f32 != 0;
  p.eps = eps;
  p.cos = cos;
  p.sin = sin;
  p.interleaved = interleaved != 0;
  p.slot_mapping = slot_mapping;
  p.cache = static_cast<uint8_t*>(cache);
  p.n_slots = n_slots;
  p.status = status;
  return cuda_rc(launch_chained(use_ue8m0 ? latent_write_kernel<true> : latent_write_kernel<false>, dim3(static_cast<unsigned>((n_tokens + kRowWarps - 1) / kRowWarps)),
                                dim3(32 * kRowWarps), 0, static_cast<cudaStream_t>(stream), p));
}

static int latent_read(LatentReadParams& p, void* stream) {
  if (reinterpret_cast<uintptr_t>(p.cache) & 15 || reinterpret_cast<uintptr_t>(p.out) & 15) {
    set_last_error("b200dsa_latent_cache_rows / _gather: cache and out must be 16-byte aligned");
    return B200DSA_EALIGN;
  }
  return cuda_rc(launch_chained(latent_read_kernel, dim3(static_cast<unsigned>((p.n_rows + kRowWarps - 1) / kRowWarps)),
                                dim3(32 * kRowWarps), 0, static_cast<cudaStream_t>(stream), p));
}

extern "C" int b200dsa_latent_cache_rows(const void* cache, int64_t n_slots, const int64_t* slots, int64_t n_rows,
                                         void* out_bf16, int32_t* status, void* stream) {
  if (n_rows == 0) return B200DSA_OK;
  if (!cache || !slots || !out_bf16 || !status || n_rows < 0 || n_rows > (1ll << 31) || n_slots < 1) {
    set_last_error("b200dsa_latent_cache_rows: bad argument");
    return B200DSA_EINVAL;
  }
  LatentReadParams p{};
  p.cache = static_cast<const uint8_t*>(cache);
  p.n_slots = n_slots;
  p.slots = slots;
  p.n_rows = n_rows;
  p.out = static_cast<__nv_bfloat16*>(out_bf16);
  p.status = status;
  return latent_read(p, stream);
}

extern "C" int b200dsa_latent_cache_gather(const void* cache, int64_t n_slots, int32_t page_size,
                                           const int32_t* block_table, int64_t table_stride, int32_t table_cols,
                                           const int32_t* cu_rows, int32_t n_requests, int64_t n_rows, void* out_bf16,
                                           int32_t* status, void* stream) {
  if (n_rows == 0 || n_requests == 0) return B200DSA_OK;
  if (!cache || !block_table || !cu_rows || !out_bf16 || !status || n_rows < 0 || n_rows > (1ll << 31) || n_slots < 1 ||
      page_size < 1 || n_requests < 0 || table_cols < 1 || table_stride < table_cols) {
    set_last_error("b200dsa_latent_cache_gather: bad argument");
    return B200DSA_EINVAL;
  }
  LatentReadParams p{};
  p.cache = static_cast<const uint8_t*>(cache);
  p.n_slots = n_slots;
  p.table = block_table;
  p.table_stride = table_stride;
  p.table_cols = table_cols;
  p.page_size = page_size;
  p.cu = cu_rows;
  p.n_requests = n_requests;
  p.n_rows = n_rows;
  p.out = static_cast<__nv_bfloat16*>(out_bf16);
  p.status = status;
  return latent_read(p, stream);
}

extern "C" int b200dsa_draft_tree_masks(const int32_t* parents, int32_t n_trees, int32_t n_nodes, int64_t* masks,
                                        int32_t* status, void* stream) {
  if (n_trees == 0 || n_nodes == 0) return B200DSA_OK;
  if (!parents || !masks || !status || n_trees < 0 || n_nodes < 0 || n_nodes > 64) {
    set_last_error("b200dsa_draft_tree_masks: bad argument (at most 64 nodes a tree)");
    return B200DSA_EINVAL;
  }
  return cuda_rc(launch_chained(draft_tree_masks_kernel, dim3(n_trees), dim3(64), 0, static_cast<cudaStream_t>(stream),
                                parents, static_cast<int>(n_nodes), masks, status));
}
