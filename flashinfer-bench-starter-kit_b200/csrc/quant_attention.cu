// quant_attention.cu -- attention over the paged latent cache in 8 bits: dense,
// for single tokens and chains of drafts, and over selected slots (sm_100a).
//
// With the cache's token k as codes c_k (512 e4m3), scale s_k and position part
// e_k (64 bf16):
//   x_k = scale * (s_k (q_nope . c_k) + q_pe . e_k)
//   lse = log2 sum_k 2^(x_k log2 e),   out = sum_k 2^(x_k log2 e - lse) s_k c_k
//
// This first form is the plain one: one CTA per query row and 16 heads, a warp
// per head, tiles of 16 tokens in shared memory, everything in fp32.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "dsa_b200.h"
#include "host.h"
#include "ptx.cuh"

namespace dsa {
namespace qattn {

constexpr int kCkv = DSA_CKV_DIM;
constexpr int kKpe = DSA_KPE_DIM;
constexpr int kPage = DSA_PAGE_SIZE;
constexpr int kPageBytes = DSA_LATENT_PAGE_BYTES;
constexpr int kKpeAt = kPage * kCkv;
constexpr int kScaleAt = kKpeAt + kPage * kKpe * 2;
constexpr int kTile = 16;
constexpr int kHeads = 16;
constexpr int kMaxRequests = 65536;
constexpr int64_t kMaxRows = 1 << 24;  // rows x heads

struct Params {
  const __nv_bfloat16* q_nope;
  const __nv_bfloat16* q_pe;
  const uint8_t* cache;
  int num_pages;
  const int32_t* seq_lens;
  const int32_t* block_table;
  const int32_t* cu;        // or nullptr: row r is request r's
  const int32_t* picked;    // sparse: [rows][topk]
  int topk;
  int num_requests, num_rows, heads, max_pages;
  float scale_log2;
  __nv_bfloat16* out;
  float* lse;
  unsigned int* status;
};

__device__ __forceinline__ float fp8(uint8_t x) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(x, __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&h));
}

__global__ void __launch_bounds__(32 * kHeads)
plain_kernel(const Params p) {
  griddep_wait();
  __shared__ float tile[kTile][kCkv + kKpe];
  __shared__ int64_t where[kTile];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x, head = blockIdx.y * kHeads + warp;
  int tokens = p.topk;
  const int32_t* table = nullptr;
  if (p.picked == nullptr) {
    int r = row;
    int len;
    if (p.cu != nullptr) {
      bool decreasing = p.cu[0] < 0 || p.cu[p.num_requests] > p.num_rows;
      for (int k = tid; k < p.num_requests; k += blockDim.x) decreasing |= p.cu[k + 1] < p.cu[k];
      if (__syncthreads_or(decreasing)) {
        if (tid == 0) atomicOr(p.status, DSA_DEV_BAD_SEQ_LEN);
        return;
      }
      if (row < p.cu[0] || row >= p.cu[p.num_requests]) return;
      int lo = 0, hi = p.num_requests;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (p.cu[mid] <= row) lo = mid;
        else hi = mid;
      }
      r = lo;
      len = p.seq_lens[r];
      if (len < 0 || len > p.max_pages * kPage) {
        if (tid == 0) atomicOr(p.status, DSA_DEV_BAD_SEQ_LEN);
        len = len < 0 ? 0 : p.max_pages * kPage;
      }
      len -= p.cu[r + 1] - 1 - row;
    } else {
      len = p.seq_lens[r];
      if (len < 0 || len > p.max_pages * kPage) {
        if (tid == 0) atomicOr(p.status, DSA_DEV_BAD_SEQ_LEN);
        len = len < 0 ? 0 : p.max_pages * kPage;
      }
    }
    tokens = max(len, 0);
    table = p.block_table + static_cast<int64_t>(r) * p.max_pages;
  }
  float q[18], o[16], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) o[k] = 0.f;
  if (head < p.heads) {
    const int64_t at = static_cast<int64_t>(row) * p.heads + head;
#pragma unroll
    for (int k = 0; k < 16; ++k) q[k] = __bfloat162float(p.q_nope[at * kCkv + lane + 32 * k]);
#pragma unroll
    for (int k = 0; k < 2; ++k) q[16 + k] = __bfloat162float(p.q_pe[at * kKpe + lane + 32 * k]);
  }
  for (int t0 = 0; t0 < tokens; t0 += kTile) {
    __syncthreads();
    if (tid < kTile) {
      int64_t w = -1;
      const int t = t0 + tid;
      if (t < tokens) {
        int64_t slot;
        if (p.picked != nullptr) {
          slot = p.picked[static_cast<int64_t>(row) * p.topk + t];
          if (slot < -1 || slot >= static_cast<int64_t>(p.num_pages) * kPage) {
            atomicOr(p.status, DSA_DEV_BAD_INDEX);
            slot = -1;
          }
        } else {
          const int page = table[t / kPage];
          slot = static_cast<int64_t>(page) * kPage + t % kPage;
          if (page < 0 || page >= p.num_pages) {
            atomicOr(p.status, DSA_DEV_BAD_PAGE);
            slot = -1;
          }
        }
        if (slot >= 0) w = slot;
      }
      where[tid] = w;
    }
    __syncthreads();
    for (int t = warp; t < kTile; t += kHeads) {
      if (where[t] < 0) continue;
      const uint8_t* page = p.cache + where[t] / kPage * kPageBytes;
      const int in = static_cast<int>(where[t] % kPage);
      const float s = *reinterpret_cast<const float*>(page + kScaleAt + 4 * in);
      for (int k = lane; k < kCkv; k += 32) tile[t][k] = s * fp8(page[in * kCkv + k]);
      for (int k = lane; k < kKpe; k += 32)
        tile[t][kCkv + k] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(page + kKpeAt)[in * kKpe + k]);
    }
    __syncthreads();
    if (head < p.heads) {
      for (int t = 0; t < kTile; ++t) {
        if (where[t] < 0) continue;
        float x = 0.f;
#pragma unroll
        for (int k = 0; k < 18; ++k) x = fmaf(q[k], tile[t][lane + 32 * k], x);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
        x *= p.scale_log2;
        const float top = fmaxf(m, x);
        if (!(x <= m)) {  // NaN too
          const float a = m == -INFINITY ? 0.f : exp2f(m - top);
          l *= a;
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] *= a;
          m = top;
        }
        const float w = x == -INFINITY ? 0.f : exp2f(x - m);
        l += w;
#pragma unroll
        for (int k = 0; k < 16; ++k) o[k] = fmaf(w, tile[t][lane + 32 * k], o[k]);
      }
    }
  }
  if (head < p.heads) {
    const int64_t at = static_cast<int64_t>(row) * p.heads + head;
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int k = 0; k < 16; ++k) p.out[at * kCkv + lane + 32 * k] = __float2bfloat16_rn(o[k] * inv);
    if (lane == 0) p.lse[at] = l == 0.f ? -INFINITY : m + log2f(l);
  }
}

struct Range {
  const void* at;
  size_t bytes;
};

// Outputs lie apart from what other CTAs still read, but for the output over
// q_nope itself, whose rows are written behind their last use.
int check_outputs(const void* output, const float* lse, size_t rows_q, const Range* in, int count) {
  const Range out[2] = {{output, rows_q * kCkv * 2}, {lse, rows_q * 4}};
  if (ranges_overlap(output, out[0].bytes, lse, out[1].bytes)) return DSA_ERR_OVERLAP;
  for (int o = 0; o < 2; ++o)
    for (int i = 0; i < count; ++i)
      if (in[i].at != nullptr && ranges_overlap(out[o].at, out[o].bytes, in[i].at, in[i].bytes) &&
          !(o == 0 && i == 0 && output == in[0].at))
        return DSA_ERR_OVERLAP;
  return DSA_OK;
}

int launch(const Params& p, cudaStream_t s) {
  if (launch_programmatic(plain_kernel, dim3(p.num_rows, (p.heads + kHeads - 1) / kHeads), dim3(32 * kHeads), 0, s, p) !=
          cudaSuccess ||
      cudaGetLastError() != cudaSuccess)
    return DSA_ERR_CUDA;
  return DSA_OK;
}

}  // namespace qattn
}  // namespace dsa

using namespace dsa;

extern "C" size_t dsa_latent_attention_workspace_bytes(void) { return kWorkspaceHeader; }

extern "C" int dsa_latent_attention_run(const void* q_nope, const void* q_pe, const void* latent_cache, int64_t num_pages,
                                        const int32_t* seq_lens, const int32_t* block_table, const int32_t* cu_rows,
                                        int32_t num_requests, int32_t num_rows, int32_t num_heads, int32_t max_pages,
                                        float sm_scale, void* output, float* lse, void* workspace, size_t workspace_bytes,
                                        void* stream) {
  if (num_rows < 0 || num_heads < 1 || num_heads > 128 || num_requests < 0 || num_requests > qattn::kMaxRequests ||
      static_cast<int64_t>(num_rows) * num_heads > qattn::kMaxRows)
    return DSA_ERR_INVALID_ARGUMENT;
  if (num_rows == 0 || num_requests == 0) return DSA_OK;
  if (!q_nope || !q_pe || !latent_cache || !seq_lens || !block_table || !output || !lse || !workspace || num_pages < 1 ||
      num_pages > 0x7FFFFFFE || max_pages < 1 || max_pages > (1 << 24) || (!cu_rows && num_rows != num_requests))
    return DSA_ERR_INVALID_ARGUMENT;
  if (!aligned16(q_nope) || !aligned16(q_pe) || !aligned16(latent_cache) || !aligned16(output) || !aligned16(workspace) ||
      ((reinterpret_cast<uintptr_t>(seq_lens) | reinterpret_cast<uintptr_t>(block_table) |
        reinterpret_cast<uintptr_t>(cu_rows) | reinterpret_cast<uintptr_t>(lse)) & 3u))
    return DSA_ERR_MISALIGNED;
  const size_t n = static_cast<size_t>(num_requests), rows_q = static_cast<size_t>(num_rows) * num_heads;
  const qattn::Range in[6] = {{q_nope, rows_q * qattn::kCkv * 2},
                              {q_pe, rows_q * qattn::kKpe * 2},
                              {latent_cache, static_cast<size_t>(num_pages) * qattn::kPageBytes},
                              {seq_lens, n * 4},
                              {block_table, n * max_pages * 4},
                              {cu_rows, (n + 1) * 4}};
  int st = qattn::check_outputs(output, lse, rows_q, in, 6);
  if (st != DSA_OK) return st;
  DeviceInfo info;
  if ((st = current_device_info(&info)) != DSA_OK) return st;
  if (workspace_bytes < dsa_latent_attention_workspace_bytes()) return DSA_ERR_WORKSPACE_TOO_SMALL;
  qattn::Params p{};
  p.q_nope = static_cast<const __nv_bfloat16*>(q_nope);
  p.q_pe = static_cast<const __nv_bfloat16*>(q_pe);
  p.cache = static_cast<const uint8_t*>(latent_cache);
  p.num_pages = static_cast<int>(num_pages);
  p.seq_lens = seq_lens;
  p.block_table = block_table;
  p.cu = cu_rows;
  p.num_requests = num_requests;
  p.num_rows = num_rows;
  p.heads = num_heads;
  p.max_pages = max_pages;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.out = static_cast<__nv_bfloat16*>(output);
  p.lse = lse;
  p.status = static_cast<unsigned int*>(workspace);
  return qattn::launch(p, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int dsa_latent_sparse_attention_run(const void* q_nope, const void* q_pe, const void* latent_cache,
                                               int64_t num_pages, const int32_t* sparse_indices, int32_t num_rows,
                                               int32_t num_heads, int32_t topk, float sm_scale, void* output, float* lse,
                                               void* workspace, size_t workspace_bytes, void* stream) {
  if (num_rows < 0 || num_heads < 1 || num_heads > 128 || static_cast<int64_t>(num_rows) * num_heads > qattn::kMaxRows ||
      topk < 1 || topk > 65536)
    return DSA_ERR_INVALID_ARGUMENT;
  if (num_rows == 0) return DSA_OK;
  if (!q_nope || !q_pe || !latent_cache || !sparse_indices || !output || !lse || !workspace || num_pages < 1 ||
      num_pages > 0x7FFFFFFF / qattn::kPage)
    return DSA_ERR_INVALID_ARGUMENT;
  if (!aligned16(q_nope) || !aligned16(q_pe) || !aligned16(latent_cache) || !aligned16(output) || !aligned16(workspace) ||
      ((reinterpret_cast<uintptr_t>(sparse_indices) | reinterpret_cast<uintptr_t>(lse)) & 3u))
    return DSA_ERR_MISALIGNED;
  const size_t rows_q = static_cast<size_t>(num_rows) * num_heads;
  const qattn::Range in[4] = {{q_nope, rows_q * qattn::kCkv * 2},
                              {q_pe, rows_q * qattn::kKpe * 2},
                              {latent_cache, static_cast<size_t>(num_pages) * qattn::kPageBytes},
                              {sparse_indices, static_cast<size_t>(num_rows) * topk * 4}};
  int st = qattn::check_outputs(output, lse, rows_q, in, 4);
  if (st != DSA_OK) return st;
  DeviceInfo info;
  if ((st = current_device_info(&info)) != DSA_OK) return st;
  if (workspace_bytes < dsa_latent_attention_workspace_bytes()) return DSA_ERR_WORKSPACE_TOO_SMALL;
  qattn::Params p{};
  p.q_nope = static_cast<const __nv_bfloat16*>(q_nope);
  p.q_pe = static_cast<const __nv_bfloat16*>(q_pe);
  p.cache = static_cast<const uint8_t*>(latent_cache);
  p.num_pages = static_cast<int>(num_pages);
  p.picked = sparse_indices;
  p.topk = topk;
  p.num_rows = num_rows;
  p.heads = num_heads;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.out = static_cast<__nv_bfloat16*>(output);
  p.lse = lse;
  p.status = static_cast<unsigned int*>(workspace);
  return qattn::launch(p, reinterpret_cast<cudaStream_t>(stream));
}
