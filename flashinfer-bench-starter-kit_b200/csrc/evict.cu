// evict.cu -- eviction from the paged caches by accumulated attention weight.
//
// Request r has L = seq_lens[r] tokens and keeps at most `budget` of them:
// the first num_sink, the last num_recent, and of the tokens between those
// with the largest accumulated weight (equal ones: the earlier; NaN counts as
// largest).  Their order stays.  Two kernels:
//
// select_kernel: one thread-block cluster per request.  Each CTA holds its
//   slice of the request's weights in shared memory, read from HBM once (4 B
//   per token).  The boundary weight is found by radix: a histogram of the
//   order key's top 11 bits, then of the next 11 and the last 10 among the
//   keys that share the boundary's bits, each added up in the first CTA's
//   shared memory with the sums of every 32 bins: a warp of each CTA finds the
//   boundary bin from those 64 sums and 32 bins, 384 bytes of remote reads
//   (all 2048 bins from one SM took 4400 clocks a pass).  The kept positions
//   then come out in order: a
//   token's place is the number kept before it, from ballots, a scan over
//   the CTA's warps and the counts of the lower CTAs.
// move_kernel: copies the kept tokens' rows of every cache to their new
//   pages, up to 1284 B per token in and out; HBM-bound.  It writes the new
//   lengths too: they may take the old ones' place, which all of a cluster's
//   threads read for themselves.
//
// Measured, 32 requests of 32768-65536 tokens to 8192: select 28 us (latency of
// its barriers and remote reads; 7 us for one request of 5001 to 1024), move
// 106 us (262144 tokens, 673 MB, 6.3 TB/s).
#include <mutex>

#include "dsa_b200.h"
#include "host.h"
#include "ptx.cuh"

namespace dsa {
namespace evict {

constexpr int kPage = DSA_PAGE_SIZE;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 16;            // beyond the portable 8, allowed below
constexpr int kMaxResident = 49152;        // weights a CTA can hold (192 KB)
constexpr int kCoarse = kBins / 32;         // sums of 32 bins each
constexpr uint32_t kZeroKey = 0x80000000u;  // score_key of 0

struct Params {
  const float* acc;
  int64_t acc_stride;
  const int32_t* seq_lens;
  const int32_t* block_table;
  const int32_t* new_block_table;
  int requests, max_pages, new_max_pages;
  int budget, num_sink, num_recent;
  int resident;                            // weights that fit the CTA's shared memory
  uint8_t* ckv;
  uint8_t* kpe;
  uint8_t* index;                          // may be null
  int64_t ckv_page, ckv_row, kpe_page, kpe_row;
  int num_pages;
  int32_t* keep;
  int32_t* new_seq_lens;
  float* new_acc;
  int64_t new_acc_stride;
  unsigned int* status;
};

__device__ __forceinline__ int length_of(const Params& p, int b, bool& bad) {
  const int L = p.seq_lens[b];
  const int cap = p.max_pages * kPage;
  bad = L < 0 || L > cap;
  return L < 0 ? 0 : (L > cap ? cap : L);
}

// Inclusive sum over the warp's lanes.
__device__ __forceinline__ int warp_scan(int v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += a;
  }
  return v;
}

__global__ void __launch_bounds__(kThreads) select_kernel(const Params p) {
  extern __shared__ uint32_t keys[];       // of this CTA's tokens, if they fit
  __shared__ __align__(16) int hist[kBins];          // this CTA's, of one pass
  __shared__ int sums[3][kBins], coarse[3][kCoarse];  // the cluster's, in its first CTA
  __shared__ int counts[2];                // tokens above the boundary key, and at it
  __shared__ int lower[2];                 // those of the lower CTAs
  __shared__ int scratch[2][kWarps];
  __shared__ int found[3];                 // boundary bin, kept ones needed from it, its size
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ctas = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
  const int b = blockIdx.x / ctas;
  griddep_wait();
  // The move kernel is not let in early: its blocks, waiting on the SMs, would
  // keep clusters out (158 against 137 us at 32 x 65536 tokens to 8192).

  bool bad;
  const int L = length_of(p, b, bad);
  if (bad && rank == 0 && tid == 0) atomicOr(p.status, DSA_DEV_BAD_SEQ_LEN);
  const float* acc = p.acc + b * p.acc_stride;
  int32_t* keep = p.keep + static_cast<int64_t>(b) * p.budget;
  float* new_acc = p.new_acc + b * p.new_acc_stride;
  const int kept = L < p.budget ? L : p.budget;
  const int t0 = rank * kThreads + tid, step = ctas * kThreads;
  // Behind what is kept.
  for (int i = kept + t0; i < p.budget; i += step) keep[i] = -1;
  for (int i = kept + t0; i < p.new_max_pages * kPage; i += step) new_acc[i] = 0.f;
  if (L <= p.budget) {
    for (int i = t0; i < L; i += step) {
      keep[i] = i;
      new_acc[i] = acc[i];
    }
    return;  // the whole cluster leaves here
  }
  int need = p.budget - p.num_sink - p.num_recent;  // from the middle; fewer than it has
  const int middle = L - p.num_sink - p.num_recent;
  const int slice = (middle + ctas - 1) / ctas;
  const int lo = min(rank * slice, middle), n = min(slice, middle - lo);
  const float* mine = acc + p.num_sink + lo;
  const bool fits = slice <= p.resident;
  if (fits && need > 0)
    for (int i = tid; i < n; i += kThreads) cp_async4(smem_u32(keys + i), mine + i);
  for (int i = t0; i < p.num_sink + p.num_recent; i += step) {
    const bool first = i < p.num_sink;
    const int pos = first ? i : L - p.num_recent + (i - p.num_sink);
    const int to = first ? i : p.budget - p.num_recent + (i - p.num_sink);
    keep[to] = pos;
    new_acc[to] = acc[pos];
  }
  if (need == 0) return;
  for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
  if (rank == 0) {
    for (int i = tid; i < 3 * kBins; i += kThreads) sums[0][i] = 0;
    if (tid < 3 * kCoarse) coarse[0][tid] = 0;
  }
  cluster_arrive();                        // waited for before the first remote access
  cp_async_wait_all();                     // each thread turns its own copies into keys below
  __syncthreads();
  auto key_of = [&](int i) { return fits ? keys[i] : score_key(mine[i]); };

  // ---- boundary key: 11 + 11 + 10 bits.
  uint32_t prefix = 0;                     // the boundary key's bits so far
  uint32_t above = 0xffffffffu;            // kept for sure: keys > above
  int ties = 0;                            // kept ones among keys == above
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const int bins = pass == 2 ? 1024 : kBins;
    const int upper = shift + (pass == 2 ? 10 : 11);
    for (int i0 = 0; i0 < n; i0 += kThreads) {
      const int i = i0 + tid;
      bool count = i < n;
      uint32_t key = 0;
      if (count) {
        if (pass == 0 && fits) {
          key = score_key(__uint_as_float(keys[i]));
          keys[i] = key;
        } else {
          key = key_of(i);
        }
      }
      count = count && (pass == 0 || (key >> upper) == prefix);
      // Tokens that were never read have exactly 0: a warp adds all of its at
      // once.
      const unsigned int zeros = __ballot_sync(0xffffffffu, count && key == kZeroKey);
      if (zeros != 0 && lane == 0) atomicAdd(&hist[(kZeroKey >> shift) & (bins - 1)], __popc(zeros));
      if (count && key != kZeroKey) atomicAdd(&hist[(key >> shift) & (bins - 1)], 1);
    }
    __syncthreads();
    if (pass == 0) cluster_wait();
    {
      // Thread t adds its bins 4t .. 4t + 3 to the first CTA's, eight threads
      // the sum of their 32, and clears them for the next pass.
      static_assert(kBins == 4 * kThreads, "four bins a thread");
      int4* own = reinterpret_cast<int4*>(hist) + tid;
      const int4 q = *own;
      *own = make_int4(0, 0, 0, 0);
      int* to = &sums[pass][4 * tid];
      if (q.x != 0) add_cluster(to, 0, q.x);
      if (q.y != 0) add_cluster(to + 1, 0, q.y);
      if (q.z != 0) add_cluster(to + 2, 0, q.z);
      if (q.w != 0) add_cluster(to + 3, 0, q.w);
      int sum = (q.x + q.y) + (q.z + q.w);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if ((tid & 7) == 0 && sum != 0) add_cluster(&coarse[pass][tid >> 3], 0, sum);
    }
    cluster_sync();
    if (warp == 0) {
      // From the largest bins down: lane l has two coarse sums, then one bin.
      const int at = bins / 32 - 1 - 2 * lane;
      const int c0 = at >= 0 ? ld_cluster(&coarse[pass][at], 0) : 0;
      const int c1 = at >= 1 ? ld_cluster(&coarse[pass][at - 1], 0) : 0;
      int before = warp_scan(c0 + c1) - (c0 + c1);
      const bool here = before < need && need <= before + c0 + c1;
      const int lead = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
      const bool second = need > before + c0;
      const int block = __shfl_sync(0xffffffffu, second ? at - 1 : at, lead);
      const int above_block = __shfl_sync(0xffffffffu, second ? before + c0 : before, lead);
      const int bin = 32 * block + 31 - lane;
      const int c = ld_cluster(&sums[pass][bin], 0);
      before = above_block + warp_scan(c) - c;
      if (before < need && need <= before + c) {
        found[0] = bin;
        found[1] = need - before;
        found[2] = c;
      }
    }
    __syncthreads();
    prefix = (prefix << (pass == 2 ? 10 : 11)) | static_cast<uint32_t>(found[0]);
    need = found[1];
    const bool all = found[2] == need;     // the whole bin is kept: no key bits below matter
    __syncthreads();
    if (all || pass == 2) {
      above = all ? (prefix << shift) - 1u : prefix;  // not below 0: some key of the middle is not kept
      ties = all ? 0 : need;
      break;
    }
  }

  // ---- counts, then the positions in order.  A warp has a run of tokens, so
  // that its first kept token's place needs one sum over the lower warps.
  const int run = (n + kWarps * 32 - 1) / (kWarps * 32) * 32;
  const int w_lo = min(warp * run, n), w_hi = min(w_lo + run, n);
  int g_at = 0, q_at = 0;                  // tokens above the boundary key, and at it, before the warp's next
#pragma unroll 4
  for (int i0 = w_lo; i0 < w_hi; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t key = i < w_hi ? key_of(i) : 0u;
    g_at += __popc(__ballot_sync(0xffffffffu, i < w_hi && key > above));
    q_at += __popc(__ballot_sync(0xffffffffu, i < w_hi && key == above));
  }
  if (lane == 0) {
    scratch[0][warp] = g_at;
    scratch[1][warp] = q_at;
  }
  __syncthreads();
  if (warp == 0) {
    int g = lane < kWarps ? scratch[0][lane] : 0, q = lane < kWarps ? scratch[1][lane] : 0;
    const int g_sum = warp_scan(g), q_sum = warp_scan(q);
    if (lane < kWarps) {
      scratch[0][lane] = g_sum - g;
      scratch[1][lane] = q_sum - q;
    }
    if (lane == kWarps - 1) {
      counts[0] = g_sum;
      counts[1] = q_sum;
    }
  }
  cluster_sync();
  if (warp == 0) {
    int g = lane < rank ? ld_cluster(&counts[0], lane) : 0, q = lane < rank ? ld_cluster(&counts[1], lane) : 0;
    g = warp_scan(g);
    q = warp_scan(q);
    if (lane == 31) {
      lower[0] = g;
      lower[1] = q;
    }
  }
  __syncthreads();
  // That was the last remote access: a CTA leaves once all have made theirs.
  cluster_arrive();
  g_at = lower[0] + scratch[0][warp];
  q_at = lower[1] + scratch[1][warp];
  const unsigned int lt = (1u << lane) - 1u;
#pragma unroll 4
  for (int i0 = w_lo; i0 < w_hi; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t key = i < w_hi ? key_of(i) : 0u;
    const bool up = i < w_hi && key > above, tie = i < w_hi && key == above;
    const unsigned int up_mask = __ballot_sync(0xffffffffu, up), tie_mask = __ballot_sync(0xffffffffu, tie);
    const int q = q_at + __popc(tie_mask & lt);  // ties before this token; the first `ties` are kept
    if (up || (tie && q < ties)) {
      const int to = p.num_sink + g_at + __popc(up_mask & lt) + min(q, ties);
      keep[to] = p.num_sink + lo + i;
      new_acc[to] = mine[i];
    }
    g_at += __popc(up_mask);
    q_at += __popc(tie_mask);
  }
  cluster_wait();
}

// A warp moves kMoveTokens tokens at a time: all their loads (5 KB) are in
// flight before the first store.
constexpr int kMoveThreads = 256;
constexpr int kMoveWarps = kMoveThreads / 32;
constexpr int kMoveTokens = 4;
constexpr int kIndexRow = DSA_INDEX_DIM;               // 128 bytes, then the page's 64 scales
constexpr int kIndexScales = kPage * kIndexRow;

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const Params p) {
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int per_row = (p.budget + kMoveTokens - 1) / kMoveTokens;
  const int64_t all = static_cast<int64_t>(p.requests) * per_row;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kMoveWarps;
  for (int64_t w = static_cast<int64_t>(blockIdx.x) * kMoveWarps + (threadIdx.x >> 5); w < all; w += step) {
    const int b = static_cast<int>(w / per_row), i0 = static_cast<int>(w % per_row) * kMoveTokens;
    if (i0 == 0 && lane == 0) {
      bool bad;  // reported by the select
      p.new_seq_lens[b] = min(length_of(p, b, bad), p.budget);
    }
    // Lane l looks up token l & 3 of the four.
    const int i = i0 + (lane & (kMoveTokens - 1));
    const int pos = i < p.budget ? __ldcg(p.keep + static_cast<int64_t>(b) * p.budget + i) : -1;
    int from = -1, to = -1;                            // pages; from < 0: nothing to move
    if (pos >= 0) {
      from = p.block_table[static_cast<int64_t>(b) * p.max_pages + pos / kPage];
      to = p.new_block_table[static_cast<int64_t>(b) * p.new_max_pages + i / kPage];
      if (from < 0 || from >= p.num_pages || to < 0 || to >= p.num_pages) {
        if (lane < kMoveTokens) atomicOr(p.status, DSA_DEV_BAD_PAGE);
        from = -1;
      }
    }
    const int row = pos & (kPage - 1);
    if (__all_sync(0xffffffffu, from < 0)) continue;
    // ckv: 64 pieces of 16 bytes a token, two a lane.
    int f[kMoveTokens], t[kMoveTokens];
    uint4 c[2 * kMoveTokens];
#pragma unroll
    for (int k = 0; k < kMoveTokens; ++k) {
      f[k] = __shfl_sync(0xffffffffu, from, k);
      t[k] = __shfl_sync(0xffffffffu, to, k);
      const int r = __shfl_sync(0xffffffffu, row, k);
      if (f[k] >= 0) {
        const uint4* src = reinterpret_cast<const uint4*>(p.ckv + f[k] * p.ckv_page + r * p.ckv_row) + lane;
        c[2 * k] = __ldcg(src);
        c[2 * k + 1] = __ldcg(src + 32);
      }
    }
    // kpe and index keys: 8 pieces a token, lane l has piece l & 7 of token l >> 3.
    const int k = lane >> 3, piece = 16 * (lane & 7);
    const int fk = __shfl_sync(0xffffffffu, from, k), tk = __shfl_sync(0xffffffffu, to, k);
    const int rk = __shfl_sync(0xffffffffu, row, k), dk = (i0 + k) & (kPage - 1);
    uint4 e = make_uint4(0u, 0u, 0u, 0u), x = e;
    uint32_t scale = 0;
    if (fk >= 0) {
      e = __ldcg(reinterpret_cast<const uint4*>(p.kpe + fk * p.kpe_page + rk * p.kpe_row + piece));
      if (p.index != nullptr) {
        const uint8_t* page = p.index + static_cast<int64_t>(fk) * DSA_INDEX_PAGE_BYTES;
        x = __ldcg(reinterpret_cast<const uint4*>(page + rk * kIndexRow + piece));
        if (piece == 0) scale = __ldcg(reinterpret_cast<const uint32_t*>(page + kIndexScales + 4 * rk));
      }
    }
#pragma unroll
    for (int q = 0; q < kMoveTokens; ++q) {
      if (f[q] >= 0) {
        uint4* dst =
            reinterpret_cast<uint4*>(p.ckv + t[q] * p.ckv_page + ((i0 + q) & (kPage - 1)) * p.ckv_row) + lane;
        dst[0] = c[2 * q];
        dst[32] = c[2 * q + 1];
      }
    }
    if (fk >= 0) {
      *reinterpret_cast<uint4*>(p.kpe + tk * p.kpe_page + dk * p.kpe_row + piece) = e;
      if (p.index != nullptr) {
        uint8_t* page = p.index + static_cast<int64_t>(tk) * DSA_INDEX_PAGE_BYTES;
        *reinterpret_cast<uint4*>(page + dk * kIndexRow + piece) = x;
        if (piece == 0) *reinterpret_cast<uint32_t*>(page + kIndexScales + 4 * dk) = scale;
      }
    }
  }
}

// CTAs per request: as many as the cluster limit, the SMs (two 512-thread CTAs
// each) and the table's width can use, down to 256 tokens a CTA.  One request of
// 65536 tokens: 14.9 us with 16, 20.0 with 8; 8 of 3000-4096: 11.3 us, 15.5 with
// 8192 tokens a CTA.
int cluster_for(int requests, int max_pages, int sms) {
  int c = kMaxCluster;
  while (c > 1 && (static_cast<int64_t>(requests) * c > 2 * sms || static_cast<int64_t>(max_pages) * kPage <= 512 * (c / 2)))
    c /= 2;
  return c;
}

std::once_flag g_once[64];
int g_status[64];

}  // namespace evict
}  // namespace dsa

using namespace dsa;

extern "C" int dsa_cache_evict_run(const float* acc, int64_t acc_stride, const int32_t* seq_lens,
                                   const int32_t* block_table, const int32_t* new_block_table, int32_t num_requests,
                                   int32_t max_pages, int32_t new_max_pages, void* ckv_cache, int64_t ckv_page_bytes,
                                   int64_t ckv_row_bytes, void* kpe_cache, int64_t kpe_page_bytes,
                                   int64_t kpe_row_bytes, void* k_index_cache_fp8, int64_t num_pages, int32_t budget,
                                   int32_t num_sink, int32_t num_recent, int32_t* keep, int32_t* new_seq_lens,
                                   float* new_acc, int64_t new_acc_stride, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  if (num_requests < 0 || num_requests > 65536) return DSA_ERR_INVALID_ARGUMENT;
  if (num_requests == 0) return DSA_OK;
  if (!acc || !seq_lens || !block_table || !new_block_table || !ckv_cache || !kpe_cache || !keep || !new_seq_lens ||
      !new_acc || !workspace)
    return DSA_ERR_INVALID_ARGUMENT;
  if (num_pages < 1 || num_pages > 0x7FFFFFFF || max_pages < 1 || max_pages > (1 << 24) || new_max_pages < 1 ||
      new_max_pages > (1 << 24))
    return DSA_ERR_INVALID_ARGUMENT;
  if (budget < 1 || budget > new_max_pages * evict::kPage || num_sink < 0 || num_recent < 0 ||
      static_cast<int64_t>(num_sink) + num_recent > budget)
    return DSA_ERR_INVALID_ARGUMENT;
  if (acc_stride < static_cast<int64_t>(max_pages) * evict::kPage ||
      new_acc_stride < static_cast<int64_t>(new_max_pages) * evict::kPage)
    return DSA_ERR_INVALID_ARGUMENT;
  if (ckv_row_bytes < DSA_CKV_DIM * 2 || kpe_row_bytes < DSA_KPE_DIM * 2 || ckv_page_bytes < 0 || kpe_page_bytes < 0)
    return DSA_ERR_INVALID_ARGUMENT;
  if (!aligned16(ckv_cache) || !aligned16(kpe_cache) || !aligned16(k_index_cache_fp8) || !aligned16(workspace) ||
      ((ckv_page_bytes | ckv_row_bytes | kpe_page_bytes | kpe_row_bytes) & 15))
    return DSA_ERR_MISALIGNED;
  if ((reinterpret_cast<uintptr_t>(acc) | reinterpret_cast<uintptr_t>(seq_lens) |
       reinterpret_cast<uintptr_t>(block_table) | reinterpret_cast<uintptr_t>(new_block_table) |
       reinterpret_cast<uintptr_t>(keep) | reinterpret_cast<uintptr_t>(new_seq_lens) |
       reinterpret_cast<uintptr_t>(new_acc)) & 3u)
    return DSA_ERR_MISALIGNED;
  if (workspace_bytes < kWorkspaceHeader) return DSA_ERR_WORKSPACE_TOO_SMALL;
  // The kernels read their inputs while they write keep and new_acc; a
  // request's length alone is read by nobody once its new one is written.
  const size_t n = static_cast<size_t>(num_requests);
  const int64_t width = static_cast<int64_t>(max_pages) * evict::kPage;
  const int64_t new_width = static_cast<int64_t>(new_max_pages) * evict::kPage;
  const struct {
    const void* at;
    size_t bytes;
  } out[3] = {{keep, n * budget * 4}, {new_seq_lens, n * 4}, {new_acc, ((n - 1) * new_acc_stride + new_width) * 4}},
    in[3] = {{seq_lens, n * 4}, {block_table, n * max_pages * 4}, {new_block_table, n * new_max_pages * 4}};
  for (int i = 0; i < 3; ++i) {
    for (int j = 0; j < 3; ++j) {
      if (i < j && ranges_overlap(out[i].at, out[i].bytes, out[j].at, out[j].bytes)) return DSA_ERR_OVERLAP;
      const bool in_place = i == 1 && j == 0 && new_seq_lens == seq_lens;
      if (!in_place && ranges_overlap(out[i].at, out[i].bytes, in[j].at, in[j].bytes)) return DSA_ERR_OVERLAP;
    }
  }
  const size_t acc_bytes = static_cast<size_t>((num_requests - 1) * acc_stride + width) * 4;
  if (ranges_overlap(keep, out[0].bytes, acc, acc_bytes) || ranges_overlap(new_seq_lens, out[1].bytes, acc, acc_bytes) ||
      rows_overlap(num_requests, acc, acc_stride, width, new_acc, new_acc_stride, new_width))
    return DSA_ERR_OVERLAP;
  DeviceInfo info;
  int st = current_device_info(&info);
  if (st != DSA_OK) return st;
  std::call_once(evict::g_once[info.device], [&]() {
    evict::g_status[info.device] =
        cudaFuncSetAttribute(evict::select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             evict::kMaxResident * 4) == cudaSuccess &&
                cudaFuncSetAttribute(evict::select_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) ==
                    cudaSuccess
            ? DSA_OK
            : DSA_ERR_CUDA;
  });
  if (evict::g_status[info.device] != DSA_OK) return evict::g_status[info.device];

  evict::Params p{};
  p.acc = acc;
  p.acc_stride = acc_stride;
  p.seq_lens = seq_lens;
  p.block_table = block_table;
  p.new_block_table = new_block_table;
  p.requests = num_requests;
  p.max_pages = max_pages;
  p.new_max_pages = new_max_pages;
  p.budget = budget;
  p.num_sink = num_sink;
  p.num_recent = num_recent;
  p.ckv = static_cast<uint8_t*>(ckv_cache);
  p.kpe = static_cast<uint8_t*>(kpe_cache);
  p.index = static_cast<uint8_t*>(k_index_cache_fp8);
  p.ckv_page = ckv_page_bytes;
  p.ckv_row = ckv_row_bytes;
  p.kpe_page = kpe_page_bytes;
  p.kpe_row = kpe_row_bytes;
  p.num_pages = static_cast<int>(num_pages);
  p.keep = keep;
  p.new_seq_lens = new_seq_lens;
  p.new_acc = new_acc;
  p.new_acc_stride = new_acc_stride;
  p.status = static_cast<unsigned int*>(workspace);

  const int ctas = evict::cluster_for(num_requests, max_pages, info.num_sms);
  const int64_t slice = (static_cast<int64_t>(max_pages) * evict::kPage + ctas - 1) / ctas;
  p.resident = static_cast<int>(slice < evict::kMaxResident ? slice : evict::kMaxResident);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned int>(num_requests) * ctas);
  cfg.blockDim = dim3(evict::kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(p.resident) * 4;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned int>(ctas);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, evict::select_kernel, p) != cudaSuccess) return DSA_ERR_CUDA;
  const int64_t warps = static_cast<int64_t>(num_requests) * ((budget + evict::kMoveTokens - 1) / evict::kMoveTokens);
  const int64_t blocks = (warps + evict::kMoveWarps - 1) / evict::kMoveWarps;
  const int64_t most = 0x7FFFFFFF;  // beyond, warps take several turns
  if (launch_programmatic(evict::move_kernel, dim3(static_cast<unsigned int>(blocks < most ? blocks : most)),
                          dim3(evict::kMoveThreads), 0, s, p) != cudaSuccess)
    return DSA_ERR_CUDA;
  if (cudaGetLastError() != cudaSuccess) return DSA_ERR_CUDA;
  return DSA_OK;
}
