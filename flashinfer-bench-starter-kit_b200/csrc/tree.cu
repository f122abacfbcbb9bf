// tree.cu -- attention for a tree of drafted tokens over the paged ckv / kpe
// cache, and the accumulation of the attention weights its rows give to the
// cached tokens (sm_100a).
//
// Request b has prefix_lens[b] cached tokens and n drafts (rows cu[b] ..
// cu[b+1]-1 of the queries), whose own cache rows follow at positions
// prefix .. prefix + n - 1.  With c_k, e_k the ckv / kpe rows of position k,
// for draft i and head h
//   s_k = scale * (q_nope . c_k + q_pe . e_k)
//   visible: k < prefix, or k = prefix + j with bit j of draft i's mask set
//   lse = log2 sum_k 2^(s_k log2 e),   out = sum_k 2^(s_k log2 e - lse) c_k
// and the weights kernel adds sum_{i,h} 2^(s_k log2 e - lse_ih) to position
// k's accumulator.
//
// All heads share one key, so the n * H (draft, head) pairs of a request are
// one tall set of query rows.  They are taken kRows = 64 at a time (a group);
// a work unit is one group against one 64-token page.  Per unit
//   S^T[64 tokens, 64 rows] = K[64, 576] . Q[64, 576]^T   36 x (M64 N64 K16)
//   O^T[512, 64] += V^T[512, 64 tokens] . P^T[64 tokens, 64] 16 x (M128 N64 K16)
// with V the ckv part of the K tile in shared memory, read MN-major.  The
// transposed form leaves O^T in 256 TMEM columns (64 rows in the plain form
// would take half the lanes of 512) and makes P an operand that the softmax
// warps write without a transpose (MN-major, one 128-byte row per token).
// K tile 72 KB x 2 stages + Q 72 KB + P 8 KB fill the shared memory, which
// is what limits a CTA to 64 rows: at 64 rows the tile's 72 KB come from L2
// or HBM in about the time of its MMAs (1152 + 768 clocks, measured 32 and 48
// a piece).
//
// Units are ordered (request, group, tile) and cut into equal contiguous
// slices, one per CTA ("stream-K").  (Ordering the groups of a request by
// chunks of tiles, so that they walk the same pages at the same time, was
// measured and is slower everywhere, 64 x 65536 tokens included: twice the
// pieces, and L2 serves the second group well enough as it is.)  A slice's
// pieces that do not cover their group's whole context are written as fp32
// records (slot 0: the piece at the slice's start, slot 1: the one at its end;
// no other can be partial) and joined by combine_kernel.
//
// Measured, attention with its join, one call a graph replay: 64 x 65536 tokens
// with 4 drafts of 16 heads 798 us (4.84 GB, 6.1 TB/s: HBM-bound); 4 x 32768
// with 64 drafts 360 us (0.80 PFLOP/s: the stages' hand-over and shared memory).
// Back to back for a second the power cap makes those 963 and 434 us.  Weights:
// 32 x 8192-65536 tokens 155 us (0.93 GB, 6.0 TB/s: HBM-bound).
#include <cuda_bf16.h>

#include <mutex>

#include "dsa_b200.h"
#include "host.h"
#include "ptx.cuh"

namespace dsa {
namespace tree {

constexpr int kCkv = DSA_CKV_DIM;            // 512
constexpr int kKpe = DSA_KPE_DIM;            // 64
constexpr int kTok = DSA_PAGE_SIZE;          // 64 tokens per tile: one page
constexpr int kRows = 64;                    // query rows per group
constexpr int kChunks = 9;                   // 8 ckv + 1 kpe pieces of 64 columns
constexpr int kChunkBytes = 64 * 128;        // 8192
constexpr int kTileBytes = kChunks * kChunkBytes;  // 73728: a K tile, or a group's Q
constexpr int kSoftWarps = 8;                // warps 0-7: two sets of four, 32 rows each
constexpr int kLoadWarp = 8;                 // TMA
constexpr int kLogitWarp = 9;                // S^T MMAs (owns TMEM)
constexpr int kValueWarp = 10;               // O^T MMAs
constexpr int kThreads = 352;
constexpr int kTmemCols = 512;
constexpr uint32_t kColS = 0;                // two S^T buffers of 64 columns, for the weights of kSumsS x 64
constexpr uint32_t kColO = 128;              // O^T: 4 blocks of 128 dims x 64 columns
constexpr float kRescaleThreshold = 8.0f;    // log2 units, see the softmax warps
constexpr int kPartFloats = kRows * kCkv;    // a partial record's O, [row][dim]
constexpr int kSumTiles = 16;                // weights: tiles whose sums wait in shared memory
constexpr int kSumTilesShared = 8;           // ... when several groups re-read them through L2

// N is the group's rows, rounded up to what the instruction takes: a group of
// 16 rows (one draft of 16 heads) costs the tensor core and shared memory
// less than one of 64.  Columns behind it are neither computed nor read.
constexpr uint32_t kIdescS = idesc_make(1, 1, false, false, 64, 0);
constexpr uint32_t kIdescO = idesc_make(1, 1, true, true, 128, 0);
__device__ __forceinline__ uint32_t with_rows(uint32_t idesc, int rows) {
  return idesc | static_cast<uint32_t>((rows + 15) / 16 * 2) << 17;
}

// A tile moves in four parts with barriers of their own: part x is the ckv
// pieces 2x and 2x + 1, which O^T's block x needs, and the last has kpe too.
// S^T starts with the first part that lands, and each block of O^T frees its
// part for the tile after next.
constexpr int kParts = 4;
// The tensor core cuts its fp32 accumulator off below the last bit at every
// step, always towards zero: after 36 steps a logit is about 5e-7 of itself too
// small, which no sum over rows takes back.  The weights, which have nothing
// coarser in them, keep kSumsS sums of kSumSteps steps and add them in
// registers (TMEM has the room: there is no O).  Weights of logits from 4 to 9
// are 6.9e-7 off (rms) with three sums, 2.0e-6 with one, 1.0e-6 with two and
// 5.5e-7 with four; 4 x 12000-16384 tokens with 32-40 drafts take 70.2, 68.0,
// 70.1 and 75.7 us.  Long contexts take the same with any.  The attention rounds
// its weights to bf16, beside which this is nothing.
constexpr int kSumsS = 3;
constexpr int kSumSteps = (kCkv + kKpe) / 16 / kSumsS;
static_assert(kSumsS * kSumSteps * 16 == kCkv + kKpe, "equal sums");
__device__ __forceinline__ constexpr uint32_t part_bytes(int x) {
  return (x == kParts - 1 ? 3 : 2) * kChunkBytes;
}

constexpr int kOffQ = 2 * kTileBytes;          // 147456
constexpr int kOffP = kOffQ + kTileBytes;      // 221184: P, or the weights' sums
constexpr int kOffBar = kOffP + kTok * 128;    // 229376
constexpr int kOffMisc = kOffBar + 256;
constexpr int kOffRed = kOffMisc + 96;         // [4][64] floats
constexpr int kOffFactor = kOffRed + 1024;     // [64]
constexpr int kOffMax = kOffFactor + 256;      // [64]
constexpr int kSmemBytes = 1024 + kOffMax + 256;
static_assert(kSmemBytes <= 232448, "shared memory of a CTA");
static_assert(2 * kSumTiles * kTok * 4 <= kTok * 128, "the weights' sums take P's place");

constexpr int kMaxRequests = 65536;
constexpr int64_t kMaxRows = 1 << 24;          // drafts x heads
constexpr int64_t kMaxUnits = 1 << 30;         // units and (request, page) places are counted in 32 bits
constexpr int kMaxCtas = 256;
// Plan, in ints: the group of each record (-1: none), then first row and rows
// of each group.
constexpr int kPlanGroups = 2 * kMaxCtas;

struct Params {
  const int32_t* prefix_lens;
  const int32_t* block_table;
  const int32_t* cu;
  const long long* mask;
  int num_requests, num_drafts, heads, max_pages, mask_words;
  int num_pages;
  float scale_log2;
  unsigned int* status;
  unsigned long long wait_limit_ns;
  // attention
  __nv_bfloat16* out;
  float* lse_out;
  float* part_o;    // [2 * grid][kPartFloats]
  float* part_ml;   // [2 * grid][kRows][4]: m, l, lr
  int* plan;        // see kPlanGroups
  // weights
  const float* lse_in;
  const float* acc;
  float* acc_out;
  int64_t acc_stride, acc_out_stride;
};

struct Request {
  int prefix, n, row0;  // cached tokens, drafts, first draft's row
  int rows, groups, tiles;
  int span;             // units per group: its tiles and, for the attention, kLead more
};

// Starting a group (its queries, the pipeline's first tile, O's way out) takes
// about as long as three more tiles.  So a group counts kLead units more than
// its tiles, at its start, when slices are cut (200 requests of 50-700 tokens:
// 48.5 us at 0, 43.2 at 1, 39.4 at 2, 38.0 at 3, 38.5 at 4; long contexts: no
// change).
constexpr int kLead = 3;

// Inputs are read with plain loads, not through the non-coherent path: a
// kernel launched programmatically may lie on an SM while the one before it
// still writes them.
//
// Request b as its inputs give it; what they give wrongly is clamped or, if
// it cannot be, taken as a request without drafts.
template <bool kWeights>
__device__ __forceinline__ Request load_request(const Params& p, int b, bool& bad) {
  Request r;
  const int lo = p.cu[b], hi = p.cu[b + 1];
  const int cap = p.max_pages * kTok;
  r.prefix = p.prefix_lens[b];
  r.row0 = lo;
  r.n = hi - lo;
  bad = false;
  if (lo < 0 || hi < lo || hi > p.num_drafts || r.n > cap) {
    r.n = 0;
    bad = true;
  }
  if (r.prefix < 0) {
    r.prefix = 0;
    bad = true;
  }
  if (r.prefix > cap - r.n) {
    r.prefix = cap - r.n;
    bad = true;
  }
  bad |= (r.n + 63) / 64 > p.mask_words;
  r.rows = r.n * p.heads;
  r.groups = (r.rows + kRows - 1) / kRows;
  r.tiles = r.n == 0 ? 0 : (r.prefix + r.n + kTok - 1) / kTok;
  r.span = r.n == 0 || kWeights ? r.tiles : r.tiles + kLead;
  return r;
}

// Slice boundaries: CTA c of `ctas` has units [start(c), start(c+1)), with
// start(c) = floor(total * c / ctas) in 32-bit steps.
__device__ __forceinline__ int slice_start(int total, int c, int ctas) {
  const int q = total / ctas;
  return q * c + (total - q * ctas) * c / ctas;
}
// Where a slice starts, as the plan found it.
struct Start {
  int b, first, first_group;  // request, its first unit and group over all requests
  Request r;
  int group, unit;            // attention: of the request; of the group
};

// A run of tiles of one group.
struct Segment {
  int b, group, t0, t1;
  __device__ int rows() const { return min(kRows, r.rows - group * kRows); }
  int group_index;        // attention: over all requests
  Request r;
  bool whole;             // attention: covers the group's whole context
  int slot;               // attention: record slot if it does not
  bool first_group, last_group;  // weights: of this run of tiles
};

// The segments of a CTA's slice, in order; every role walks its own copy.
template <bool kWeights>
struct Walker {
  const Params& p;
  int u, u0, u1;
  int b, first;           // request and its first unit
  int first_group;        // its first group, over all requests
  Request r;
  int group, unit;        // attention: of the next unit
  int run0, run1, end, g; // weights: current run of tiles, end of the slice's tiles, next group

  __device__ Walker(const Params& prm, int u0_, int u1_, const Start& st)
      : p(prm), u(u0_), u0(u0_), u1(u1_), b(st.b), first(st.first), first_group(st.first_group) {
    if (u0 >= u1) return;
    r = st.r;
    group = st.group;
    unit = st.unit;
    if constexpr (kWeights) start_tiles();
  }

  __device__ void start_tiles() {
    // A tile belongs to the slice that its first unit falls into.
    const int lo = u0 - first, hi = u1 - first;
    run0 = lo <= 0 ? 0 : (lo + r.groups - 1) / r.groups;
    end = (hi + r.groups - 1) / r.groups;
    if (end > r.tiles) end = r.tiles;
    start_run();
  }
  __device__ void start_run() {
    const int most = r.groups > 1 ? kSumTilesShared : kSumTiles;
    run1 = run0 + most < end ? run0 + most : end;
    g = 0;
  }
  __device__ bool leave() {  // to the next request that has units in the slice
    for (;;) {
      first += r.groups * r.span;
      first_group += r.groups;
      ++b;
      if (b >= p.num_requests || first >= u1) return false;
      bool bad;
      r = load_request<kWeights>(p, b, bad);
      if (r.tiles == 0) continue;
      if constexpr (kWeights) {
        start_tiles();
      } else {
        group = unit = 0;
      }
      return true;
    }
  }

  __device__ bool next(Segment& s) {
    if constexpr (kWeights) {
      if (u0 >= u1) return false;
      while (run0 >= run1)
        if (b >= p.num_requests || !leave()) return false;
      s.b = b;
      s.r = r;
      s.group = g;
      s.t0 = run0;
      s.t1 = run1;
      s.first_group = g == 0;
      s.last_group = g == r.groups - 1;
      if (++g == r.groups) {
        run0 = run1;
        start_run();
      }
      return true;
    } else {
      while (u < u1) {
        s.b = b;
        s.r = r;
        s.group = group;
        s.group_index = first_group + group;
        const int len = min(r.span - unit, u1 - u);
        s.t0 = unit < kLead ? 0 : unit - kLead;
        s.t1 = unit + len - kLead;
        s.whole = s.t0 == 0 && s.t1 == r.tiles;
        s.slot = u == u0 ? 0 : 1;
        u += len;
        unit = 0;
        if (u < u1 && ++group == r.groups && !leave()) u = u1;
        if (s.t1 > s.t0) return true;  // else a slice's end within the lead
      }
      return false;
    }
  }
};

// Weights: what no unit writes, the tiles behind each request's tokens.  The
// (request, tile) places are spread over the CTAs; a CTA's warps take 32 of
// its places at a time from a counter in shared memory: the value warp, which
// the weights leave idle, from the start, the others when their tiles are done.
__device__ __forceinline__ void copy_behind(const Params& p, bool nothing, int* counter) {
  const int lane = threadIdx.x & 31;
  const int places = p.num_requests * p.max_pages;
  const int lo = slice_start(places, blockIdx.x, gridDim.x), hi = slice_start(places, blockIdx.x + 1, gridDim.x);
  for (;;) {
    int q0 = 0;
    if (lane == 0) q0 = lo + 32 * atomicAdd(counter, 1);
    q0 = __shfl_sync(0xffffffffu, q0, 0);
    if (q0 >= hi) break;
    const int q = q0 + lane;
    const int b = q / p.max_pages, t = q - b * p.max_pages;
    bool copy = q < hi;
    if (copy && !nothing) {
      bool bad;
      copy = t >= load_request<true>(p, b, bad).tiles;
    }
    const int64_t from = b * p.acc_stride + static_cast<int64_t>(t) * kTok;
    const int64_t to = b * p.acc_out_stride + static_cast<int64_t>(t) * kTok;
    unsigned int todo = __ballot_sync(0xffffffffu, copy);
    while (todo != 0) {
      constexpr int kAtOnce = 8;
      float v[kAtOnce][2];
      unsigned int bits = todo;
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int l = bits != 0 ? __ffs(bits) - 1 : 0;
        const float* src = p.acc + __shfl_sync(0xffffffffu, from, l);
        if (bits != 0) {
          v[j][0] = src[lane];
          v[j][1] = src[lane + 32];
        }
        bits &= bits - 1;
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int l = todo != 0 ? __ffs(todo) - 1 : 0;
        float* dst = p.acc_out + __shfl_sync(0xffffffffu, to, l);
        if (todo != 0) {
          dst[lane] = v[j][0];
          dst[lane + 32] = v[j][1];
        }
        todo &= todo - 1;
      }
    }
  }
}

// Bits of one thread's 8 columns (rows of Q) that see position pos, which
// lies at or behind the prefix.
__device__ __forceinline__ uint32_t visible_columns(const Params& p, const Segment& s, int pos, const int (&draft)[8]) {
  const int j = pos - s.r.prefix;
  uint32_t m = 0;
  if (j < s.r.n && j < 64 * p.mask_words) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const long long w = p.mask[static_cast<int64_t>(s.r.row0 + draft[k]) * p.mask_words + (j >> 6)];
      m |= static_cast<uint32_t>((w >> (j & 63)) & 1) << k;
    }
  }
  return m;
}

template <bool kWeights>
__global__ void __launch_bounds__(kThreads, 1)
tree_kernel(const __grid_constant__ CUtensorMap ckv_map, const __grid_constant__ CUtensorMap kpe_map,
            const __grid_constant__ CUtensorMap qn_map, const __grid_constant__ CUtensorMap qp_map, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* q_mem = smem + kOffQ;
  uint8_t* p_mem = smem + kOffP;
  float* sums = reinterpret_cast<float*>(p_mem);  // weights: [2 sets][kSumTiles][64]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint64_t* kv_full = bars;                  // [2 stages][kParts]
  uint64_t* kv_free = bars + 2 * kParts;     // [2][kParts]: the part's block of O^T is done
  uint64_t* q_full = bars + 4 * kParts;      // [kParts]
  uint64_t* q_empty = bars + 5 * kParts;
  uint64_t* s_full = q_empty + 1;            // [2]
  uint64_t* s_empty = q_empty + 3;           // [2]
  uint64_t* p_full = q_empty + 5;
  uint64_t* o_empty = q_empty + 6;
  uint64_t* drain = q_empty + 7;             // [2]
  constexpr int kBars = 5 * kParts + 9;
  static_assert(kBars * 8 <= kOffMisc - kOffBar, "barriers");
  // O^T's last block frees the stage's last part: all of PV(i) is done.
  auto pv_done = [&](int i) { return &kv_free[(i & 1) * kParts + kParts - 1]; };
  int* misc = reinterpret_cast<int*>(smem + kOffMisc);
  uint32_t* tmem_base_smem = reinterpret_cast<uint32_t*>(misc);
  int* abort_flag = misc + 1;
  int* copied = misc + 2;                    // weights: see copy_behind
  Start* found = reinterpret_cast<Start*>(misc + 3);
  static_assert(12 + sizeof(Start) <= kOffRed - kOffMisc, "misc");
  float* red = reinterpret_cast<float*>(smem + kOffRed);
  int* warp_sums = reinterpret_cast<int*>(red);  // planning: [11] units, [11] groups
  float* factor_s = reinterpret_cast<float*>(smem + kOffFactor);  // O's rescaling; at the end 1 / l
  float* max_s = reinterpret_cast<float*>(smem + kOffMax);

  const int tid = threadIdx.x;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int lane = tid & 31;

  if (tid == 0) {
    for (int x = 0; x < kBars; ++x) mbar_init(&bars[x], 1);
    for (int s = 0; s < 2; ++s) mbar_init(&s_empty[s], kSoftWarps);
    mbar_init(p_full, kSoftWarps);
    mbar_init(o_empty, kSoftWarps);
    *abort_flag = 0;
    *copied = 0;
    fence_mbar_init();
  }
  if (warp == kLoadWarp && elect_one()) {
    prefetch_tensor_map(&ckv_map);
    prefetch_tensor_map(&kpe_map);
    prefetch_tensor_map(&qn_map);
    prefetch_tensor_map(&qp_map);
  }
  if (warp == kLogitWarp) tmem_alloc(tmem_base_smem, kTmemCols);
  griddep_launch_dependents();
  griddep_wait();

  // ---- plan: total units, and the request that holds this slice's first one.
  // Every CTA sums all requests (one or two loads a thread for ordinary
  // batches) instead of waiting for a planning launch.
  const int per = (p.num_requests + kThreads - 1) / kThreads;
  const int b_lo = min(tid * per, p.num_requests), b_hi = min(b_lo + per, p.num_requests);
  int units = 0, groups = 0;
  bool any_bad = false, decreasing = false;
  Request mine;  // the thread's first (for ordinary batches its only) request
  for (int b = b_lo; b < b_hi; ++b) {
    bool bad;
    const Request r = load_request<kWeights>(p, b, bad);
    if (b == b_lo) mine = r;
    decreasing |= p.cu[b + 1] < p.cu[b];
    units += r.groups * r.span;
    groups += r.groups;
    any_bad |= bad;
  }
  if (any_bad && blockIdx.x == 0) atomicOr(p.status, DSA_DEV_BAD_SEQ_LEN);
  int iu = units, ig = groups;  // inclusive over the warp
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, iu, o), c = __shfl_up_sync(0xffffffffu, ig, o);
    if (lane >= o) {
      iu += a;
      ig += c;
    }
  }
  if (lane == 31) {
    warp_sums[warp] = iu;
    warp_sums[11 + warp] = ig;
  }
  tc_fence_before();
  // Where cu_drafts decreases, requests could share rows, and the sums below
  // exceed what the host checked: such a call does nothing.
  const bool nothing = __syncthreads_or(decreasing);
  tc_fence_after();
  int total = 0, before = iu - units, gbefore = ig - groups;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) {
      before += warp_sums[w];
      gbefore += warp_sums[11 + w];
    }
    total += warp_sums[w];
  }
  if (nothing) total = units = 0;
  const int ctas = gridDim.x;
  const int u0 = slice_start(total, blockIdx.x, ctas), u1 = slice_start(total, blockIdx.x + 1, ctas);
  const bool keeper = !kWeights && blockIdx.x == 0;  // writes the groups for combine_kernel
  if (!nothing && (keeper || (u0 >= before && u0 < before + units))) {
    for (int b = b_lo; b < b_hi; ++b) {
      bool bad;
      const Request r = b == b_lo ? mine : load_request<kWeights>(p, b, bad);
      const int un = r.groups * r.span;
      if (u0 >= before && u0 < before + un) {
        const int group = (u0 - before) / r.span;
        *found = Start{b, before, gbefore, r, group, u0 - before - group * r.span};
      }
      if (keeper) {
        int2* to = reinterpret_cast<int2*>(p.plan + kPlanGroups) + gbefore;
        for (int g = 0; g < r.groups; ++g)
          to[g] = make_int2(r.row0 * p.heads + g * kRows, min(kRows, r.rows - g * kRows));
      }
      before += un;
      gbefore += r.groups;
    }
  }
  __syncthreads();

  const uint32_t tmem_base = *tmem_base_smem;
  const WaitCtx wctx{abort_flag, p.status, p.wait_limit_ns};
  Walker<kWeights> walk(p, u0, u1, *found);
  Segment s;

  if (warp == kLoadWarp) {
    // ------------------------------------------------------------ loads
    // This role and the next two are one thread each: a warp-wide wait before
    // every issue (vote, re-election) costs some 250 clocks, a thread's own
    // about 60, and the tensor pipe idles meanwhile.
    if (elect_one()) {
      int i = 0, segs = 0;
      int parts = 0;  // issued
      bool ok = true;
      while (ok && walk.next(s)) {
        const int32_t* row = p.block_table + static_cast<int64_t>(s.b) * p.max_pages;
        int next_page = row[s.t0];
        for (int t = s.t0; t < s.t1; ++t, ++i) {
          // A page outside the pool reads as zeros (a box outside the tensor
          // is filled with them); its tokens are masked below.
          const int page = next_page < 0 || next_page >= p.num_pages ? p.num_pages : next_page;
          if (t + 1 < s.t1) next_page = row[t + 1];
          const int st = i & 1;
          const uint32_t parity = ((i >> 1) & 1) ^ 1;
          uint8_t* dst = smem + st * kTileBytes;
#pragma unroll
          for (int x = 0; x < kParts; ++x) {
            // The weights' S^T alone reads a stage.
            ok = ok && mbar_wait(kWeights ? &s_full[st] : &kv_free[st * kParts + x], parity, wctx);
            if (!ok) break;
            uint64_t* bar = &kv_full[st * kParts + x];
            mbar_arrive_expect_tx(bar, part_bytes(x));
            tma_load_3d(dst + 2 * x * kChunkBytes, &ckv_map, bar, 128 * x, 0, page);
            tma_load_3d(dst + (2 * x + 1) * kChunkBytes, &ckv_map, bar, 128 * x + 64, 0, page);
            if (x == kParts - 1) tma_load_3d(dst + 8 * kChunkBytes, &kpe_map, bar, 0, 0, page);
            ++parts;
          }
          if (t == s.t0 && ok) {
            // The group's queries, behind its first tile.  Rows behind the
            // request's own are another's or zeros; their columns are never
            // written out.
            const int row_q = s.r.row0 * p.heads + s.group * kRows;
            ok = mbar_wait(q_empty, (segs & 1) ^ 1, wctx);
            if (ok) {
#pragma unroll
              for (int x = 0; x < kParts; ++x) {
                mbar_arrive_expect_tx(&q_full[x], part_bytes(x));
                tma_load_2d(q_mem + 2 * x * kChunkBytes, &qn_map, &q_full[x], 128 * x, row_q);
                tma_load_2d(q_mem + (2 * x + 1) * kChunkBytes, &qn_map, &q_full[x], 128 * x + 64, row_q);
                if (x == kParts - 1) tma_load_2d(q_mem + 8 * kChunkBytes, &qp_map, &q_full[x], 0, row_q);
              }
              ++segs;
            }
          }
          if (!ok) break;
        }
      }
      // Copies still in flight (after an abort) land before the CTA exits: of
      // each part the last two, whose phases nothing refills.
      for (int x = 0; x < kParts; ++x) {
        const int tiles = (parts + kParts - 1 - x) / kParts;
        for (int k = tiles - 1; k >= 0 && k >= tiles - 2; --k)
          mbar_drain(&kv_full[(k & 1) * kParts + x], (k >> 1) & 1, p.status);
        if (segs >= 1) mbar_drain(&q_full[x], (segs - 1) & 1, p.status);
      }
    }
    __syncwarp();
  } else if (warp == kLogitWarp) {
    // ------------------------------------------------------------ S^T = K Q^T
    if (elect_one()) {
      const uint64_t k_desc = sdesc_sw128(smem_u32(smem), 16, 1024);
      const uint64_t q_desc = sdesc_sw128(smem_u32(q_mem), 16, 1024);
      int i = 0, segs = 0;
      bool ok = true;
      while (ok && walk.next(s)) {
        const uint32_t idesc = with_rows(kIdescS, s.rows());
        for (int t = s.t0; t < s.t1; ++t, ++i) {
          const int st = i & 1;
          const uint64_t a = k_desc + st * (kTileBytes >> 4);
          const uint32_t d = tmem_base + kColS + 64u * st * (kWeights ? kSumsS : 1);
          ok = mbar_wait(&s_empty[st], ((i >> 1) & 1) ^ 1, wctx);
#pragma unroll
          for (int x = 0; x < kParts; ++x) {
            if (t == s.t0) ok = ok && mbar_wait(&q_full[x], segs & 1, wctx);
            ok = ok && mbar_wait(&kv_full[st * kParts + x], (i >> 1) & 1, wctx);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int k = 8 * x; k < 8 * x + (x == kParts - 1 ? 12 : 8); ++k) {
              // +8192 bytes per 64 columns, +32 per K16 step (>> 4)
              const uint32_t at = (k >> 2) * (kChunkBytes >> 4) + (k & 3) * 2;
              if (kWeights)
                umma_bf16(d + 64u * (k / kSumSteps), a + at, q_desc + at, idesc, k % kSumSteps > 0 ? 1u : 0u);
              else
                umma_bf16(d, a + at, q_desc + at, idesc, k > 0 ? 1u : 0u);
            }
          }
          if (!ok) break;
          umma_commit(&s_full[st]);
          if (t == s.t1 - 1) umma_commit(q_empty);
        }
        ++segs;
      }
      umma_commit(&drain[0]);
      mbar_drain(&drain[0], 0, p.status);
    }
    __syncwarp();
  } else if (warp == kValueWarp) {
    // ------------------------------------------------------------ O^T += V^T P^T
    if (kWeights && p.acc_out != p.acc) copy_behind(p, nothing, copied);
    if (!kWeights && elect_one()) {
      const uint64_t v_desc = sdesc_sw128(smem_u32(smem), kChunkBytes, 1024);
      const uint64_t p_desc = sdesc_sw128(smem_u32(p_mem), kChunkBytes, 1024);
      int i = 0, segs = 0;
      bool ok = true;
      while (ok && walk.next(s)) {
        const uint32_t idesc = with_rows(kIdescO, s.rows());
        for (int t = s.t0; t < s.t1; ++t, ++i) {
          const int st = i & 1;
          if (t == s.t0) ok = mbar_wait(o_empty, (segs & 1) ^ 1, wctx);
          ok = ok && mbar_wait(p_full, i & 1, wctx);
          if (!ok) break;
          tc_fence_after();
          const uint32_t more = t == s.t0 ? 0u : 1u;
          const uint64_t a = v_desc + st * (kTileBytes >> 4);
#pragma unroll
          for (int mb = 0; mb < 4; ++mb) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)  // 128 dims are two pieces; a K16 step is 16 token rows of 128 bytes
              umma_bf16(tmem_base + kColO + 64u * mb, a + mb * (2 * kChunkBytes >> 4) + kk * (2048 >> 4),
                        p_desc + kk * (2048 >> 4), idesc, kk > 0 ? 1u : more);
            umma_commit(&kv_free[st * kParts + mb]);
          }
        }
        ++segs;
      }
      umma_commit(&drain[1]);
      mbar_drain(&drain[1], 0, p.status);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax
    // Set `set` of four warps has the columns (query rows) 32 set .. +31 of
    // S^T; in it, warp sp reads tokens 16 sp .. +15 (the M = 64 accumulator
    // has them in lanes 0-15 of its sub-partition), thread (lane) the tokens
    // r0 and r0 + 8 and the columns col(k), k = 0..7.
    const int set = warp >> 2, sp = warp & 3;
    const int r0 = 16 * sp + (lane >> 2);
    const int c0 = 32 * set + 2 * (lane & 3);
    auto col = [&](int k) { return c0 + 8 * (k >> 1) + (k & 1); };
    const uint32_t lane_base = static_cast<uint32_t>(32 * sp) << 16;
    const int e = tid & 127;  // thread of the set
    int i = 0;
    bool ok = true;

    if constexpr (kWeights) {
      // The accumulators that a run of tiles will be added to, read at its start.
      constexpr int kOld = kSumTiles * kTok / (32 * kSoftWarps);
      float old[kOld];
      while (walk.next(s)) {
        if (s.first_group) {
          const float* acc = p.acc + s.b * p.acc_stride + static_cast<int64_t>(s.t0) * kTok;
#pragma unroll
          for (int k = 0; k < kOld; ++k) {
            const int q = tid + k * 32 * kSoftWarps;
            old[k] = q < (s.t1 - s.t0) * kTok ? acc[q] : 0.f;
          }
        }
        float lse[8];
        int draft[8];
        uint32_t live = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int row = s.group * kRows + col(k);
          const bool in = row < s.r.rows;
          lse[k] = in ? p.lse_in[static_cast<int64_t>(s.r.row0) * p.heads + row] : 0.f;
          draft[k] = in ? row / p.heads : 0;
          if (in && lse[k] != -INFINITY) live |= 1u << k;  // a row that saw nothing gives nothing
        }
        const bool all_live = __all_sync(0xffffffffu, live == 0xffu);
        const int32_t* bt = p.block_table + static_cast<int64_t>(s.b) * p.max_pages;
        int next_page = bt[s.t0];
        for (int t = s.t0; t < s.t1; ++t, ++i) {
          const int st = i & 1;
          const int page = next_page;
          if (t + 1 < s.t1) next_page = bt[t + 1];
          uint32_t see0 = live, see1 = live;
          const bool lost = page < 0 || page >= p.num_pages;
          const bool tail = (t + 1) * kTok > s.r.prefix;
          if (lost) {
            see0 = see1 = 0;
            if (e == 0) atomicOr(p.status, DSA_DEV_BAD_PAGE);
          } else if (tail) {
            const int pos = t * kTok + r0;
            if (pos >= s.r.prefix) see0 &= visible_columns(p, s, pos, draft);
            if (pos + 8 >= s.r.prefix) see1 &= visible_columns(p, s, pos + 8, draft);
          }
          ok = ok && mbar_wait(&s_full[st], (i >> 1) & 1, wctx);
          tc_fence_after();
          float v[16];
          tmem_ld_16x32_sum3_wait(tmem_base + lane_base + kColS + 64u * kSumsS * st + 32u * set, v);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[st]);
          float w0 = 0.f, w1 = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int f = 4 * (k >> 1) + (k & 1);
            v[f] = ex2_approx(fmaf(v[f], p.scale_log2, -lse[k]));
            v[f + 2] = ex2_approx(fmaf(v[f + 2], p.scale_log2, -lse[k]));
          }
          if (all_live && !tail && !lost) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              w0 += v[4 * (k >> 1) + (k & 1)];
              w1 += v[4 * (k >> 1) + (k & 1) + 2];
            }
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              w0 += (see0 >> k) & 1 ? v[4 * (k >> 1) + (k & 1)] : 0.f;
              w1 += (see1 >> k) & 1 ? v[4 * (k >> 1) + (k & 1) + 2] : 0.f;
            }
          }
          w0 += __shfl_xor_sync(0xffffffffu, w0, 1);
          w1 += __shfl_xor_sync(0xffffffffu, w1, 1);
          w0 += __shfl_xor_sync(0xffffffffu, w0, 2);
          w1 += __shfl_xor_sync(0xffffffffu, w1, 2);
          if ((lane & 3) == 0) {
            // The same thread adds a token's groups one after the other.
            float* to = sums + (set * kSumTiles + (t - s.t0)) * kTok + r0;
            to[0] = s.first_group ? w0 : to[0] + w0;
            to[8] = s.first_group ? w1 : to[8] + w1;
          }
        }
        if (s.last_group) {
          named_barrier_sync(3, 32 * kSoftWarps);
          float* out = p.acc_out + s.b * p.acc_out_stride + static_cast<int64_t>(s.t0) * kTok;
#pragma unroll
          for (int k = 0; k < kOld; ++k) {
            const int q = tid + k * 32 * kSoftWarps;
            if (q < (s.t1 - s.t0) * kTok) out[q] = old[k] + (sums[q] + sums[kSumTiles * kTok + q]);
          }
          named_barrier_sync(3, 32 * kSoftWarps);
        }
      }
      if (p.acc_out != p.acc) copy_behind(p, nothing, copied);
    } else {
      // Online softmax in base 2.  The running max m[k] of a column is the
      // same in every thread that has it.  It moves only when some token of
      // the tile exceeds it by more than kRescaleThreshold (always at a
      // segment's first tile), which one OR-barrier per tile tells the set;
      // only then is the tile's max reduced over the tokens and O rescaled.
      // P <= 2^8 then.  P is rounded to bf16 for the MMA (off by at most 2^-8
      // of itself), as any bf16 tensor-core product needs.  O is divided by
      // lr, the fp32 sum of the rounded weights, so that a row that hangs on a
      // few tokens does not inherit their rounding; lse comes from l, the sum
      // of the unrounded ones (both sums: under 1 % of the time).
      // A tile's path from S^T to P is what its K stage waits for, so the
      // ordinary tile takes one FMA, one max and one exponential a value:
      // d = s * scale - m, masked in the tiles that need it only.
      int* group_of = p.plan + 2 * blockIdx.x;  // of this CTA's records
      if (tid == 0) group_of[0] = group_of[1] = -1;
      while (walk.next(s)) {
        float m[8], minus[8], l[8], lr[8];  // minus: -m, or 0 while the column has seen nothing
        int draft[8];
        bool unset = false;          // some column of this thread has seen nothing yet
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int row = s.group * kRows + col(k);
          const bool in = row < s.r.rows;
          m[k] = in ? -INFINITY : 0.f;
          minus[k] = in ? 0.f : -INFINITY;  // no row of the group: all weights 0
          l[k] = lr[k] = 0.f;
          draft[k] = in ? row / p.heads : 0;
          unset |= in;
        }
        const int32_t* bt = p.block_table + static_cast<int64_t>(s.b) * p.max_pages;
        int next_page = bt[s.t0];
        for (int t = s.t0; t < s.t1; ++t, ++i) {
          const int st = i & 1;
          const int page = next_page;
          if (t + 1 < s.t1) next_page = bt[t + 1];
          uint32_t see0 = 0xffu, see1 = 0xffu;
          const bool tail = (t + 1) * kTok > s.r.prefix;
          const bool lost = page < 0 || page >= p.num_pages;
          if (lost) {
            see0 = see1 = 0;
            if (e == 0) atomicOr(p.status, DSA_DEV_BAD_PAGE);
          } else if (tail) {
            const int pos = t * kTok + r0;
            if (pos >= s.r.prefix) see0 = visible_columns(p, s, pos, draft);
            if (pos + 8 >= s.r.prefix) see1 = visible_columns(p, s, pos + 8, draft);
          }
          ok = ok && mbar_wait(&s_full[st], (i >> 1) & 1, wctx);
          tc_fence_after();
          float v[16];
          tmem_ld_16x32_wait(tmem_base + lane_base + kColS + 64u * st + 32u * set, v);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[st]);
          float d0[8], d1[8];  // tokens r0 and r0 + 8
          auto differences = [&]() {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int f = 4 * (k >> 1) + (k & 1);
              d0[k] = fmaf(v[f], p.scale_log2, minus[k]);
              d1[k] = fmaf(v[f + 2], p.scale_log2, minus[k]);
            }
            if (tail || lost) {
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                if (!((see0 >> k) & 1)) d0[k] = -INFINITY;
                if (!((see1 >> k) & 1)) d1[k] = -INFINITY;
              }
            }
          };
          differences();
          float most = d0[0];
#pragma unroll
          for (int k = 0; k < 8; ++k) most = fmaxf(most, fmaxf(d0[k], d1[k]));
          if (named_barrier_or(1 + set, 128, unset || most > kRescaleThreshold)) {
            {
              // Over the warp's 8 token pairs (lane bits 2-4): at each step a
              // lane keeps half of its columns and sends the others.
              float mt[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) mt[k] = fmaxf(d0[k], d1[k]) - minus[k];
              int k0 = 0;  // the column that is left
#pragma unroll
              for (int half = 4; half >= 1; half /= 2) {
                const bool up = lane & (4 * half);
#pragma unroll
                for (int k = 0; k < half; ++k) {
                  const float send = up ? mt[k] : mt[k + half];
                  mt[k] = fmaxf(up ? mt[k + half] : mt[k], __shfl_xor_sync(0xffffffffu, send, 4 * half));
                }
                if (up) k0 += half;
              }
              red[kRows * sp + col(k0)] = mt[0];
            }
            named_barrier_sync(1 + set, 128);
            unset = false;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float* r = red + col(k);
              const float mt = fmaxf(fmaxf(r[0], r[kRows]), fmaxf(r[2 * kRows], r[3 * kRows]));
              float alpha = 1.f;
              if (mt > m[k] + kRescaleThreshold) {
                alpha = exp2f(m[k] - mt);  // 0 when m was -inf
                m[k] = mt;
                minus[k] = -mt;
              }
              l[k] *= alpha;
              lr[k] *= alpha;
              unset |= m[k] == -INFINITY;
              if (sp == 0 && lane < 4) factor_s[col(k)] = alpha;
            }
            differences();
            named_barrier_sync(1 + set, 128);
            if (t > s.t0) {
              // O holds PV(i - 1) before it is rescaled.
              ok = ok && mbar_wait(pv_done(i - 1), ((i - 1) >> 1) & 1, wctx);
              tc_fence_after();
#pragma unroll 1
              for (int mb = 0; mb < 4; ++mb) {
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                  const uint32_t at = tmem_base + lane_base + kColO + 64u * mb + 32u * set + 16u * h;
                  float o[16];
                  tmem_ld16_wait(at, o);
#pragma unroll
                  for (int c = 0; c < 16; ++c) o[c] *= factor_s[32 * set + 16 * h + c];
                  tmem_st16(at, o);
                }
              }
              tmem_wait_st();
            }
          }
          if (tail) {
            // Cache rows at and behind the prefix may be masked and hold
            // anything; a zero weight would still turn an infinity or NaN
            // among them into NaN.  The logits have been read (S^T is done),
            // so such values are zeroed in the V tile; a row that does see
            // one has its NaN from the logit (or, where the logit is -inf,
            // the weight 0 and nothing of the value; before the prefix's end,
            // where nothing is zeroed, 0 times infinity: callers are told
            // that this is not defined).
#pragma unroll
            for (int x = 0; x < kParts; ++x) ok = ok && mbar_wait(&kv_full[st * kParts + x], (i >> 1) & 1, wctx);
            const int from = s.r.prefix > t * kTok ? s.r.prefix - t * kTok : 0;
            for (int q = tid; q < (kTok - from) * 64; q += 32 * kSoftWarps) {
              // 16-byte piece q & 7 of row from + (q >> 6) in piece (q >> 3) & 7
              uint4* at = reinterpret_cast<uint4*>(smem + st * kTileBytes + ((q >> 3) & 7) * kChunkBytes +
                                                   (from + (q >> 6)) * 128 + (q & 7) * 16);
              uint4 w = *at;
              uint32_t* ww = reinterpret_cast<uint32_t*>(&w);
              bool changed = false;
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                if ((ww[z] & 0x7F80u) == 0x7F80u) {
                  ww[z] &= 0xFFFF0000u;
                  changed = true;
                }
                if ((ww[z] & 0x7F800000u) == 0x7F800000u) {
                  ww[z] &= 0x0000FFFFu;
                  changed = true;
                }
              }
              if (changed) *at = w;
            }
          }
          uint32_t p0[4], p1[4];
#pragma unroll
          for (int k = 0; k < 8; k += 2) {
            float a[2], c[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              // A column that has seen nothing has only -inf (weight 0) and
              // NaN (kept) here.
              a[h] = ex2_approx(d0[k + h]);
              c[h] = ex2_approx(d1[k + h]);
              l[k + h] += a[h] + c[h];
            }
            const __nv_bfloat162 pa = __floats2bfloat162_rn(a[0], a[1]), pc = __floats2bfloat162_rn(c[0], c[1]);
            p0[k >> 1] = *reinterpret_cast<const uint32_t*>(&pa);
            p1[k >> 1] = *reinterpret_cast<const uint32_t*>(&pc);
            lr[k] += __uint_as_float(p0[k >> 1] << 16) + __uint_as_float(p1[k >> 1] << 16);
            lr[k + 1] += __uint_as_float(p0[k >> 1] & 0xFFFF0000u) + __uint_as_float(p1[k >> 1] & 0xFFFF0000u);
          }
          // P was last read by PV(i - 1).
          if (i > 0) ok = ok && mbar_wait(pv_done(i - 1), ((i - 1) >> 1) & 1, wctx);
          {
            // One 128-byte row per token, 16-byte pieces swizzled by token & 7
            // (the same for r0 and r0 + 8): a warp's stores meet no bank twice.
            uint8_t* at = p_mem + r0 * 128 + 4 * (lane & 3);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int piece = ((4 * set + j) ^ (r0 & 7)) << 4;
              *reinterpret_cast<uint32_t*>(at + piece) = p0[j];
              *reinterpret_cast<uint32_t*>(at + 1024 + piece) = p1[j];
            }
          }
          fence_proxy_async_smem();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(p_full);
        }

        // ---- the segment's end: denominators over the tokens (while the last
        // PV runs), then O.
        auto over_tokens = [&](const float (&sum)[8]) {  // of column 32 set + e, for e < 32
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float v = sum[k];
            v += __shfl_xor_sync(0xffffffffu, v, 4);
            v += __shfl_xor_sync(0xffffffffu, v, 8);
            v += __shfl_xor_sync(0xffffffffu, v, 16);
            if (lane < 4) red[kRows * sp + col(k)] = v;
          }
          named_barrier_sync(1 + set, 128);
          const float* r = red + 32 * set + (e & 31);
          const float v = (r[0] + r[kRows]) + (r[2 * kRows] + r[3 * kRows]);
          named_barrier_sync(1 + set, 128);
          return v;
        };
        if (sp == 0 && lane < 4) {
#pragma unroll
          for (int k = 0; k < 8; ++k) max_s[col(k)] = m[k];
        }
        const float sum = over_tokens(l), sum_r = over_tokens(lr);
        const int64_t row_q = static_cast<int64_t>(s.r.row0) * p.heads + s.group * kRows;
        const int rows = s.rows();
        const int64_t rec = static_cast<int64_t>(blockIdx.x) * 2 + s.slot;
        if (tid == 0 && !s.whole) group_of[s.slot] = s.group_index;
        if (e < 32) {
          const int c = 32 * set + e;
          if (s.whole) {
            factor_s[c] = sum_r == 0.f ? 0.f : 1.f / sum_r;
            if (c < rows) p.lse_out[row_q + c] = sum == 0.f ? -INFINITY : max_s[c] + log2f(sum);
          } else {
            *reinterpret_cast<float4*>(p.part_ml + (rec * kRows + c) * 4) = make_float4(max_s[c], sum, sum_r, 0.f);
          }
        }
        ok = ok && mbar_wait(pv_done(i - 1), ((i - 1) >> 1) & 1, wctx);
        named_barrier_sync(1 + set, 128);
        tc_fence_after();
#pragma unroll 1
        for (int mb = 0; mb < 4; ++mb) {
          const int dim = 128 * mb + 32 * sp + lane;
          float o[32];
          tmem_ld32_wait(tmem_base + lane_base + kColO + 64u * mb + 32u * set, o);
          if (s.whole) {
            // Neighbouring lanes swap halves, so that each stores two dims
            // of one row.
            const bool odd = lane & 1;
            __nv_bfloat16* out = p.out + row_q * kCkv + (dim & ~1);
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              const float a = o[c] * factor_s[32 * set + c], b = o[c + 1] * factor_s[32 * set + c + 1];
              const float got = __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
              const int row = 32 * set + c + (odd ? 1 : 0);
              if (row < rows)
                *reinterpret_cast<__nv_bfloat162*>(out + static_cast<int64_t>(row) * kCkv) =
                    odd ? __floats2bfloat162_rn(got, b) : __floats2bfloat162_rn(a, got);
            }
          } else {
            float* to = p.part_o + rec * kPartFloats + 32 * set * kCkv + dim;
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (32 * set + c < rows) to[c * kCkv] = o[c];
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_empty);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kLogitWarp) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// Joins the records of a group that several slices share: per row
//   M = max m_i, L = sum l_i 2^(m_i - M), lse = M + log2 L,
//   out = sum O_i 2^(m_i - M) / sum lr_i 2^(m_i - M),
// in an order that the slices alone give.  Block x has the group x, or where
// groups outnumber records the group of record x if x is its first one;
// block y its rows y * rows_per_block ...  Each kParts-th of the block takes every
// kParts-th record of a row, a thread four dims: the loads are latency-bound,
// so many are in flight at once.
constexpr int kJoinRows = 4;       // most rows per block
constexpr int kJoinDepth = 8;      // records whose loads a thread has in flight

template <int kParts>
__global__ void __launch_bounds__(128 * kParts)
combine_kernel(const Params p, int ctas, int rows_per_block, bool by_record) {
  griddep_wait();
  constexpr int kJoinThreads = 128 * kParts;
  constexpr int kLooks = 2 * kMaxCtas / kJoinThreads;  // records a thread looks at
  __shared__ int recs[2 * kMaxCtas];
  __shared__ float weight[kJoinRows][2 * kMaxCtas];
  __shared__ int warp_count[kLooks][kJoinThreads / 32];
  __shared__ float4 other[kParts > 1 ? kParts - 1 : 1][kCkv / 4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int x = blockIdx.x;
  const int group = by_record ? __ldcg(p.plan + x) : x;
  int mine[kLooks];
#pragma unroll
  for (int k = 0; k < kLooks; ++k) {
    const int r = tid + k * kJoinThreads;
    mine[k] = r < 2 * ctas ? __ldcg(p.plan + r) : -1;
  }
  if (group < 0) return;
  const int2 info = __ldcg(reinterpret_cast<const int2*>(p.plan + kPlanGroups) + group);
  unsigned int votes[kLooks];
#pragma unroll
  for (int k = 0; k < kLooks; ++k) {
    votes[k] = __ballot_sync(0xffffffffu, mine[k] == group);
    if (lane == 0) warp_count[k][warp] = __popc(votes[k]);
  }
  __syncthreads();
  int count = 0;
#pragma unroll
  for (int k = 0; k < kLooks; ++k) {
    int at = count + __popc(votes[k] & ((1u << lane) - 1u));
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) {
      if (w < warp) at += warp_count[k][w];
      count += warp_count[k][w];
    }
    if (mine[k] == group) recs[at] = tid + k * kJoinThreads;
  }
  __syncthreads();
  if (count == 0 || (by_record && recs[0] != x)) return;  // written whole; or another block's
  const int y0 = blockIdx.y * rows_per_block;
  const int rows = min(rows_per_block, info.y - y0);
  if (rows <= 0) return;
  // The first records' loads of the first row need no weights: they go first.
  const int part = tid >> 7, d4 = tid & 127;
  const float4* src = reinterpret_cast<const float4*>(p.part_o) + y0 * (kCkv / 4) + d4;
  float4 v[kJoinDepth];
  auto load = [&](int k0) {
#pragma unroll
    for (int j = 0; j < kJoinDepth; ++j)
      if (k0 + kParts * j < count)
        v[j] = __ldcg(src + static_cast<int64_t>(recs[k0 + kParts * j]) * (kPartFloats / 4));
  };
  load(part);
  for (int y = warp; y < rows; y += kJoinThreads / 32) {
    float M = -INFINITY, L = 0.f, R = 0.f;
    const float4* ml = reinterpret_cast<const float4*>(p.part_ml) + y0 + y;
    for (int k = lane; k < count; k += 32) {
      const float m = __ldcg(&ml[static_cast<int64_t>(recs[k]) * kRows].x);
      M = fmaxf(M, m);
      weight[y][k] = m;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    for (int k = lane; k < count; k += 32) {
      const float4 q = __ldcg(ml + static_cast<int64_t>(recs[k]) * kRows);
      const float w = q.x == -INFINITY ? 0.f : exp2f(q.x - M);
      L = fmaf(q.y, w, L);
      R = fmaf(q.z, w, R);
      weight[y][k] = w;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      L += __shfl_xor_sync(0xffffffffu, L, o);
      R += __shfl_xor_sync(0xffffffffu, R, o);
    }
    const float inv = R == 0.f ? 0.f : 1.f / R;
    __syncwarp();
    for (int k = lane; k < count; k += 32) weight[y][k] *= inv;
    if (lane == 0) p.lse_out[info.x + y0 + y] = L == 0.f ? -INFINITY : M + log2f(L);
  }
  __syncthreads();
  for (int y = 0; y < rows; ++y) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = part; k0 < count; k0 += kParts * kJoinDepth) {
      if (y > 0 || k0 > part) load(k0);
#pragma unroll
      for (int j = 0; j < kJoinDepth; ++j) {
        if (k0 + kParts * j < count) {
          const float w = weight[y][k0 + kParts * j];
          acc.x = fmaf(v[j].x, w, acc.x);
          acc.y = fmaf(v[j].y, w, acc.y);
          acc.z = fmaf(v[j].z, w, acc.z);
          acc.w = fmaf(v[j].w, w, acc.w);
        }
      }
    }
    src += kCkv / 4;
    if (part > 0) other[part - 1][d4] = acc;
    __syncthreads();
    if (part == 0) {
#pragma unroll
      for (int k = 0; k < kParts - 1; ++k) {
        const float4 o = other[k][d4];
        acc.x += o.x;
        acc.y += o.y;
        acc.z += o.z;
        acc.w += o.w;
      }
      __nv_bfloat162 h[2] = {__floats2bfloat162_rn(acc.x, acc.y), __floats2bfloat162_rn(acc.z, acc.w)};
      *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(info.x) + y0 + y) * kCkv + 4 * d4) =
          *reinterpret_cast<const uint2*>(h);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ host
std::once_flag g_once[64];
int g_status[64];

struct Layout {
  size_t part_ml, part_o, plan, bytes;
};

// Upper bound of the groups of all requests: sum ceil(n_b H / 64).
inline int64_t groups_bound(int64_t drafts, int64_t heads, int64_t requests) {
  return drafts * heads / kRows + requests;
}

// The same for every call that is accepted, so that a workspace never has to
// move (a captured graph would go on using the old one).
inline Layout layout(int sms) {
  Layout a;
  a.part_ml = kWorkspaceHeader;
  a.part_o = a.part_ml + static_cast<size_t>(2 * sms) * kRows * 4 * sizeof(float);
  a.plan = a.part_o + static_cast<size_t>(2 * sms) * kPartFloats * sizeof(float);
  a.bytes = a.plan + (kPlanGroups + 2 * static_cast<size_t>(groups_bound(kMaxRows, 1, kMaxRequests))) * sizeof(int);
  return a;
}

inline bool sizes_ok(int64_t drafts, int64_t heads, int64_t requests) {
  return drafts >= 0 && heads >= 1 && heads <= 128 && requests >= 0 && requests <= kMaxRequests &&
         drafts * heads <= kMaxRows;
}

struct Range {
  const void* at;
  size_t bytes;
};

// `more`: the attention's output and lse; the weights' accumulators and lse,
// which is an input.
int check_and_setup(const void* q_nope, const void* q_pe, const void* ckv, int64_t ckv_page, int64_t ckv_row,
                    const void* kpe, int64_t kpe_page, int64_t kpe_row, int64_t num_pages,
                    const int32_t* prefix_lens, const int32_t* block_table, const int32_t* cu, const int64_t* mask,
                    int32_t requests, int32_t drafts, int32_t heads, int32_t max_pages, int32_t mask_words,
                    float sm_scale, void* workspace, size_t workspace_bytes, bool records, const Range (&more)[2],
                    DeviceInfo* info, Params* prm, CUtensorMap (&maps)[4]) {
  if (!q_nope || !q_pe || !ckv || !kpe || !prefix_lens || !block_table || !cu || !mask || !workspace)
    return DSA_ERR_INVALID_ARGUMENT;
  if (num_pages < 1 || num_pages > 0x7FFFFFFE || max_pages < 1 || max_pages > (1 << 24) || mask_words < 1 ||
      mask_words > 64)
    return DSA_ERR_INVALID_ARGUMENT;
  if (groups_bound(drafts, heads, requests) * (max_pages + kLead) > kMaxUnits) return DSA_ERR_INVALID_ARGUMENT;
  if (ckv_row < kCkv * 2 || kpe_row < kKpe * 2 || ckv_page < 0 || kpe_page < 0) return DSA_ERR_INVALID_ARGUMENT;
  if (!aligned16(q_nope) || !aligned16(q_pe) || !aligned16(ckv) || !aligned16(kpe) || !aligned16(workspace) ||
      ((ckv_page | ckv_row | kpe_page | kpe_row) & 15))
    return DSA_ERR_MISALIGNED;
  if ((reinterpret_cast<uintptr_t>(prefix_lens) | reinterpret_cast<uintptr_t>(block_table) |
       reinterpret_cast<uintptr_t>(cu)) & 3u)
    return DSA_ERR_MISALIGNED;
  if (reinterpret_cast<uintptr_t>(mask) & 7u) return DSA_ERR_MISALIGNED;
  // Outputs lie apart from what other CTAs still read.  The attention's output
  // may be q_nope: a group's rows are written behind its queries' last use, by
  // the CTA that read them or by the join.
  const size_t n = static_cast<size_t>(requests), rows_q = static_cast<size_t>(drafts) * heads;
  const Range in[8] = {{q_nope, rows_q * kCkv * 2},
                       {q_pe, rows_q * kKpe * 2},
                       {ckv, static_cast<size_t>(num_pages - 1) * ckv_page + (kTok - 1) * ckv_row + kCkv * 2},
                       {kpe, static_cast<size_t>(num_pages - 1) * kpe_page + (kTok - 1) * kpe_row + kKpe * 2},
                       {prefix_lens, n * 4},
                       {block_table, n * max_pages * 4},
                       {cu, (n + 1) * 4},
                       {mask, static_cast<size_t>(drafts) * mask_words * 8}};
  if (ranges_overlap(more[0].at, more[0].bytes, more[1].at, more[1].bytes)) return DSA_ERR_OVERLAP;
  for (int o = 0; o < (records ? 2 : 1); ++o)
    for (int i = 0; i < 8; ++i)
      if (ranges_overlap(more[o].at, more[o].bytes, in[i].at, in[i].bytes) &&
          !(records && o == 0 && i == 0 && more[o].at == q_nope))
        return DSA_ERR_OVERLAP;
  int st = current_device_info(info);
  if (st != DSA_OK) return st;
  if (static_cast<size_t>(kSmemBytes) > info->max_smem_optin || info->num_sms > kMaxCtas)
    return DSA_ERR_UNSUPPORTED_DEVICE;
  const Layout a = layout(info->num_sms);
  if (workspace_bytes < (records ? a.bytes : kWorkspaceHeader)) return DSA_ERR_WORKSPACE_TOO_SMALL;
  std::call_once(g_once[info->device], [&]() {
    g_status[info->device] =
        cudaFuncSetAttribute(tree_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) ==
                    cudaSuccess &&
                cudaFuncSetAttribute(tree_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) ==
                    cudaSuccess
            ? DSA_OK
            : DSA_ERR_CUDA;
  });
  if (g_status[info->device] != DSA_OK) return g_status[info->device];
  const uint64_t rows = static_cast<uint64_t>(drafts) * heads;
  if ((st = encode_tmap_3d(&maps[0], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, ckv, kCkv, kTok, num_pages, ckv_row, ckv_page,
                           64, kTok)) != DSA_OK)
    return st;
  if ((st = encode_tmap_3d(&maps[1], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, kpe, kKpe, kTok, num_pages, kpe_row, kpe_page,
                           64, kTok)) != DSA_OK)
    return st;
  if ((st = encode_tmap_2d(&maps[2], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, q_nope, kCkv, rows, kCkv * 2, 64, kRows)) !=
      DSA_OK)
    return st;
  if ((st = encode_tmap_2d(&maps[3], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, q_pe, kKpe, rows, kKpe * 2, 64, kRows)) !=
      DSA_OK)
    return st;
  *prm = Params{};
  prm->prefix_lens = prefix_lens;
  prm->block_table = block_table;
  prm->cu = cu;
  prm->mask = reinterpret_cast<const long long*>(mask);
  prm->num_requests = requests;
  prm->num_drafts = drafts;
  prm->heads = heads;
  prm->max_pages = max_pages;
  prm->mask_words = mask_words;
  prm->num_pages = static_cast<int>(num_pages);
  prm->scale_log2 = sm_scale * 1.4426950408889634f;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  prm->status = reinterpret_cast<unsigned int*>(ws);
  prm->wait_limit_ns = kWaitLimitNs;
  if (records) {
    prm->part_ml = reinterpret_cast<float*>(ws + a.part_ml);
    prm->part_o = reinterpret_cast<float*>(ws + a.part_o);
    prm->plan = reinterpret_cast<int*>(ws + a.plan);
  }
  return DSA_OK;
}

}  // namespace tree
}  // namespace dsa

using namespace dsa;

extern "C" size_t dsa_tree_attention_workspace_bytes(void) {
  DeviceInfo info;
  // Without a usable device, size for the largest SM count of the family.
  const int sms = current_device_info(&info) == DSA_OK ? info.num_sms : 160;
  return tree::layout(sms).bytes;
}

extern "C" int dsa_tree_attention_run(const void* q_nope, const void* q_pe, const void* ckv_cache,
                                      int64_t ckv_page_bytes, int64_t ckv_row_bytes, const void* kpe_cache,
                                      int64_t kpe_page_bytes, int64_t kpe_row_bytes, int64_t num_pages,
                                      const int32_t* prefix_lens, const int32_t* block_table,
                                      const int32_t* cu_drafts, const int64_t* tree_mask, int32_t num_requests,
                                      int32_t num_drafts, int32_t num_heads, int32_t max_pages, int32_t mask_words,
                                      float sm_scale, void* output, float* lse, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  if (!tree::sizes_ok(num_drafts, num_heads, num_requests)) return DSA_ERR_INVALID_ARGUMENT;
  if (num_drafts == 0 || num_requests == 0) return DSA_OK;
  if (!output || !lse) return DSA_ERR_INVALID_ARGUMENT;
  if (!aligned16(output) || (reinterpret_cast<uintptr_t>(lse) & 3u)) return DSA_ERR_MISALIGNED;
  DeviceInfo info;
  tree::Params prm;
  CUtensorMap maps[4];
  const size_t rows_q = static_cast<size_t>(num_drafts) * num_heads;
  const int st = tree::check_and_setup(q_nope, q_pe, ckv_cache, ckv_page_bytes, ckv_row_bytes, kpe_cache,
                                       kpe_page_bytes, kpe_row_bytes, num_pages, prefix_lens, block_table, cu_drafts,
                                       tree_mask, num_requests, num_drafts, num_heads, max_pages, mask_words, sm_scale,
                                       workspace, workspace_bytes, true,
                                       {{output, rows_q * tree::kCkv * 2}, {lse, rows_q * 4}}, &info, &prm, maps);
  if (st != DSA_OK) return st;
  prm.out = static_cast<__nv_bfloat16*>(output);
  prm.lse_out = lse;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const std::lock_guard<std::mutex> turn(turn_of(workspace));  // the attention and its join share the records
  if (launch_programmatic(tree::tree_kernel<false>, dim3(info.num_sms), dim3(tree::kThreads), tree::kSmemBytes, s,
                          maps[0], maps[1], maps[2], maps[3], prm) != cudaSuccess)
    return DSA_ERR_CUDA;
  // Up to 10 groups (by their bound): a row a block of 512 threads, so that a
  // long context's many records are read by many SMs with many loads in flight.
  // More: a group has few records, and blocks of 128 threads and up to four
  // rows cost less.  Whole calls in us, requests of 4 drafts x 16 heads with
  // 2000-16000 tokens, from 64 groups on 1000-8000, at 200 500-6000:
  //   groups            8    10    12    16    32    48    64    96   128   200
  //   1 row, 512     26.2  25.0  28.8  32.7  50.0  67.5  63.3  86.1 107.5 127.9
  //   1 row, 128     29.9  26.5  27.0  28.8  41.7  53.7  45.4  57.7  71.9  77.8
  //   2 rows         35.9  31.0  31.0  32.9  43.2  53.5  44.0  55.6  68.7  73.3
  //   4 rows         44.0  37.9  39.1  40.6  47.8  56.7  47.0  55.4  67.6  71.8
  //   8 rows         61.9  55.9  56.1  57.5  57.8  64.5  54.1  61.2  72.2  73.7
  const int64_t groups = tree::groups_bound(num_drafts, num_heads, num_requests);
  const bool by_record = groups > 2 * info.num_sms;
  const unsigned int across = static_cast<unsigned int>(by_record ? 2 * info.num_sms : groups);
  const int rows = across <= 32 ? 1 : (across <= 96 ? 2 : tree::kJoinRows);
  const bool deep = across <= 10;
  if (launch_programmatic(deep ? tree::combine_kernel<4> : tree::combine_kernel<1>, dim3(across, tree::kRows / rows),
                          dim3(deep ? 512 : 128), 0, s, prm, info.num_sms, rows, by_record) != cudaSuccess)
    return DSA_ERR_CUDA;
  if (cudaGetLastError() != cudaSuccess) return DSA_ERR_CUDA;
  return DSA_OK;
}

extern "C" int dsa_tree_weights_run(const void* q_nope, const void* q_pe, const void* ckv_cache,
                                    int64_t ckv_page_bytes, int64_t ckv_row_bytes, const void* kpe_cache,
                                    int64_t kpe_page_bytes, int64_t kpe_row_bytes, int64_t num_pages,
                                    const int32_t* prefix_lens, const int32_t* block_table, const int32_t* cu_drafts,
                                    const int64_t* tree_mask, int32_t num_requests, int32_t num_drafts,
                                    int32_t num_heads, int32_t max_pages, int32_t mask_words, float sm_scale,
                                    const float* lse, const float* acc, int64_t acc_stride, float* acc_out,
                                    int64_t acc_out_stride, void* workspace, size_t workspace_bytes, void* stream) {
  if (!tree::sizes_ok(num_drafts, num_heads, num_requests)) return DSA_ERR_INVALID_ARGUMENT;
  if (num_requests == 0) return DSA_OK;
  if (!lse || !acc || !acc_out) return DSA_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(acc) | reinterpret_cast<uintptr_t>(acc_out)) & 3u)
    return DSA_ERR_MISALIGNED;
  const int64_t width = static_cast<int64_t>(max_pages) * tree::kTok;
  if (max_pages < 1 || acc_stride < width || acc_out_stride < width || (acc == acc_out && acc_stride != acc_out_stride))
    return DSA_ERR_INVALID_ARGUMENT;
  if (acc != acc_out && rows_overlap(num_requests, acc, acc_stride, width, acc_out, acc_out_stride, width))
    return DSA_ERR_OVERLAP;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (num_drafts == 0) {  // nothing to add
    if (acc != acc_out &&
        cudaMemcpy2DAsync(acc_out, acc_out_stride * 4, acc, acc_stride * 4, static_cast<size_t>(max_pages) * tree::kTok * 4,
                          num_requests, cudaMemcpyDeviceToDevice, s) != cudaSuccess)
      return DSA_ERR_CUDA;
    return DSA_OK;
  }
  DeviceInfo info;
  tree::Params prm;
  CUtensorMap maps[4];
  const int st = tree::check_and_setup(q_nope, q_pe, ckv_cache, ckv_page_bytes, ckv_row_bytes, kpe_cache,
                                       kpe_page_bytes, kpe_row_bytes, num_pages, prefix_lens, block_table, cu_drafts,
                                       tree_mask, num_requests, num_drafts, num_heads, max_pages, mask_words, sm_scale,
                                       workspace, workspace_bytes, false,
                                       {{acc_out, static_cast<size_t>((num_requests - 1) * acc_out_stride + width) * 4},
                                        {lse, static_cast<size_t>(num_drafts) * num_heads * 4}},
                                       &info, &prm, maps);
  if (st != DSA_OK) return st;
  prm.lse_in = lse;
  prm.acc = acc;
  prm.acc_stride = acc_stride;
  prm.acc_out = acc_out;
  prm.acc_out_stride = acc_out_stride;
  if (launch_programmatic(tree::tree_kernel<true>, dim3(info.num_sms), dim3(tree::kThreads), tree::kSmemBytes, s,
                          maps[0], maps[1], maps[2], maps[3], prm) != cudaSuccess)
    return DSA_ERR_CUDA;
  if (cudaGetLastError() != cudaSuccess) return DSA_ERR_CUDA;
  return DSA_OK;
}
