// quant_attention.cu -- attention over the paged latent cache in 8 bits: dense,
// for single tokens and chains of drafts, and over selected slots (sm_100a).
//
// With the cache's token k as codes c_k (512 e4m3), scale s_k and position part
// e_k (64 bf16):
//   x_k = scale * (s_k (q_nope . c_k) + q_pe . e_k)
//   lse = log2 sum_k 2^(x_k log2 e),   out = sum_k 2^(x_k log2 e - lse) s_k c_k
//
// The codes go to the tensor core as they are: a token's scale is taken out of
// both products.  For that the other operands have to be 8 bits too, and are, in
// parts that add up to what they were:
//   q_nope f = a + b / 16 with a, b e4m3 and f a power of two for each row (its
//     largest value to 128 .. 256).  a takes the upper 4 of the 8 bits of a bf16,
//     b the other 4: exact from 2^-13 of the row's largest up, to 2^-21 of that
//     below.
//   w = p s (weight by scale, the row's largest so far 2^5 or more) = a + b +
//     (c + d) / 128 with e5m2 parts, each to nearest: 3 bits, then 4 more each (what
//     is left has a sign and is less than the last step).  Within 2^-14 of w (6e-6 in
//     the mean) from 2^15 down to 2^-9, and within 2^-23 below: many light tokens
//     beside a heavy one still count.
//     Three parts, 2^-11 (1.2e-4), would make a difference that outputs show: bf16
//     has 2^-9, and one in fifteen was rounded to a neighbour (one in 300).
// Per tile of 128 tokens and group of R rows (token, head)
//   S^T[128, 2R] = C[128, 512] . [a b]^T    16 x (M128 N2R K32, e4m3)
//   E^T[128, R]  = E[128, 64] . (q_pe f)^T   4 x (M128 NR K16, bf16)
//   O^T += C^T[512, 128] . [a c b d]^T       4 x 4 x (M128 N64 K32, e4m3 x e5m2)
// so the parts lie along N, which costs the tensor core nothing up to N = 64: it
// is fed at 128 bytes of A a clock.  Of 16 rows each part has its own 16 columns
// of O^T; of 32, whose 128 would leave TMEM no room for S^T, a product of a and c
// is followed by one of b and d into the same 64.  A tile's 82 KB cross shared
// memory once in, and once and a half out (twice and a half of 32 rows), against
// three and a half times for bf16 copies of it (225 KB, 1750 clocks, where its share
// of the HBM rate takes 3500).
//
// Units of work are (request, group, tile), cut into equal contiguous slices, one
// per CTA; slices' pieces that do not cover their group's whole context are
// written as fp32 records (slot 0: at the slice's start, slot 1: at its end) and
// joined by join_kernel.  Small calls give each group to a cluster of CTAs, which
// join their pieces through shared memory (together_for).
//
// Measured, attention with its join in replayed graphs: one row of 16 heads over
// 64 x 65536 tokens 416 us (2.70 GB, 6.5 TB/s: HBM-bound; 443-480 back to back under
// the power cap); 16 x 4096-16384 tokens, 1-4 rows 38 us (96 MB: start, end and join,
// see below); 1-2 rows of 128 heads over 5 x 8000-30001 tokens 65 us (35 GFLOP: a
// tile's way through its stage takes 5600 clocks, load 800, S^T 1800, softmax 1800,
// O^T 1200, and two stages fit; the products alone take 1660 a tile); 300 x 2048
// selected slots of 16 heads 95 us (406 MB; a kernel that only reads these rows takes
// 87: half-kilobyte pieces at random, and 14 us of it the scales, a sector each).
// About 8 us are a call's start (plan, page ids, first tile, its maxima) and end,
// 3.5-9 its join.  With weights in three parts, and the product of 32 rows in one, the
// four took 406, 36, 62 and 93 us.  (Comparisons beside choices below that do not
// choose between 16 rows and 32, or clusters and slices, are of that time.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <mutex>

#include "dsa_b200.h"
#include "host.h"
#include "ptx.cuh"

namespace dsa {
namespace qattn {

constexpr int kCkv = DSA_CKV_DIM;            // 512
constexpr int kKpe = DSA_KPE_DIM;            // 64
constexpr int kPage = DSA_PAGE_SIZE;
constexpr int kPageBytes = DSA_LATENT_PAGE_BYTES;
constexpr int kKpeAt = kPage * kCkv;
constexpr int kScaleAt = kKpeAt + kPage * kKpe * 2;
constexpr int kTok = 128;                    // tokens per tile: two pages
constexpr int kBlockBytes = kTok * 128;      // 16384: 128 dims of a tile's codes, or its position part
constexpr int kParts = 4;                    // blocks of codes
constexpr int kStageBytes = (kParts + 1) * kBlockBytes;  // 81920
constexpr int kTmemCols = 512;
// A rescale of O costs its tile some 2300 clocks, and of two sets whichever needs one
// holds up the other: at a threshold of 8 log2 units 2 of 34 tiles need one (normal
// logits of spread 2.5, scales spread by e^0.3), at 6 four, at 4 six.  Graph replays
// at 8, 9 and 10: 128 heads 66.9, 65.7 and 65.0 us, 16 x 4096-16384 tokens 38.6, 38.3
// and 38.3; each halves the unit that is left for light weights.
constexpr float kRescaleThreshold = 10.0f;
constexpr float kUnit = 32.0f;               // of weights: 2^10 x 32 = 2^15 is the largest, e5m2 goes to 57344
constexpr float kUnitLog2 = 5.0f;
constexpr float kScaleRange = 60.0f;         // log2 units from a segment's unit of scales
constexpr float kLeastRef = 0x1p-100f;       // of that unit: kUnit over it has to be a number
constexpr float kLowUnit = 1.0f / 128.0f;    // of their last two parts: what the first two leave is below 2^-7 of a weight
constexpr int kMostRows = 32;
constexpr int kColsO = 64;                   // of O^T for 128 dims

// R = 16 rows with two buffers of queries and of S^T, or 32 with one.  Softmax
// warps come in two sets of four, which have half of the columns each and a token
// a thread.
template <int kR, bool kSparse>
struct Shape {
  // Columns (rows of Q) of a softmax thread.  32 rows as four sets of 8 columns, 16
  // warps in 80 registers, take 63.6 us for 62 (128 heads), 31.7 for 29.9 (16 x 2
  // rows of 16 heads, 4000-12000 tokens): what a warp does once a tile is half of it.
  static constexpr int kCols = kR / 2;
  static constexpr int kSets = kR / kCols;
  static constexpr int kSoftWarps = 4 * kSets;
  static constexpr int kLogitWarp = kSoftWarps;          // S^T, E^T (owns TMEM)
  static constexpr int kValueWarp = kSoftWarps + 1;      // O^T
  static constexpr int kQueryWarps = kSparse ? 2 : 4;    // queries into parts
  static constexpr int kQueryWarp = kSoftWarps + 2;
  static constexpr int kLoadWarp = kQueryWarp + kQueryWarps;    // dense: TMA
  static constexpr int kGatherWarp = kQueryWarp + kQueryWarps;  // sparse
  // Two groups, one for each stage: four warps each, or two for 32 rows, whose softmax
  // warps need the registers (with four 188 bytes spill; 64 rows of 128 heads 111.6 us for 106.3).
  static constexpr int kGatherWarps = kR == 16 ? 8 : 4;
  static constexpr int kThreads = 32 * (kSparse ? kGatherWarp + kGatherWarps : kLoadWarp + 1);
  // Warps that take queries at the first segment.
  static constexpr int kFirstWarps = kQueryWarps + kSoftWarps;
  static_assert(kFirstWarps % kQueryWarps == 0 && (kCols == 8 || kCols == 16), "shape");
  static constexpr int kQBufs = kR == 16 ? 2 : 1;
  static constexpr int kSBufs = kR == 16 ? 2 : 1;
  static constexpr int kQBlock = 2 * kR * 128;           // 128 dims of both parts
  static constexpr int kQBytes = kParts * kQBlock + kR * 128;
  static constexpr uint32_t kColS = 0;                   // a: 0, b: R, e: 2R of each buffer
  static constexpr uint32_t kColO = kSBufs * 3 * kR;     // 4 blocks of 128 dims x 64 columns
  static constexpr int kSums = kColsO / kR;              // of a row: of a, c, b, d, or of a + b, c + d
  static_assert(kColO + kParts * kColsO <= kTmemCols && kSums * kCols == 32, "TMEM");
  static constexpr uint32_t kIdescS = idesc_make(0, 0, false, false, 128, 2 * kR);
  static constexpr uint32_t kIdescE = idesc_make(1, 1, false, false, 128, kR);
  static constexpr uint32_t kIdescO = idesc_make(0, 1, true, true, 128, kColsO);  // e4m3 codes, e5m2 weights
};

constexpr int kOffQ = 2 * kStageBytes;                 // 163840
constexpr int kOffP = kOffQ + 36864;                   // either shape's queries
static_assert(Shape<16, false>::kQBufs * Shape<16, false>::kQBytes == 36864 && Shape<32, false>::kQBytes == 36864,
              "queries");
constexpr int kOffScale = kOffP + kTok * 128;          // [2][128]
constexpr int kOffBar = kOffScale + 2 * kTok * 4;
constexpr int kOffMisc = kOffBar + 256;
constexpr int kOffRed = kOffMisc + 128;                // [sets][4 warps][columns], planning: warp sums
constexpr int kOffFactor = kOffRed + 512;              // [32]
constexpr int kOffMax = kOffFactor + 128;              // [32] running maxima
constexpr int kOffMinus = kOffMax + 128;               // [32] what is added to logits
constexpr int kOffMost = kOffMinus + 128;              // [4][4] largest scales
constexpr int kOffC = kOffMost + 64;                   // [2][32] logits' factors
constexpr int kOffInfo = kOffC + 256;                  // what the softmax warps need of the segments, 4 in turn
constexpr int kSmemBytes = 1024 + kOffInfo + 4 * 48;
static_assert(kSmemBytes <= 232448, "shared memory of a CTA");

constexpr int kMaxRequests = 65536;
constexpr int64_t kMaxRows = 1 << 24;          // rows x heads
constexpr int64_t kMaxUnits = 1 << 30;
constexpr int kMaxCtas = 256;
constexpr int kPlanGroups = 2 * kMaxCtas;      // the plan: groups of the records, then first row and rows of each group
constexpr int kPartFloats = kMostRows * kCkv;

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
  double by_ctas;           // 1 / CTAs
  __nv_bfloat16* out;
  float* lse;
  unsigned int* status;
  unsigned long long wait_limit_ns;
  float* part_o;            // [2 * grid][kMostRows][512]
  float2* part_ml;          // [2 * grid][kMostRows]: m, l
  int* plan;
};

struct Request {
  int row0, n;              // first row, rows (tokens)
  int length;               // cached tokens; row j of n sees length - n + 1 + j
  int rows, groups, tiles;  // (token, head) rows
  int span;                 // units per group: its tiles and kLead<kR> more for its start
};

// What starting a group costs, in tiles (of 16 rows; of 32, whose tiles take longer
// but whose start and end do as well): requests of 1000-3000 tokens, 64 of one row
// of 16 heads 30.1 us at 1, 29.6 at 2, 30.6 at 3, 31.3 at 4; 64 of four rows of
// 300-900 tokens 31.3, 31.2, 29.7, 29.6; 4 of 128 heads and 4000-12000 tokens 28.4,
// 26.9, 25.6, 25.7.
template <int kR>
constexpr int kLead = kR == 16 ? 2 : 3;
constexpr int kMostLead = 3;
constexpr int kMostTogether = 8;             // CTAs of a cluster that share a group

template <int kR, bool kSparse>
__device__ __forceinline__ Request load_request(const Params& p, int b, bool& bad) {
  Request r;
  bad = false;
  if (kSparse) {
    r.row0 = b;
    r.n = 1;
    r.length = p.topk;
  } else {
    const int cap = p.max_pages * kPage;
    r.row0 = b;
    r.n = 1;
    if (p.cu != nullptr) {
      const int lo = p.cu[b], hi = p.cu[b + 1];
      r.row0 = lo;
      r.n = hi - lo;
      if (lo < 0 || hi < lo || hi > p.num_rows) {
        r.n = 0;
        bad = true;
      }
    }
    r.length = p.seq_lens[b];
    if (r.length < 0 || r.length > cap) {
      r.length = r.length < 0 ? 0 : cap;
      bad = true;
    }
  }
  r.rows = r.n * p.heads;
  r.groups = (r.rows + kR - 1) / kR;
  // A row that sees nothing is written by a tile whose tokens are all masked.
  r.tiles = r.n == 0 ? 0 : max(1, (r.length + kTok - 1) / kTok);
  r.span = r.n == 0 ? 0 : r.tiles + kLead<kR>;
  return r;
}

// CTA c of `ctas` has the units [start(c), start(c+1)), start(c) = floor(total c /
// ctas); by_ctas is 1 / ctas.  In 64-bit floating point the quotient, at most 2^30,
// is within 2^-21 of the exact one, whose fraction is a multiple of 1 / 256 or more.
__device__ __forceinline__ int slice_start(int total, int c, double by_ctas) {
  return static_cast<int>(fma(static_cast<double>(total) * c, by_ctas, 1.0 / 1024.0));
}

struct Start {
  int b, first, first_group;  // request, its first unit and group over all requests
  Request r;
  int group, unit;
};

// A run of tiles of one group.
struct Segment {
  int b, group, t0, t1, group_index;
  Request r;
  bool whole;  // covers the group's whole context
  int slot;    // of its record if it does not
};

// The same as the softmax warps read it from shared memory, where it takes none of
// their registers.  t0 == t1: the end.
struct SegmentInfo {
  int b, t0, t1, row_q, rows, length, n, group, group_index, whole, slot, unused;
};
static_assert(sizeof(SegmentInfo) == 48, "segment");

template <int kR, bool kSparse>
struct Walker {
  const Params& p;
  int u, u0, u1, b, first, first_group;
  Request r;
  int group, unit;

  __device__ Walker(const Params& prm, int u0_, int u1_, const Start& st)
      : p(prm), u(u0_), u0(u0_), u1(u1_), b(st.b), first(st.first), first_group(st.first_group) {
    if (u0 >= u1) return;
    r = st.r;
    group = st.group;
    unit = st.unit;
  }
  __device__ bool leave() {  // to the next request that has units in the slice
    for (;;) {
      first += r.groups * r.span;
      first_group += r.groups;
      ++b;
      if (b >= p.num_requests || first >= u1) return false;
      bool bad;
      r = load_request<kR, kSparse>(p, b, bad);
      if (r.tiles == 0) continue;
      group = unit = 0;
      return true;
    }
  }
  __device__ bool next(Segment& s) {
    while (u < u1) {
      s.b = b;
      s.r = r;
      s.group = group;
      s.group_index = first_group + group;
      const int len = min(r.span - unit, u1 - u);
      s.t0 = unit < kLead<kR> ? 0 : unit - kLead<kR>;
      s.t1 = unit + len - kLead<kR>;
      s.whole = s.t0 == 0 && s.t1 == r.tiles;
      s.slot = u == u0 ? 0 : 1;
      u += len;
      unit = 0;
      if (u < u1 && ++group == r.groups && !leave()) u = u1;
      if (s.t1 > s.t0) return true;  // else a slice's end within the lead
    }
    return false;
  }
};

// `count` arrivals at once.
__device__ __forceinline__ void mbar_arrive_many(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}

// Three blocks of 8 or 16 consecutive columns of 32 lanes, with the wait for them
// in the same statement.
__device__ __forceinline__ void tmem_ld_three(uint32_t a0, uint32_t b0, uint32_t c0, float (&a)[8], float (&b)[8],
                                              float (&c)[8]) {
  uint32_t r[24];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%24];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8, %9, %10, %11, %12, %13, %14, %15}, [%25];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%16, %17, %18, %19, %20, %21, %22, %23}, [%26];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23])
      : "r"(a0), "r"(b0), "r"(c0)
      : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[i] = __uint_as_float(r[i]);
    b[i] = __uint_as_float(r[8 + i]);
    c[i] = __uint_as_float(r[16 + i]);
  }
}

__device__ __forceinline__ void tmem_ld_three(uint32_t a0, uint32_t b0, uint32_t c0, float (&a)[16], float (&b)[16],
                                              float (&c)[16]) {
  uint32_t r[48];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%48];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%49];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47}, [%50];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]),
        "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]),
        "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47])
      : "r"(a0), "r"(b0), "r"(c0)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    a[i] = __uint_as_float(r[i]);
    b[i] = __uint_as_float(r[16 + i]);
    c[i] = __uint_as_float(r[32 + i]);
  }
}

// A row's sums of 8 or 16 columns: 4 blocks of 8, 16 apart, or 2 of 16, 32 apart.
__device__ __forceinline__ void tmem_ld_sums(uint32_t at, float (&v)[4][8]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8, %9, %10, %11, %12, %13, %14, %15}, [%33];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%16, %17, %18, %19, %20, %21, %22, %23}, [%34];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%24, %25, %26, %27, %28, %29, %30, %31}, [%35];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at), "r"(at + 16), "r"(at + 32), "r"(at + 48)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i / 8][i % 8] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_ld_sums(uint32_t at, float (&v)[2][16]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%33];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at), "r"(at + 32)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i / 16][i % 16] = __uint_as_float(r[i]);
}

// The row's O from its sums.
__device__ __forceinline__ float whole_sum(const float (&v)[4][8], int k) {
  return fmaf(v[1][k] + v[3][k], kLowUnit, v[0][k] + v[2][k]);
}
__device__ __forceinline__ float whole_sum(const float (&v)[2][16], int k) { return fmaf(v[1][k], kLowUnit, v[0][k]); }

__device__ __forceinline__ void tmem_st(uint32_t at, const float (&v)[16]) { tmem_st16(at, v); }
__device__ __forceinline__ void tmem_st(uint32_t at, const float (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at),
               "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])),
               "r"(__float_as_uint(v[3])), "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])),
               "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7]))
               : "memory");
}

// kN values of each lane reduced over the warp: at each step a lane keeps half of
// its columns and sends the others.  Lanes end with column `k`'s result.
template <int kN, typename Op>
__device__ __forceinline__ float over_tokens(float (&v)[kN], int lane, int& k, Op op) {
  k = 0;
#pragma unroll
  for (int half = kN / 2, o = 16; half >= 1; half /= 2, o /= 2) {
    const bool up = lane & o;
#pragma unroll
    for (int j = 0; j < half; ++j) {
      const float send = up ? v[j] : v[j + half];
      v[j] = op(up ? v[j + half] : v[j], __shfl_xor_sync(0xffffffffu, send, o));
    }
    if (up) k += half;
  }
#pragma unroll
  for (int o = 16 / kN; o >= 1; o /= 2) v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
  return v[0];
}

template <int kN>
__device__ __forceinline__ void load_cols(const float* from, float (&v)[kN]) {
#pragma unroll
  for (int k = 0; k < kN / 4; ++k) {
    const float4 x = reinterpret_cast<const float4*>(from)[k];
    v[4 * k] = x.x;
    v[4 * k + 1] = x.y;
    v[4 * k + 2] = x.z;
    v[4 * k + 3] = x.w;
  }
}

// 16 bytes with cp.async, or zeros.
__device__ __forceinline__ void cp_async16_or_zeros(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4_or_zeros(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(real ? 4 : 0) : "memory");
}

// What CTA `rank` of the cluster has at this address of its shared memory, or zeros
// (where it may be no rank of the cluster: its address is not formed then).
__device__ __forceinline__ float2 ld_cluster_or_zeros(uint32_t at, int rank, bool real) {
  float2 v;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 a;\n\t"
      "setp.ne.u32 p, %4, 0;\n\tmov.u32 a, %2;\n\t@p mapa.shared::cluster.u32 a, %2, %3;\n\tmov.f32 %0, 0f00000000;\n\tmov.f32 %1, 0f00000000;\n\t"
      "@p ld.shared::cluster.v2.f32 {%0, %1}, [a];\n\t}"
      : "=&f"(v.x), "=&f"(v.y)
      : "r"(at), "r"(rank), "r"(static_cast<uint32_t>(real))
      : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4_or_zeros(uint32_t at, int rank, bool real) {
  float4 v;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 a;\n\t"
      "setp.ne.u32 p, %6, 0;\n\tmov.u32 a, %4;\n\t@p mapa.shared::cluster.u32 a, %4, %5;\n\tmov.f32 %0, 0f00000000;\n\tmov.f32 %1, 0f00000000;\n\t"
      "mov.f32 %2, 0f00000000;\n\tmov.f32 %3, 0f00000000;\n\t"
      "@p ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
      : "=&f"(v.x), "=&f"(v.y), "=&f"(v.z), "=&f"(v.w)
      : "r"(at), "r"(rank), "r"(static_cast<uint32_t>(real))
      : "memory");
  return v;
}

// Eight weights (at most 2^15) into their four e5m2 parts a + b + (c + d) / 128, in
// the order a, c, b, d.  In half precision: the weight's upper 11 bits, from which
// a and b are taken without rounding, and what they leave with its lower bits, to
// 11 bits more.  An e5m2 value is the upper byte of the same value in half
// precision; half a step added below it rounds (a carry moves the exponent), in two
// integer operations (by conversions 128 heads took 1 us more).  (NaN may become 0
// here; its row's sum l is NaN.)
__device__ __forceinline__ void in_parts(const float* w, uint2 (&out)[4]) {
  uint32_t part[4][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float u0 = __uint_as_float(__float_as_uint(w[2 * k]) & 0xFFFFE000u);
    const float u1 = __uint_as_float(__float_as_uint(w[2 * k + 1]) & 0xFFFFE000u);
    __half2 h = __floats2half2_rn(u0, u1);
    const __half2 lower = __floats2half2_rn(w[2 * k] - u0, w[2 * k + 1] - u1);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (x == 2) h = __hmul2(__hadd2(h, lower), __float2half2_rn(1.0f / kLowUnit));
      uint32_t two = *reinterpret_cast<const uint32_t*>(&h) + 0x00800080u;
      if (x < 3) two &= 0xFF00FF00u;
      part[x < 2 ? 2 * x : 2 * x - 3][k] = two;
      if (x < 3) h = __hsub2(h, *reinterpret_cast<const __half2*>(&two));  // exact
    }
  }
#pragma unroll
  for (int x = 0; x < 4; ++x)
    out[x] = make_uint2(__byte_perm(part[x][0], part[x][1], 0x7531), __byte_perm(part[x][2], part[x][3], 0x7531));
}

// kTogether: each cluster of CTAs has one group, whose tiles they share alike and
// whose pieces they join through shared memory.
template <int kR, bool kSparse, bool kTogether>
__global__ void __launch_bounds__(Shape<kR, kSparse>::kThreads, 1)
attend_kernel(const __grid_constant__ CUtensorMap codes_map, const __grid_constant__ CUtensorMap kpe_map, const Params p) {
  using Sh = Shape<kR, kSparse>;
  constexpr int C = Sh::kCols;
  constexpr int kThreads = Sh::kThreads;
  constexpr int kWarps = kThreads / 32;
  constexpr int kSoftWarps = Sh::kSoftWarps, kLoadWarp = Sh::kLoadWarp, kLogitWarp = Sh::kLogitWarp;
  constexpr int kValueWarp = Sh::kValueWarp, kQueryWarp = Sh::kQueryWarp, kGatherWarp = Sh::kGatherWarp;
  constexpr int kQueryWarps = Sh::kQueryWarps;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);  // (an offset: the compiler still knows it as shared)
  uint8_t* q_mem = smem + kOffQ;
  uint8_t* p_mem = smem + kOffP;
  float* scale_s = reinterpret_cast<float*>(smem + kOffScale);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint64_t* kv_full = bars;                // [2 stages][kParts]; sparse: the last of each only
  uint64_t* kv_free = bars + 2 * kParts;   // [2][kParts]: the block's part of O^T is done
  uint64_t* q_full = bars + 4 * kParts;    // [2]
  uint64_t* q_empty = q_full + 2;          // [2]
  uint64_t* s_full = q_full + 4;           // [2]
  uint64_t* s_empty = q_full + 6;          // [2]
  uint64_t* p_full = q_full + 8;
  uint64_t* o_empty = q_full + 9;
  uint64_t* drain = q_full + 10;           // [2]
  constexpr int kBars = 4 * kParts + 12;
  static_assert(kBars * 8 <= kOffMisc - kOffBar, "barriers");
  auto pv_done = [&](int i) { return &kv_free[(i & 1) * kParts + kParts - 1]; };
  int* misc = reinterpret_cast<int*>(smem + kOffMisc);
  uint32_t* tmem_base_smem = reinterpret_cast<uint32_t*>(misc);
  int* abort_flag = misc + 1;
  Start* found = reinterpret_cast<Start*>(misc + 2);
  static_assert(8 + sizeof(Start) <= kOffRed - kOffMisc, "misc");
  float* red = reinterpret_cast<float*>(smem + kOffRed);
  int* warp_sums = reinterpret_cast<int*>(red);  // planning: units, groups of each warp
  static_assert(2 * kWarps * 4 <= 512, "warp sums");
  float* factor_s = reinterpret_cast<float*>(smem + kOffFactor);
  float* max_s = reinterpret_cast<float*>(smem + kOffMax);
  float* minus_s = reinterpret_cast<float*>(smem + kOffMinus);
  float* most_s = reinterpret_cast<float*>(smem + kOffMost);
  float* c_s = reinterpret_cast<float*>(smem + kOffC);
  // kTogether: the CTA's piece, over the first stage: O over the codes once its last
  // product is done, m and l over the position part, which the last logits have used.
  float* together_o = reinterpret_cast<float*>(smem);  // [kR][512]
  float2* together_ml = reinterpret_cast<float2*>(smem + kParts * kBlockBytes);
  static_assert(kR * kCkv * 4 <= kParts * kBlockBytes, "a piece");
  // Entry x & 3 is written again behind q_empty of segment x + 2, at which all softmax warps are done with segment x.
  SegmentInfo* info_s = reinterpret_cast<SegmentInfo*>(smem + kOffInfo);

  const int tid = threadIdx.x;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int lane = tid & 31;

  if (tid == 0) {
    for (int x = 0; x < kBars; ++x) mbar_init(&bars[x], 1);
    for (int s = 0; s < 2; ++s) {
      if (kSparse) mbar_init(&kv_full[s * kParts + kParts - 1], Sh::kGatherWarps / 2);
      mbar_init(&q_full[s], Sh::kFirstWarps);
      mbar_init(&q_empty[s], 1 + kSoftWarps);
      mbar_init(&s_empty[s], kSoftWarps);
    }
    mbar_init(p_full, kSoftWarps);
    mbar_init(o_empty, kSoftWarps);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (!kSparse && warp == kLoadWarp && elect_one()) {
    prefetch_tensor_map(&codes_map);
    prefetch_tensor_map(&kpe_map);
  }
  if (warp == kLogitWarp) tmem_alloc(tmem_base_smem, kTmemCols);
  griddep_launch_dependents();
  griddep_wait();

  // ---- plan: total units, and the request that holds this slice's first one.
  // (kTogether: the total of groups, and the request that holds the cluster's.)
  const unsigned int ctas = kTogether ? cluster_size() : 1u;
  const int rank = kTogether ? static_cast<int>(cluster_rank()) : 0;
  const int cluster = static_cast<int>(blockIdx.x / ctas);
  auto each_of = [&](int tiles) { return static_cast<int>((static_cast<unsigned int>(tiles) + ctas - 1u) / ctas); };
  const bool keeper = blockIdx.x == 0;  // writes the groups for join_kernel
  int2* groups_out = reinterpret_cast<int2*>(p.plan + kPlanGroups);
  int total = 0;
  if constexpr (kSparse) {
    bool bad;
    const Request r = load_request<kR, true>(p, 0, bad);
    total = p.num_rows * r.groups * (kTogether ? 1 : r.span);  // every row alike
    if (!kTogether && keeper)
      for (int x = tid; x < p.num_rows * r.groups; x += kThreads)
        groups_out[x] = make_int2(x / r.groups * p.heads + x % r.groups * kR, min(kR, r.rows - x % r.groups * kR));
    if (kTogether && tid == 0) {
      const int b = cluster / r.groups;
      Request mine = r;
      mine.row0 = b;
      *found = Start{b, 0, 0, mine, cluster - b * r.groups, kLead<kR> + min(rank * each_of(r.tiles), r.tiles)};
    } else if (tid == 0) {
      const int u0 = slice_start(total, blockIdx.x, p.by_ctas);
      const int b = u0 / (r.groups * r.span), in = u0 - b * r.groups * r.span;
      Request mine = r;
      mine.row0 = b;
      *found = Start{b, b * r.groups * r.span, b * r.groups, mine, in / r.span, in % r.span};
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  } else {
    // Every CTA sums all requests (one or two loads a thread for ordinary
    // batches) instead of waiting for a planning launch.
    const int per = (p.num_requests + kThreads - 1) / kThreads;
    const int b_lo = min(tid * per, p.num_requests), b_hi = min(b_lo + per, p.num_requests);
    int units = 0, groups = 0;
    bool any_bad = false, decreasing = false;
    Request mine;  // the thread's first (for ordinary batches its only) request
    for (int b = b_lo; b < b_hi; ++b) {
      bool bad;
      const Request r = load_request<kR, false>(p, b, bad);
      if (b == b_lo) mine = r;
      if (p.cu != nullptr) decreasing |= p.cu[b + 1] < p.cu[b];
      units += r.groups * (kTogether ? 1 : r.span);
      groups += r.groups;
      any_bad |= bad;
    }
    if (any_bad && keeper) atomicOr(p.status, DSA_DEV_BAD_SEQ_LEN);
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
      warp_sums[kWarps + warp] = ig;
    }
    tc_fence_before();
    // Where cu_rows decreases, requests could share rows, and the sums exceed
    // what the host checked: such a call does nothing.
    const bool nothing = __syncthreads_or(decreasing);
    tc_fence_after();
    int before = iu - units, gbefore = ig - groups;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) {
        before += warp_sums[w];
        gbefore += warp_sums[kWarps + w];
      }
      total += warp_sums[w];
    }
    if (nothing) total = units = 0;
    const int u0 = kTogether ? cluster : slice_start(total, blockIdx.x, p.by_ctas);
    if (!nothing && ((!kTogether && keeper) || (u0 >= before && u0 < before + units))) {
      for (int b = b_lo; b < b_hi; ++b) {
        bool bad;
        const Request r = b == b_lo ? mine : load_request<kR, false>(p, b, bad);
        const int un = r.groups * (kTogether ? 1 : r.span);
        if (kTogether && u0 >= before && u0 < before + un) {
          *found = Start{b, 0, 0, r, u0 - before, kLead<kR> + min(rank * each_of(r.tiles), r.tiles)};
        } else if (u0 >= before && u0 < before + un) {
          const int group = (u0 - before) / r.span;
          *found = Start{b, before, gbefore, r, group, u0 - before - group * r.span};
        }
        if (!kTogether && keeper)
          for (int g = 0; g < r.groups; ++g)
            groups_out[gbefore + g] = make_int2(r.row0 * p.heads + g * kR, min(kR, r.rows - g * kR));
        before += un;
        gbefore += r.groups;
      }
    }
    __syncthreads();
  }
  int u0 = 0, u1 = 0;
  if constexpr (kTogether) {
    if (cluster < total) u1 = max(min(each_of(found->r.tiles), found->r.tiles + kLead<kR> - found->unit), 0);
  } else {
    u0 = slice_start(total, blockIdx.x, p.by_ctas);
    u1 = slice_start(total, blockIdx.x + 1, p.by_ctas);
  }
  const uint32_t tmem_base = *tmem_base_smem;
  const WaitCtx wctx{abort_flag, p.status, p.wait_limit_ns};
  Walker<kR, kSparse> walk(p, u0, u1, *found);
  Segment s;

  // ------------------------------------------------------------ queries into parts
  // The query warps do it for all segments, a segment ahead of the softmax where
  // there are two buffers; at the first one the softmax warps, which have nothing
  // to do yet, take their share of the rows.  Lane l has a row's dims 16 l .. +15.
  if (warp < kSoftWarps || (warp >= kQueryWarp && warp < kQueryWarp + kQueryWarps)) {
    const bool helper = warp < kSoftWarps;
    Walker<kR, kSparse> ahead = walk;
    int segs = 0;
    for (;;) {
      const bool more = ahead.next(s);
      const int qb = segs % Sh::kQBufs;
      const int rows = more ? min(kR, s.r.rows - s.group * kR) : 0;
      const int64_t row_q = more ? static_cast<int64_t>(s.r.row0) * p.heads + s.group * kR : 0;
      const int step = segs == 0 ? Sh::kFirstWarps : kQueryWarps;
      uint8_t* to = q_mem + qb * Sh::kQBytes;
      struct Raw {
        uint4 c[2], pe;
      };
      auto load = [&](int r) {
        Raw x;
        x.c[0] = x.c[1] = x.pe = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows) {
          const uint4* src = reinterpret_cast<const uint4*>(p.q_nope + (row_q + r) * kCkv) + 2 * lane;
          x.c[0] = src[0];
          x.c[1] = src[1];
          if (lane < 8) x.pe = *(reinterpret_cast<const uint4*>(p.q_pe + (row_q + r) * kKpe) + lane);
        }
        return x;
      };
      int r = helper ? warp : warp - kQueryWarp + step - kQueryWarps;
      Raw first = load(r), second = load(r + step);
      // All lanes leave together.
      if (!__all_sync(0xffffffffu, mbar_wait(&q_empty[qb], ((segs / Sh::kQBufs) & 1) ^ 1, wctx))) break;
      if (warp == kQueryWarp && lane == 0) {
        SegmentInfo x = {};
        if (more)
          x = SegmentInfo{s.b, s.t0, s.t1, static_cast<int>(row_q), rows, s.r.length, s.r.n, s.group, s.group_index, s.whole, s.slot, 0};
        info_s[segs & 3] = x;
      }
#pragma unroll 1
      for (; more && r < kR; r += step) {
        const uint32_t x[8] = {first.c[0].x, first.c[0].y, first.c[0].z, first.c[0].w,
                               first.c[1].x, first.c[1].y, first.c[1].z, first.c[1].w};
        const uint4 now_pe = first.pe;
        first = second;
        second = load(r + 2 * step);  // two rows ahead
        uint32_t most = 0u;
#pragma unroll
        for (int k = 0; k < 8; ++k) most = max(most, max((x[k] << 16) & 0x7FFFFFFFu, x[k] & 0x7FFF0000u));
        most = __reduce_max_sync(0xffffffffu, most);
        // f = 2^7 over the largest value's power of two, at most 2^30: the
        // logits of queries below that are 0 to all purposes.
        const int exponent = most == 0u || most >= 0x7F800000u ? 127 : min(max(261 - static_cast<int>(most >> 23), 1), 157);
        const float f = __uint_as_float(static_cast<uint32_t>(exponent) << 23);
        uint32_t pa[4], pb[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t a4 = 0u, b4 = 0u;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // In half precision: its 11 bits hold q f down to 2^-24.
            const uint32_t w = x[2 * k + h];
            const __half2 v = __floats2half2_rn(__uint_as_float(w << 16) * f, __uint_as_float(w & 0xFFFF0000u) * f);
            const __nv_fp8x2_storage_t a2 =
                __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(v), __NV_SATFINITE, __NV_E4M3);
            const __half2 back = __half2(__nv_cvt_fp8x2_to_halfraw2(a2, __NV_E4M3));
            const __half2 rest = __hmul2(__hsub2(v, back), __floats2half2_rn(16.f, 16.f));
            const __nv_fp8x2_storage_t b2 =
                __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(rest), __NV_SATFINITE, __NV_E4M3);
            a4 |= static_cast<uint32_t>(a2) << (16 * h);
            b4 |= static_cast<uint32_t>(b2) << (16 * h);
          }
          pa[k] = a4;
          pb[k] = b4;
        }
        if (most >= 0x7F800000u) {  // an infinity or NaN: the row's logits are NaN
#pragma unroll
          for (int k = 0; k < 4; ++k) pa[k] = pb[k] = 0x7F7F7F7Fu;
        }
        uint8_t* at = to + (lane >> 3) * Sh::kQBlock + r * 128 + (((lane & 7) ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>(at) = make_uint4(pa[0], pa[1], pa[2], pa[3]);
        *reinterpret_cast<uint4*>(at + kR * 128) = make_uint4(pb[0], pb[1], pb[2], pb[3]);
        if (lane < 8) {
          uint32_t y[4] = {now_pe.x, now_pe.y, now_pe.z, now_pe.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(y[k] << 16) * f,
                                                           __uint_as_float(y[k] & 0xFFFF0000u) * f);
            y[k] = *reinterpret_cast<const uint32_t*>(&h);
          }
          *reinterpret_cast<uint4*>(to + kParts * Sh::kQBlock + r * 128 + ((lane ^ (r & 7)) << 4)) =
              make_uint4(y[0], y[1], y[2], y[3]);
        }
        if (lane == 0) c_s[qb * kMostRows + r] = p.scale_log2 / f;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive_many(&q_full[qb], segs == 0 ? 1 : Sh::kFirstWarps / kQueryWarps);
      ++segs;
      if (helper || !more) break;
    }
  }

  if (!kSparse && warp == kLoadWarp) {
    // ------------------------------------------------------------ loads (dense)
    if (elect_one()) {
      int i = 0;
      int parts = 0;  // issued
      bool ok = true;
      while (ok && walk.next(s)) {
        const int32_t* row = p.block_table + static_cast<int64_t>(s.b) * p.max_pages;
        // A page outside of the pool or behind the tokens reads as zeros (a box
        // outside of the tensor is filled with them); its tokens are masked.
        auto page_at = [&](int x) {
          const int page = x * kPage < s.r.length ? row[x] : -1;
          return page < 0 || page >= p.num_pages ? p.num_pages : page;
        };
        int n0 = page_at(2 * s.t0), n1 = page_at(2 * s.t0 + 1);
        for (int t = s.t0; t < s.t1; ++t, ++i) {
          const int p0 = n0, p1 = n1;
          if (t + 1 < s.t1) {
            n0 = page_at(2 * t + 2);
            n1 = page_at(2 * t + 3);
          }
          const int st = i & 1;
          uint8_t* dst = smem + st * kStageBytes;
#pragma unroll
          for (int x = 0; x < kParts; ++x) {
            ok = ok && mbar_wait(&kv_free[st * kParts + x], ((i >> 1) & 1) ^ 1, wctx);
            if (!ok) break;
            uint64_t* bar = &kv_full[st * kParts + x];
            mbar_arrive_expect_tx(bar, x == 0 ? 2 * kBlockBytes + kTok * 4 : kBlockBytes);
            tma_load_3d(dst + x * kBlockBytes, &codes_map, bar, 128 * x, 0, p0);
            tma_load_3d(dst + x * kBlockBytes + kBlockBytes / 2, &codes_map, bar, 128 * x, 0, p1);
            // The position part and the scales with the first block: what read those of tile i - 2 was done before its O^T.
            if (x == 0) {
              tma_load_3d(dst + kParts * kBlockBytes, &kpe_map, bar, 0, 0, p0);
              tma_load_3d(dst + kParts * kBlockBytes + kBlockBytes / 2, &kpe_map, bar, 0, 0, p1);
              const uint8_t* s0 = p.cache + static_cast<int64_t>(p0 < p.num_pages ? p0 : 0) * kPageBytes + kScaleAt;
              const uint8_t* s1 = p.cache + static_cast<int64_t>(p1 < p.num_pages ? p1 : 0) * kPageBytes + kScaleAt;
              bulk_load(scale_s + st * kTok, s0, kPage * 4, bar);
              bulk_load(scale_s + st * kTok + kPage, s1, kPage * 4, bar);
            }
            ++parts;
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
      }
    }
    __syncwarp();
  } else if (warp == kLogitWarp) {
    // ------------------------------------------------------------ S^T and E^T
    if (elect_one()) {
      const uint64_t k_desc = sdesc_sw128(smem_u32(smem), 16, 1024);
      const uint64_t q_desc = sdesc_sw128(smem_u32(q_mem), 16, 1024);
      int i = 0, segs = 0;
      bool ok = true;
      while (ok && walk.next(s)) {
        const int qb = segs % Sh::kQBufs;
        const uint64_t bq = q_desc + qb * (Sh::kQBytes >> 4);
        for (int t = s.t0; t < s.t1; ++t, ++i) {
          const int st = i & 1, sb = i % Sh::kSBufs;
          const uint64_t a = k_desc + st * (kStageBytes >> 4);
          const uint32_t d = tmem_base + Sh::kColS + 3u * kR * sb;
          ok = mbar_wait(&s_empty[sb], ((i / Sh::kSBufs) & 1) ^ 1, wctx);
          if (t == s.t0) ok = ok && mbar_wait(&q_full[qb], (segs / Sh::kQBufs) & 1, wctx);
#pragma unroll
          for (int x = 0; x < kParts; ++x) {
            if (!kSparse || x == 0)
              ok = ok && mbar_wait(&kv_full[st * kParts + (kSparse ? kParts - 1 : x)], (i >> 1) & 1, wctx);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < 4; ++k)  // +32 bytes per K32 step
              umma_f8(d, a + x * (kBlockBytes >> 4) + 2 * k, bq + x * (Sh::kQBlock >> 4) + 2 * k, Sh::kIdescS,
                      x + k > 0 ? 1u : 0u);
            if (x == 0) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_bf16(d + 2u * kR, a + kParts * (kBlockBytes >> 4) + 2 * k, bq + kParts * (Sh::kQBlock >> 4) + 2 * k,
                          Sh::kIdescE, k > 0 ? 1u : 0u);
            }
          }
          if (!ok) break;
          umma_commit(&s_full[sb]);
          if (t == s.t1 - 1) umma_commit(&q_empty[qb]);
        }
        ++segs;
      }
      umma_commit(&drain[0]);
      mbar_drain(&drain[0], 0, p.status);
    }
    __syncwarp();
  } else if (warp == kValueWarp) {
    // ------------------------------------------------------------ O^T
    if (elect_one()) {
      const uint64_t v_desc = sdesc_sw128(smem_u32(smem), kBlockBytes, 1024);
      const uint64_t p_desc = sdesc_sw128(smem_u32(p_mem), kBlockBytes, 1024);
      int i = 0, segs = 0;
      bool ok = true;
      while (ok && walk.next(s)) {
        for (int t = s.t0; t < s.t1; ++t, ++i) {
          const int st = i & 1;
          if (t == s.t0) ok = mbar_wait(o_empty, (segs & 1) ^ 1, wctx);
          ok = ok && mbar_wait(p_full, i & 1, wctx);
          if (!ok) break;
          tc_fence_after();
          const uint32_t more = t == s.t0 ? 0u : 1u;
          const uint64_t a = v_desc + st * (kStageBytes >> 4);
#pragma unroll
          for (int mb = 0; mb < kParts; ++mb) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {  // a K32 step is 32 token rows of 128 bytes
              const uint32_t d = tmem_base + Sh::kColO + kColsO * mb;
              const uint64_t ak = a + mb * (kBlockBytes >> 4) + kk * (4096 >> 4), pk = p_desc + kk * (4096 >> 4);
              umma_f8(d, ak, pk, Sh::kIdescO, kk > 0 ? 1u : more);
              if (kR == 32) umma_f8(d, ak, pk + (kColsO >> 4), Sh::kIdescO, 1u);  // the rows' other 64 bytes
            }
            umma_commit(&kv_free[st * kParts + mb]);
          }
        }
        ++segs;
      }
      umma_commit(&drain[1]);
      mbar_drain(&drain[1], 0, p.status);
    }
    __syncwarp();
  } else if (kSparse && warp >= kGatherWarp) {
    // ------------------------------------------------------------ gather (sparse)
    // A group of warps for each stage; a warp copies 32 of its tile's tokens at a
    // time, 16 bytes a lane: a token's codes with one instruction, four position
    // parts with one.
    constexpr int kEach = Sh::kGatherWarps / 2, kTurns = kTok / 32 / kEach;
    const int group = (warp - kGatherWarp) / kEach, part = (warp - kGatherWarp) % kEach;
    int i = 0;
    bool ok = true;
    while (ok && walk.next(s)) {
      const int32_t* row = p.picked + static_cast<int64_t>(s.b) * p.topk;
      for (int t = s.t0; t < s.t1; ++t, ++i) {
        if ((i & 1) != group) continue;
        int slots[kTurns];
#pragma unroll
        for (int c = 0; c < kTurns; ++c) {
          const int pos = t * kTok + 32 * (part * kTurns + c) + lane;
          slots[c] = pos < p.topk ? row[pos] : -1;
          if (slots[c] < -1 || slots[c] >= p.num_pages * kPage) {
            atomicOr(p.status, DSA_DEV_BAD_INDEX);
            slots[c] = -1;
          }
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&kv_free[group * kParts + kParts - 1], ((i >> 1) & 1) ^ 1, wctx));
        if (!ok) break;
        const uint32_t to = smem_u32(smem + group * kStageBytes);
#pragma unroll
        for (int c = 0; c < kTurns; ++c) {
          const int first = 32 * (part * kTurns + c), slot = slots[c];
          auto page = [&](int x) { return p.cache + static_cast<int64_t>(max(x, 0) >> 6) * kPageBytes; };
#pragma unroll 8
          for (int n = 0; n < 32; ++n) {
            const int x = __shfl_sync(0xffffffffu, slot, n), r = first + n;
            cp_async16_or_zeros(to + (lane >> 3) * kBlockBytes + r * 128 + (((lane & 7) ^ (r & 7)) << 4),
                                page(x) + (max(x, 0) & 63) * kCkv + 16 * lane, x >= 0);
          }
#pragma unroll
          for (int n = 0; n < 32; n += 4) {
            const int x = __shfl_sync(0xffffffffu, slot, n + (lane >> 3)), r = first + n + (lane >> 3);
            cp_async16_or_zeros(to + kParts * kBlockBytes + r * 128 + (((lane & 7) ^ (r & 7)) << 4),
                                page(x) + kKpeAt + (max(x, 0) & 63) * (kKpe * 2) + 16 * (lane & 7), x >= 0);
          }
          cp_async4_or_zeros(smem_u32(scale_s + group * kTok + first + lane),
                             page(slot) + kScaleAt + 4 * (max(slot, 0) & 63), slot >= 0);
        }
        cp_async_wait_all();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kv_full[group * kParts + kParts - 1]);
      }
    }
  } else if (warp < kSoftWarps) {
    // ------------------------------------------------------------ softmax
    // Set `set` of four warps has the columns C set .. C set + C - 1 (rows of Q); in
    // it thread (sp, lane) has token 32 sp + lane.
    const int set = warp >> 2, sp = warp & 3;
    const int tok = 32 * sp + lane;
    const uint32_t lane_base = static_cast<uint32_t>(32 * sp) << 16;
    const int e = tid & 127;  // thread of the set
    float* red_set = red + 4 * C * set;  // [4][C]
    float* my_max = max_s + C * set;
    float* my_minus = minus_s + C * set;  // -m, or 0 where m is -inf
    float* my_factor = factor_s + C * set;
    int* group_of = p.plan + 2 * blockIdx.x;  // of this CTA's records
    if (!kTogether && tid == 0) group_of[0] = group_of[1] = -1;
    int i = 0, segs = 0;
    bool ok = true;
    // Online softmax in base 2.  A weight by its scale is 2^(x - m) s, and what a
    // column's reference m follows is that product, not the logit alone: m is the
    // running maximum of x + log2(s / ref), ref the power of two of the largest scale
    // in the segment's first tile.  So the column's largest product is kUnit or more,
    // and no token takes from the others' precision but by its own weight (with maxima
    // of x and s apart, a token of a scale 2^24 times the others' and no weight left
    // them 3 bits).  The sums l of 2^(x - m), in 32 bits, need no such reference: scales
    // within 2^60 of ref cannot drive them out of the range.  Smaller ones (zeros
    // among them) count as 2^-60 in m, larger ones move ref.
    // m (-inf: the column has seen nothing; +inf: no row of the group, all weights 0)
    // is the same in every thread that has the column.  It moves only when some token
    // of the tile exceeds it by more than kRescaleThreshold (always at a segment's
    // first tile), which one OR-barrier per tile tells the set; only then is the
    // tile's max reduced over the tokens and O rescaled.
    for (;;) {
      const int qb = segs % Sh::kQBufs;
      ok = ok && mbar_wait(&q_full[qb], (segs / Sh::kQBufs) & 1, wctx);
      // All warps of the set leave together.
      if (!named_barrier_and(1 + set, 128, ok)) break;
      const SegmentInfo& seg = info_s[segs & 3];
      const int t0 = seg.t0, t1 = seg.t1, rows = seg.rows, length = seg.length;
      if (t0 == t1) break;
      float l[C];
      bool unset = C * set < rows;  // some column has seen nothing yet
      float ref = 0.f, by_ref = 0.f;
      if (e < C) {
        my_max[e] = C * set + e < rows ? -INFINITY : INFINITY;
        my_minus[e] = C * set + e < rows ? 0.f : -INFINITY;
      }
      // The power of two at or below the tile's largest scale of those that count (the set waits for one another).
      auto unit_of_tile = [&](float scale, bool counts) {
        const uint32_t largest = __reduce_max_sync(0xffffffffu, counts ? __float_as_uint(fabsf(scale)) : 0u);
        if (lane == 0) most_s[4 * set + sp] = __uint_as_float(largest);
        named_barrier_sync(1 + set, 128);
        const float4 m4 = *reinterpret_cast<const float4*>(most_s + 4 * set);
        const float largest4 = fmaxf(fmaxf(m4.x, m4.y), fmaxf(m4.z, m4.w));
        return fmaxf(__uint_as_float(__float_as_uint(largest4) & 0x7F800000u), kLeastRef);
      };
      // log2(s / ref) of a scale in units (s kUnit / ref).
      auto log_of = [](float by) { return fmaxf(lg2_approx(fabsf(by)) - kUnitLog2, -kScaleRange); };
      const float* my_c = c_s + qb * kMostRows + C * set;
#pragma unroll
      for (int k = 0; k < C; ++k) l[k] = 0.f;
      const int sure = length - seg.n + 1;  // tokens that every row sees
      const int32_t* bt = kSparse ? p.picked + static_cast<int64_t>(seg.b) * p.topk
                                  : p.block_table + static_cast<int64_t>(seg.b) * p.max_pages;
      // Dense: the token's page; sparse: its slot.  -1 behind the context.
      auto place = [&](int t) {
        const int pos = t * kTok + tok;
        return pos < length ? bt[kSparse ? pos : pos / kPage] : -1;
      };
      const int places = kSparse ? p.num_pages * kPage : p.num_pages;
      int next_place = place(t0);
      for (int t = t0; t < t1; ++t, ++i) {
        const int st = i & 1, sb = i % Sh::kSBufs;
        const int pos = t * kTok + tok;
        const int at_place = next_place;
        if (t + 1 < t1) next_place = place(t + 1);
        const bool hidden = at_place < 0 || at_place >= places;  // seen by no row
        const bool tail = !kSparse && (t + 1) * kTok > sure;
        if (!kSparse && hidden && pos < length && (e & 63) == 0) atomicOr(p.status, DSA_DEV_BAD_PAGE);
        ok = ok && mbar_wait(&kv_full[st * kParts + (kSparse ? kParts - 1 : 0)], (i >> 1) & 1, wctx);
        const float scale = scale_s[st * kTok + tok];
        // A scale that is no number has made the token's logits NaN, and with them l, where it is seen; it counts as 0 here.
        bool counts = !hidden && fabsf(scale) < INFINITY;
        if (t == t0) {  // (while S^T is computed)
          ref = unit_of_tile(scale, counts);
          by_ref = kUnit / ref;
        }
        float by = counts ? scale * by_ref : 0.f, log_by = log_of(by);
        ok = ok && mbar_wait(&s_full[sb], (i / Sh::kSBufs) & 1, wctx);
        tc_fence_after();
        float x[C];  // logits
        {
          float b[C], pe[C], c[C];
          load_cols(my_c, c);
          const uint32_t at = tmem_base + lane_base + Sh::kColS + 3u * kR * sb + C * set;
          tmem_ld_three(at, at + kR, at + 2 * kR, x, b, pe);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[sb]);
#pragma unroll
          for (int k = 0; k < C; ++k) x[k] = fmaf(fmaf(b[k], 0.0625f, x[k]), scale, pe[k]) * c[k];
        }
        if (t == t1 - 1) {  // the queries' factors have been read
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_empty[qb]);
        }
        if (__any_sync(0xffffffffu, hidden || (tail && pos >= sure))) {
          int row = seg.group * kR + C * set;
          int draft = row / p.heads, left = (draft + 1) * p.heads - row;
#pragma unroll
          for (int k = 0; k < C; ++k) {
            if (hidden || (tail && pos >= sure + draft)) x[k] = -INFINITY;
            if (--left == 0) {
              ++draft;
              left = p.heads;
            }
          }
        }
        float d[C];
        load_cols(my_minus, d);
#pragma unroll
        for (int k = 0; k < C; ++k) d[k] += x[k];
        float most = fmaxf(d[0], d[1]);
#pragma unroll
        for (int k = 2; k < C; k += 2) most = fmaxf(most, fmaxf(d[k], d[k + 1]));
        if (named_barrier_or(1 + set, 128,
                             unset || most + log_by > kRescaleThreshold || log_by > kScaleRange)) {
          // A row of zeros has no weight, whatever its scale; those that are written here have 1, which may be
          // far above the scales of small latents.
          if (__any_sync(0xffffffffu, counts && scale == 1.f)) {
#pragma unroll
            for (int y = 0; y < kParts; ++y)
              if (!kSparse || y == kParts - 1) ok = ok && mbar_wait(&kv_full[st * kParts + y], (i >> 1) & 1, wctx);
            if (counts && scale == 1.f) {
              const uint8_t* codes = smem + st * kStageBytes + tok * 128;
              uint32_t any = 0u;
#pragma unroll 1
              for (int q = 0; q < 32; ++q) {
                const uint4 w = *reinterpret_cast<const uint4*>(codes + (q >> 3) * kBlockBytes + (q & 7) * 16);
                any |= (w.x | w.y) | (w.z | w.w);
              }
              if ((any & 0x7F7F7F7Fu) == 0u) {
                counts = false;
                by = 0.f;
                log_by = -kScaleRange;
              }
            }
          }
          int col;
          auto tile_maxima = [&]() {
            float v[C];
#pragma unroll
            for (int k = 0; k < C; ++k) v[k] = x[k] + log_by;
            // (fmaxf passes over NaN, which moves no maximum.)
            const float mt = over_tokens(v, lane, col, [](float a, float b) { return fmaxf(a, b); });
            red_set[C * sp + col] = mt == mt ? mt : -INFINITY;
          };
          tile_maxima();
          float shrink = 1.f;
          if (named_barrier_or(1 + set, 128, log_by > kScaleRange)) {
            const float now = unit_of_tile(scale, counts);
            shrink = ref / now;
            ref = now;
            by_ref = kUnit / now;
            by = counts ? scale * by_ref : 0.f;
            log_by = log_of(by);
            tile_maxima();
            named_barrier_sync(1 + set, 128);
          }
          if (sp == 0) {
            const float mt = fmaxf(fmaxf(red_set[col], red_set[C + col]), fmaxf(red_set[2 * C + col], red_set[3 * C + col]));
            const float m = my_max[col];
            const bool moves = mt > m + kRescaleThreshold;
            __syncwarp();
            const float now = moves ? mt : m;
            my_max[col] = now;
            my_minus[col] = now == -INFINITY ? 0.f : -now;
            my_factor[col] = moves ? ex2_approx(m - mt) : 1.f;  // 0 when m was -inf
          }
          named_barrier_sync(1 + set, 128);
          float alpha[C];
          load_cols(my_max, alpha);
          unset = false;
#pragma unroll
          for (int k = 0; k < C; ++k) unset |= alpha[k] == -INFINITY;
          load_cols(my_factor, alpha);
          load_cols(my_minus, d);
#pragma unroll
          for (int k = 0; k < C; ++k) {
            l[k] *= alpha[k];
            alpha[k] *= shrink;
            d[k] += x[k];
          }
          if (t > t0) {
            // O holds PV(i - 1) before it is rescaled.
            ok = ok && mbar_wait(pv_done(i - 1), ((i - 1) >> 1) & 1, wctx);
            tc_fence_after();
#pragma unroll 1
            for (int mb = 0; mb < kParts; ++mb) {
              const uint32_t at = tmem_base + lane_base + Sh::kColO + kColsO * mb + C * set;
              float o[Sh::kSums][C];
              tmem_ld_sums(at, o);
#pragma unroll
              for (int x = 0; x < Sh::kSums; ++x) {
#pragma unroll
                for (int k = 0; k < C; ++k) o[x][k] *= alpha[k];
                tmem_st(at + kR * x, o[x]);
              }
            }
            tmem_wait_st();
          }
        }
        if (tail) {
          // Tokens that some row does not see may hold anything; a zero weight
          // would still turn a NaN code of theirs into NaN.  Their logits have
          // been read (S^T is done), so such codes are zeroed; a row that does
          // see one has its NaN from the logit.
#pragma unroll
          for (int y = 0; y < kParts; ++y) ok = ok && mbar_wait(&kv_full[st * kParts + y], (i >> 1) & 1, wctx);
          const int from = max(sure - t * kTok, 0);
          for (int q = tid; q < (kTok - from) * 32; q += 32 * kSoftWarps) {
            uint4* at = reinterpret_cast<uint4*>(smem + st * kStageBytes + ((q >> 3) & 3) * kBlockBytes +
                                                 (from + (q >> 5)) * 128 + (q & 7) * 16);
            uint4 w = *at;
            uint32_t* ww = reinterpret_cast<uint32_t*>(&w);
            bool changed = false;
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const uint32_t nan = ((ww[z] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
              ww[z] &= ~((nan >> 7) * 0xFFu);
              changed |= nan != 0u;
            }
            if (changed) *at = w;
          }
        }
        // Weights (of d = -inf, 0; NaN stays), and their products with the scale in
        // four parts.
        uint2 part[C / 8][4];
#pragma unroll
        for (int k = 0; k < C; ++k) {
          d[k] = ex2_approx(d[k]);
          l[k] += d[k];
          d[k] *= by;
        }
#pragma unroll
        for (int k = 0; k < C / 8; ++k) in_parts(d + 8 * k, part[k]);
        // P was last read by PV(i - 1).
        if (i > 0) ok = ok && mbar_wait(pv_done(i - 1), ((i - 1) >> 1) & 1, wctx);
        {
          // One 128-byte row per token: column n of part x at byte x R + n, 16-byte pieces swizzled by token & 7.
          uint8_t* at = p_mem + tok * 128;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int byte = kR * x + C * set;
            uint8_t* to = at + (((byte >> 4) ^ (tok & 7)) << 4) + (byte & 8);
            if constexpr (C == 16)
              *reinterpret_cast<uint4*>(to) = make_uint4(part[0][x].x, part[0][x].y, part[1][x].x, part[1][x].y);
            else
              *reinterpret_cast<uint2*>(to) = part[0][x];
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
      }
      ++segs;

      // ---- the segment's end: denominators over the tokens (while the last PV
      // runs), then O.
      {
        int col;
        const float sum = over_tokens(l, lane, col, [](float a, float b) { return a + b; });
        red_set[C * sp + col] = sum;
      }
      named_barrier_sync(1 + set, 128);
      const int64_t row_q = seg.row_q;
      const int64_t rec = static_cast<int64_t>(blockIdx.x) * 2 + seg.slot;
      if (!kTogether && tid == 0 && !seg.whole) group_of[seg.slot] = seg.group_index;
      if (e < C) {
        const int col = C * set + e;
        const float sum = (red_set[e] + red_set[C + e]) + (red_set[2 * C + e] + red_set[3 * C + e]);
        // A piece is normalised too: its sum of scaled codes alone could leave the range.
        factor_s[col] = sum == 0.f ? 0.f : ref * (1.f / kUnit) / sum;
        if (!seg.whole)
          (kTogether ? together_ml : p.part_ml + rec * kMostRows)[col] = make_float2(max_s[col], sum);
        else if (col < rows)
          p.lse[row_q + col] = sum == 0.f ? -INFINITY : max_s[col] + log2f(sum);
      }
      ok = ok && mbar_wait(pv_done(i - 1), ((i - 1) >> 1) & 1, wctx);
      named_barrier_sync(1 + set, 128);
      tc_fence_after();
#pragma unroll 1
      for (int mb = 0; mb < kParts; ++mb) {
        const int dim = 128 * mb + 32 * sp + lane;
        float o[C];
        {
          float sums[Sh::kSums][C];
          tmem_ld_sums(tmem_base + lane_base + Sh::kColO + kColsO * mb + C * set, sums);
#pragma unroll
          for (int k = 0; k < C; ++k) o[k] = whole_sum(sums, k) * factor_s[C * set + k];
        }
        if (seg.whole) {
          // Neighbouring lanes swap halves, so that each stores two dims of one row.
          const bool odd = lane & 1;
          __nv_bfloat16* out = p.out + row_q * kCkv + (dim & ~1);
#pragma unroll
          for (int k = 0; k < C; k += 2) {
            const float got = __shfl_xor_sync(0xffffffffu, odd ? o[k] : o[k + 1], 1);
            const int row = C * set + k + (odd ? 1 : 0);
            if (row < rows)
              *reinterpret_cast<__nv_bfloat162*>(out + static_cast<int64_t>(row) * kCkv) =
                  odd ? __floats2bfloat162_rn(got, o[k + 1]) : __floats2bfloat162_rn(o[k], got);
          }
        } else {
          float* to = (kTogether ? together_o : p.part_o + rec * kPartFloats) + C * set * kCkv + dim;
#pragma unroll
          for (int k = 0; k < C; ++k)
            if (C * set + k < rows) to[k * kCkv] = o[k];
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_empty);
    }
  }

  tc_fence_before();
  if constexpr (kTogether)
    cluster_sync();
  else
    __syncthreads();
  if (warp == kLogitWarp) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
  if constexpr (kTogether) {
    // The pieces as join_kernel joins records, in the order of the ranks; a CTA has
    // its share of the rows' 16-byte pieces.
    const int tiles = cluster < total ? found->r.tiles : 0, share = each_of(tiles);
    if (share < tiles) {  // else written whole
      const Start& st = *found;
      const int rows = min(kR, st.r.rows - st.group * kR);
      const int64_t row_q = static_cast<int64_t>(st.r.row0) * p.heads + st.group * kR;
      const int all = rows * (kCkv / 4), each = each_of(all);
      const uint32_t o_at = smem_u32(together_o), ml_at = smem_u32(together_ml);
      for (int x = rank * each + tid; x < min((rank + 1) * each, all); x += kThreads) {
        const int y = x / (kCkv / 4), d4 = x % (kCkv / 4);
        float2 ml[kMostTogether];
        float4 o[kMostTogether];
#pragma unroll
        for (int k = 0; k < kMostTogether; ++k) ml[k] = ld_cluster_or_zeros(ml_at + y * 8, k, k * share < tiles);
#pragma unroll
        for (int k = 0; k < kMostTogether; ++k) o[k] = ld_cluster4_or_zeros(o_at + x * 16, k, k * share < tiles);
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int k = 0; k < kMostTogether; ++k) {
          if (k * share >= tiles) ml[k].x = -INFINITY;
          M = fmaxf(M, ml[k].x);
        }
#pragma unroll
        for (int k = 0; k < kMostTogether; ++k) {
          ml[k].y = ml[k].x == -INFINITY ? (ml[k].y == ml[k].y ? 0.f : ml[k].y) : ml[k].y * exp2f(ml[k].x - M);
          L += ml[k].y;
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < kMostTogether; ++k) {
          const float w = ml[k].y * inv;
          acc.x = fmaf(o[k].x, w, acc.x);
          acc.y = fmaf(o[k].y, w, acc.y);
          acc.z = fmaf(o[k].z, w, acc.z);
          acc.w = fmaf(o[k].w, w, acc.w);
        }
        const __nv_bfloat162 h[2] = {__floats2bfloat162_rn(acc.x, acc.y), __floats2bfloat162_rn(acc.z, acc.w)};
        *reinterpret_cast<uint2*>(p.out + (row_q + y) * kCkv + 4 * d4) = *reinterpret_cast<const uint2*>(h);
        if (d4 == 0) p.lse[row_q + y] = L == 0.f ? -INFINITY : M + log2f(L);
      }
    }
    cluster_sync();  // no CTA leaves while another reads its piece
  }
}

// Joins the records of a group that several slices share: per row
//   M = max m_i, w_i = l_i 2^(m_i - M), L = sum w_i, lse = M + log2 L, out = sum O_i w_i / L,
// in an order that the slices alone give.  Block x has the group x, or where
// groups outnumber records the group of record x if x is its first one; block y
// its rows y * rows_per_block ...  Each kSplit-th of the block takes every
// kSplit-th record of a row, a thread four dims, many loads in flight.
constexpr int kJoinRows = 4;       // most rows per block
constexpr int kJoinDepth = 8;      // records whose loads a thread has in flight
constexpr int kJoinFew = 4;        // records of a row that are loaded for all of the block's rows at once

template <int kSplit>
__global__ void __launch_bounds__(128 * kSplit)
join_kernel(const Params p, int ctas, int rows_per_block, bool by_record) {
  griddep_wait();
  constexpr int kThreads = 128 * kSplit;
  constexpr int kLooks = 2 * kMaxCtas / kThreads;  // records a thread looks at
  __shared__ int recs[2 * kMaxCtas];
  __shared__ float weight[kJoinRows][2 * kMaxCtas];
  __shared__ int warp_count[kLooks][kThreads / 32];
  __shared__ float4 other[kSplit > 1 ? kSplit - 1 : 1][kCkv / 4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int x = blockIdx.x;
  const int group = by_record ? __ldcg(p.plan + x) : x;
  int mine[kLooks];
#pragma unroll
  for (int k = 0; k < kLooks; ++k) {
    const int r = tid + k * kThreads;
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
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) at += warp_count[k][w];
      count += warp_count[k][w];
    }
    if (mine[k] == group) recs[at] = tid + k * kThreads;
  }
  __syncthreads();
  if (count == 0 || (by_record && recs[0] != x)) return;  // written whole; or another block's
  const int y0 = blockIdx.y * rows_per_block;
  const int rows = min(rows_per_block, info.y - y0);
  if (rows <= 0) return;
  // The loads that need no weights go first: all rows' where they have few
  // records, or the first records of the first row.
  const int part = tid >> 7, d4 = tid & 127;
  const float4* src = reinterpret_cast<const float4*>(p.part_o) + y0 * (kCkv / 4) + d4;
  constexpr int kHeld = kSplit == 1 ? kJoinRows * kJoinFew : kJoinDepth;
  static_assert(kHeld >= kJoinDepth, "loads");
  const bool few = kSplit == 1 && count <= kJoinFew;
  float4 v[kHeld];
  auto load = [&](int k0) {
#pragma unroll
    for (int j = 0; j < kJoinDepth; ++j)
      if (k0 + kSplit * j < count)
        v[j] = __ldcg(src + static_cast<int64_t>(recs[k0 + kSplit * j]) * (kPartFloats / 4));
  };
  if (few) {
#pragma unroll
    for (int k = 0; k < kJoinFew; ++k) {
      if (k < count) {
        const float4* from = src + static_cast<int64_t>(recs[k]) * (kPartFloats / 4);
#pragma unroll
        for (int y = 0; y < kHeld / kJoinFew; ++y)
          if (y < rows) v[y * kJoinFew + k] = __ldcg(from + y * (kCkv / 4));
      }
    }
  } else {
    load(part);
  }
  for (int y = warp; y < rows; y += kThreads / 32) {
    float M = -INFINITY, L = 0.f;
    const float2* ml = p.part_ml + y0 + y;
    float2 first = make_float2(-INFINITY, 0.f);  // of the lane's first record
    for (int k = lane; k < count; k += 32) {
      const float2 q = __ldcg(&ml[static_cast<int64_t>(recs[k]) * kMostRows]);
      if (k == lane) first = q;
      M = fmaxf(M, q.x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    for (int k = lane; k < count; k += 32) {
      const float2 q = k == lane ? first : __ldcg(ml + static_cast<int64_t>(recs[k]) * kMostRows);
      // NaN sums have a place even where the max of what is left of a piece is -inf.
      const float w = q.x == -INFINITY ? (q.y == q.y ? 0.f : q.y) : q.y * exp2f(q.x - M);
      L += w;
      weight[y][k] = w;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    __syncwarp();
    for (int k = lane; k < count; k += 32) weight[y][k] *= inv;
    if (lane == 0) p.lse[info.x + y0 + y] = L == 0.f ? -INFINITY : M + log2f(L);
  }
  __syncthreads();
  auto add = [](float4& acc, const float4& x, float w) {
    acc.x = fmaf(x.x, w, acc.x);
    acc.y = fmaf(x.y, w, acc.y);
    acc.z = fmaf(x.z, w, acc.z);
    acc.w = fmaf(x.w, w, acc.w);
  };
  auto store = [&](const float4& acc, int y) {
    const __nv_bfloat162 h[2] = {__floats2bfloat162_rn(acc.x, acc.y), __floats2bfloat162_rn(acc.z, acc.w)};
    *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(info.x) + y0 + y) * kCkv + 4 * d4) =
        *reinterpret_cast<const uint2*>(h);
  };
  if (few) {
#pragma unroll
    for (int y = 0; y < kHeld / kJoinFew; ++y) {
      if (y < rows) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < kJoinFew; ++k)
          if (k < count) add(acc, v[y * kJoinFew + k], weight[y][k]);
        store(acc, y);
      }
    }
    return;
  }
  for (int y = 0; y < rows; ++y) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = part; k0 < count; k0 += kSplit * kJoinDepth) {
      if (y > 0 || k0 > part) load(k0);
#pragma unroll
      for (int j = 0; j < kJoinDepth; ++j)
        if (k0 + kSplit * j < count) add(acc, v[j], weight[y][k0 + kSplit * j]);
    }
    src += kCkv / 4;
    if (kSplit > 1) {
      if (part > 0) other[part - 1][d4] = acc;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kSplit - 1; ++k)
        if (part == 0) add(acc, other[k][d4], 1.f);
      __syncthreads();
    }
    if (part == 0) store(acc, y);
  }
}

// ------------------------------------------------------------------ host
std::once_flag g_once[64];
int g_status[64];
constexpr int kTogetherSizes = 4;       // clusters of 8, 4, 2 and 1 CTAs
int g_clusters[64][kTogetherSizes];     // of each size, how many run at once

struct Layout {
  size_t part_ml, part_o, plan, bytes;
};

// Upper bound of the groups of R rows of all requests.
inline int64_t groups_bound(int64_t rows, int64_t heads, int64_t requests, int r) { return rows * heads / r + requests; }

// The same for every call that is accepted, so that a workspace never has to
// move (a captured graph would go on using the old one).
inline Layout layout(int sms) {
  Layout a;
  a.part_ml = kWorkspaceHeader;
  a.part_o = a.part_ml + static_cast<size_t>(2 * sms) * kMostRows * sizeof(float2);
  a.plan = a.part_o + static_cast<size_t>(2 * sms) * kPartFloats * sizeof(float);
  a.bytes = a.plan + (kPlanGroups + 2 * static_cast<size_t>(groups_bound(kMaxRows, 1, kMaxRequests, 16))) * sizeof(int);
  return a;
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

cudaLaunchConfig_t together_config(bool sparse, unsigned int grid, int ctas, cudaLaunchAttribute (&attr)[2]) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(sparse ? Shape<16, true>::kThreads : Shape<16, false>::kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned int>(ctas);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cfg;
}

int setup(const DeviceInfo& info) {
  if (static_cast<size_t>(kSmemBytes) > info.max_smem_optin || info.num_sms > kMaxCtas) return DSA_ERR_UNSUPPORTED_DEVICE;
  std::call_once(g_once[info.device], [&]() {
    auto large = [](const void* f) {
      return cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) == cudaSuccess;
    };
    const void* all[] = {reinterpret_cast<const void*>(attend_kernel<16, false, false>),
                         reinterpret_cast<const void*>(attend_kernel<32, false, false>),
                         reinterpret_cast<const void*>(attend_kernel<16, true, false>),
                         reinterpret_cast<const void*>(attend_kernel<32, true, false>),
                         reinterpret_cast<const void*>(attend_kernel<16, false, true>),
                         reinterpret_cast<const void*>(attend_kernel<16, true, true>)};
    g_status[info.device] = DSA_OK;
    for (const void* f : all)
      if (!large(f)) g_status[info.device] = DSA_ERR_CUDA;
    for (int x = 0; x < kTogetherSizes && g_status[info.device] == DSA_OK; ++x) {
      const int ctas = kMostTogether >> x;
      cudaLaunchAttribute attr[2];
      int dense = 0, sparse = 0;
      cudaLaunchConfig_t cfg = together_config(false, ctas, ctas, attr);
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&dense, attend_kernel<16, false, true>, &cfg) != cudaSuccess)
        g_status[info.device] = DSA_ERR_CUDA;
      cfg.blockDim = dim3(Shape<16, true>::kThreads);
      if (cudaOccupancyMaxActiveClusters(&sparse, attend_kernel<16, true, true>, &cfg) != cudaSuccess)
        g_status[info.device] = DSA_ERR_CUDA;
      g_clusters[info.device][x] = dense < sparse ? dense : sparse;
    }
  });
  return g_status[info.device];
}

// Upper bound of the groups of R rows of a call: with one row for each request
// (all of sparse calls) what they are.
int64_t most_groups(const Params& p, int r) {
  return p.cu == nullptr ? static_cast<int64_t>(p.num_rows) * ((p.heads + r - 1) / r)
                         : (static_cast<int64_t>(p.num_rows) * p.heads + static_cast<int64_t>(p.num_requests) * (r - 1)) / r;
}

// CTAs of the clusters that have a group of 16 rows each, or 0: slices.  Clusters,
// as large as all groups' fit at once (15 of 8 CTAs, 33 of 4, 74 of 2, 148 of 1),
// have no second launch, no records and no join (3.5 us and more on the device,
// 3.5 on the host); slices even out what they have to do.  So clusters are taken
// where a CTA has four tiles at most, and at most two and a half more than a slice
// would (two where slots are gathered).  Their number is bounded by the width of
// the table, which is what the host knows; lengths well below it lose little, as
// a CTA's tiles end with its group's.  Graph replays in us, slices against clusters:
//   requests of one row of 16 heads x tokens: 1 x 128 9.3 and 8.1, 1 x 1024 11.1 and
//   9.3, 1 x 4096 (not taken) 12.2 and 13.1; 14 x 2048 14.5 and 11.7; 16 x 4096 (not
//   taken) 17.8 and 19.9; 32 x 1024 15.3 and 12.7; 128 x 512 20.1 and 14.2
//   1 x 1024 of four rows 14.3 and 9.5, of 128 heads 14.8 and 10.1; 16 x 300 of 128
//   heads 21.3 and 13.2; 4 x 4096 of 128 (not taken) 21.0 and 20.3
//   rows of 2048 selected slots of 16 heads: 1 11.1 and 10.8, 5 12.1 and 10.9, 14 13.8
//   and 11.6, 16 (not taken) 13.7 and 14.8, 32 18.9 and 16.6
// Sixteen CTAs (7 such clusters run at once) joined slower than they saved.
int together_for(const Params& p, const DeviceInfo& info) {
  const int64_t groups = most_groups(p, 16);
  const int64_t tiles = p.picked != nullptr ? (p.topk + kTok - 1) / kTok : (p.max_pages + 1) / 2;
  int turn = 0;
  while (turn < kTogetherSizes && groups > g_clusters[info.device][turn]) ++turn;
  if (turn == kTogetherSizes) return 0;
  const int ctas = kMostTogether >> turn;
  const int64_t each = (tiles + ctas - 1) / ctas, slice = groups * (tiles + kLead<16>);
  return each <= 4 && 2 * (each * info.num_sms - slice) <= (p.picked != nullptr ? 4 : 5) * info.num_sms ? ctas : 0;
}

// The attention and its join; `p` without what the workspace gives.
int launch(Params& p, const DeviceInfo& info, bool wide, void* workspace, cudaStream_t s) {
  CUtensorMap maps[2] = {};
  const bool sparse = p.picked != nullptr;
  if (!sparse) {
    int st = encode_tmap_3d(&maps[0], CU_TENSOR_MAP_DATA_TYPE_UINT8, p.cache, kCkv, kPage, p.num_pages, kCkv, kPageBytes,
                            128, kPage);
    if (st != DSA_OK) return st;
    st = encode_tmap_3d(&maps[1], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.cache + kKpeAt, kKpe, kPage, p.num_pages, kKpe * 2,
                        kPageBytes, kKpe, kPage);
    if (st != DSA_OK) return st;
  }
  const int together = together_for(p, info);
  const Layout a = layout(info.num_sms);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.status = reinterpret_cast<unsigned int*>(ws);
  p.wait_limit_ns = kWaitLimitNs;
  p.by_ctas = 1.0 / info.num_sms;
  p.part_ml = reinterpret_cast<float2*>(ws + a.part_ml);
  p.part_o = reinterpret_cast<float*>(ws + a.part_o);
  p.plan = reinterpret_cast<int*>(ws + a.plan);
  const std::lock_guard<std::mutex> turn(turn_of(workspace));  // the attention and its join share the records
  if (together > 0) {
    // All groups of 16, and the most tiles one can have.
    const int64_t groups = most_groups(p, 16);
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = together_config(sparse, static_cast<unsigned int>(groups * together), together, attr);
    cfg.stream = s;
    const cudaError_t e = sparse ? cudaLaunchKernelEx(&cfg, attend_kernel<16, true, true>, maps[0], maps[1], p)
                                 : cudaLaunchKernelEx(&cfg, attend_kernel<16, false, true>, maps[0], maps[1], p);
    return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? DSA_OK : DSA_ERR_CUDA;
  }
  auto go = [&](auto kernel, int threads) {
    return launch_programmatic(kernel, dim3(info.num_sms), dim3(threads), kSmemBytes, s, maps[0], maps[1], p);
  };
  const cudaError_t err = sparse && wide ? go(attend_kernel<32, true, false>, Shape<32, true>::kThreads)
                          : sparse       ? go(attend_kernel<16, true, false>, Shape<16, true>::kThreads)
                          : wide         ? go(attend_kernel<32, false, false>, Shape<32, false>::kThreads)
                                         : go(attend_kernel<16, false, false>, Shape<16, false>::kThreads);
  if (err != cudaSuccess) return DSA_ERR_CUDA;
  const int r = wide ? 32 : 16;
  const int64_t groups = most_groups(p, r);
  const bool by_record = groups > 2 * info.num_sms;
  const unsigned int across = static_cast<unsigned int>(by_record ? 2 * info.num_sms : groups);
  const int rows = across <= 32 ? 1 : (across <= 96 ? 2 : kJoinRows);
  const bool deep = across <= 10;
  if (launch_programmatic(deep ? join_kernel<4> : join_kernel<1>, dim3(across, r / rows), dim3(deep ? 512 : 128), 0, s, p,
                          info.num_sms, rows, by_record) != cudaSuccess ||
      cudaGetLastError() != cudaSuccess)
    return DSA_ERR_CUDA;
  return DSA_OK;
}

}  // namespace qattn
}  // namespace dsa

using namespace dsa;

extern "C" size_t dsa_latent_attention_workspace_bytes(void) {
  DeviceInfo info;
  // Without a usable device, size for the largest SM count of the family.
  const int sms = current_device_info(&info) == DSA_OK ? info.num_sms : 160;
  return qattn::layout(sms).bytes;
}

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
  if (qattn::groups_bound(num_rows, num_heads, num_requests, 16) * (max_pages / 2 + 1 + qattn::kMostLead) > qattn::kMaxUnits)
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
  if ((st = qattn::setup(info)) != DSA_OK) return st;
  if (workspace_bytes < qattn::layout(info.num_sms).bytes) return DSA_ERR_WORKSPACE_TOO_SMALL;
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
  // Groups of 16 rows or 32: 32 where requests have more than 16 rows on average, since a group reads the whole context.
  // Graph replays in us, 16 rows against 32: 64 x 1000-3000 tokens of two rows of 16 heads 37.2 and 34.1, of 64 x 300-900
  // of four 32.6 and 28.4, of 64 x 1000-3000 of one row of 24 heads 36.7 and 35.0, of one row of 128 heads and 64 x
  // 500-1500 tokens 63.3 and 54.0.
  const bool wide = static_cast<int64_t>(num_rows) * num_heads > 16 * static_cast<int64_t>(num_requests);
  return qattn::launch(p, info, wide, workspace, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int dsa_latent_sparse_attention_run(const void* q_nope, const void* q_pe, const void* latent_cache,
                                               int64_t num_pages, const int32_t* sparse_indices, int32_t num_rows,
                                               int32_t num_heads, int32_t topk, float sm_scale, void* output, float* lse,
                                               void* workspace, size_t workspace_bytes, void* stream) {
  if (num_rows < 0 || num_heads < 1 || num_heads > 128 || static_cast<int64_t>(num_rows) * num_heads > qattn::kMaxRows ||
      topk < 1 || topk > 65536)
    return DSA_ERR_INVALID_ARGUMENT;
  const int64_t groups = static_cast<int64_t>(num_rows) * ((num_heads + 15) / 16);
  static_assert(qattn::kMaxRows / 16 * (65536 / qattn::kTok + qattn::kMostLead) <= qattn::kMaxUnits, "units");
  if (groups > qattn::kMaxRows / 16) return DSA_ERR_INVALID_ARGUMENT;
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
  if ((st = qattn::setup(info)) != DSA_OK) return st;
  if (workspace_bytes < qattn::layout(info.num_sms).bytes) return DSA_ERR_WORKSPACE_TOO_SMALL;
  qattn::Params p{};
  p.q_nope = static_cast<const __nv_bfloat16*>(q_nope);
  p.q_pe = static_cast<const __nv_bfloat16*>(q_pe);
  p.cache = static_cast<const uint8_t*>(latent_cache);
  p.num_pages = static_cast<int>(num_pages);
  p.picked = sparse_indices;
  p.topk = topk;
  p.num_requests = num_rows;
  p.num_rows = num_rows;
  p.heads = num_heads;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.out = static_cast<__nv_bfloat16*>(output);
  p.lse = lse;
  // Groups of 16 heads or 32: 32 where a row has more than 16 and groups of 16 make more than 8 tiles an SM.  A group
  // gathers its row's slots anew; where there are few, the shorter start and end of 16 win.  Graph replays in us, 16
  // against 32, 2048 slots, rows x heads (tiles an SM at 16): 16 x 64 (6.9) 25.2 and 25.4, 8 x 128 (6.9) 24.8 and 24.9,
  // 64 x 24 (14) 45.1 and 42.0, 64 x 32 (14) 45.6 and 43.8, 64 x 64 (28) 76.5 and 63.4, 64 x 128 (55) 133.3 and 109.2,
  // 256 x 32 (55) 146.7 and 115.1.
  const int64_t tiles = groups * ((topk + qattn::kTok - 1) / qattn::kTok);
  const bool wide = num_heads > 16 && tiles > 8 * static_cast<int64_t>(info.num_sms);
  return qattn::launch(p, info, wide, workspace, reinterpret_cast<cudaStream_t>(stream));
}
