// quant.cu -- the paged latent cache in 8 bits: writing new tokens' rows, with
// the latent's norm and the position part's rotation in the same pass, and
// reading ranges of tokens back as bf16 (sm_100a).
//
// A page of 64 tokens is 41216 bytes: 64 x 512 e4m3 codes (the ckv part), 64 x
// 64 bf16 (the kpe part), 64 fp32 scales, one for each token.  A token's latent
// is code * scale.
//
// Writing: with c the 512 latent values, e the 64 position values of a token,
//   t_d = c_d * norm_d,  M = max |t_d|,  r = 1 / sqrt(mean c^2 + eps)
//   code_d = e4m3(448 t_d / M),  scale = r M / 448
//   e rotated by the angles of its position, rounded to bf16
// (norm absent: t = c, r = 1).  The row's r is left to the scale, so the codes
// do not depend on a sum: t is the exact product of two bf16, and the quotient
// of two integers of 16 bits by 448 is a border of e4m3 or at least 2^-21 of
// itself away from one.  A correctly rounded quotient (2^-24) therefore rounds
// to the code that exact arithmetic gives.  Rows whose squares or products leave
// fp32's range are scaled by powers of two first (write_far_row).
//
// One scale a token, not one for each 128 values: e4m3 keeps its three bits down
// to 2^-15 of the row's largest value, and the attention over this cache can
// then take the scale out of both products (see quant_attention.cu).
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "dsa_b200.h"
#include "host.h"
#include "ptx.cuh"

namespace dsa {
namespace quant {

constexpr int kCkv = DSA_CKV_DIM;                 // 512
constexpr int kKpe = DSA_KPE_DIM;                 // 64
constexpr int kPage = DSA_PAGE_SIZE;              // 64
constexpr int kPageBytes = DSA_LATENT_PAGE_BYTES; // 41216
constexpr int kKpeAt = kPage * kCkv;              // offsets in a page
constexpr int kScaleAt = kKpeAt + kPage * kKpe * 2;
static_assert(kScaleAt + kPage * 4 == kPageBytes, "page layout");
constexpr int kWarps = 8;
constexpr float kMostCode = 448.0f;
constexpr float kLeastScale = 1.1754943508222875e-38f;  // 2^-126
constexpr float kMostScale = 3.4028234663852886e38f;
constexpr uint32_t kSmall = (127u - 100u) << 23;        // the bits of 2^-100

__device__ __forceinline__ float2 bf16x2(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ uint32_t to_bf16x2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// ------------------------------------------------------------------ write
struct WriteParams {
  const uint8_t* kv;
  int64_t kv_row;           // bytes
  const int64_t* slots;
  int num_tokens;
  const __nv_bfloat16* norm;  // or nullptr
  float eps;
  const int64_t* positions;   // or nullptr: no rotation
  const float* cos_sin;       // [max_positions][32 cos, 32 sin]
  int64_t max_positions;
  int interleaved;
  uint8_t* cache;
  int64_t num_slots;
  unsigned int* status;       // or nullptr
};

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// M / 2^9 of 7/8 M, M = max |c w|, exactly: a first quotient, its remainder by one
// FMA, and the sum of both rounded.
__device__ __forceinline__ float most_over_512(float top7) {
  const float first = top7 * (1.f / kMostCode);
  return fmaf(fmaf(-first, kMostCode, top7), 1.f / kMostCode, first);
}

// 2^n in 64 bits, -1022 <= n <= 1023.
__device__ __forceinline__ double power_of_two(int n) { return __hiloint2double((n + 1023) << 20, 0); }

// Codes e4m3(t / D) of a lane's 16 values, D = 7/8 M / 448 of a row.
__device__ __forceinline__ void codes_of(float (&t)[16], float D, uint32_t (&code)[4]) {
  if (D < 1e-18f || D > 1e18f) {  // by a power of two, so that no reciprocal or quotient leaves the range
    const float by = D < 1.f ? 1.8446744073709552e19f : 5.421010862427522e-20f;  // 2^64, 2^-64
    D *= by;
#pragma unroll
    for (int k = 0; k < 16; ++k) t[k] *= by;
  }
  // t / D = 448 c w / M in the same way as D (a quotient corrected by its remainder:
  // P. Markstein, as in cache_write.cu): within 2^-44 of itself before it is rounded,
  // so exact where it is a border of e4m3 (what underflows is far below half of the
  // smallest code).
  float rcp;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rcp) : "f"(D));
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float v[4];
#pragma unroll
    for (int z = 0; z < 4; ++z) {
      const float q = __fmul_rn(t[4 * k + z], rcp);
      v[z] = __fmaf_rn(__fmaf_rn(q, D, -t[4 * k + z]), -rcp, q);  // (signs that keep -0)
    }
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[2], v[3]), __NV_SATFINITE, __NV_E4M3);
    code[k] = lo | (hi << 16);
  }
}

__device__ __forceinline__ void store_codes(uint8_t* codes, const uint32_t (&code)[4], float* to_scale, float scale) {
  const int lane = threadIdx.x & 31;
  *reinterpret_cast<uint2*>(codes + 8 * lane) = make_uint2(code[0], code[1]);
  *reinterpret_cast<uint2*>(codes + 256 + 8 * lane) = make_uint2(code[2], code[3]);
  if (lane == 0) *to_scale = scale;
}

// The latent of a row whose squares or products leave the range of fp32, or its
// normal numbers, of a row of zeros and of one that is not finite: again, with c and
// the weights scaled by powers of two to magnitudes of 1 (the codes are the same),
// and the scale in 64 bits.  For a whole warp.
__device__ __forceinline__ void write_far_row(const uint8_t* row, const __nv_bfloat16* norm, float eps, uint8_t* codes, float* to_scale) {
  const int lane = threadIdx.x & 31;
  uint4 c_raw[2], w_raw[2];
  c_raw[0] = *reinterpret_cast<const uint4*>(row + 16 * lane);
  c_raw[1] = *reinterpret_cast<const uint4*>(row + 512 + 16 * lane);
  w_raw[0] = w_raw[1] = make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u);  // ones
  if (norm != nullptr) {
    w_raw[0] = *reinterpret_cast<const uint4*>(norm + 8 * lane);
    w_raw[1] = *reinterpret_cast<const uint4*>(norm + 256 + 8 * lane);
  }
  const uint32_t* x = reinterpret_cast<const uint32_t*>(c_raw);
  const uint32_t* y = reinterpret_cast<const uint32_t*>(w_raw);
  uint32_t c_top = 0u, w_top = 0u;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    c_top = max(c_top, max((x[k] << 16) & 0x7FFFFFFFu, x[k] & 0x7FFF0000u));
    w_top = max(w_top, max((y[k] << 16) & 0x7FFFFFFFu, y[k] & 0x7FFF0000u));
  }
  c_top = __reduce_max_sync(0xffffffffu, c_top);
  w_top = __reduce_max_sync(0xffffffffu, w_top);
  // Exponents of the largest values (of subnormal ones the least), and what brings them to 1.
  const int c_exp = min(max(static_cast<int>(c_top >> 23), 1), 253) - 127;
  const int w_exp = min(max(static_cast<int>(w_top >> 23), 1), 253) - 127;
  const float by_c = __uint_as_float(static_cast<uint32_t>(127 - c_exp) << 23);
  const float by_w = __uint_as_float(static_cast<uint32_t>(127 - w_exp) << 23) * (kMostCode / 512.f);
  float t[16];
  float sum = 0.f, most = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float2 c = bf16x2(x[k]), w = bf16x2(y[k]);
    const float a = c.x * by_c, b = c.y * by_c;
    sum = fmaf(a, a, sum);
    sum = fmaf(b, b, sum);
    t[2 * k] = a * (w.x * by_w);
    t[2 * k + 1] = b * (w.y * by_w);
    most = fmaxf(most, fmaxf(fabsf(t[2 * k]), fabsf(t[2 * k + 1])));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float D = most_over_512(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most))));
  double scale = static_cast<double>(D * (512.f / kMostCode)) * power_of_two(c_exp) * power_of_two(w_exp);
  if (norm != nullptr) {
    // 1 / sqrt of v = m 4^n with 1 <= m < 4.
    const double v = static_cast<double>(sum) * (1.0 / kCkv) * power_of_two(2 * c_exp) + static_cast<double>(eps);
    const int n = ((__double2hiint(v) >> 20) - 1023) >> 1;
    scale = v > 0.0 ? scale * power_of_two(-n) * static_cast<double>(rsqrtf(static_cast<float>(v * power_of_two(-n) * power_of_two(-n))))
                    : 0.0;
  }
  float to_store = static_cast<float>(scale);
  uint32_t code[4];
  if (c_top >= 0x7F800000u || w_top >= 0x7F800000u || to_store > kMostScale) {  // the whole row is NaN
    to_store = 1.f;
    code[0] = code[1] = code[2] = code[3] = 0x7F7F7F7Fu;
  } else if (!(to_store >= kLeastScale)) {  // zeros, or too small for a scale
    to_store = 1.f;
    code[0] = code[1] = code[2] = code[3] = 0u;
  } else {
    codes_of(t, D, code);
  }
  store_codes(codes, code, to_scale, to_store);
}

// A lane's weights times 7/8 (ones without a norm).
__device__ __forceinline__ void load_weights(const __nv_bfloat16* norm, float (&w78)[16]) {
  const int lane = threadIdx.x & 31;
  uint4 raw[2] = {make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u),
                  make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u)};  // ones
  if (norm != nullptr) {
    raw[0] = *reinterpret_cast<const uint4*>(norm + 8 * lane);
    raw[1] = *reinterpret_cast<const uint4*>(norm + 256 + 8 * lane);
  }
  const uint32_t* x = reinterpret_cast<const uint32_t*>(raw);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float2 w = bf16x2(x[k]);
    w78[2 * k] = w.x * (kMostCode / 512.f);
    w78[2 * k + 1] = w.y * (kMostCode / 512.f);
  }
}

// Of a row in the ordinary way: a lane's t = 7/8 c w, exact; the largest |t| as
// bits, whose order is that of non-negative floats with NaN on top; the sum of c^2
// (with a norm).  The last two are the same in every lane.
__device__ __forceinline__ void row_sums(const uint4 (&c_raw)[2], const float (&w78)[16], bool norm, float (&t)[16], uint32_t& top,
                                         float& sum) {
  const uint32_t* x = reinterpret_cast<const uint32_t*>(c_raw);
  float most = 0.f;
  sum = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float2 c = bf16x2(x[k]);
    sum = fmaf(c.x, c.x, sum);
    sum = fmaf(c.y, c.y, sum);
    t[2 * k] = c.x * w78[2 * k];
    t[2 * k + 1] = c.y * w78[2 * k + 1];
    most = max3_nan(most, fabsf(t[2 * k]), fabsf(t[2 * k + 1]));
  }
  top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
  if (norm) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
}

// For a whole warp: whether a row's latent is zeros, of either sign.
__device__ __forceinline__ bool is_zero(const uint4 (&c_raw)[2]) {
  const uint32_t any = (c_raw[0].x | c_raw[0].y) | (c_raw[0].z | c_raw[0].w) | (c_raw[1].x | c_raw[1].y) | (c_raw[1].z | c_raw[1].w);
  return !__any_sync(0xffffffffu, (any & 0x7FFF7FFFu) != 0u);
}

// Whether the ordinary way serves: t and squares in the range of normal fp32 numbers (a mean square is its own
// measure), and so the scale; rows of zeros are told apart before.
// (Comparisons of bits: negative numbers and NaN are above infinity.)
__device__ __forceinline__ bool is_far(uint32_t top, float mean, float scale) {
  constexpr uint32_t kRange = 0x7F800000u - kSmall, kScaleRange = 0x7F800000u - 0x00800000u;
  return top - kSmall >= kRange || __float_as_uint(scale) - 0x00800000u >= kScaleRange || __float_as_uint(mean) - kSmall >= kRange;
}

// A warp that met rows out of range goes over its tokens again, for these alone.  Behind the others and not inlined:
// as a branch for each row, their registers cost every row (94 us for 74).
__device__ __noinline__ void far_rows(const uint8_t* kv, int64_t kv_row, const int64_t* slots, int num_tokens,
                                      const __nv_bfloat16* norm, float eps, const int64_t* positions, int64_t max_positions,
                                      uint8_t* cache, int64_t num_slots) {
  const int lane = threadIdx.x & 31;
  float w78[16];
  load_weights(norm, w78);
  const uint32_t stride = gridDim.x * kWarps;
  for (uint32_t token = blockIdx.x * kWarps + (threadIdx.x >> 5); token < static_cast<uint32_t>(num_tokens); token += stride) {
    const int64_t slot = slots[token];
    if (slot < 0 || slot >= num_slots) continue;
    if (positions != nullptr && (positions[token] < 0 || positions[token] >= max_positions)) continue;
    const uint8_t* row = kv + static_cast<int64_t>(token) * kv_row;
    const uint4 c[2] = {*reinterpret_cast<const uint4*>(row + 16 * lane), *reinterpret_cast<const uint4*>(row + 512 + 16 * lane)};
    float t[16], sum;
    uint32_t top;
    row_sums(c, w78, norm != nullptr, t, top, sum);
    const float mean = norm != nullptr ? fmaf(sum, 1.f / kCkv, eps) : 1.f;
    const float scale = most_over_512(__uint_as_float(top)) * (512.f / kMostCode) * rsqrtf(mean);
    if ((top == 0u && is_zero(c)) || !is_far(top, mean, scale)) continue;
    const int64_t page = slot / kPage;
    const int in_page = static_cast<int>(slot - page * kPage);
    uint8_t* base = cache + page * kPageBytes;
    write_far_row(row, norm, eps, base + in_page * kCkv, reinterpret_cast<float*>(base + kScaleAt + 4 * in_page));
  }
}

// Warps walk the tokens; of a token a lane has the values 8 l .. 8 l + 7 and 256
// + 8 l .. of the latent (16-byte loads, 8-byte stores, each of a warp's in one
// piece) and the pair 2 l, 2 l + 1 of the position part.  A warp loads its next
// token before it works on the one it has: 24 warps an SM of 80 registers have
// 33 KB on their way.  About 300 instructions a token, three quarters of the issue
// slots; DRAM at 56 % of its peak.  Packed FMAs save 40 of them and 0.3 us; a load
// two tokens ahead needs 122 registers, 16 warps: 85 us.  200003 tokens with norm
// and rotation: 76 us, 5.2 TB/s (60 us at the copy's rate; 74 without the look for
// rows out of range); without the load ahead 86, two tokens a warp 88, four in 159 registers (8 warps an SM) 185; two
// blocks an SM 88, four (spilling) 98.
constexpr int kBlocksPerSm = 3;

// What a lane loads of a token.
struct TokenPart {
  uint4 c[2];
  uint32_t pe;
  float2 cs, sn;
  int64_t slot;
};

__global__ void __launch_bounds__(32 * kWarps, kBlocksPerSm)
write_kernel(const WriteParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  __shared__ bool met_far[kWarps];
  met_far[threadIdx.x >> 5] = false;
  float w78[16];
  load_weights(p.norm, w78);
  // Unsigned 32 bits hold a token and 32 strides beyond.
  const uint32_t stride = gridDim.x * kWarps;
  uint32_t t_next = blockIdx.x * kWarps + (threadIdx.x >> 5);
  // Lane x has slot and position of the warp's x-th token from here on, so that
  // no load waits for another but once in 32 tokens.
  int64_t lane_slot = -1, lane_pos = 0;
  int turn = 0;
  auto load = [&]() {
    if (turn == 0) {
      const uint32_t at = t_next + lane * stride;
      lane_slot = -1;
      lane_pos = 0;
      if (at < static_cast<uint32_t>(p.num_tokens)) {
        lane_slot = p.slots[at];
        if (p.positions != nullptr) lane_pos = p.positions[at];
        const bool outside = p.positions != nullptr && (lane_pos < 0 || lane_pos >= p.max_positions);
        if (lane_slot >= p.num_slots || (lane_slot >= 0 && outside)) {
          lane_slot = -1;
          if (p.status != nullptr) atomicOr(p.status, DSA_DEV_BAD_INDEX);
        }
        if (outside) lane_pos = 0;
      }
    }
    TokenPart n;
    n.c[0] = n.c[1] = make_uint4(0u, 0u, 0u, 0u);
    n.pe = 0u;
    n.cs = n.sn = make_float2(0.f, 0.f);
    n.slot = __shfl_sync(0xffffffffu, lane_slot, turn);
    if (n.slot >= 0) {
      const uint8_t* row = p.kv + static_cast<int64_t>(t_next) * p.kv_row;
      n.c[0] = *reinterpret_cast<const uint4*>(row + 16 * lane);
      n.c[1] = *reinterpret_cast<const uint4*>(row + 512 + 16 * lane);
      n.pe = *reinterpret_cast<const uint32_t*>(row + 2 * kCkv + 4 * lane);
      if (p.positions != nullptr) {
        // cos and sin: of the pair's frequency (interleaved), or of the two
        // frequencies 2 l, 2 l + 1 (mod 32) that the lane's values have.
        const float* angles = p.cos_sin + __shfl_sync(0xffffffffu, lane_pos, turn) * kKpe;
        if (p.interleaved) {
          n.cs.x = angles[lane];
          n.sn.x = angles[32 + lane];
        } else {
          n.cs = *reinterpret_cast<const float2*>(angles + 2 * (lane & 15));
          n.sn = *reinterpret_cast<const float2*>(angles + 32 + 2 * (lane & 15));
        }
      }
    }
    turn = (turn + 1) & 31;
    t_next += stride;
    return n;
  };
  if (t_next >= static_cast<uint32_t>(p.num_tokens)) return;
  TokenPart next = load();
  for (;;) {
    const TokenPart now = next;
    const bool more = t_next < static_cast<uint32_t>(p.num_tokens);
    if (more) next = load();
    if (now.slot >= 0) {  // the whole warp
      float t[16], sum;
      uint32_t top;
      row_sums(now.c, w78, p.norm != nullptr, t, top, sum);
      const int64_t page = now.slot / kPage;
      const int row = static_cast<int>(now.slot - page * kPage);
      uint8_t* base = p.cache + page * kPageBytes;
      uint8_t* codes = base + row * kCkv;
      float* to_scale = reinterpret_cast<float*>(base + kScaleAt + 4 * row);
      const float mean = p.norm != nullptr ? fmaf(sum, 1.f / kCkv, p.eps) : 1.f;
      const float D = most_over_512(__uint_as_float(top));
      const float scale = D * (512.f / kMostCode) * rsqrtf(mean);
      if (top == 0u && is_zero(now.c)) {
        const uint32_t code[4] = {0u, 0u, 0u, 0u};
        store_codes(codes, code, to_scale, 1.f);
      } else if (is_far(top, mean, scale)) {
        met_far[threadIdx.x >> 5] = true;  // behind all others
      } else {
        uint32_t code[4];
        codes_of(t, D, code);
        store_codes(codes, code, to_scale, scale);
      }
      uint32_t rotated = now.pe;
      if (p.positions != nullptr) {
        const float2 v = bf16x2(now.pe);
        if (p.interleaved) {
          rotated = to_bf16x2(fmaf(v.x, now.cs.x, -(v.y * now.sn.x)), fmaf(v.y, now.cs.x, v.x * now.sn.x));
        } else {
          // Lanes 0-15 have the first halves a of the pairs, lanes 16-31 the
          // second ones b: a cos - b sin, and b cos + a sin.
          const float2 o = bf16x2(__shfl_xor_sync(0xffffffffu, now.pe, 16));
          const float sign = lane < 16 ? -1.f : 1.f;
          rotated = to_bf16x2(fmaf(v.x, now.cs.x, sign * (o.x * now.sn.x)), fmaf(v.y, now.cs.y, sign * (o.y * now.sn.y)));
        }
      }
      *reinterpret_cast<uint32_t*>(base + kKpeAt + row * kKpe * 2 + 4 * lane) = rotated;
    }
    if (!more) break;
  }
  __syncwarp();
  if (!met_far[threadIdx.x >> 5]) return;
  far_rows(p.kv, p.kv_row, p.slots, p.num_tokens, p.norm, p.eps, p.positions, p.max_positions, p.cache, p.num_slots);
}

// ------------------------------------------------------------------ read
struct ReadParams {
  const uint8_t* cache;
  int num_pages;
  const int32_t* block_table;
  const int32_t* starts;
  const int32_t* cu;
  int num_requests, max_pages, num_rows;
  uint8_t* ckv;
  uint8_t* kpe;
  int64_t ckv_row, kpe_row;  // bytes
  unsigned int* status;
};

// The request of row `row` (the last r with cu[r] <= row; cu ascends), found 32
// requests at a time by the whole warp.  Always in [0, n).
__device__ __forceinline__ int request_of(const int32_t* cu, int n, int row, int lane) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + (lane + 1) * step;
    const bool below = at < hi && cu[at] <= row;
    const int k = __popc(__ballot_sync(0xffffffffu, below));
    lo += k * step;
    hi = min(lo + step, hi);
  }
  return lo;
}

constexpr int kReadTok = 4;

__global__ void __launch_bounds__(32 * kWarps)
read_kernel(const ReadParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int row0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * kReadTok;
  if (row0 >= p.num_rows) return;
  int r = request_of(p.cu, p.num_requests, row0, lane);
  // Lane i resolves row i: its page's first byte and its row in it; -1: zeros, -2: not written.
  int64_t at = -2;
  int in_page = 0;
  const int mine = row0 + lane;
  if (lane < kReadTok && mine < p.num_rows && mine >= p.cu[0] && mine < p.cu[p.num_requests]) {
    while (r + 1 < p.num_requests && p.cu[r + 1] <= mine) ++r;
    const int64_t pos = static_cast<int64_t>(p.starts[r]) + (mine - p.cu[r]);
    at = -1;
    if (pos < 0 || pos >= static_cast<int64_t>(p.max_pages) * kPage) {
      atomicOr(p.status, DSA_DEV_BAD_SEQ_LEN);
    } else {
      const int page = p.block_table[static_cast<int64_t>(r) * p.max_pages + pos / kPage];
      in_page = static_cast<int>(pos % kPage);
      if (page < 0 || page >= p.num_pages)
        atomicOr(p.status, DSA_DEV_BAD_PAGE);
      else
        at = static_cast<int64_t>(page) * kPageBytes;
    }
  }
  uint2 code[kReadTok][2];
  uint32_t pe[kReadTok];
  float scale[kReadTok];
  bool write[kReadTok];
#pragma unroll
  for (int i = 0; i < kReadTok; ++i) {
    const int64_t a = __shfl_sync(0xffffffffu, at, i);
    const int row = __shfl_sync(0xffffffffu, in_page, i);
    write[i] = a != -2;
    code[i][0] = code[i][1] = make_uint2(0u, 0u);
    pe[i] = 0u;
    scale[i] = 0.f;
    if (a >= 0) {
      const uint8_t* page = p.cache + a;
      code[i][0] = *reinterpret_cast<const uint2*>(page + row * kCkv + 8 * lane);
      code[i][1] = *reinterpret_cast<const uint2*>(page + row * kCkv + 256 + 8 * lane);
      pe[i] = *reinterpret_cast<const uint32_t*>(page + kKpeAt + row * kKpe * 2 + 4 * lane);
      scale[i] = *reinterpret_cast<const float*>(page + kScaleAt + 4 * row);
    }
  }
#pragma unroll
  for (int i = 0; i < kReadTok; ++i) {
    if (!write[i]) continue;
    uint8_t* to = p.ckv + static_cast<int64_t>(row0 + i) * p.ckv_row;
    const uint32_t x[4] = {code[i][0].x, code[i][0].y, code[i][1].x, code[i][1].y};
    uint32_t y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const __nv_fp8x2_storage_t two = static_cast<__nv_fp8x2_storage_t>(x[k >> 1] >> (16 * (k & 1)));
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3);  // exact
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      y[k] = to_bf16x2(f.x * scale[i], f.y * scale[i]);
    }
    *reinterpret_cast<uint4*>(to + 16 * lane) = make_uint4(y[0], y[1], y[2], y[3]);
    *reinterpret_cast<uint4*>(to + 512 + 16 * lane) = make_uint4(y[4], y[5], y[6], y[7]);
    *reinterpret_cast<uint32_t*>(p.kpe + static_cast<int64_t>(row0 + i) * p.kpe_row + 4 * lane) = pe[i];
  }
}

}  // namespace quant
}  // namespace dsa

using namespace dsa;

extern "C" int dsa_latent_cache_write(const void* kv, int64_t kv_row_bytes, const int64_t* slot_mapping,
                                      int32_t num_tokens, const void* norm_weight, float eps,
                                      const int64_t* positions, const float* cos_sin, int64_t max_positions,
                                      int32_t interleaved, void* latent_cache, int64_t num_pages, uint32_t* status,
                                      void* stream) {
  if (num_tokens < 0 || num_pages < 0 || num_pages > 0x7FFFFFFE) return DSA_ERR_INVALID_ARGUMENT;
  if (num_tokens == 0) return DSA_OK;
  constexpr int64_t kRow = 2 * (quant::kCkv + quant::kKpe);
  if (!kv || !slot_mapping || !latent_cache || kv_row_bytes < kRow || (positions == nullptr) != (cos_sin == nullptr) ||
      (positions && max_positions < 1))
    return DSA_ERR_INVALID_ARGUMENT;
  if (!aligned16(kv) || (kv_row_bytes & 15) || !aligned16(latent_cache) || !aligned16(norm_weight) ||
      (reinterpret_cast<uintptr_t>(slot_mapping) & 7u) || (reinterpret_cast<uintptr_t>(positions) & 7u) ||
      (reinterpret_cast<uintptr_t>(cos_sin) & 7u) || (reinterpret_cast<uintptr_t>(status) & 3u))
    return DSA_ERR_MISALIGNED;
  const size_t cache_bytes = static_cast<size_t>(num_pages) * quant::kPageBytes, n = static_cast<size_t>(num_tokens);
  if (ranges_overlap(latent_cache, cache_bytes, kv, (n - 1) * kv_row_bytes + kRow) ||
      ranges_overlap(latent_cache, cache_bytes, slot_mapping, n * 8) ||
      (norm_weight && ranges_overlap(latent_cache, cache_bytes, norm_weight, quant::kCkv * 2)) ||
      (positions && (ranges_overlap(latent_cache, cache_bytes, positions, n * 8) ||
                     ranges_overlap(latent_cache, cache_bytes, cos_sin, static_cast<size_t>(max_positions) * quant::kKpe * 4))))
    return DSA_ERR_OVERLAP;
  DeviceInfo info;
  const int st = current_device_info(&info);
  if (st != DSA_OK) return st;
  const quant::WriteParams p{static_cast<const uint8_t*>(kv), kv_row_bytes, slot_mapping, num_tokens,
                             static_cast<const __nv_bfloat16*>(norm_weight), eps, positions, cos_sin, max_positions,
                             interleaved, static_cast<uint8_t*>(latent_cache), num_pages * quant::kPage,
                             reinterpret_cast<unsigned int*>(status)};
  const int64_t need = (static_cast<int64_t>(num_tokens) + quant::kWarps - 1) / quant::kWarps;
  const int64_t most = static_cast<int64_t>(info.num_sms) * quant::kBlocksPerSm;
  if (launch_programmatic(quant::write_kernel, dim3(static_cast<unsigned int>(need < most ? need : most)),
                          dim3(32 * quant::kWarps), 0, reinterpret_cast<cudaStream_t>(stream), p) != cudaSuccess ||
      cudaGetLastError() != cudaSuccess)
    return DSA_ERR_CUDA;
  return DSA_OK;
}

extern "C" int dsa_latent_cache_read(const void* latent_cache, int64_t num_pages, const int32_t* block_table,
                                     const int32_t* starts, const int32_t* cu_rows, int32_t num_requests,
                                     int32_t max_pages, int32_t num_rows, void* ckv, int64_t ckv_row_bytes, void* kpe,
                                     int64_t kpe_row_bytes, uint32_t* status, void* stream) {
  if (num_rows < 0 || num_requests < 0) return DSA_ERR_INVALID_ARGUMENT;
  if (num_rows == 0 || num_requests == 0) return DSA_OK;
  constexpr int kC = quant::kCkv * 2, kE = quant::kKpe * 2;
  if (!latent_cache || !block_table || !starts || !cu_rows || !ckv || !kpe || !status || num_pages < 1 ||
      num_pages > 0x7FFFFFFE || max_pages < 1 || max_pages > (1 << 24) || ckv_row_bytes < kC || kpe_row_bytes < kE)
    return DSA_ERR_INVALID_ARGUMENT;
  if (!aligned16(latent_cache) || !aligned16(ckv) || !aligned16(kpe) || ((ckv_row_bytes | kpe_row_bytes) & 15) ||
      ((reinterpret_cast<uintptr_t>(block_table) | reinterpret_cast<uintptr_t>(starts) |
        reinterpret_cast<uintptr_t>(cu_rows) | reinterpret_cast<uintptr_t>(status)) & 3u))
    return DSA_ERR_MISALIGNED;
  const size_t rows = static_cast<size_t>(num_rows), n = static_cast<size_t>(num_requests);
  struct {
    const void* at;
    size_t bytes;
  } in[4] = {{latent_cache, static_cast<size_t>(num_pages) * quant::kPageBytes},
             {block_table, n * max_pages * 4},
             {starts, n * 4},
             {cu_rows, (n + 1) * 4}};
  for (const auto& x : in)
    if (ranges_overlap(ckv, (rows - 1) * ckv_row_bytes + kC, x.at, x.bytes) ||
        ranges_overlap(kpe, (rows - 1) * kpe_row_bytes + kE, x.at, x.bytes))
      return DSA_ERR_OVERLAP;
  // ckv and kpe may be columns of one buffer; widths and pitches as fp32 for rows_overlap.
  if (rows_overlap(num_rows, static_cast<const float*>(ckv), ckv_row_bytes / 4, kC / 4, static_cast<const float*>(kpe),
                   kpe_row_bytes / 4, kE / 4))
    return DSA_ERR_OVERLAP;
  DeviceInfo info;
  const int st = current_device_info(&info);
  if (st != DSA_OK) return st;
  const quant::ReadParams p{static_cast<const uint8_t*>(latent_cache), static_cast<int>(num_pages), block_table, starts,
                            cu_rows, num_requests, max_pages, num_rows, static_cast<uint8_t*>(ckv),
                            static_cast<uint8_t*>(kpe), ckv_row_bytes, kpe_row_bytes,
                            reinterpret_cast<unsigned int*>(status)};
  constexpr int kRows = quant::kWarps * quant::kReadTok;
  const int64_t blocks = (static_cast<int64_t>(num_rows) + kRows - 1) / kRows;
  if (launch_programmatic(quant::read_kernel, dim3(static_cast<unsigned int>(blocks)), dim3(32 * quant::kWarps), 0,
                          reinterpret_cast<cudaStream_t>(stream), p) != cudaSuccess ||
      cudaGetLastError() != cudaSuccess)
    return DSA_ERR_CUDA;
  return DSA_OK;
}
