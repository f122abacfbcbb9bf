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
// to the code that exact arithmetic gives.
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

// Warps walk the tokens; of a token a lane has the values 8 l .. 8 l + 7 and 256
// + 8 l .. of the latent (16-byte loads, 8-byte stores, each of a warp's in one
// piece) and the pair 2 l, 2 l + 1 of the position part.  A warp loads its next
// token before it works on the one it has: 24 warps an SM of 79 registers have
// 33 KB on their way.  About 300 instructions a token, three quarters of the issue
// slots; DRAM at 57 % of its peak.  Packed FMAs save 40 of them and 0.3 us; a load
// two tokens ahead needs 122 registers, 16 warps: 85 us.  200003 tokens with norm
// and rotation: 74 us, 5.4 TB/s (60 us at the copy's rate); without the load
// ahead 86, two tokens a warp 88, four in 159 registers (8 warps an SM) 185; two
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
  float w78[16];
  {
    uint4 raw[2] = {make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u),
                    make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u)};  // ones
    if (p.norm != nullptr) {
      raw[0] = *reinterpret_cast<const uint4*>(p.norm + 8 * lane);
      raw[1] = *reinterpret_cast<const uint4*>(p.norm + 256 + 8 * lane);
    }
    const uint32_t* x = reinterpret_cast<const uint32_t*>(raw);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float2 w = bf16x2(x[k]);
      w78[2 * k] = w.x * (kMostCode / 512.f);
      w78[2 * k + 1] = w.y * (kMostCode / 512.f);
    }
  }
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kWarps;
  int64_t t_next = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  // Lane x has slot and position of the warp's x-th token from here on, so that
  // no load waits for another but once in 32 tokens.
  int64_t lane_slot = -1, lane_pos = 0;
  int turn = 0;
  auto load = [&]() {
    if (turn == 0) {
      const int64_t at = t_next + lane * stride;
      lane_slot = -1;
      lane_pos = 0;
      if (at < p.num_tokens) {
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
      const uint8_t* row = p.kv + t_next * p.kv_row;
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
  if (t_next >= p.num_tokens) return;
  TokenPart next = load();
  for (;;) {
    const TokenPart now = next;
    const bool more = t_next < p.num_tokens;
    if (more) next = load();
    if (now.slot >= 0) {  // the whole warp
      const uint32_t* x = reinterpret_cast<const uint32_t*>(now.c);
      float t[16];  // 7/8 c w, exact
      float sum = 0.f, most = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float2 c = bf16x2(x[k]);
        sum = fmaf(c.x, c.x, sum);
        sum = fmaf(c.y, c.y, sum);
        t[2 * k] = c.x * w78[2 * k];
        t[2 * k + 1] = c.y * w78[2 * k + 1];
        most = max3_nan(most, fabsf(t[2 * k]), fabsf(t[2 * k + 1]));
      }
      // The order of non-negative floats is that of their bits, NaN on top.
      const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
      if (p.norm != nullptr) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      }
      const float r = p.norm != nullptr ? rsqrtf(fmaf(sum, 1.f / kCkv, p.eps)) : 1.f;
      // M / 2^9 with M = max |c w|, and the row's scale.  That quotient is exact:
      // a first one, its remainder by one FMA, and the sum of both rounded.
      const float top7 = __uint_as_float(top), first = top7 * (1.f / kMostCode);
      float D = fmaf(fmaf(-first, kMostCode, top7), 1.f / kMostCode, first);
      float scale = D * (512.f / kMostCode) * r;
      uint32_t code[4];
      if (top >= 0x7F800000u) {  // an infinity or NaN: the whole row is NaN
        scale = 1.f;
        code[0] = code[1] = code[2] = code[3] = 0x7F7F7F7Fu;
      } else if (!(scale >= kLeastScale)) {  // zeros, or too small for a scale
        scale = 1.f;
        code[0] = code[1] = code[2] = code[3] = 0u;
      } else {
        if (D < 1e-18f || D > 1e18f) {  // by a power of two, so that no reciprocal or quotient leaves the range
          const float by = D < 1.f ? 1.8446744073709552e19f : 5.421010862427522e-20f;  // 2^64, 2^-64
          D *= by;
#pragma unroll
          for (int k = 0; k < 16; ++k) t[k] *= by;
        }
        // t / D = 448 c w / M in the same way: within 2^-44 of itself before it is
        // rounded, so exact where it is a border of e4m3 (what underflows is far
        // below half of the smallest code).
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
      const int64_t page = now.slot / kPage;
      const int row = static_cast<int>(now.slot - page * kPage);
      uint8_t* base = p.cache + page * kPageBytes;
      uint8_t* codes = base + row * kCkv;
      *reinterpret_cast<uint2*>(codes + 8 * lane) = make_uint2(code[0], code[1]);
      *reinterpret_cast<uint2*>(codes + 256 + 8 * lane) = make_uint2(code[2], code[3]);
      if (lane == 0) *reinterpret_cast<float*>(base + kScaleAt + 4 * row) = scale;
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
