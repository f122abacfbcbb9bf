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

// A warp takes kTok tokens at a time, a lane values 8 l .. 8 l + 7 and 256 + 8 l
// .. of the latent (16-byte loads, 8-byte stores, each of a warp's in one piece)
// and the pair 2 l, 2 l + 1 of the position part.  All loads of the kTok tokens
// are made before any is used.
template <int kTok>
__global__ void __launch_bounds__(32 * kWarps)
write_kernel(const WriteParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int stride = gridDim.x * kWarps * kTok;
  uint4 wraw[2] = {make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u),
                   make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u)};  // ones
  if (p.norm != nullptr) {
    wraw[0] = *reinterpret_cast<const uint4*>(p.norm + 8 * lane);
    wraw[1] = *reinterpret_cast<const uint4*>(p.norm + 256 + 8 * lane);
  }
  const uint32_t* w32 = reinterpret_cast<const uint32_t*>(wraw);
  const int64_t stride64 = stride;
  for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * kTok; t0 < p.num_tokens;
       t0 += stride64) {
    const int n = p.num_tokens - t0 < kTok ? static_cast<int>(p.num_tokens - t0) : kTok;
    uint4 raw[kTok][2];
    uint32_t pe[kTok];
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      if (i < n) {
        const uint8_t* row = p.kv + (t0 + i) * p.kv_row;
        raw[i][0] = *reinterpret_cast<const uint4*>(row + 16 * lane);
        raw[i][1] = *reinterpret_cast<const uint4*>(row + 512 + 16 * lane);
        pe[i] = *reinterpret_cast<const uint32_t*>(row + 2 * kCkv + 4 * lane);
      } else {
        raw[i][0] = raw[i][1] = make_uint4(0u, 0u, 0u, 0u);
        pe[i] = 0u;
      }
    }
    // Lane i has what is token i's own: where it goes, its position.
    int64_t slot = -1, pos = 0;
    if (lane < n) {
      slot = p.slots[t0 + lane];
      bool bad = slot >= p.num_slots;
      if (p.positions != nullptr) {
        pos = p.positions[t0 + lane];
        bad |= slot >= 0 && (pos < 0 || pos >= p.max_positions);
      }
      if (bad) {
        slot = -1;
        if (p.status != nullptr) atomicOr(p.status, DSA_DEV_BAD_INDEX);
      }
    }
    // cos and sin: of the pair's frequency (interleaved), or of the two
    // frequencies 2 l, 2 l + 1 (mod 32) that the lane's values have.
    float2 cs[kTok], sn[kTok];
    if (p.positions != nullptr) {
#pragma unroll
      for (int i = 0; i < kTok; ++i) {
        const int64_t at = __shfl_sync(0xffffffffu, slot >= 0 ? pos : 0, i);
        if (i < n) {
          const float* row = p.cos_sin + at * kKpe;
          if (p.interleaved) {
            cs[i] = make_float2(row[lane], 0.f);
            sn[i] = make_float2(row[32 + lane], 0.f);
          } else {
            cs[i] = *reinterpret_cast<const float2*>(row + 2 * (lane & 15));
            sn[i] = *reinterpret_cast<const float2*>(row + 32 + 2 * (lane & 15));
          }
        }
      }
    }
    float sum[kTok];
    uint32_t most[kTok];  // bits of the largest |t|: their order is that of the values, NaN on top
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      const uint32_t* x = reinterpret_cast<const uint32_t*>(raw[i]);
      float s = 0.f;
      uint32_t m = 0u;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float2 c = bf16x2(x[k]), w = bf16x2(w32[k]);
        s = fmaf(c.x, c.x, s);
        s = fmaf(c.y, c.y, s);
        m = max(m, max(__float_as_uint(c.x * w.x) & 0x7FFFFFFFu, __float_as_uint(c.y * w.y) & 0x7FFFFFFFu));
      }
      sum[i] = s;
      most[i] = __reduce_max_sync(0xffffffffu, m);
    }
    if (p.norm != nullptr) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
        for (int i = 0; i < kTok; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
      }
    }
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      const int64_t to = __shfl_sync(0xffffffffu, slot, i);
      if (to < 0) continue;
      const int64_t page = to / kPage;
      const int row = static_cast<int>(to - page * kPage);
      uint8_t* base = p.cache + page * kPageBytes;
      const float M = __uint_as_float(most[i]);
      const float r = p.norm != nullptr ? 1.f / sqrtf(fmaf(sum[i], 1.f / kCkv, p.eps)) : 1.f;
      float scale = M * r / kMostCode;
      uint32_t code[4];
      if (most[i] >= 0x7F800000u) {  // an infinity or NaN: the whole row is NaN
        scale = 1.f;
        code[0] = code[1] = code[2] = code[3] = 0x7F7F7F7Fu;
      } else if (!(scale >= kLeastScale)) {  // zeros, or too small for a scale
        scale = 1.f;
        code[0] = code[1] = code[2] = code[3] = 0u;
      } else {
        // Powers of two bring M to [1, 2), exactly; then 448 t / M as the
        // correctly rounded reciprocal and an FMA-corrected quotient (P.
        // Markstein, IBM J. Res. Dev. 34(1), 1990: equal to IEEE division here;
        // what underflows is far below half of the smallest code).
        const int exponent = static_cast<int>(most[i] >> 23);  // biased; 0: M is subnormal
        const float by = __uint_as_float(static_cast<uint32_t>(min(max(254 - exponent, 1), 254)) << 23);
        const float Mn = M * by, rcp = __frcp_rn(Mn), by448 = by;
        const uint32_t* x = reinterpret_cast<const uint32_t*>(raw[i]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float v[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 c = bf16x2(x[2 * k + h]), w = bf16x2(w32[2 * k + h]);
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const float t = (z ? c.y * w.y : c.x * w.x) * by448 * kMostCode;  // exact: 19 bits
              const float q = __fmul_rn(t, rcp);
              v[2 * h + z] = __fmaf_rn(__fmaf_rn(-q, Mn, t), rcp, q);
            }
          }
          const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E4M3);
          const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[2], v[3]), __NV_SATFINITE, __NV_E4M3);
          code[k] = lo | (hi << 16);
        }
      }
      uint8_t* codes = base + row * kCkv;
      *reinterpret_cast<uint2*>(codes + 8 * lane) = make_uint2(code[0], code[1]);
      *reinterpret_cast<uint2*>(codes + 256 + 8 * lane) = make_uint2(code[2], code[3]);
      if (lane == 0) *reinterpret_cast<float*>(base + kScaleAt + 4 * row) = scale;
      uint32_t rotated = pe[i];
      if (p.positions != nullptr) {
        const float2 v = bf16x2(pe[i]);
        if (p.interleaved) {
          rotated = to_bf16x2(fmaf(v.x, cs[i].x, -(v.y * sn[i].x)), fmaf(v.y, cs[i].x, v.x * sn[i].x));
        } else {
          // Lanes 0-15 have the first halves a of the pairs, lanes 16-31 the
          // second ones b: a cos - b sin, and b cos + a sin.
          const float2 o = bf16x2(__shfl_xor_sync(0xffffffffu, pe[i], 16));
          const float sign = lane < 16 ? -1.f : 1.f;
          rotated = to_bf16x2(fmaf(v.x, cs[i].x, sign * (o.x * sn[i].x)), fmaf(v.y, cs[i].y, sign * (o.y * sn[i].y)));
        }
      }
      *reinterpret_cast<uint32_t*>(base + kKpeAt + row * kKpe * 2 + 4 * lane) = rotated;
    }
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

template <int kTok>
__global__ void __launch_bounds__(32 * kWarps)
read_kernel(const ReadParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int row0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * kTok;
  if (row0 >= p.num_rows) return;
  int r = request_of(p.cu, p.num_requests, row0, lane);
  // Lane i resolves row i: its page's first byte and its row in it; -1: zeros, -2: not written.
  int64_t at = -2;
  int in_page = 0;
  const int mine = row0 + lane;
  if (lane < kTok && mine < p.num_rows && mine >= p.cu[0] && mine < p.cu[p.num_requests]) {
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
  uint2 code[kTok][2];
  uint32_t pe[kTok];
  float scale[kTok];
  bool write[kTok];
#pragma unroll
  for (int i = 0; i < kTok; ++i) {
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
  for (int i = 0; i < kTok; ++i) {
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
  constexpr int kTok = 4;
  const int64_t blocks = (static_cast<int64_t>(num_tokens) + quant::kWarps * kTok - 1) / (quant::kWarps * kTok);
  if (launch_programmatic(quant::write_kernel<kTok>, dim3(static_cast<unsigned int>(blocks)), dim3(32 * quant::kWarps), 0,
                          reinterpret_cast<cudaStream_t>(stream), p) != cudaSuccess ||
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
  constexpr int kTok = 4;
  const int64_t blocks = (static_cast<int64_t>(num_rows) + quant::kWarps * kTok - 1) / (quant::kWarps * kTok);
  if (launch_programmatic(quant::read_kernel<kTok>, dim3(static_cast<unsigned int>(blocks)), dim3(32 * quant::kWarps), 0,
                          reinterpret_cast<cudaStream_t>(stream), p) != cudaSuccess ||
      cudaGetLastError() != cudaSuccess)
    return DSA_ERR_CUDA;
  return DSA_OK;
}
