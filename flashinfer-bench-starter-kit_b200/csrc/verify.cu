// verify.cu -- verification of drafted tokens against the target's
// probabilities, from given random numbers (sm_100a).
//
// Request r has the rows cu[r] .. cu[r+1]-1, a tree: row 0 is its last certain
// token, every other row a draft whose parent comes before it.  With p the
// target's distribution after a node (row of target_probs) and q the one that
// the node's children were drawn from (row of draft_probs), the walk starts at
// row 0; at a node it looks at the children in the order of their rows.  Child
// x is taken with probability min(1, p'(x) / q(x)), where p' is p at first and,
// after each rejection, what is left of it: p' := max(p' - q, 0), normalised.
// The tokens that come out are distributed as if the target had drawn them.
//
// Normalising is kept in two numbers: after k rejections
//   p' = max(p - c_k q, 0) / R_k,  c_0 = 0, R_0 = 1,
//   c_{k+1} = c_k + R_k,  R_{k+1} = sum_v max(p_v - c_{k+1} q_v, 0)
// since max(max(p - c q, 0) / R - q, 0) = max(p - (c + R) q, 0) / R for q >= 0.
// Child x is accepted if u q(x) R_k < max(p(x) - c_k q(x), 0).  Where no child
// is taken, the next token is drawn from p': the first v whose running sum of
// max(p - c q, 0) exceeds u times the sum of all (p itself where that is 0).
// Without draft_probs, q is 1 at the drafted token: a rejected x is struck out of
// p and R is reduced by its weight.  All of it is computed in 64 bits: the
// comparisons decide whole tokens, and running sums over a vocabulary in 32 bits
// would move one draw in a hundred to a neighbour.
//
// One cluster of CTAs per request.  Every warp walks the tree by itself, from
// p(x), q(x) of all rows that the CTA fetched in one round; only a rejection
// that is followed by another child, and the draw at the end, read whole rows:
// each warp of the cluster has one segment of the vocabulary, segment sums are
// exchanged through shared memory (two buffers in turn, one cluster barrier a
// sum), and the warp whose segment holds the drawn token looks at it again.
// What bounds it: two dependent loads and a barrier for the short cases; for
// large vocabularies the rows, read once or twice from L2.
#include <cstdint>

#include "dsa_b200.h"
#include "host.h"
#include "ptx.cuh"

namespace dsa {
namespace verify {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kMaxRows = 4096;   // of a request
constexpr int kStep = 128;       // values a warp reads at once: four a lane
constexpr int kDepth = 4;        // steps whose loads are in flight together
constexpr double kWide = 0x1p896;  // see difference()

struct Params {
  const float* target;
  const float* draft;        // or nullptr
  int64_t target_pitch, draft_pitch;  // values
  const int32_t* tokens;
  const int32_t* parents;
  const int32_t* cu;
  const float* accept_u;
  const float* sample_u;
  int num_requests, num_rows, vocab, width;
  int most;                  // rows that the shared memory holds
  int32_t* path;
  int32_t* accepted;
  int32_t* next;
  unsigned int* status;
};

struct Row {
  int parent, token;
  float u, p, q;
};

__device__ __forceinline__ double ld_cluster_f64(const double* p, int rank) {
  uint32_t a;
  double v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(a) : "memory");
  return v;
}

// Four values of a row from v on (zeros behind the vocabulary).
template <bool kWide>
__device__ __forceinline__ float4 load4(const float* row, int v, int vocab) {
  if (kWide && v + 4 <= vocab) return *reinterpret_cast<const float4*>(row + v);
  float4 x;
  x.x = v < vocab ? row[v] : 0.f;
  x.y = v + 1 < vocab ? row[v + 1] : 0.f;
  x.z = v + 2 < vocab ? row[v + 2] : 0.f;
  x.w = v + 3 < vocab ? row[v + 3] : 0.f;
  return x;
}

// What is left of p at the walk's place: rows of p and q, c, and (without q)
// the children that are struck out, those of `node` before row `stop`.
struct Left {
  const float* p;
  const float* q;   // or nullptr
  double c;
  const Row* rows;
  int node, stop;   // stop = 0: none
};

__device__ __forceinline__ double left_of(float p, float q, double c) {
  const double w = fma(-c, static_cast<double>(q), static_cast<double>(p));
  return w <= 0.0 ? 0.0 : w;  // NaN stays
}

// The same before the maximum, for whole rows, where conversions to 64 bits would
// bound it (one takes 8 clocks of its unit): q is widened by three integer
// instructions instead, without its sign (of 0) and without another exponent: that
// double, a subnormal one if q is 0 or subnormal, is q 2^-896 exactly, and `c_wide`
// is c 2^896.  An infinity comes out as 2^128, more than any p; NaN is looked for in
// another way (segment_sum).
__device__ __forceinline__ double difference(float p, float q, double c_wide) {
  const uint32_t b = __float_as_uint(q);
  const double wide = __hiloint2double(static_cast<int>((b >> 3) & 0x0FFFFFFFu), static_cast<int>(b << 29));
  return fma(-c_wide, wide, static_cast<double>(p));
}

// The largest of three, NaN if any is.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// Weights of the four values from v on, doubled where q counts (max(w, 0) is half
// of w + |w|, which takes no selection); `struck`: whether any child's token may
// lie in the warp's segment.
__device__ __forceinline__ void weights(const Left& s, float4 p, float4 q, int v, bool struck, double (&w)[4]) {
  if (s.q != nullptr && s.c != 0.0) {
    const double c = s.c * kWide;
    w[0] = difference(p.x, q.x, c);
    w[1] = difference(p.y, q.y, c);
    w[2] = difference(p.z, q.z, c);
    w[3] = difference(p.w, q.w, c);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] += fabs(w[e]);
    return;
  }
  w[0] = p.x;
  w[1] = p.y;
  w[2] = p.z;
  w[3] = p.w;
  if (struck) {
    for (int k = 1; k < s.stop; ++k) {
      if (s.rows[k].parent != s.node) continue;
      const int at = s.rows[k].token - v;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (at == e) w[e] = 0.0;
    }
  }
}

// Sum of these over the warp's segment [from, to), in every lane; NaN where p holds
// one, or q where it counts.
template <bool kWide>
__device__ double segment_sum(const Left& s, int from, int to, int vocab, bool struck) {
  const int lane = threadIdx.x & 31;
  double sum = 0.0;
  float most = 0.f;  // of q
  for (int v0 = from; v0 < to; v0 += kStep * kDepth) {
    float4 p[kDepth], q[kDepth];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int v = v0 + d * kStep + 4 * lane;
      p[d] = q[d] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (v < to) {
        p[d] = load4<kWide>(s.p, v, vocab);
        if (s.q != nullptr && s.c != 0.0) q[d] = load4<kWide>(s.q, v, vocab);
      }
    }
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int v = v0 + d * kStep + 4 * lane;
      if (v < to) {
        double w[4];
        weights(s, p[d], q[d], v, struck, w);
        sum += (w[0] + w[1]) + (w[2] + w[3]);
        most = max_nan(max_nan(most, q[d].x, q[d].y), q[d].z, q[d].w);
      }
    }
  }
  if (most != most) sum = most;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

// The first value of the segment whose running sum, from `before` on, exceeds
// `target`; the last one of any weight if rounding leaves none (the segment's
// own sum did exceed it).
template <bool kWide>
__device__ int find_in_segment(const Left& s, int from, int to, int vocab, bool struck, double before, double target) {
  const int lane = threadIdx.x & 31;
  int last = -1;
  for (int v0 = from; v0 < to; v0 += kStep) {
    const int v = v0 + 4 * lane;
    double w[4] = {0.0, 0.0, 0.0, 0.0};
    if (v < to) {
      float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 p = load4<kWide>(s.p, v, vocab);
      if (s.q != nullptr && s.c != 0.0) q = load4<kWide>(s.q, v, vocab);
      weights(s, p, q, v, struck, w);
    }
    double up = (w[0] + w[1]) + (w[2] + w[3]);
    const double mine = up;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += x;
    }
    const double all = __shfl_sync(0xffffffffu, up, 31);
    const unsigned int above = __ballot_sync(0xffffffffu, before + up > target && mine > 0.0);
    int weighted = -1;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (w[e] > 0.0) weighted = v + e;
    if (above != 0) {
      const int at = __ffs(above) - 1;
      double run = before + (up - mine);
      int found = weighted;
#pragma unroll
      for (int e = 3; e >= 0; --e) {
        double upto = run;
#pragma unroll
        for (int z = 0; z <= e; ++z) upto += w[z];
        if (upto > target && w[e] > 0.0) found = v + e;
      }
      return __shfl_sync(0xffffffffu, found, at);
    }
    last = max(last, static_cast<int>(__reduce_max_sync(0xffffffffu, static_cast<unsigned int>(weighted + 1))) - 1);
    before += all;
  }
  return last;
}

template <bool kWide>
__global__ void __launch_bounds__(kThreads, 2)
verify_kernel(const Params p) {
  extern __shared__ Row rows[];
  __shared__ double sums[2][kWarps];
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int ctas = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
  const int b = blockIdx.x / ctas;
  griddep_wait();
  griddep_launch_dependents();

  const int lo = p.cu[b], hi = p.cu[b + 1];
  int n = hi - lo;
  bool bad = lo < 0 || hi < lo || hi > p.num_rows;
  if (bad) n = 0;
  if (n > p.most) {
    n = p.most;
    bad = true;
  }
  if (bad && rank == 0 && tid == 0) atomicOr(p.status, DSA_DEV_BAD_SEQ_LEN);

  // ---- every row's parent and token, and p, q at the token after the parent
  for (int k = 1 + tid; k < n; k += kThreads) {
    Row r{p.parents[lo + k], p.tokens[lo + k], p.accept_u[lo + k], 0.f, 0.f};
    if (r.parent >= k) r.parent = -1;  // no parent: never looked at
    if (r.token < 0 || r.token >= p.vocab) {
      if (rank == 0) atomicOr(p.status, DSA_DEV_BAD_INDEX);  // never accepted
      r.token = -1;
    } else if (r.parent >= 0) {
      r.p = p.target[static_cast<int64_t>(lo + r.parent) * p.target_pitch + r.token];
      r.q = p.draft != nullptr ? p.draft[static_cast<int64_t>(lo + r.parent) * p.draft_pitch + r.token] : 1.f;
    }
    rows[k] = r;
  }
  __syncthreads();

  // The warp's segment of the vocabulary, and the exchange of segment sums.
  const int segments = ctas * kWarps;
  const int per = ((p.vocab + segments - 1) / segments + kStep - 1) / kStep * kStep;
  const int segment = rank * kWarps + warp;
  const int from = min(static_cast<int>(min(static_cast<int64_t>(segment) * per, static_cast<int64_t>(p.vocab))), p.vocab);
  const int to = min(from + per, p.vocab);
  const int each = (segments + 31) / 32;  // segments that a lane adds up, at most 4
  int turn = 0;
  double part[4], upto = 0.0;  // the lane's segments; running sum up to their end
  auto exchange = [&](double mine) {
    if (lane == 0) sums[turn][warp] = mine;
    // Buffer `turn` is written again behind the next barrier but one, which no
    // CTA passes before all have read it.
    cluster_sync();
    double total = 0.0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int x = lane * each + k;
      part[k] = k < each && x < segments ? ld_cluster_f64(&sums[turn][x % kWarps], x / kWarps) : 0.0;
      total += part[k];
    }
    upto = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    turn ^= 1;
    return __shfl_sync(0xffffffffu, upto, 31);
  };

  // ---- the walk, by every warp alike
  int32_t* path = p.path + static_cast<int64_t>(b) * p.width;
  const bool writer = rank == 0 && tid == 0;
  int node = 0, taken = 0, looked = 1;
  double c = 0.0, R = 1.0;
  bool open = false;  // R has to be summed before it is used
  auto left = [&](double cc, int stop) {
    return Left{p.target + static_cast<int64_t>(lo + node) * p.target_pitch,
                p.draft != nullptr ? p.draft + static_cast<int64_t>(lo + node) * p.draft_pitch : nullptr, cc, rows, node,
                p.draft != nullptr ? 0 : stop};
  };
  while (looked < n && taken < p.width) {
    int k = -1;  // the node's next child
    for (int k0 = looked; k0 < n && k < 0; k0 += 32) {
      const unsigned int hit = __ballot_sync(0xffffffffu, k0 + lane < n && rows[k0 + lane].parent == node);
      if (hit != 0) k = k0 + __ffs(hit) - 1;
    }
    if (k < 0) break;
    const Row r = rows[k];
    looked = k + 1;
    double w = r.p;
    if (p.draft != nullptr) {
      if (open) {
        R = 0.5 * exchange(segment_sum<kWide>(left(c, 0), from, to, p.vocab, false));
        open = false;
      }
      w = left_of(r.p, r.q, c);
    } else {
      for (int z = 1; z < k; ++z)  // struck out already
        if (rows[z].parent == node && rows[z].token == r.token) w = 0.0;
    }
    if (static_cast<double>(r.u) * static_cast<double>(r.q) * R < w) {
      if (writer) path[taken] = k;
      ++taken;
      node = k;
      c = 0.0;
      R = 1.0;
      open = false;
    } else if (p.draft != nullptr) {
      c += R;
      open = true;
    } else {
      R -= w;
      c = 1.0;  // something is struck out
    }
  }
  if (rank == 0) {
    for (int k = taken + tid; k < p.width; k += kThreads) path[k] = -1;
    if (tid == 0) p.accepted[b] = taken;
  }

  // ---- the token that follows
  if (n > 0) {
    Left s = left(c, c != 0.0 ? looked : 0);
    // Without q: whether a struck token lies in this segment.
    bool struck = false;
    for (int k0 = 1; k0 < s.stop; k0 += 32) {
      const int k = k0 + lane;
      struck |= __any_sync(0xffffffffu, k < s.stop && rows[k].parent == node && rows[k].token >= from && rows[k].token < to);
    }
    double total = exchange(segment_sum<kWide>(s, from, to, p.vocab, struck));
    if (total == 0.0 && c != 0.0) {  // nothing is left of p: p itself
      s = left(0.0, 0);
      struck = false;
      total = exchange(segment_sum<kWide>(s, from, to, p.vocab, false));
    }
    const double target = static_cast<double>(p.sample_u[b]) * total;
    // The first segment whose running sum exceeds it.
    double run = __shfl_up_sync(0xffffffffu, upto, 1);
    if (lane == 0) run = 0.0;
    int mine = -1;
    double before = 0.0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const double after = run + part[k];
      if (mine < 0 && after > target && part[k] > 0.0) {
        mine = lane * each + k;
        before = run;
      }
      run = after;
    }
    const unsigned int hit = __ballot_sync(0xffffffffu, mine >= 0);
    if (hit == 0) {
      if (writer) p.next[b] = -1;
    } else {
      const int at = __ffs(hit) - 1;
      mine = __shfl_sync(0xffffffffu, mine, at);
      before = __shfl_sync(0xffffffffu, before, at);
      if (mine == segment) {
        const int token = find_in_segment<kWide>(s, from, to, p.vocab, struck, before, target);
        if (lane == 0) p.next[b] = token;
      }
    }
  } else if (writer) {
    p.next[b] = -1;
  }
  cluster_sync();  // no CTA leaves while another reads its sums
}

// CTAs per request: enough that each SM has about two, at most one for every
// 2048 values of the vocabulary.
int cluster_for(int requests, int vocab, int sms) {
  const int fit = 2 * sms / requests, fill = (vocab + 2047) / 2048;
  const int c = fit < fill ? fit : fill;
  return c < 1 ? 1 : (c < kMaxCluster ? c : kMaxCluster);
}

}  // namespace verify
}  // namespace dsa

using namespace dsa;

extern "C" int dsa_verify_run(const float* target_probs, int64_t target_stride, const float* draft_probs,
                              int64_t draft_stride, const int32_t* draft_tokens, const int32_t* parents,
                              const int32_t* cu_drafts, const float* accept_u, const float* sample_u,
                              int32_t num_requests, int32_t num_rows, int32_t vocab, int32_t path_width, int32_t* path,
                              int32_t* num_accepted, int32_t* next_token, uint32_t* status, void* stream) {
  if (num_requests < 0 || num_rows < 0) return DSA_ERR_INVALID_ARGUMENT;
  if (num_requests == 0) return DSA_OK;
  if (num_rows > (1 << 24) || num_requests > 65536 || vocab < 1 || vocab > (1 << 28) || path_width < 1 ||
      path_width > (1 << 16) || target_stride < vocab || (draft_probs && draft_stride < vocab))
    return DSA_ERR_INVALID_ARGUMENT;
  if (!target_probs || !draft_tokens || !parents || !cu_drafts || !accept_u || !sample_u || !path || !num_accepted ||
      !next_token || !status)
    return DSA_ERR_INVALID_ARGUMENT;
  const void* all[] = {target_probs, draft_probs, draft_tokens, parents, cu_drafts, accept_u,
                       sample_u,     path,        num_accepted, next_token, status};
  for (const void* x : all)
    if (reinterpret_cast<uintptr_t>(x) & 3u) return DSA_ERR_MISALIGNED;
  const size_t n = static_cast<size_t>(num_requests), t = static_cast<size_t>(num_rows);
  struct Range {
    const void* at;
    size_t bytes;
  };
  const Range in[7] = {{target_probs, t == 0 ? 0 : ((t - 1) * target_stride + vocab) * 4},
                       {draft_probs, draft_probs && t ? ((t - 1) * draft_stride + vocab) * 4 : 0},
                       {draft_tokens, t * 4},
                       {parents, t * 4},
                       {cu_drafts, (n + 1) * 4},
                       {accept_u, t * 4},
                       {sample_u, n * 4}};
  const Range out[3] = {{path, n * path_width * 4}, {num_accepted, n * 4}, {next_token, n * 4}};
  for (int i = 0; i < 3; ++i) {
    for (int j = 0; j < i; ++j)
      if (ranges_overlap(out[i].at, out[i].bytes, out[j].at, out[j].bytes)) return DSA_ERR_OVERLAP;
    for (const Range& x : in)
      if (x.bytes != 0 && ranges_overlap(out[i].at, out[i].bytes, x.at, x.bytes)) return DSA_ERR_OVERLAP;
  }
  DeviceInfo info;
  const int st = current_device_info(&info);
  if (st != DSA_OK) return st;
  const int most = num_rows < verify::kMaxRows ? num_rows : verify::kMaxRows;
  const bool wide = !((reinterpret_cast<uintptr_t>(target_probs) | reinterpret_cast<uintptr_t>(draft_probs)) & 15u) &&
                    !((target_stride | (draft_probs ? draft_stride : 0)) & 3);
  const verify::Params p{target_probs, draft_probs, target_stride, draft_stride, draft_tokens, parents, cu_drafts,
                         accept_u,     sample_u,    num_requests,  num_rows,     vocab,        path_width, most,
                         path,         num_accepted, next_token,   reinterpret_cast<unsigned int*>(status)};
  auto kernel = wide ? verify::verify_kernel<true> : verify::verify_kernel<false>;
  static std::once_flag once[64];
  static int ready[64];
  std::call_once(once[info.device], [&]() {
    const int bytes = verify::kMaxRows * static_cast<int>(sizeof(verify::Row));
    ready[info.device] = cudaFuncSetAttribute(verify::verify_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                              bytes) == cudaSuccess &&
                                 cudaFuncSetAttribute(verify::verify_kernel<false>,
                                                      cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess
                             ? DSA_OK
                             : DSA_ERR_CUDA;
  });
  if (ready[info.device] != DSA_OK) return ready[info.device];
  const int ctas = verify::cluster_for(num_requests, vocab, info.num_sms);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned int>(num_requests) * ctas);
  cfg.blockDim = dim3(verify::kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(most > 0 ? most : 1) * sizeof(verify::Row);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned int>(ctas);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess || cudaGetLastError() != cudaSuccess) return DSA_ERR_CUDA;
  return DSA_OK;
}
