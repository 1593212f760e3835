// Verification of drafted tokens against the target's probabilities, from
// given random numbers, for gfx950.
//
// Request r has the target rows cu[r] .. cu[r + 1): one for each of its n
// drafts, in order, and one more.  Draft i, the token x with the draft
// model's probability q(x) and the target's p(x), is taken while
//   u_i * q(x) < p(x)           (fp32; q = 1 where drafts have no probabilities)
// The first one that is not is replaced by a token drawn from max(p - q, 0)
// (from p without x); where all are taken one more is drawn from the last
// row's p.  The draw is the inverse of the distribution function on whole
// numbers: token v weighs floor(max(p - q, 0) * 2^40), W is their sum, and the
// token is the first whose weights up to and with it pass floor(s * W), s the
// request's second random number.  Whole sums have no rounding, so the answer
// does not depend on the order in which they are taken.  Where all weights
// are 0 the weights of p itself serve; where those are 0 too the token is -1.
//
// Two launches: every workgroup of the first decides its request (a few
// dependent loads, the same for all of them) and sums the weights of its
// chunk of the vocabulary; a workgroup of the second finds its request's
// chunk and the token in it.  Bound by the latency of these chains for small
// batches and by reading two rows of each request for large ones.
#include "glm53_common.h"

namespace glm53 {
namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 16;
constexpr int kChunk = kThreads * kPerThread;   // vocabulary entries of a workgroup

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

struct VerifyArgs {
  const float* target;
  int64_t st;
  const float* draft;    // or null
  int64_t sd;
  const void* ids;
  int ids_i64;
  const int32_t* cu;
  const float* accept_u;
  const double* sample_u;
  int64_t rows, drafts;
  int vocab, max_drafts, chunks;
  int32_t* tokens;       // [requests][max_drafts + 1]
  int32_t* accepted;
  int64_t* sums;         // [requests][chunks][2]: of max(p - q, 0), of p
};

__device__ __forceinline__ int64_t token_at(const VerifyArgs& a, int64_t i) {
  return a.ids_i64 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<int64_t>(static_cast<const int32_t*>(a.ids)[i]);
}

// floor(min(max(x, 0), 1) * 2^40), NaN as 0: the two products by 2^20 and the
// remainder between them are exact.
__device__ __forceinline__ uint64_t weight(float x) {
  x = x > 0.f ? fminf(x, 1.f) : 0.f;
  const float t = x * 1048576.f;
  const uint32_t hi = static_cast<uint32_t>(t);
  const uint32_t lo = static_cast<uint32_t>((t - static_cast<float>(hi)) * 1048576.f);
  return (static_cast<uint64_t>(hi) << 20) + lo;
}

// What a request's rows say: how many drafts are taken, and whose weights the
// next token is drawn from.
struct Decision {
  int64_t row;      // target row, -1: the request has none
  int64_t place;    // the rejected draft's row of `draft`, -1: none was rejected
  int64_t token;    // that draft
  int64_t first;    // the request's first draft
  int count;
};

// All 64 lanes of a wave call it and get the same answer.
__device__ __forceinline__ Decision decide(const VerifyArgs& a, int r, int lane) {
  const int64_t c0 = a.cu[r], c1 = a.cu[r + 1];
  Decision d = {-1, -1, -1, c0 - r, 0};
  int64_t n = c1 - c0 - 1;
  if (n > a.max_drafts) n = a.max_drafts;
  if (c0 < 0 || c1 > a.rows || n < 0 || d.first < 0 || d.first + n > a.drafts) return d;
  for (int i0 = 0; i0 < n; i0 += 64) {
    const int i = i0 + lane;
    bool ok = false;
    if (i < n) {
      const int64_t x = token_at(a, d.first + i);
      const float u = a.accept_u[d.first + i];
      if (x >= 0 && x < a.vocab) {
        const float p = a.target[(c0 + i) * a.st + x];
        const float q = a.draft ? a.draft[(d.first + i) * a.sd + x] : 1.f;
        ok = u * q < p;
      }
    }
    const uint64_t taken = __ballot(ok);
    const int lead = taken == ~0ull ? 64 : __builtin_ctzll(~taken);
    d.count += lead;
    if (lead < 64) break;
  }
  d.row = c0 + d.count;
  if (d.count < n) {
    d.place = d.first + d.count;
    d.token = token_at(a, d.place);
  }
  return d;
}

// The weights of kPerThread entries from `at` of the decided row: of what is
// left of the target (rest) and of the target itself (whole).
__device__ __forceinline__ void load_weights(const VerifyArgs& a, const Decision& d, int at, uint64_t (&rest)[kPerThread],
                                             uint64_t (&whole)[kPerThread]) {
  const float* p = a.target + d.row * a.st;
  const bool minus = d.place >= 0 && a.draft;
  const float* q = minus ? a.draft + d.place * a.sd : nullptr;
  float ps[kPerThread], qs[kPerThread];
  if (at + kPerThread <= a.vocab) {
#pragma unroll
    for (int k = 0; k < kPerThread; k += 4) {
      const f32x4u v = *reinterpret_cast<const f32x4u*>(p + at + k);
      ps[k] = v.x, ps[k + 1] = v.y, ps[k + 2] = v.z, ps[k + 3] = v.w;
    }
    if (minus) {
#pragma unroll
      for (int k = 0; k < kPerThread; k += 4) {
        const f32x4u v = *reinterpret_cast<const f32x4u*>(q + at + k);
        qs[k] = v.x, qs[k + 1] = v.y, qs[k + 2] = v.z, qs[k + 3] = v.w;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < kPerThread; k++) {
      ps[k] = at + k < a.vocab ? p[at + k] : 0.f;
      qs[k] = minus && at + k < a.vocab ? q[at + k] : 0.f;
    }
  }
#pragma unroll
  for (int k = 0; k < kPerThread; k++) {
    whole[k] = weight(ps[k]);
    rest[k] = minus ? weight(ps[k] - qs[k]) : d.place >= 0 && at + k == d.token ? 0 : whole[k];
  }
}

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

__global__ __launch_bounds__(kThreads) void verify_sums_kernel(const VerifyArgs a) {
  __shared__ uint64_t part[kThreads / 64][2];
  const int r = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const Decision d = decide(a, r, lane);
  if (d.row < 0) return;   // uniform
  uint64_t rest[kPerThread], whole[kPerThread], s0 = 0, s1 = 0;
  load_weights(a, d, blockIdx.x * kChunk + threadIdx.x * kPerThread, rest, whole);
#pragma unroll
  for (int k = 0; k < kPerThread; k++) s0 += rest[k], s1 += whole[k];
  s0 = wave_sum_u64(s0), s1 = wave_sum_u64(s1);
  if (lane == 0) part[w][0] = s0, part[w][1] = s1;
  __syncthreads();
  if (threadIdx.x < 2) {
    uint64_t s = 0;
    for (int i = 0; i < kThreads / 64; i++) s += part[i][threadIdx.x];
    a.sums[(static_cast<int64_t>(r) * a.chunks + blockIdx.x) * 2 + threadIdx.x] = static_cast<int64_t>(s);
  }
}

// Inclusive scan over the workgroup.
__device__ __forceinline__ uint64_t scan_u64(uint64_t v, uint64_t* part, int lane, int w, uint64_t& total) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t t = __shfl_up(v, d);
    if (lane >= d) v += t;
  }
  __syncthreads();   // an earlier scan's reads of `part`
  if (lane == 63) part[w] = v;
  __syncthreads();
  total = 0;
  uint64_t before = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; i++) {
    if (i < w) before += part[i];
    total += part[i];
  }
  return v + before;
}

__global__ __launch_bounds__(kThreads) void verify_draw_kernel(const VerifyArgs a) {
  __shared__ uint64_t part[kThreads / 64];
  __shared__ int found_chunk, found;
  __shared__ uint64_t below;
  const int r = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const Decision d = decide(a, r, lane);
  int32_t* out = a.tokens + static_cast<int64_t>(r) * (a.max_drafts + 1);
  if (threadIdx.x == 0) found = -1;
  int token = -1;
  if (d.row >= 0) {
    const int64_t* sums = a.sums + static_cast<int64_t>(r) * a.chunks * 2;
    uint64_t total = 0;
    int which = 0;
    for (; which < 2; which++) {   // the rest's weights, else the target's
      total = 0;
      for (int i = threadIdx.x; i < a.chunks; i += kThreads) total += static_cast<uint64_t>(sums[2 * i + which]);
      uint64_t all;
      scan_u64(total, part, lane, w, all);
      total = all;
      if (total) break;
    }
    if (total) {
      const double f = floor(a.sample_u[r] * static_cast<double>(total));
      uint64_t mark = f > 0. ? (f < static_cast<double>(total) ? static_cast<uint64_t>(f) : total - 1) : 0;
      if (mark >= total) mark = total - 1;
      uint64_t base = 0;
      for (int c0 = 0; c0 < a.chunks; c0 += kThreads) {
        const int i = c0 + static_cast<int>(threadIdx.x);
        const uint64_t v = i < a.chunks ? static_cast<uint64_t>(sums[2 * i + which]) : 0;
        uint64_t all;
        const uint64_t upto = base + scan_u64(v, part, lane, w, all);
        if (upto > mark && upto - v <= mark) found_chunk = i, below = upto - v;
        base += all;
      }
      __syncthreads();
      const int at = found_chunk * kChunk + threadIdx.x * kPerThread;
      uint64_t rest[kPerThread], whole[kPerThread], s = 0, all;
      load_weights(a, d, at, rest, whole);
#pragma unroll
      for (int k = 0; k < kPerThread; k++) s += which ? whole[k] : rest[k];
      uint64_t upto = below + scan_u64(s, part, lane, w, all) - s;
#pragma unroll
      for (int k = 0; k < kPerThread; k++) {
        const uint64_t v = which ? whole[k] : rest[k];
        if (upto <= mark && mark < upto + v) found = at + k;
        upto += v;
      }
    }
  }
  __syncthreads();
  token = found;
  for (int j = threadIdx.x; j <= a.max_drafts; j += kThreads)
    out[j] = d.row < 0 || j > d.count ? -1 : j == d.count ? token : static_cast<int32_t>(token_at(a, d.first + j));
  if (threadIdx.x == 0) a.accepted[r] = d.count;
}

}  // namespace
}  // namespace glm53

using namespace glm53;

extern "C" int64_t glm53_verify_drafts_workspace_bytes(int64_t num_requests, int64_t vocab) {
  if (num_requests <= 0 || vocab <= 0) return 0;
  return num_requests * ((vocab + kChunk - 1) / kChunk) * 16;
}

extern "C" int glm53_verify_drafts(const float* target_probs, int64_t st, int64_t num_rows, const float* draft_probs,
                                   int64_t sd, const void* draft_ids, int ids_is_i64, int64_t num_drafts,
                                   const int32_t* cu_rows, const float* accept_u, const double* sample_u,
                                   int64_t num_requests, int64_t vocab, int64_t max_drafts, void* workspace,
                                   int64_t workspace_bytes, int32_t* tokens, int32_t* accepted, void* stream) {
  if (num_rows < 0 || num_drafts < 0 || num_requests < 0 || vocab <= 0 || max_drafts < 0 || num_requests > 65535 ||
      vocab > 0x7fffffff - kChunk || max_drafts > 0x7ffffffe)
    return GLM53_ERR_BAD_SHAPE;
  if (num_requests == 0) return 0;
  if (!cu_rows || !sample_u || !tokens || !accepted || (num_rows && !target_probs) ||
      (num_drafts && (!draft_ids || !accept_u)))
    return GLM53_ERR_NULL_POINTER;
  if (!workspace || workspace_bytes < glm53_verify_drafts_workspace_bytes(num_requests, vocab)) return GLM53_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 8) return GLM53_ERR_MISALIGNED;
  VerifyArgs a = {};
  a.target = target_probs, a.st = st, a.draft = draft_probs, a.sd = sd;
  a.ids = draft_ids, a.ids_i64 = ids_is_i64, a.cu = cu_rows, a.accept_u = accept_u, a.sample_u = sample_u;
  a.rows = num_rows, a.drafts = num_drafts;
  a.vocab = static_cast<int>(vocab), a.max_drafts = static_cast<int>(max_drafts);
  a.chunks = static_cast<int>((vocab + kChunk - 1) / kChunk);
  a.tokens = tokens, a.accepted = accepted, a.sums = static_cast<int64_t*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  hipLaunchKernelGGL(verify_sums_kernel, dim3(a.chunks, static_cast<unsigned>(num_requests)), dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL(verify_draw_kernel, dim3(static_cast<unsigned>(num_requests)), dim3(kThreads), 0, s, a);
  return static_cast<int>(hipGetLastError());
}
