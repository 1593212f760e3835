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
// Two launches: every wave of the first decides its request (four dependent
// loads, the same for all of them) and sums the weights of its 1024 entries of
// the vocabulary, in whole numbers of 20 bits and 20 bits; a wave of the second
// finds, from those sums, the 1024 entries that hold the token and the token in
// them.  The target's own weights are summed only where the others are all 0,
// by the eight waves of the second launch: they would double the first's
// arithmetic, and draws from a distribution do not need them.
//
// Bound by the chain of dependent loads and the two launches for small batches
// (three drafts over 32000 tokens: 7.0 us, 4.2 and 3.0 the kernels alone), by
// reading two rows of each request for large ones (64 requests over 131072: 67
// MB in 15.7 us, 4.3 TB/s; 12.1 the sums).  A wave a chunk needs no barrier, and
// 20 + 20 bits in 32-bit sums half the instructions of 64-bit ones: 10.6 and
// 19.8 us before both.  Scans by lane shifts instead of LDS permutes: 7.4 and
// 16.3 before.
#include "glm53_common.h"

namespace glm53 {
namespace {

constexpr int kThreads = 256;
constexpr int kPerLane = 16;
constexpr int kChunk = 64 * kPerLane;      // vocabulary entries of a wave
constexpr int kDrawWaves = 8;

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
  struct Decision* decisions;   // [requests]
  uint64_t* sums;               // [requests][chunks]
};

__device__ __forceinline__ int64_t token_at(const VerifyArgs& a, int64_t i) {
  return a.ids_i64 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<int64_t>(static_cast<const int32_t*>(a.ids)[i]);
}

// floor(min(max(x, 0), 1) * 2^40), NaN as 0, as hi * 2^20 + lo: the products by
// 2^20 and the remainder between them are exact.
struct Weight {
  uint32_t hi, lo;
};
__device__ __forceinline__ Weight weight(float x) {
  const float t = fminf(fmaxf(x, 0.f), 1.f) * 1048576.f;
  return {static_cast<uint32_t>(t), static_cast<uint32_t>(__builtin_amdgcn_fractf(t) * 1048576.f)};
}
__device__ __forceinline__ uint64_t weight_of(Weight w) { return (static_cast<uint64_t>(w.hi) << 20) + w.lo; }

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
__device__ __forceinline__ Decision decide(const VerifyArgs& a, const int32_t* cu, int r, int lane) {
  const int64_t c0 = cu[r], c1 = cu[r + 1];
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

// Four entries from `at` on of what the next token is drawn from: of what is
// left of the target's row, or (`whole`) of the row itself.
struct Four {
  float v[4];
};
__device__ __forceinline__ Four load_four(const VerifyArgs& a, const Decision& d, int at, bool whole) {
  const float* p = a.target + d.row * a.st;
  const bool minus = !whole && d.place >= 0 && a.draft;
  const float* q = minus ? a.draft + d.place * a.sd : nullptr;
  Four r;
  if (at + 4 <= a.vocab) {
    const f32x4u v = *reinterpret_cast<const f32x4u*>(p + at);
    f32x4u u = {0.f, 0.f, 0.f, 0.f};
    if (minus) u = *reinterpret_cast<const f32x4u*>(q + at);
#pragma unroll
    for (int k = 0; k < 4; k++) r.v[k] = v[k] - u[k];
  } else {
#pragma unroll
    for (int k = 0; k < 4; k++) r.v[k] = at + k < a.vocab ? minus ? p[at + k] - q[at + k] : p[at + k] : 0.f;
  }
  if (!whole && d.place >= 0 && !a.draft) {
#pragma unroll
    for (int k = 0; k < 4; k++) r.v[k] = at + k == d.token ? 0.f : r.v[k];
  }
  return r;
}

template <int kCtrl>
__device__ __forceinline__ uint32_t add_dpp(uint32_t v) {
  return v + static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, 0xf, 0xf, true));
}
__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v) {
  v = add_dpp<0xb1>(v);    // lanes 1 apart, 2 apart (quad_perm),
  v = add_dpp<0x4e>(v);
  v = add_dpp<0x141>(v);   // the other four of eight, the other eight of a row (mirrors)
  v = add_dpp<0x140>(v);
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = a[0] + a[1];
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return b[0] + b[1];
}
// Inclusive sum over the wave: within rows of 16 lanes by shifts, then the last
// lane of row 0 (2) into row 1 (3) and that of row 1 into rows 2 and 3.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint64_t add_from(uint64_t v) {
  const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, kRows, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), kCtrl, kRows, 0xf, true);
  return v + (static_cast<uint32_t>(lo) | static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32);
}
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {
  v = add_from<0x111, 0xf>(v);
  v = add_from<0x112, 0xf>(v);
  v = add_from<0x114, 0xf>(v);
  v = add_from<0x118, 0xf>(v);
  v = add_from<0x142, 0xa>(v);
  return add_from<0x143, 0xc>(v);
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {   // of a lane that is the same in all
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane)) |
         static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane))) << 32;
}

// The sum of a wave's 1024 weights from `at` on.  1024 * 2^20 fits 32 bits.
__device__ __forceinline__ uint64_t chunk_sum(const VerifyArgs& a, const Decision& d, int at, bool whole, int lane) {
  Four v[kPerLane / 4];
#pragma unroll
  for (int k = 0; k < kPerLane / 4; k++) v[k] = load_four(a, d, at + 256 * k + 4 * lane, whole);
  uint32_t hi = 0, lo = 0;
#pragma unroll
  for (int k = 0; k < kPerLane / 4; k++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const Weight t = weight(v[k].v[e]);
      hi += t.hi, lo += t.lo;
    }
  return weight_of({wave_sum_u32(hi), wave_sum_u32(lo)});
}

// (The kernels' first loads' arguments lead: they come preloaded in registers.)
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(const int32_t* cu, int chunks, const VerifyArgs a) {
  const int r = blockIdx.y, lane = threadIdx.x & 63;
  const int chunk = blockIdx.x * (kThreads / 64) + uniform(threadIdx.x >> 6);
  if (chunk >= chunks) return;
  const Decision d = decide(a, cu, r, lane);
  if (chunk == 0 && lane == 0) a.decisions[r] = d;
  if (d.row < 0) return;
  const uint64_t s = chunk_sum(a, d, chunk * kChunk, false, lane);
  if (lane == 0) a.sums[static_cast<int64_t>(r) * a.chunks + chunk] = s;
}

// Where the running sum of `chunks` sums passes mark: the chunk, and the sum below it.
struct Place {
  int chunk;
  uint64_t below;
};
__device__ __forceinline__ Place find_chunk(const uint64_t* sums, int chunks, uint64_t mark, int lane) {
  uint64_t base = 0;
  for (int c0 = 0; c0 < chunks; c0 += 64) {
    const uint64_t v = c0 + lane < chunks ? sums[c0 + lane] : 0;
    const uint64_t upto = base + wave_scan_u64(v);
    const uint64_t past = __ballot(upto > mark);
    if (past) {
      const int l = __builtin_ctzll(past);
      return {c0 + l, lane_u64(upto - v, l)};
    }
    base = lane_u64(upto, 63);
  }
  return {-1, 0};
}

__global__ __launch_bounds__(64 * kDrawWaves) void verify_draw_kernel(const Decision* decisions, const double* sample_u, uint64_t* all_sums,
                                                                      int chunks, const VerifyArgs a) {
  __shared__ uint64_t part[kDrawWaves];
  const int r = blockIdx.x, lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
  uint64_t* sums = all_sums + static_cast<int64_t>(r) * chunks;
  uint64_t total = 0;
  const Decision d = decisions[r];
  const double s = sample_u[r];
  int token = -1;
  if (d.row >= 0) {   // uniform over the workgroup
    for (int i = lane; i < chunks; i += 64) total += sums[i];
    total = lane_u64(wave_scan_u64(total), 63);
    const bool whole = total == 0 && d.place >= 0;
    if (whole) {
      // nothing is left: the target's own weights, into the sums of the others
      __syncthreads();   // (which every wave has read)
      for (int c = w; c < chunks; c += kDrawWaves) {
        const uint64_t v = chunk_sum(a, d, c * kChunk, true, lane);
        total += v;
        if (lane == 0) sums[c] = v;
      }
      if (lane == 0) part[w] = total;
      __syncthreads();   // and so are the sums in memory, for this workgroup
      total = 0;
      for (int i = 0; i < kDrawWaves; i++) total += part[i];
    }
    if (w == 0 && total) {
      const double f = floor(s * static_cast<double>(total));
      uint64_t mark = f > 0. ? (f < static_cast<double>(total) ? static_cast<uint64_t>(f) : total - 1) : 0;
      if (mark >= total) mark = total - 1;
      const Place at = find_chunk(sums, chunks, mark, lane);
      // in the chunk (none only if the sums passed 64 bits): 16 entries a lane, in order
      const int first = at.chunk < 0 ? a.vocab : at.chunk * kChunk + kPerLane * lane;
      uint64_t v[kPerLane], sum = 0;
#pragma unroll
      for (int k = 0; k < kPerLane; k += 4) {
        const Four t = load_four(a, d, first + k, whole);
#pragma unroll
        for (int e = 0; e < 4; e++) sum += v[k + e] = weight_of(weight(t.v[e]));
      }
      uint64_t upto = at.below + wave_scan_u64(sum) - sum;
      int found = -1;
#pragma unroll
      for (int k = 0; k < kPerLane; k++) {
        if (upto <= mark && mark < upto + v[k]) found = first + k;
        upto += v[k];
      }
      const uint64_t has = __ballot(found >= 0);
      token = has ? __builtin_amdgcn_readlane(found, __builtin_ctzll(has)) : -1;
    }
  }
  if (w) return;
  int32_t* out = a.tokens + static_cast<int64_t>(r) * (static_cast<int64_t>(a.max_drafts) + 1);
  for (int64_t j = lane; j <= a.max_drafts; j += 64)
    out[j] = d.row < 0 || j > d.count ? -1 : j == d.count ? token : static_cast<int32_t>(token_at(a, d.first + j));
  if (lane == 0) a.accepted[r] = d.count;
}

}  // namespace
}  // namespace glm53

using namespace glm53;

extern "C" int64_t glm53_verify_drafts_workspace_bytes(int64_t num_requests, int64_t vocab) {
  if (num_requests <= 0 || vocab <= 0) return 0;
  return num_requests * (static_cast<int64_t>(sizeof(Decision)) + (vocab + kChunk - 1) / kChunk * 8);
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
  a.tokens = tokens, a.accepted = accepted, a.decisions = static_cast<Decision*>(workspace);
  a.sums = reinterpret_cast<uint64_t*>(a.decisions + num_requests);
  hipStream_t s = static_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  hipLaunchKernelGGL(verify_sums_kernel, dim3((a.chunks + kThreads / 64 - 1) / (kThreads / 64), static_cast<unsigned>(num_requests)),
                     dim3(kThreads), 0, s, a.cu, a.chunks, a);
  hipLaunchKernelGGL(verify_draw_kernel, dim3(static_cast<unsigned>(num_requests)), dim3(64 * kDrawWaves), 0, s,
                     a.decisions, a.sample_u, a.sums, a.chunks, a);
  return static_cast<int>(hipGetLastError());
}
