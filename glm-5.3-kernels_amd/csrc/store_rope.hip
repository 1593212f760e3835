// Appending to a paged bf16 latent cache with the rotation on the way, for
// gfx950.
//
// Token i with position p = pos[i] and slot s = slots[i]: the 576-wide row s
// of the cache becomes
//   [ y(512) | rotate(k_pe[i], p) ],   y = x                                 (no norm)
//                                      y = x * w / sqrt(mean(x^2) + eps)     (RMS norm)
// and the queries' rotary parts q_out[i, h] = rotate(q_pe[i, h], p).  With the
// table's row p = (cos_0 .. cos_31 | sin_0 .. sin_31), rotate turns the pairs
// (a_k, b_k) - values k and 32 + k, or 2k and 2k + 1 (interleaved) - into
// (a cos - b sin, b cos + a sin).  All in fp32, rounded to bf16 once.
//
// Layout: a wave takes the latents of kRows tokens (lane l: values 8l .. 8l + 7
// of each, all loaded before any is stored) and, eight lanes a token, their
// rotary keys; further waves take eight query heads of the tokens each, eight
// lanes a head, four pairs a lane.  The table's row is read where it is used
// (it stays in the L2).
//
// Bound by memory from some thousand tokens on, by the launch and one chain of
// dependent loads (the position, then its table row) below.  From kManyTokens
// on a wave takes four tokens, so that more loads are on their way, and what
// passes through does so non-temporally: 65536 tokens without queries, from
// inputs that no cache holds, 39.8 us with one token a wave, 34.1 with four,
// 30.5 non-temporally too (5.3 TB/s); 8192 tokens 6.8, 6.6 and 5.4 us, with
// normalised latents and 16 query heads 14.0, 11.7 and 12.0.  Fewer tokens are
// better spread over more waves (2048 with 16 heads: 4.7 us with one, 5.5 with
// four) and left in the caches for the attention that reads them next.
#include "glm53_common.h"

namespace glm53 {
namespace {

constexpr int kLatent = 512;
constexpr int kRope = 64;
constexpr int kWavesPerBlock = 4;
constexpr int kHeadsPerWave = 8;
constexpr int kManyRows = 4;             // tokens of a wave in calls of at least
constexpr int64_t kManyTokens = 8192;    // so many tokens, which pass through non-temporally

struct RopeArgs {
  const uint16_t* x;
  int64_t sx;
  const uint16_t* k_pe;
  int64_t sk;
  const void* pos;
  const void* slots;
  int pos_i64, slots_i64, table_f32, interleaved;
  const void* table;   // [max_pos][64]
  int64_t max_pos;
  const uint16_t* norm;   // 512 weights, or null
  float eps;
  uint8_t* cache;
  int64_t page_bytes, row_bytes, capacity;
  uint32_t block_size;
  Divider by_block;
  const uint16_t* q_pe;
  int64_t sq_t, sq_h;
  uint16_t* q_out;
  int64_t so_t, so_h;
  int heads;
  int64_t n;
};

__device__ __forceinline__ int64_t index_at(const void* p, int i64, int64_t i) {
  return i64 ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}

template <int kCtrl>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), kCtrl, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float v) {
  v = add_dpp<0xb1>(v);    // lanes 1 apart, 2 apart (quad_perm),
  v = add_dpp<0x4e>(v);
  v = add_dpp<0x141>(v);   // the other four of eight, the other eight of a row (mirrors)
  v = add_dpp<0x140>(v);
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

template <bool kStream, class T>
__device__ __forceinline__ T load(const T* p) {
  if constexpr (kStream) return __builtin_nontemporal_load(p);
  return *p;
}
template <bool kStream, class T>
__device__ __forceinline__ void store(T* p, T v) {
  if constexpr (kStream)
    __builtin_nontemporal_store(v, p);
  else
    *p = v;
}

struct Pairs {
  float a[4], b[4];
};

// Pairs 4j .. 4j + 3 of the 64 values at p.
template <bool kStream>
__device__ __forceinline__ Pairs load_pairs(const uint16_t* p, int j, int interleaved) {
  u32x2 u, v;
  if (interleaved) {
    const u32x4 t = load<kStream>(reinterpret_cast<const u32x4*>(p + 8 * j));
    u = u32x2{__builtin_amdgcn_perm(t.y, t.x, 0x05040100u), __builtin_amdgcn_perm(t.w, t.z, 0x05040100u)};
    v = u32x2{__builtin_amdgcn_perm(t.y, t.x, 0x07060302u), __builtin_amdgcn_perm(t.w, t.z, 0x07060302u)};
  } else {
    u = load<kStream>(reinterpret_cast<const u32x2*>(p + 4 * j));
    v = load<kStream>(reinterpret_cast<const u32x2*>(p + kRope / 2 + 4 * j));
  }
  Pairs r;
  r.a[0] = bf16_bits_to_f32(u.x & 0xffffu), r.a[1] = __uint_as_float(u.x & 0xffff0000u);
  r.a[2] = bf16_bits_to_f32(u.y & 0xffffu), r.a[3] = __uint_as_float(u.y & 0xffff0000u);
  r.b[0] = bf16_bits_to_f32(v.x & 0xffffu), r.b[1] = __uint_as_float(v.x & 0xffff0000u);
  r.b[2] = bf16_bits_to_f32(v.y & 0xffffu), r.b[3] = __uint_as_float(v.y & 0xffff0000u);
  return r;
}

__device__ __forceinline__ Pairs load_angles(const RopeArgs& a, int64_t pos, int j) {
  Pairs r;
  if (a.table_f32) {
    const float* t = static_cast<const float*>(a.table) + pos * kRope + 4 * j;
    const float4 u = *reinterpret_cast<const float4*>(t), v = *reinterpret_cast<const float4*>(t + kRope / 2);
    r.a[0] = u.x, r.a[1] = u.y, r.a[2] = u.z, r.a[3] = u.w;
    r.b[0] = v.x, r.b[1] = v.y, r.b[2] = v.z, r.b[3] = v.w;
    return r;
  }
  return load_pairs<false>(static_cast<const uint16_t*>(a.table) + pos * kRope, j, 0);
}

template <bool kStream>
__device__ __forceinline__ void store_rotated(uint16_t* o, int j, int interleaved, const Pairs& p, const Pairs& t) {
  float u[4], v[4];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    u[k] = p.a[k] * t.a[k] - p.b[k] * t.b[k];
    v[k] = p.b[k] * t.a[k] + p.a[k] * t.b[k];
  }
  if (interleaved) {
    store<kStream>(reinterpret_cast<u32x4*>(o + 8 * j), u32x4{pack_bf16x2(u[0], v[0]), pack_bf16x2(u[1], v[1]),
                                                              pack_bf16x2(u[2], v[2]), pack_bf16x2(u[3], v[3])});
  } else {
    store<kStream>(reinterpret_cast<u32x2*>(o + 4 * j), u32x2{pack_bf16x2(u[0], u[1]), pack_bf16x2(u[2], u[3])});
    store<kStream>(reinterpret_cast<u32x2*>(o + kRope / 2 + 4 * j), u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])});
  }
}

// (The arguments of the first loads lead: they come preloaded in registers.)
template <int kRows, bool kStream>
__global__ __launch_bounds__(64 * kWavesPerBlock) void store_rope_kernel(const void* positions, const void* slots, int64_t n,
                                                                       const uint16_t* x, int64_t sx, int wide,
                                                                       const RopeArgs a) {
  static_assert(kRows <= 8, "eight lanes a token's rotary key");
  const int lane = threadIdx.x & 63, part = blockIdx.y;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + uniform(threadIdx.x >> 6)) * kRows;
  if (first >= n) return;
  const int count = n - first < kRows ? static_cast<int>(n - first) : kRows;
  const int j = lane & 7;
  if (part == 0) {
    // lanes 8 k .. 8 k + 7 look after token k (the last ones after the last)
    const int mine = min(lane >> 3, count - 1);
    const int64_t pos = index_at(positions, wide & 1, first + mine);
    const int64_t slot = index_at(slots, wide & 2, first + mine);
    u32x4 v[kRows], weight = {};
#pragma unroll
    for (int k = 0; k < kRows; k++)
      v[k] = load<kStream>(reinterpret_cast<const u32x4*>(x + (first + min(k, count - 1)) * sx + 8 * lane));
    if (a.norm) weight = *reinterpret_cast<const u32x4*>(a.norm + 8 * lane);
    Pairs key = {};
    if (lane < 8 * count) key = load_pairs<kStream>(a.k_pe + (first + mine) * a.sk, j, a.interleaved);
    // a position outside the table, a slot outside the cache: the row stays
    const bool ok = pos >= 0 && pos < a.max_pos && slot >= 0 && slot < a.capacity;
    const uint32_t at = ok ? static_cast<uint32_t>(slot) : 0, page = divide(at, a.by_block);
    const int64_t row = page * a.page_bytes + (at - page * a.block_size) * a.row_bytes;
    if (lane < 8 * count && ok)
      store_rotated<kStream>(reinterpret_cast<uint16_t*>(a.cache + row) + kLatent, j, a.interleaved, key, load_angles(a, pos, j));
    const uint64_t there = __ballot(ok && lane < 8 * count);
    const int row_lo = static_cast<int>(row), row_hi = static_cast<int>(row >> 32);
#pragma unroll
    for (int k = 0; k < kRows; k++) {
      if (!(there >> (8 * k) & 1)) continue;   // uniform
      u32x4 o = v[k];
      if (a.norm) {
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float lo = __uint_as_float(o[i] << 16), hi = __uint_as_float(o[i] & 0xffff0000u);
          sq += lo * lo;
          sq += hi * hi;
        }
        const float inv = 1.f / sqrtf(wave_sum(sq) * (1.f / kLatent) + a.eps);
#pragma unroll
        for (int i = 0; i < 4; i++)
          o[i] = pack_bf16x2(__uint_as_float(o[i] << 16) * inv * __uint_as_float(weight[i] << 16),
                             __uint_as_float(o[i] & 0xffff0000u) * inv * __uint_as_float(weight[i] & 0xffff0000u));
      }
      const int64_t to = static_cast<uint32_t>(__builtin_amdgcn_readlane(row_lo, 8 * k)) |
                         static_cast<int64_t>(__builtin_amdgcn_readlane(row_hi, 8 * k)) << 32;
      store<kStream>(reinterpret_cast<u32x4*>(a.cache + to) + lane, o);
    }
    return;
  }
  const int head = kHeadsPerWave * (part - 1) + (lane >> 3);
  if (head >= a.heads) return;
  int64_t pos[kRows];
  Pairs q[kRows];
#pragma unroll
  for (int k = 0; k < kRows; k++) {
    const int64_t tok = first + min(k, count - 1);
    pos[k] = index_at(positions, wide & 1, tok);
    q[k] = load_pairs<kStream>(a.q_pe + tok * a.sq_t + head * a.sq_h, j, a.interleaved);
  }
#pragma unroll
  for (int k = 0; k < kRows; k++) {
    if (k >= count) break;
    uint16_t* o = a.q_out + (first + k) * a.so_t + head * a.so_h;
    if (pos[k] >= 0 && pos[k] < a.max_pos)
      store_rotated<kStream>(o, j, a.interleaved, q[k], load_angles(a, pos[k], j));
    else
      store<kStream>(reinterpret_cast<u32x4*>(o + 8 * j), u32x4{0, 0, 0, 0});
  }
}

template <int kRows, bool kStream>
int launch(const RopeArgs& a, hipStream_t st) {
  const int64_t rows = kRows * kWavesPerBlock, grid = (a.n + rows - 1) / rows;
  if (grid > 0x7fffffff) return GLM53_ERR_BAD_SHAPE;
  const unsigned parts = 1 + (a.heads + kHeadsPerWave - 1) / kHeadsPerWave;
  (void)hipGetLastError();
  hipLaunchKernelGGL((store_rope_kernel<kRows, kStream>), dim3(static_cast<unsigned>(grid), parts), dim3(64 * kWavesPerBlock), 0,
                     st, a.pos, a.slots, a.n, a.x, a.sx, (a.pos_i64 ? 1 : 0) | (a.slots_i64 ? 2 : 0), a);
  return static_cast<int>(hipGetLastError());
}

}  // namespace
}  // namespace glm53

using namespace glm53;

extern "C" int glm53_store_rope(const void* x, int64_t x_row_stride, const void* k_pe, int64_t k_row_stride,
                                const void* positions, int positions_is_i64, const void* cos_sin, int cos_sin_is_f32,
                                int64_t max_pos, int interleaved, const void* norm_weight, float eps, void* cache,
                                int64_t cache_stride_block, int64_t cache_stride_slot, int64_t block_size,
                                int64_t capacity, const void* slots, int slots_is_i64, int64_t n_slots,
                                const void* q_pe, int64_t sq_t, int64_t sq_h, void* q_out, int64_t so_t, int64_t so_h,
                                int64_t num_heads, void* stream) {
  if (n_slots < 0 || block_size <= 0 || max_pos < 0 || num_heads < 0 || capacity < 0 || num_heads > 65536)
    return GLM53_ERR_BAD_SHAPE;
  // rows of a cache are counted in 32 bits (so many rows of 1152 bytes are 4.9 TB)
  if (capacity > 0xffffffffll || block_size > 0xffffffffll) return GLM53_ERR_BAD_SHAPE;
  if (n_slots == 0) return 0;
  if (!x || !k_pe || !positions || (max_pos && !cos_sin) || (capacity && !cache) || !slots || (num_heads && (!q_pe || !q_out)))
    return GLM53_ERR_NULL_POINTER;
  const auto off = [](const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % 16 || n % 16; };
  if (off(x, 2 * x_row_stride) || off(k_pe, 2 * k_row_stride) || off(cos_sin, 0) || off(norm_weight, 0) ||
      off(cache, cache_stride_block) || off(cache, cache_stride_slot))
    return GLM53_ERR_MISALIGNED;
  if (num_heads && (off(q_pe, 2 * sq_t) || off(q_pe, 2 * sq_h) || off(q_out, 2 * so_t) || off(q_out, 2 * so_h)))
    return GLM53_ERR_MISALIGNED;
  RopeArgs a = {};
  a.x = static_cast<const uint16_t*>(x), a.sx = x_row_stride;
  a.k_pe = static_cast<const uint16_t*>(k_pe), a.sk = k_row_stride;
  a.pos = positions, a.pos_i64 = positions_is_i64;
  a.slots = slots, a.slots_i64 = slots_is_i64;
  a.table = cos_sin, a.table_f32 = cos_sin_is_f32, a.max_pos = max_pos;
  a.interleaved = interleaved;
  a.norm = static_cast<const uint16_t*>(norm_weight), a.eps = eps;
  a.cache = static_cast<uint8_t*>(cache);
  a.page_bytes = cache_stride_block, a.row_bytes = cache_stride_slot, a.capacity = capacity;
  a.block_size = static_cast<uint32_t>(block_size), a.by_block = divider(block_size);
  a.q_pe = static_cast<const uint16_t*>(q_pe), a.sq_t = sq_t, a.sq_h = sq_h;
  a.q_out = static_cast<uint16_t*>(q_out), a.so_t = so_t, a.so_h = so_h;
  a.heads = static_cast<int>(num_heads);
  a.n = n_slots;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return n_slots >= kManyTokens ? launch<kManyRows, true>(a, st) : launch<1, false>(a, st);
}
