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
// Layout: a wave takes a token's latent (lane l: values 8l .. 8l + 7) and, in
// lanes 0 .. 7, its rotary key; further waves take eight query heads of the
// token each, eight lanes a head, four pairs a lane.  The table's row is read
// where it is used (it stays in the L2).
#include "glm53_common.h"

namespace glm53 {
namespace {

constexpr int kLatent = 512;
constexpr int kRope = 64;
constexpr int kWidth = kLatent + kRope;
constexpr int kWavesPerBlock = 4;
constexpr int kHeadsPerWave = 8;

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
  int64_t page_bytes, row_bytes, block_size, capacity;
  const uint16_t* q_pe;
  int64_t sq_t, sq_h;
  uint16_t* q_out;
  int64_t so_t, so_h;
  int heads;
  int parts;   // waves per token: 1 + ceil(heads / 8)
  int64_t n;
};

__device__ __forceinline__ int64_t index_at(const void* p, int i64, int64_t i) {
  return i64 ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

struct Pairs {
  float a[4], b[4];
};

// Pairs 4j .. 4j + 3 of the 64 values at p.
__device__ __forceinline__ Pairs load_pairs(const uint16_t* p, int j, int interleaved) {
  uint2 u, v;
  if (interleaved) {
    const uint4 t = *reinterpret_cast<const uint4*>(p + 8 * j);
    u = make_uint2(__builtin_amdgcn_perm(t.y, t.x, 0x05040100u), __builtin_amdgcn_perm(t.w, t.z, 0x05040100u));
    v = make_uint2(__builtin_amdgcn_perm(t.y, t.x, 0x07060302u), __builtin_amdgcn_perm(t.w, t.z, 0x07060302u));
  } else {
    u = *reinterpret_cast<const uint2*>(p + 4 * j);
    v = *reinterpret_cast<const uint2*>(p + kRope / 2 + 4 * j);
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
  return load_pairs(static_cast<const uint16_t*>(a.table) + pos * kRope, j, 0);
}

__device__ __forceinline__ void store_rotated(uint16_t* o, int j, int interleaved, const Pairs& p, const Pairs& t) {
  float u[4], v[4];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    u[k] = p.a[k] * t.a[k] - p.b[k] * t.b[k];
    v[k] = p.b[k] * t.a[k] + p.a[k] * t.b[k];
  }
  if (interleaved) {
    *reinterpret_cast<uint4*>(o + 8 * j) = make_uint4(pack_bf16x2(u[0], v[0]), pack_bf16x2(u[1], v[1]),
                                                      pack_bf16x2(u[2], v[2]), pack_bf16x2(u[3], v[3]));
  } else {
    *reinterpret_cast<uint2*>(o + 4 * j) = make_uint2(pack_bf16x2(u[0], u[1]), pack_bf16x2(u[2], u[3]));
    *reinterpret_cast<uint2*>(o + kRope / 2 + 4 * j) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  }
}

__global__ __launch_bounds__(64 * kWavesPerBlock) void store_rope_kernel(const RopeArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + uniform(threadIdx.x >> 6);
  const int64_t tok = unit / a.parts;
  const int part = static_cast<int>(unit - tok * a.parts);
  if (tok >= a.n) return;
  const int64_t pos = index_at(a.pos, a.pos_i64, tok);
  const bool known = pos >= 0 && pos < a.max_pos;   // a position outside the table
  const int j = lane & 7;
  if (part == 0) {
    const uint4 v = *reinterpret_cast<const uint4*>(a.x + tok * a.sx + 8 * lane);
    const int64_t slot = index_at(a.slots, a.slots_i64, tok);
    if (!known || slot < 0 || slot >= a.capacity) return;
    uint16_t* row = reinterpret_cast<uint16_t*>(a.cache + slot / a.block_size * a.page_bytes +
                                                slot % a.block_size * a.row_bytes);
    if (lane < 8) {
      const Pairs k = load_pairs(a.k_pe + tok * a.sk, j, a.interleaved);
      store_rotated(row + kLatent, j, a.interleaved, k, load_angles(a, pos, j));
    }
    uint4 o = v;
    if (a.norm) {
      const uint4 w = *reinterpret_cast<const uint4*>(a.norm + 8 * lane);
      const uint32_t vs[4] = {v.x, v.y, v.z, v.w}, ws[4] = {w.x, w.y, w.z, w.w};
      float sq = 0.f;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float lo = __uint_as_float(vs[k] << 16), hi = __uint_as_float(vs[k] & 0xffff0000u);
        sq += lo * lo;
        sq += hi * hi;
      }
      const float inv = 1.f / sqrtf(wave_sum(sq) * (1.f / kLatent) + a.eps);
      uint32_t os[4];
#pragma unroll
      for (int k = 0; k < 4; k++)
        os[k] = pack_bf16x2(__uint_as_float(vs[k] << 16) * inv * __uint_as_float(ws[k] << 16),
                            __uint_as_float(vs[k] & 0xffff0000u) * inv * __uint_as_float(ws[k] & 0xffff0000u));
      o = make_uint4(os[0], os[1], os[2], os[3]);
    }
    *reinterpret_cast<uint4*>(row + 8 * lane) = o;
    return;
  }
  const int head = kHeadsPerWave * (part - 1) + (lane >> 3);
  if (head >= a.heads) return;
  uint16_t* o = a.q_out + tok * a.so_t + head * a.so_h;
  if (!known) {
    *reinterpret_cast<uint4*>(o + 8 * j) = make_uint4(0, 0, 0, 0);
    return;
  }
  const Pairs q = load_pairs(a.q_pe + tok * a.sq_t + head * a.sq_h, j, a.interleaved);
  store_rotated(o, j, a.interleaved, q, load_angles(a, pos, j));
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
  if (n_slots == 0) return 0;
  if (!x || !k_pe || !positions || !cos_sin || !cache || !slots || (num_heads && (!q_pe || !q_out)))
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
  a.page_bytes = cache_stride_block, a.row_bytes = cache_stride_slot, a.block_size = block_size, a.capacity = capacity;
  a.q_pe = static_cast<const uint16_t*>(q_pe), a.sq_t = sq_t, a.sq_h = sq_h;
  a.q_out = static_cast<uint16_t*>(q_out), a.so_t = so_t, a.so_h = so_h;
  a.heads = static_cast<int>(num_heads);
  a.parts = static_cast<int>(1 + (num_heads + kHeadsPerWave - 1) / kHeadsPerWave);
  a.n = n_slots;
  if (n_slots > (INT64_C(1) << 40) / a.parts) return GLM53_ERR_BAD_SHAPE;
  const int64_t grid = (n_slots * a.parts + kWavesPerBlock - 1) / kWavesPerBlock;
  if (grid > 0x7fffffff) return GLM53_ERR_BAD_SHAPE;
  (void)hipGetLastError();
  hipLaunchKernelGGL(store_rope_kernel, dim3(static_cast<unsigned>(grid)), dim3(64 * kWavesPerBlock), 0,
                     static_cast<hipStream_t>(stream), a);
  return static_cast<int>(hipGetLastError());
}
