// Shared device helpers for the gfx950 kernels of libglm53_hip.so.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

#include "glm53.h"

namespace glm53 {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4;
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short i16x4;
typedef __attribute__((__vector_size__(2 * sizeof(int)))) int i32x2;
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

#define GLM53_LDS(T, p) ((__attribute__((address_space(3))) T*)(p))

__device__ __forceinline__ float bf16_bits_to_f32(uint32_t h) { return __uint_as_float(h << 16); }

// fp32 -> bf16 bits, round to nearest even (finite inputs).
__device__ __forceinline__ uint32_t f32_to_bf16_bits(float f) {
  uint32_t u = __float_as_uint(f);
  return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}

// Pack two fp32 into a dword of two bf16 (lo in bits 0..15), round to
// nearest even: one v_cvt_pk_bf16_f32 on gfx950 (same bits as
// f32_to_bf16_bits for finite inputs; NaN stays NaN).
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t f = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2_t));
}

// Wave-uniform value in a scalar register.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Maximum over the wave, returned to every lane, without LDS traffic: DPP
// quad permutes and row rotations inside each 16-lane row, then
// v_permlane16_swap / v_permlane32_swap across the four rows.
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  auto mx = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  v = mx(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xB1, 0xF, 0xF, false)));   // lane ^ 1
  v = mx(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4E, 0xF, 0xF, false)));   // lane ^ 2
  v = mx(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x124, 0xF, 0xF, false)));  // row_ror 4
  v = mx(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x128, 0xF, 0xF, false)));  // row_ror 8
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = mx(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return mx(b[0], b[1]);
}

// n / d of 32-bit numbers by multiplication (Granlund and Montgomery's method):
// with l = ceil(log2 d), mul = floor(2^32 (2^l - d) / d) + 1.
struct Divider {
  uint32_t mul;
  int sh1, sh2;
};
inline Divider divider(int64_t d) {
  int l = 0;
  while ((INT64_C(1) << l) < d) l++;
  const uint64_t mul = ((uint64_t(1) << l) - static_cast<uint64_t>(d)) * (uint64_t(1) << 32) / static_cast<uint64_t>(d) + 1;
  return {static_cast<uint32_t>(mul), l < 1 ? l : 1, l > 1 ? l - 1 : 0};
}
__device__ __forceinline__ uint32_t divide(uint32_t n, const Divider& d) {
  const uint32_t t = static_cast<uint32_t>(static_cast<uint64_t>(d.mul) * n >> 32);
  return (t + ((n - t) >> d.sh1)) >> d.sh2;
}

// Compute units of the current device (looked up once per device).
inline int num_cus() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (!n) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1) n = 256;
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace glm53
