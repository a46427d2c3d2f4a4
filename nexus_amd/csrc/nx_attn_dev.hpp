// nx_attn_dev.hpp — what the attention (nx_attn.hip) and the weight that it gives each cached
// token (nx_mass.hip) share: f32 queries as two f16 halves, operands out of the cache, and
// exchanges between a wave's lane groups.
#pragma once

#include "nx_kv_dev.hpp"
#include "nx_split_dev.hpp"

namespace nx {

// row / group for 0 <= row < 2^31, by magic = ceil(2^(31 + shift) / group) and shift =
// ceil(log2 group): magic group - 2^(31 + shift) < 2^shift, so the
// quotient's excess row (magic group - 2^(31 + shift)) / 2^(31 + shift) is below 1 / group's step
__device__ __forceinline__ int by_group(int row, uint32_t magic, int shift) {
  return (int)(__umulhi(2u * (uint32_t)row, magic) >> shift);
}
inline int group_shift(int group) { return group > 1 ? 32 - __builtin_clz(group - 1) : 0; }
inline uint32_t group_magic(int group) {
  return (uint32_t)((((uint64_t)1 << (31 + group_shift(group))) + group - 1) / group);
}

constexpr float kLog2e = 1.4426950408889634f;

// int8 code -> f16 q 2^-9, exact: 0x80 ^ code as the low bits of a subnormal half
__device__ __forceinline__ f16x8 from_codes(uint32_t lo, uint32_t hi) { return operand8(lo, hi); }

__device__ __forceinline__ float ldexp1(float x, int e) { return __builtin_amdgcn_ldexpf(x, e); }

// 8 values as two halves each, x = hi + lo to 22 bits.  `one` is 1 that the compiler
// does not know: x one - hi is then one instruction that reads the packed half.
__device__ __forceinline__ void split2(const float (&x)[8], float one, f16x8 &h, f16x8 &l) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  f16x2 hi[4], lo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hi[i] = __builtin_convertvector((f32x2{x[2 * i], x[2 * i + 1]}), f16x2);
    asm("" : "+v"(hi[i]));  // converted once, packed
    lo[i] = __builtin_convertvector(
        (f32x2{fmaf(x[2 * i], one, -(float)hi[i][0]), fmaf(x[2 * i + 1], one, -(float)hi[i][1])}), f16x2);
  }
  h = f16x8{hi[0][0], hi[0][1], hi[1][0], hi[1][1], hi[2][0], hi[2][1], hi[3][0], hi[3][1]};
  l = f16x8{lo[0][0], lo[0][1], lo[1][0], lo[1][1], lo[2][0], lo[2][1], lo[3][0], lo[3][1]};
}
__device__ __forceinline__ void load8(const float *p, bool wide, float (&x)[8]) {
  if (wide) {
    const f32x4 lo = *reinterpret_cast<const f32x4 *>(p), hi = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = lo[i];
      x[4 + i] = hi[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[i];
  }
}
__device__ __forceinline__ float opaque_one() {
  float one = 1.f;
  asm("" : "+s"(one));
  return one;
}

// the largest (sum) over the four lane groups, in all of them
template <typename Op>
__device__ __forceinline__ float across_groups(float v, Op op) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float max_groups(float v) {
  return across_groups(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float sum_groups(float v) {
  return across_groups(v, [](float a, float b) { return a + b; });
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

// the other half of the wave's value
template <typename Op>
__device__ __forceinline__ float across_halves(float v, Op op) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

__device__ __forceinline__ float max_halves(float v) {
  return across_halves(v, [](float x, float y) { return fmaxf(x, y); });
}

}  // namespace nx
