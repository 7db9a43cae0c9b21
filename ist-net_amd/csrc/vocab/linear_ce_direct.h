// Shared by the paths of the cross entropy that read their operands as they lie (linear_ce_few.hip, linear_ce_classes.hip): products of
// 16 x 16 straight from memory.
#pragma once
#include "vocab_common.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

// one step of K: 64 bytes of a row, lane group g = lane / 16 has sixteen of them; which K they are does not matter as long as both
// operands agree
template <typename T> constexpr int kStep = 64 / (int)sizeof(T);
template <typename T> __device__ __forceinline__ f32x4 multiply(const u32x4& a, const u32x4& b, f32x4 c) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[k]), __uint_as_float(b[k]), c, 0, 0, 0);
    return c;
  } else if constexpr (__is_same(T, bf16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
  }
}
// sixteen bytes of which `left` elements belong to the row, zeros behind them
template <typename T> __device__ __forceinline__ u32x4 load_raw(const T* p, int left) {
  float f[kVec<T>];
  load_part(p, left, f);
  return pack<T>(f);
}

inline long long round_up(long long x, long long m) { return (x + m - 1) / m * m; }

}  // namespace
