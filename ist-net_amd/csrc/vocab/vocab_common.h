// Shared by the kernels of include/istnet_vocab.h: element types, unaligned 16-byte accesses, wave and workgroup reductions.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../../include/istnet_vocab.h"

// The cross entropy of few rows (linear_ce_few.hip), of few classes (linear_ce_classes.hip) and of small problems
// (linear_ce_small.hip), called by the entry points of linear_ce.hip.
constexpr int kFewRowsCe = 32;
long long vocab_few_ce_keep(long long n, int v, int train);
long long vocab_few_ce_scratch(long long n, int d, int v, int dtype, int backward);
int vocab_few_ce_forward(int n, int d, int v, int dtype, int idx64, int train, const void* x, long long ldx, const void* w,
                         long long ldw, const void* bias, const void* target, long long ignore, int reduction, float* loss, void* keep,
                         void* ws, hipStream_t st);
int vocab_few_ce_backward(int n, int d, int v, int dtype, const void* x, long long ldx, const void* w, long long ldw, int reduction,
                          const float* gout, const void* keep, void* ws, void* dx, void* dw, void* db, hipStream_t st);
long long vocab_class_ce_keep(long long n, int v, int train);
long long vocab_class_ce_scratch(long long n, int d, int v, int dtype, int backward);
int vocab_class_ce_forward(int n, int d, int v, int dtype, int idx64, int train, const void* x, long long ldx, const void* w,
                           long long ldw, const void* bias, const void* target, long long ignore, int reduction, float* loss, void* keep,
                           void* ws, hipStream_t st);
int vocab_class_ce_backward(int n, int d, int v, int dtype, const void* x, long long ldx, const void* w, long long ldw, int reduction,
                            const float* gout, const void* keep, void* ws, void* dx, void* dw, void* db, hipStream_t st);
long long vocab_small_ce_keep(long long n, int v);
int vocab_small_ce_forward(int n, int d, int v, int dtype, int idx64, const void* x, long long ldx, const void* w, long long ldw,
                           const void* bias, const void* target, long long ignore, int reduction, float* loss, void* keep, hipStream_t st);
int vocab_small_ce_backward(int n, int d, int v, int dtype, const void* x, long long ldx, const void* w, long long ldw, int reduction,
                            const float* gout, const void* keep, void* dx, void* dw, void* db, hipStream_t st);

namespace {

constexpr float kNaN = __builtin_nanf("");

typedef _Float16 f16;
struct bf16 { uint16_t u; };

// sixteen and eight bytes at any element boundary: gfx950 loads and stores them with one instruction whatever the address
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
struct __attribute__((packed, aligned(2))) Raw16 { u32x4 v; };
struct __attribute__((packed, aligned(2))) Raw8 { u32x2 v; };

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(f16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __uint_as_float((uint32_t)x.u << 16); }
// float -> bf16 to nearest even (NaN stays NaN)
__device__ __forceinline__ uint16_t bf16_bits(float x) {
  uint32_t u = __float_as_uint(x);
  const uint32_t r = u + 0x7fffu + ((u >> 16) & 1u);
  return (x != x) ? (uint16_t)0x7fc0u : (uint16_t)(r >> 16);
}
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ f16 from_f32<f16>(float x) { return (f16)x; }
template <> __device__ __forceinline__ bf16 from_f32<bf16>(float x) { return bf16{bf16_bits(x)}; }

// elements in sixteen bytes
template <typename T> constexpr int kVec = 16 / (int)sizeof(T);

template <typename T> __device__ __forceinline__ void unpack(const u32x4& r, float (&f)[kVec<T>]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(r[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (__is_same(T, bf16)) {
        f[2 * i] = __uint_as_float(r[i] << 16);
        f[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
      } else {
        f[2 * i] = (float)__builtin_bit_cast(f16, (uint16_t)(r[i] & 0xffffu));
        f[2 * i + 1] = (float)__builtin_bit_cast(f16, (uint16_t)(r[i] >> 16));
      }
    }
  }
}
template <typename T> __device__ __forceinline__ u32x4 pack(const float (&f)[kVec<T>]) {
  u32x4 r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t a = __builtin_bit_cast(uint16_t, from_f32<T>(f[2 * i]));
      const uint16_t b = __builtin_bit_cast(uint16_t, from_f32<T>(f[2 * i + 1]));
      r[i] = (uint32_t)a | ((uint32_t)b << 16);
    }
  }
  return r;
}
template <typename T> __device__ __forceinline__ u32x4 load16(const T* p) { return reinterpret_cast<const Raw16*>(p)->v; }
template <typename T> __device__ __forceinline__ void store16(T* p, const u32x4& r) { reinterpret_cast<Raw16*>(p)->v = r; }

// `left` >= kVec: sixteen bytes at once; less: element by element (nothing behind the row is touched)
template <typename T> __device__ __forceinline__ void load_part(const T* p, int left, float (&f)[kVec<T>]) {
  if (left >= kVec<T>) {
    unpack<T>(load16(p), f);
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) f[i] = i < left ? to_f32(p[i]) : 0.f;
  }
}
template <typename T> __device__ __forceinline__ void store_part(T* p, int left, const float (&f)[kVec<T>]) {
  if (left >= kVec<T>) {
    store16(p, pack<T>(f));
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i)
      if (i < left) p[i] = from_f32<T>(f[i]);
  }
}

__device__ __forceinline__ long long load_index(const void* p, long long i, int idx64) {
  return idx64 ? ((const long long*)p)[i] : (long long)((const int*)p)[i];
}

// one instruction; results below 2^-126 are zero
__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// A row from its other classes (largest logit m, sum s of exp(z - m)) and its target's logit: probabilities inv exp(z - top), p - 1 of the
// target from the sum over the others, so that it and the loss keep their relative precision where the target is almost certain.
struct __attribute__((aligned(16))) Row { float top, inv, at_target, loss; };
__device__ __forceinline__ Row row_of(float m, float s, float zt) {
  const float d = zt - m;
  Row r;
  if (m == -INFINITY) {
    r.loss = s + 0.f * zt;      // zero, or NaN
    r.at_target = -r.loss;
    r.top = zt;
  } else if (d < -60.f) {
    r.loss = logf(s) - d;
    r.at_target = d == -INFINITY ? -1.f : -1.f + 0.f * r.loss;
    r.top = m;
  } else {
    const float rest = d == INFINITY ? kNaN : d > 0.f ? s * expf(-d) : s / expf(d);
    r.loss = log1pf(rest);
    r.at_target = -rest / (1.f + rest);
    r.top = fmaxf(m, zt);
  }
  r.inv = 1.f / ((m == -INFINITY ? s : s * expf(m - r.top)) + expf(zt - r.top));
  return r;
}

inline int launch_status() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : (int)e;
}

// f(T()) for the element type `dtype` names
#define VOCAB_DISPATCH(dtype, T, ...)                                    \
  do {                                                                   \
    if ((dtype) == ISTNET_VOCAB_F32) { typedef float T; __VA_ARGS__; }   \
    else if ((dtype) == ISTNET_VOCAB_BF16) { typedef bf16 T; __VA_ARGS__; } \
    else { typedef f16 T; __VA_ARGS__; }                                 \
  } while (0)

}  // namespace
