// Element types and 64-lane reductions shared by the kernels of ic_score.hip, ic_optim.hip and
// ic_grouped.hip.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ic_internal.h"

namespace ic {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// 16 bytes hold kVec<T> elements
struct bf16_t { unsigned short bits; };
struct f16_t { _Float16 v; };

template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
  static __device__ __forceinline__ void unpack(u32x4 w, float* out) {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = __uint_as_float(w[i]);
  }
  static __device__ __forceinline__ u32x4 pack(const float* v) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[i]);
    return w;
  }
};
// float -> bfloat16, round to nearest even (one rounding, at the end of a float32 computation);
// a NaN stays one
__device__ __forceinline__ unsigned bf16_bits(float f) {
  const __bf16 b = (__bf16)f;
  return (unsigned)__builtin_bit_cast(unsigned short, b);
}
__device__ __forceinline__ unsigned f16_bits(float f) {
  const _Float16 h = (_Float16)f;   // round to nearest even, overflow to infinity
  return (unsigned)__builtin_bit_cast(unsigned short, h);
}
template <> struct Elem<bf16_t> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float load(const bf16_t* p) {
    return __uint_as_float((unsigned)p->bits << 16);
  }
  static __device__ __forceinline__ void store(bf16_t* p, float v) {
    p->bits = (unsigned short)bf16_bits(v);
  }
  static __device__ __forceinline__ void unpack(u32x4 w, float* out) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[2 * i] = __uint_as_float(w[i] << 16);
      out[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float* v) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = bf16_bits(v[2 * i]) | (bf16_bits(v[2 * i + 1]) << 16);
    return w;
  }
};
template <> struct Elem<f16_t> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float load(const f16_t* p) { return (float)p->v; }
  static __device__ __forceinline__ void store(f16_t* p, float v) { p->v = (_Float16)v; }
  static __device__ __forceinline__ void unpack(u32x4 w, float* out) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[2 * i] = (float)__builtin_bit_cast(_Float16, (unsigned short)(w[i] & 0xffffu));
      out[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (unsigned short)(w[i] >> 16));
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float* v) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = f16_bits(v[2 * i]) | (f16_bits(v[2 * i + 1]) << 16);
    return w;
  }
};

// One step of a 64-lane reduction inside the vector ALU (no LDS): row_shr 1, 2, 4, 8 fold the
// rows of 16 lanes, the two broadcasts fold the rows into each other, lane 63 then holds the
// result.  `idle` is what lanes without a source see.
template <int CTRL>
__device__ __forceinline__ unsigned dpp_u32(unsigned idle, unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp((int)idle, (int)v, CTRL, 0xf, 0xf, false);
}
template <typename F>
__device__ __forceinline__ unsigned wave_fold(unsigned v, unsigned idle, F op) {
  v = op(v, dpp_u32<0x111>(idle, v));
  v = op(v, dpp_u32<0x112>(idle, v));
  v = op(v, dpp_u32<0x114>(idle, v));
  v = op(v, dpp_u32<0x118>(idle, v));
  v = op(v, dpp_u32<0x142>(idle, v));
  v = op(v, dpp_u32<0x143>(idle, v));
  return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ unsigned wave_max_u32(unsigned v) {
  return wave_fold(v, 0u, [](unsigned a, unsigned b) { return a > b ? a : b; });
}
__device__ __forceinline__ unsigned wave_min_u32(unsigned v) {
  return wave_fold(v, 0xffffffffu, [](unsigned a, unsigned b) { return a < b ? a : b; });
}
// largest of the lanes' values; a NaN is passed over
__device__ __forceinline__ float wave_max_f32(float v) {
  return __uint_as_float(wave_fold(__float_as_uint(v), 0xff800000u, [](unsigned a, unsigned b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
// the lanes' sum in a fixed order
__device__ __forceinline__ float wave_sum_f32(float v) {
  return __uint_as_float(wave_fold(__float_as_uint(v), 0u, [](unsigned a, unsigned b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

}  // namespace ic
