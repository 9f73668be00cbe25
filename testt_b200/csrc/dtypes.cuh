// Element types of the kernels that take fp16, bf16 and fp32 tensors (TB_FP16 / TB_BF16 / TB_FP32
// of the C ABI): single values and 8-value vectors, widened to and rounded from fp32.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace tb {

template <int T>
struct Elem;

template <>
struct Elem<TB_FP16> {
  using type = uint16_t;
  static __device__ __forceinline__ float get(type v) { return __half2float(__ushort_as_half(v)); }
  static __device__ __forceinline__ type put(float f) {
    return __half_as_ushort(__float2half_rn(f));
  }
  static __device__ __forceinline__ float2 get2(uint32_t v) { return unpack_half2(v); }
  static __device__ __forceinline__ uint32_t put2(float lo, float hi) { return pack_half2(lo, hi); }
};

template <>
struct Elem<TB_BF16> {
  using type = uint16_t;
  static __device__ __forceinline__ float get(type v) { return __uint_as_float((uint32_t)v << 16); }
  static __device__ __forceinline__ type put(float f) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(f));
  }
  static __device__ __forceinline__ float2 get2(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t put2(float lo, float hi) {
    __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&b);
  }
};

template <>
struct Elem<TB_FP32> {
  using type = float;
  static __device__ __forceinline__ float get(type v) { return v; }
  static __device__ __forceinline__ type put(float f) { return f; }
};

template <int T>
__host__ __device__ constexpr int elem_size() {
  return T == TB_FP32 ? 4 : 2;
}

inline int elem_size_of(int t) { return t == TB_FP32 ? 4 : 2; }
inline bool elem_type_ok(int t) { return t == TB_FP16 || t == TB_BF16 || t == TB_FP32; }

// Element i of an array of type T.
template <int T>
__device__ __forceinline__ float load1(const void *p, int64_t i) {
  return Elem<T>::get(static_cast<const typename Elem<T>::type *>(p)[i]);
}

template <int T>
__device__ __forceinline__ void store1(void *p, int64_t i, float f) {
  static_cast<typename Elem<T>::type *>(p)[i] = Elem<T>::put(f);
}

// Eight values at element i (16-byte aligned): one 16-byte access, two for fp32.
template <int T>
__device__ __forceinline__ void load8(const void *p, int64_t i, float (&f)[8]) {
  if constexpr (T == TB_FP32) {
    load8f(static_cast<const float *>(p) + i, f);
  } else {
    const uint4 v = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i));
    const float2 a = Elem<T>::get2(v.x), b = Elem<T>::get2(v.y), c = Elem<T>::get2(v.z),
                 d = Elem<T>::get2(v.w);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
    f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
  }
}

template <int T>
__device__ __forceinline__ void store8(void *p, int64_t i, const float (&f)[8]) {
  if constexpr (T == TB_FP32) {
    store8f(static_cast<float *>(p) + i, f);
  } else {
    uint4 v;
    v.x = Elem<T>::put2(f[0], f[1]);
    v.y = Elem<T>::put2(f[2], f[3]);
    v.z = Elem<T>::put2(f[4], f[5]);
    v.w = Elem<T>::put2(f[6], f[7]);
    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + i) = v;
  }
}

// Two fp32 values in one 64-bit register pair: sm_100's packed fp32 instructions do two
// multiply-adds in one issue slot (each rounded as the scalar one).
struct F2 {
  uint64_t v;
};

__device__ __forceinline__ F2 make_f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}

__device__ __forceinline__ F2 both(float x) { return make_f2(x, x); }

__device__ __forceinline__ float2 parts(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}

__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

__device__ __forceinline__ F2 neg2(F2 a) { return F2{a.v ^ 0x8000000080000000ull}; }

// Runs the statement with the constant `T` bound to the element type `t` (already checked).
#define TB_WITH_TYPE(t, T, ...)                                 \
  do {                                                          \
    if ((t) == TB_FP16) {                                       \
      constexpr int T = TB_FP16;                                \
      __VA_ARGS__;                                              \
    } else if ((t) == TB_BF16) {                                \
      constexpr int T = TB_BF16;                                \
      __VA_ARGS__;                                              \
    } else {                                                    \
      constexpr int T = TB_FP32;                                \
      __VA_ARGS__;                                              \
    }                                                           \
  } while (0)

}  // namespace tb
