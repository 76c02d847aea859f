// Element types of the operators around the INT8 projections: fp32, fp16 and bf16 rows
// read and written in vectors of eight values, computed on in fp32.
#pragma once

#include <cuda_bf16.h>

#include "h3_common.cuh"

namespace h3 {

H3_DEV float to_f32(float v) { return v; }
H3_DEV float to_f32(__half v) { return __half2float(v); }
H3_DEV float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
H3_DEV T from_f32(float v);
template <>
H3_DEV float from_f32<float>(float v) { return v; }
template <>
H3_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
H3_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two 16-bit values of one 32-bit word, and back.
template <typename T>
H3_DEV float2 unpack2(uint32_t w);
template <>
H3_DEV float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
H3_DEV float2 unpack2<__nv_bfloat16>(uint32_t w) {  // a bf16 is the upper half of its fp32
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
H3_DEV uint32_t pack2(float lo, float hi);
template <>
H3_DEV uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
H3_DEV uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

H3_DEV void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
H3_DEV void cp_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
H3_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
H3_DEV void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// N consecutive values (a multiple of 16 / sizeof(T) for `Words` of 16 bytes, or four
// 16-bit values in 8) as they lie in memory, unpacked to fp32 and packed from it.
template <typename T, int N>
struct Raw {
  static constexpr int kWords = N * (int)sizeof(T) / 4;
  uint32_t w[kWords];

  H3_DEV void load(const T* p) {
    if (kWords == 2) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      w[0] = u.x; w[1] = u.y;
    } else {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 u = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
      }
    }
  }
  H3_DEV void store(T* p) const {
    if (kWords == 2) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  }
  H3_DEV void unpack(float* v) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float2 f = unpack2<T>(w[i]);
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
      }
    }
  }
  H3_DEV void pack(const float* v) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    }
  }
};

}  // namespace h3
