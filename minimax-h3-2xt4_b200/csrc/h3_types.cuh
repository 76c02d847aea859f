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

}  // namespace h3
