// Few rows times a 4-bit weight with group scales:
//   y[m][n] = sum_g scale[n][g] * sum_{k in g} x[m][k] (code[n][k] - zero[n][g]) + bias[n]
// code k of a row is the low nibble of byte k / 2 for even k, the high one for odd k.
#include "h3_types.cuh"

namespace h3 {

struct Int4Args {
  const void* x;
  int64_t x_ld, m, k, n;
  const uint8_t* w;
  const void* scales;
  const uint8_t* zeros;
  const float* bias;
  void* out;
  int64_t groups;
  int group, scale_type, out_type;
};

H3_DEV float load_typed(const void* p, int type, int64_t i) {
  if (type == H3_TYPE_F32) return __ldg(reinterpret_cast<const float*>(p) + i);
  if (type == H3_TYPE_F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}

H3_DEV void store_typed(void* p, int type, int64_t i, float v) {
  if (type == H3_TYPE_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (type == H3_TYPE_F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// One warp an output column and row.
template <typename T>
__global__ void __launch_bounds__(256) int4_kernel(const Int4Args a) {
  const int lane = threadIdx.x & 31;
  const int64_t items = a.m * a.n;
  const int64_t pitch = (a.k + 1) / 2;
  const T* x = reinterpret_cast<const T*>(a.x);
  for (int64_t i = blockIdx.x * 8ll + (threadIdx.x >> 5); i < items; i += gridDim.x * 8ll) {
    const int64_t n = i / a.m, m = i - n * a.m;
    float acc = 0.0f;
    for (int64_t k = lane; k < a.k; k += 32) {
      const uint8_t b = __ldg(a.w + n * pitch + k / 2);
      const int64_t g = n * a.groups + k / a.group;
      const int zero = a.zeros != nullptr ? (int)__ldg(a.zeros + g) : 8;
      const int code = (k & 1) ? b >> 4 : b & 15;
      acc = __fmaf_rn(load_typed(a.scales, a.scale_type, g),
                      to_f32(x[m * a.x_ld + k]) * (float)(code - zero), acc);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (a.bias != nullptr) acc += __ldg(a.bias + n);
    if (lane == 0) store_typed(a.out, a.out_type, m * a.n + n, acc);
  }
}

}  // namespace h3

extern "C" int h3_int4_linear(const void* x, int x_type, int64_t x_ld, int64_t m, int64_t k,
                              const uint8_t* w, int64_t n, const void* scales, int scale_type,
                              const uint8_t* zeros, int group, const float* bias, void* out,
                              int out_type, void* stream) {
  using namespace h3;
  const auto type_ok = [](int t) {
    return t == H3_TYPE_F32 || t == H3_TYPE_F16 || t == H3_TYPE_BF16;
  };
  if (x == nullptr || w == nullptr || scales == nullptr || out == nullptr || m < 0 || k < 1 ||
      n < 1 || x_ld < k || k > (1 << 24) || n > (1 << 24) ||
      (group != 32 && group != 64 && group != 128) || !type_ok(scale_type) ||
      (out_type != H3_TYPE_F32 && out_type != x_type))
    return H3_ERR_INVALID;
  if (x_type != H3_TYPE_F16 && x_type != H3_TYPE_BF16) return H3_ERR_INVALID;
  if (m == 0) return H3_OK;
  int dev;
  h3host::DeviceScope scope;
  if (int s = scope.bind(x, &dev)) return s;
  const Int4Args a{x, x_ld, m, k, n, w, scales, zeros, bias, out, (k + group - 1) / group,
                   group, scale_type, out_type};
  const int grid = (int)std::min<int64_t>((m * n + 7) / 8, (int64_t)h3host::sm_count(dev) * 8);
  cudaStream_t st = (cudaStream_t)stream;
  if (x_type == H3_TYPE_F16) int4_kernel<__half><<<grid, 256, 0, st>>>(a);
  else int4_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
  return h3host::check_launch();
}
