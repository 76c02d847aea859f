// Residual update joined with the norms around it:
//   b  = norm_post(branch)                          (none, RMS or LayerNorm)
//   x' = residual_scale * x + gate[l] * b
//   h  = norm_pre(x') * (1 + scale[l]) + shift[l]   (none, RMS or LayerNorm)
// with x' rounded once to the residual's type, and h either rounded once to that type or
// (rotated by ConvRot256 and) quantised per row to INT8.  Statistics, x' and h are held
// in fp32 between the two roundings.
#include "h3_types.cuh"

namespace h3 {

struct ResidualNorm {
  const void* x;
  const void* branch;
  int64_t rows, width;
  float residual_scale, inv_width;
  const float* gate;
  const float* shift;
  const float* scale;
  int64_t gate_ld, shift_ld, scale_ld, mod_rows;
  const int32_t* labels;
  const float* post_weight;
  const float* post_bias;
  const float* pre_weight;
  const float* pre_bias;
  float post_eps, pre_eps;
  int post_kind, pre_kind, convrot;
  void* out;
  void* h;
  int8_t* q;
  float* row_scale;
  int* err;
};

H3_DEV float norm_block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.0f;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) t += red[w];
  return t;
}

H3_DEV float norm_block_max(float v, float* red) {
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.0f;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) t = fmaxf(t, red[w]);
  return t;
}

// Normalises row[0, width) in place (each thread its own elements).
H3_DEV void norm_row(float* row, int64_t width, float inv_width, int kind, const float* w,
                     const float* b, float eps, float* red) {
  if (kind == H3_NORM_NONE) return;
  float mean = 0.0f;
  if (kind == H3_NORM_LAYER) {
    float s = 0.0f;
    for (int64_t c = threadIdx.x; c < width; c += blockDim.x) s += row[c];
    mean = norm_block_sum(s, red) * inv_width;
  }
  float s = 0.0f;
  for (int64_t c = threadIdx.x; c < width; c += blockDim.x) {
    const float d = row[c] - mean;
    s = __fmaf_rn(d, d, s);
  }
  const float inv = __frsqrt_rn(__fmaf_rn(norm_block_sum(s, red), inv_width, eps));
  for (int64_t c = threadIdx.x; c < width; c += blockDim.x) {
    float v = (row[c] - mean) * inv;
    if (w != nullptr) v *= __ldg(w + c);
    if (b != nullptr) v += __ldg(b + c);
    row[c] = v;
  }
}

template <typename XT, typename BT>
__global__ void __launch_bounds__(256) residual_norm_kernel(const ResidualNorm a) {
  extern __shared__ __align__(16) float row[];
  __shared__ float red[8];
  const XT* x = reinterpret_cast<const XT*>(a.x);
  const BT* branch = reinterpret_cast<const BT*>(a.branch);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    int64_t lab = a.labels != nullptr ? (int64_t)__ldg(a.labels + r) : 0;
    if (lab < 0 || lab >= a.mod_rows) {
      report_error(a.err, H3_ERR_INVALID);
      lab = 0;
    }
    const int64_t base = r * a.width;
    if (branch != nullptr) {
      for (int64_t c = threadIdx.x; c < a.width; c += blockDim.x) row[c] = to_f32(branch[base + c]);
      norm_row(row, a.width, a.inv_width, a.post_kind, a.post_weight, a.post_bias, a.post_eps, red);
    }
    for (int64_t c = threadIdx.x; c < a.width; c += blockDim.x) {
      float v = to_f32(x[base + c]);
      if (branch != nullptr) {
        const float g = a.gate != nullptr ? __ldg(a.gate + lab * a.gate_ld + c) : 1.0f;
        v = __fmaf_rn(g, row[c], a.residual_scale * v);
        reinterpret_cast<XT*>(a.out)[base + c] = from_f32<XT>(v);
      }
      row[c] = v;
    }
    if (a.pre_kind == H3_NORM_NONE) continue;
    norm_row(row, a.width, a.inv_width, a.pre_kind, a.pre_weight, a.pre_bias, a.pre_eps, red);
    for (int64_t c = threadIdx.x; c < a.width; c += blockDim.x) {
      float v = row[c];
      const float f = a.scale != nullptr ? 1.0f + __ldg(a.scale + lab * a.scale_ld + c) : 1.0f;
      v = __fmaf_rn(v, f, a.shift != nullptr ? __ldg(a.shift + lab * a.shift_ld + c) : 0.0f);
      row[c] = v;
      if (a.h != nullptr) reinterpret_cast<XT*>(a.h)[base + c] = from_f32<XT>(v);
    }
    if (a.q == nullptr) continue;
    if (a.convrot) {
      for (int s = 1; s < 256; s *= 4) {
        __syncthreads();
        for (int64_t i = threadIdx.x; i < a.width / 4; i += blockDim.x) {
          float* p = row + (i / s) * (4 * s) + i % s;
          const float v0 = p[0], v1 = p[s], v2 = p[2 * s], v3 = p[3 * s];
          p[0] = v0 + v1 + v2 - v3;
          p[s] = v0 + v1 - v2 + v3;
          p[2 * s] = v0 - v1 + v2 + v3;
          p[3 * s] = v1 - v0 + v2 + v3;
        }
      }
      __syncthreads();
      for (int64_t c = threadIdx.x; c < a.width; c += blockDim.x) row[c] *= 0.0625f;
    }
    float m = 0.0f;
    for (int64_t c = threadIdx.x; c < a.width; c += blockDim.x) m = fmaxf(m, fabsf(row[c]));
    const float scale = row_scale_from_max(norm_block_max(m, red));
    const float inv = __fdiv_rn(1.0f, scale);
    for (int64_t c = threadIdx.x; c < a.width; c += blockDim.x)
      a.q[base + c] = quantize_code_rn(row[c], scale, inv);
    if (threadIdx.x == 0) a.row_scale[r] = scale;
  }
}

template <typename XT, typename BT>
int launch_residual_norm(const ResidualNorm& a, cudaStream_t stream) {
  const size_t smem = (size_t)a.width * sizeof(float);
  auto kern = residual_norm_kernel<XT, BT>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
      cudaSuccess) {
    cudaGetLastError();
    return H3_ERR_CUDA;
  }
  kern<<<(int)std::min<int64_t>(a.rows, 1 << 20), 256, smem, stream>>>(a);
  return h3host::check_launch();
}

}  // namespace h3

extern "C" int h3_residual_norm(const void* x, int x_type, const void* branch, int branch_type,
                                int64_t rows, int64_t width, float residual_scale,
                                const float* gate, int64_t gate_ld, const float* shift,
                                int64_t shift_ld, const float* scale, int64_t scale_ld,
                                int64_t mod_rows, const int32_t* labels, int post_kind,
                                const float* post_weight, const float* post_bias, float post_eps,
                                int pre_kind, const float* pre_weight, const float* pre_bias,
                                float pre_eps, void* out, void* h, int convrot, int8_t* q,
                                float* row_scale, void* stream) {
  using namespace h3;
  const bool quant = q != nullptr || row_scale != nullptr;
  const auto kind_ok = [](int k) { return k >= H3_NORM_NONE && k <= H3_NORM_LAYER; };
  if (x == nullptr || rows < 0 || width < 1 || width > 32768 || mod_rows < 1 ||
      (labels == nullptr && mod_rows != 1) || !kind_ok(post_kind) || !kind_ok(pre_kind) ||
      (branch == nullptr) != (out == nullptr) ||
      (branch == nullptr && (gate != nullptr || post_kind != H3_NORM_NONE ||
                             residual_scale != 1.0f || pre_kind == H3_NORM_NONE)) ||
      (quant && (q == nullptr || row_scale == nullptr)) ||
      (pre_kind == H3_NORM_NONE ? (quant || h != nullptr) : (quant == (h != nullptr))) ||
      (quant && convrot && width % 256 != 0))
    return H3_ERR_INVALID;
  if (rows == 0) return H3_OK;
  int dev;
  h3host::DeviceScope scope;
  if (int s = scope.bind(x, &dev)) return s;
  int* err = nullptr;
  if (labels != nullptr && (err = h3host::error_word(dev)) == nullptr) return H3_ERR_CUDA;
  const ResidualNorm a{x, branch, rows, width, residual_scale, (float)(1.0 / (double)width),
                       gate, shift, scale, gate_ld, shift_ld, scale_ld, mod_rows, labels,
                       post_weight, post_bias, pre_weight, pre_bias, post_eps, pre_eps,
                       post_kind, pre_kind, convrot, out, h, q, row_scale, err};
  cudaStream_t st = (cudaStream_t)stream;
  if (branch == nullptr) branch_type = x_type;
  if (x_type == H3_TYPE_F32 && branch_type == H3_TYPE_F32)
    return launch_residual_norm<float, float>(a, st);
  if (x_type == H3_TYPE_F16 && branch_type == H3_TYPE_F16)
    return launch_residual_norm<__half, __half>(a, st);
  if (x_type == H3_TYPE_F16 && branch_type == H3_TYPE_F32)
    return launch_residual_norm<__half, float>(a, st);
  if (x_type == H3_TYPE_BF16 && branch_type == H3_TYPE_BF16)
    return launch_residual_norm<__nv_bfloat16, __nv_bfloat16>(a, st);
  if (x_type == H3_TYPE_BF16 && branch_type == H3_TYPE_F32)
    return launch_residual_norm<__nv_bfloat16, float>(a, st);
  return H3_ERR_INVALID;
}
