// Per-head RMS norm and rotary positions over several axes, on the q and k heads of a
// projection's output.  Pair p of a head turns by pos[token][axis[p]] * frequency[p]:
//   (v1, v2) <- (v1 cos - v2 sin, v2 cos + v1 sin)
#include "h3_types.cuh"

namespace h3 {

constexpr int kMaxPairs = 128;  // head_dim <= 256

struct HeadView {
  const void* in;
  void* out;
  int64_t in_token, in_head, out_token, out_head;  // strides in elements
  int heads;
  const float* weight;
};

// The plan travels by value with the launch, so it has no device buffer whose lifetime
// or stream a caller would have to mind.
struct RopeArgs {
  HeadView q, k;
  int64_t tokens;
  int dim, pairs, axes, pos_kind, half, norm;
  float eps, inv_dim;
  const void* positions;
  double turns[kMaxPairs];      // frequency / (2 pi)
  unsigned char axis[kMaxPairs];
};

// Angles of far positions need more than 24 bits: the turns are reduced to a fraction of
// one in 64 bits, and the sine and cosine of that fraction taken in 32.
H3_DEV void pair_angle(const RopeArgs& a, int64_t token, int p, float& c, float& s) {
  const int64_t at = token * a.axes + a.axis[p];
  double pos;
  if (a.pos_kind == H3_POS_I32) pos = (double)__ldg(reinterpret_cast<const int32_t*>(a.positions) + at);
  else if (a.pos_kind == H3_POS_I64) pos = (double)reinterpret_cast<const int64_t*>(a.positions)[at];
  else pos = (double)__ldg(reinterpret_cast<const float*>(a.positions) + at);
  const double t = pos * a.turns[p];
  sincospif(2.0f * (float)(t - rint(t)), &s, &c);
}

template <typename T>
__global__ void __launch_bounds__(256) rope_kernel(const __grid_constant__ RopeArgs a) {
  const int lane = threadIdx.x & 31;
  const int heads = a.q.heads + a.k.heads;
  const int64_t items = a.tokens * heads;
  for (int64_t i = blockIdx.x * 8ll + (threadIdx.x >> 5); i < items; i += gridDim.x * 8ll) {
    const int64_t token = i / heads;
    int head = (int)(i - token * heads);
    const bool is_k = head >= a.q.heads;
    const HeadView& v = is_k ? a.k : a.q;
    if (is_k) head -= a.q.heads;
    const T* in = reinterpret_cast<const T*>(v.in) + token * v.in_token + head * v.in_head;
    T* out = reinterpret_cast<T*>(v.out) + token * v.out_token + head * v.out_head;
    float x[8];
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = lane + 32 * j;
      x[j] = c < a.dim ? to_f32(in[c]) : 0.0f;
      sum = __fmaf_rn(x[j], x[j], sum);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float inv = a.norm ? __frsqrt_rn(__fmaf_rn(sum, a.inv_dim, a.eps)) : 1.0f;
    __shared__ float row[8][256];
    float* w = row[threadIdx.x >> 5];
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = lane + 32 * j;
      if (c < a.dim) w[c] = x[j] * inv * (a.norm && v.weight != nullptr ? __ldg(v.weight + c) : 1.0f);
    }
    __syncwarp();
    for (int p = lane; p < a.pairs; p += 32) {
      float cs, sn;
      pair_angle(a, token, p, cs, sn);
      const int c1 = a.half ? p : 2 * p, c2 = a.half ? p + a.pairs : 2 * p + 1;
      const float v1 = w[c1], v2 = w[c2];
      out[c1] = from_f32<T>(__fmaf_rn(v1, cs, -(v2 * sn)));
      out[c2] = from_f32<T>(__fmaf_rn(v2, cs, v1 * sn));
    }
    for (int c = 2 * a.pairs + lane; c < a.dim; c += 32) out[c] = from_f32<T>(w[c]);
  }
}

}  // namespace h3

extern "C" int h3_qk_norm_rope(const void* q, int64_t q_token, int64_t q_head, int64_t q_heads,
                               void* q_out, int64_t qo_token, int64_t qo_head, const void* k,
                               int64_t k_token, int64_t k_head, int64_t k_heads, void* k_out,
                               int64_t ko_token, int64_t ko_head, int64_t tokens,
                               int64_t head_dim, int type, const void* positions, int pos_kind,
                               int axes, const double* turns, const uint8_t* axis, int64_t pairs,
                               int half, int norm, const float* q_weight, const float* k_weight,
                               float eps, void* stream) {
  using namespace h3;
  if (k == nullptr) k_heads = 0;
  if (q == nullptr || q_out == nullptr || (k != nullptr && k_out == nullptr) || tokens < 0 ||
      q_heads < 1 || q_heads > 65536 || k_heads < 0 || k_heads > 65536 || head_dim < 2 ||
      head_dim > 2 * kMaxPairs || positions == nullptr || axes < 1 || axes > 255 ||
      turns == nullptr || axis == nullptr || pairs < 1 || 2 * pairs > head_dim ||
      pos_kind < H3_POS_I32 || pos_kind > H3_POS_F32)
    return H3_ERR_INVALID;
  RopeArgs a;
  a.q = HeadView{q, q_out, q_token, q_head, qo_token, qo_head, (int)q_heads, q_weight};
  a.k = HeadView{k, k_out, k_token, k_head, ko_token, ko_head, (int)k_heads, k_weight};
  a.tokens = tokens;
  a.dim = (int)head_dim;
  a.pairs = (int)pairs;
  a.axes = axes;
  a.pos_kind = pos_kind;
  a.half = half != 0;
  a.norm = norm != 0;
  a.eps = eps;
  a.inv_dim = (float)(1.0 / (double)head_dim);
  a.positions = positions;
  for (int p = 0; p < kMaxPairs; ++p) {
    a.turns[p] = p < pairs ? turns[p] : 0.0;
    a.axis[p] = p < pairs ? axis[p] : 0;
    if (a.axis[p] >= axes) return H3_ERR_INVALID;
  }
  if (tokens == 0) return H3_OK;
  int dev;
  h3host::DeviceScope scope;
  if (int s = scope.bind(q, &dev)) return s;
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t ctas = (tokens * (q_heads + k_heads) + 7) / 8;
  const int grid = (int)std::min<int64_t>(ctas, (int64_t)h3host::sm_count(dev) * 8);
  if (type == H3_TYPE_F32) rope_kernel<float><<<grid, 256, 0, st>>>(a);
  else if (type == H3_TYPE_F16) rope_kernel<__half><<<grid, 256, 0, st>>>(a);
  else if (type == H3_TYPE_BF16) rope_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
  else return H3_ERR_INVALID;
  return h3host::check_launch();
}
