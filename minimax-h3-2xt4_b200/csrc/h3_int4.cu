// Few rows times a 4-bit weight with group scales:
//   y[m][n] = sum_g scale[n][g] * sum_{k in g} x[m][k] (code[n][k] - zero[n][g]) + bias[n]
// code k of a row is the low nibble of byte k / 2 for even k, the high one for odd k.
//
// Bound by the weight's bytes: each is read once.  What stands between that and a plain
// product is the unpacking (one weight in half a byte) and, for more than a row or two, the
// multiplications.  Both go to where they cost least: a warp takes 16 output columns and
// runs m16n8k16 products with the unpacked weights as the 16-row operand and eight rows of
// x as the other, so a weight is unpacked once for eight rows, two at a time, exactly
// (code - zero is a small integer in either 16-bit type), and the group's scale is applied
// to the fp32 sum of the group.  (The fifth-generation tensor cores would want the unpacked
// weights in shared memory, four times the bytes of the packed ones; at so few rows the
// older instruction is far from its limit.)
//
// The order of k inside a product does not matter as long as both operands agree, so the
// weights need no layout of their own: in a block of 32 k, lane t of a row's four takes the
// 4-byte word t of the packed row, codes 8 t to 8 t + 7, and the x staged in shared memory
// is permuted to match the pairs that the unpacking yields, (0, 4), (1, 5), (2, 6), (3, 7).
#include "h3_types.cuh"

namespace h3 {

struct Int4Args {
  const void* x;
  int64_t x_ld, m;
  int k, n;
  const uint8_t* w;
  const void* scales;
  const uint8_t* zeros;
  const float* bias;
  void* out;
  int groups, pitch;  // of a weight row: groups, bytes
  int group_shift;    // log2(group) - 5
  int chunk;          // k of a chunk of staged x, a multiple of kStageK
  int out_type;
};

constexpr int kInt4Warps = 8;
constexpr int kStageK = 256;                   // k of one stage of packed weights
constexpr int kStagePitch = kStageK / 2 + 16;  // bytes of a stage's row: the eight rows that a
                                               // load touches start in different banks
constexpr int kStageBytes = 16 * kStagePitch;

template <typename T>
struct Unpack;

// Eight codes of a word as four pairs (code i, code i + 4) of exact integers code - zero.
// A 16-bit float whose mantissa's low bits are the code is a power of two plus the code:
// 1024 + c in fp16 (or 1024 + 16 c for the upper nibble, scaled back in the subtraction) and
// 128 + c in bf16, so one logical operation and one exact fma unpack two codes.
template <>
struct Unpack<__half> {
  uint32_t low, high;  // -(1024 + zero) and -(64 + zero) in both halves

  H3_DEV explicit Unpack(int zero) {
    const __half2 a = __half2half2(__float2half_rn(-(1024.0f + (float)zero)));
    const __half2 b = __half2half2(__float2half_rn(-(64.0f + (float)zero)));
    low = *reinterpret_cast<const uint32_t*>(&a);
    high = *reinterpret_cast<const uint32_t*>(&b);
  }
  H3_DEV void operator()(uint32_t w, uint32_t (&p)[4]) const {
    const uint32_t v = w >> 8;
    p[0] = add((w & 0x000f000fu) | 0x64006400u, low);
    p[1] = fma((w & 0x00f000f0u) | 0x64006400u, high);
    p[2] = add((v & 0x000f000fu) | 0x64006400u, low);
    p[3] = fma((v & 0x00f000f0u) | 0x64006400u, high);
  }
  H3_DEV static uint32_t add(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  H3_DEV static uint32_t fma(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(0x2c002c00u), "r"(b));  // a / 16 + b
    return r;
  }
  H3_DEV static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

template <>
struct Unpack<__nv_bfloat16> {
  uint32_t low;  // -(128 + zero) in both halves

  H3_DEV explicit Unpack(int zero) {
    const __nv_bfloat162 a = __bfloat162bfloat162(__float2bfloat16_rn(-(128.0f + (float)zero)));
    low = *reinterpret_cast<const uint32_t*>(&a);
  }
  H3_DEV void operator()(uint32_t w, uint32_t (&p)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      asm("fma.rn.bf16x2 %0, %1, %2, %3;"
          : "=r"(p[i])
          : "r"(((w >> (4 * i)) & 0x000f000fu) | 0x43004300u), "r"(0x3f803f80u), "r"(low));
  }
  H3_DEV static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

template <typename S>
H3_DEV float load_scale(const void* s, int64_t i) {
  return to_f32(reinterpret_cast<const S*>(s)[i]);
}

// A CTA: MT * 8 rows of x times 16 * WN columns, eight warps as WN column tiles by WK slices
// of k (every WK-th stage), the slices added in order through shared memory at the end.
// VEC: rows of packed weights start on 16-byte boundaries (k a multiple of 32), so they are
// fetched by cp.async; else byte by byte.
template <typename T, typename S, bool ZEROS, int MT, int WN, bool VEC, int STAGES>
__global__ void __launch_bounds__(kInt4Warps * 32) int4_kernel(const __grid_constant__ Int4Args a) {
  constexpr int WK = kInt4Warps / WN;
  constexpr int kRows = 8 * MT;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int wn = warp % WN, wk = warp / WN;
  uint8_t* const ring = smem + warp * STAGES * kStageBytes;
  // x: kRows rows of `chunk` values, neighbouring rows half the banks apart, so that two
  // rows' four 16-byte words of a k block fill all banks
  const int x_pitch = a.chunk * 2 + 64;
  uint8_t* const xs = smem + kInt4Warps * STAGES * kStageBytes;
  const int n0 = (blockIdx.x * WN + wn) * 16;
  const int64_t m0 = (int64_t)blockIdx.y * kRows;
  const int rows = (int)min((int64_t)kRows, a.m - m0);
  const int stages = (a.k + kStageK - 1) / kStageK;

  // fetches this warp's stage `s` (its 16 columns, kStageK codes) into slot s / WK % STAGES
  const auto fetch = [&](int s) {
    if (s < stages && n0 < a.n) {
      uint8_t* dst = ring + (s / WK) % STAGES * kStageBytes;
      if (VEC) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = i * 4 + (lane >> 3), byte = s * (kStageK / 2) + (lane & 7) * 16;
          uint8_t* p = dst + row * kStagePitch + (lane & 7) * 16;
          if (n0 + row < a.n && byte < a.pitch)
            cp_async16((uint32_t)__cvta_generic_to_shared(p), a.w + (int64_t)(n0 + row) * a.pitch + byte);
          else *reinterpret_cast<uint4*>(p) = make_uint4(0, 0, 0, 0);
        }
      } else {
        for (int i = lane; i < 16 * kStageK / 8; i += 32) {
          const int row = i / (kStageK / 8), word = i % (kStageK / 8), byte = s * (kStageK / 2) + word * 4;
          uint32_t v = 0;
          for (int b = 0; b < 4; ++b)
            if (n0 + row < a.n && byte + b < a.pitch)
              v |= (uint32_t)a.w[(int64_t)(n0 + row) * a.pitch + byte + b] << (8 * b);
          *reinterpret_cast<uint32_t*>(dst + row * kStagePitch + word * 4) = v;
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(wk + i * WK);

  float acc[MT][4];
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;

  const int col0 = min(n0 + g, a.n - 1), col1 = min(n0 + g + 8, a.n - 1);
  const int64_t gi0 = (int64_t)col0 * a.groups, gi1 = (int64_t)col1 * a.groups;
  int s = wk;  // this warp's next stage
  for (int k0 = 0; k0 < a.k; k0 += a.chunk) {
    if (k0 > 0) __syncthreads();
    // x of the chunk, zeros behind its rows and columns; the eight values of a word's codes
    // in the order 0 4 1 5 2 6 3 7
    const int words = a.chunk / 8;
    for (int i = threadIdx.x; i < kRows * words; i += kInt4Warps * 32) {
      const int row = i / words, w = i - row * words, k = k0 + w * 8;
      T v[8];
      const T* src = reinterpret_cast<const T*>(a.x) + (m0 + row) * a.x_ld + k;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = row < rows && k + e < a.k ? src[e] : from_f32<T>(0.0f);
      T o[8] = {v[0], v[4], v[1], v[5], v[2], v[6], v[3], v[7]};
      *reinterpret_cast<uint4*>(xs + row * x_pitch + w * 16) = *reinterpret_cast<uint4*>(o);
    }
    __syncthreads();
    const int end = min(stages, (k0 + a.chunk) / kStageK);
    for (; s < end; s += WK) {
      cp_async_wait<STAGES - 2>();
      __syncwarp();
      const uint8_t* stage = ring + (s / WK) % STAGES * kStageBytes;
      const uint8_t* xk = xs + (s * kStageK - k0) * 2 + t * 16;
      const int blocks = min(kStageK, a.k - s * kStageK + 31) / 32;
      int b = 0;
      while (b < blocks) {
        // one group: its scales and zeros, the products of its blocks, the scaled sum
        const int gr = (s * (kStageK / 32) + b) >> a.group_shift;
        const int stop = min(blocks, ((gr + 1) << a.group_shift) - s * (kStageK / 32));
        const float s0 = load_scale<S>(a.scales, gi0 + gr), s1 = load_scale<S>(a.scales, gi1 + gr);
        const Unpack<T> u0(ZEROS ? a.zeros[gi0 + gr] : 8), u1(ZEROS ? a.zeros[gi1 + gr] : 8);
        float part[MT][4];
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) part[j][i] = 0.0f;
        for (; b < stop; ++b) {
          const uint32_t w0 = *reinterpret_cast<const uint32_t*>(stage + g * kStagePitch + b * 16 + t * 4);
          const uint32_t w1 = *reinterpret_cast<const uint32_t*>(stage + (g + 8) * kStagePitch + b * 16 + t * 4);
          uint32_t p0[4], p1[4];
          u0(w0, p0);
          u1(w1, p1);
          const uint32_t first[4] = {p0[0], p1[0], p0[1], p1[1]}, second[4] = {p0[2], p1[2], p0[3], p1[3]};
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            const uint4 xv = *reinterpret_cast<const uint4*>(xk + (j * 8 + g) * x_pitch + b * 64);
            Unpack<T>::mma(part[j], first, xv.x, xv.y);
            Unpack<T>::mma(part[j], second, xv.z, xv.w);
          }
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          acc[j][0] = __fmaf_rn(s0, part[j][0], acc[j][0]);
          acc[j][1] = __fmaf_rn(s0, part[j][1], acc[j][1]);
          acc[j][2] = __fmaf_rn(s1, part[j][2], acc[j][2]);
          acc[j][3] = __fmaf_rn(s1, part[j][3], acc[j][3]);
        }
      }
      __syncwarp();
      fetch(s + (STAGES - 1) * WK);
    }
  }
  cp_async_wait<0>();

  // the slices' sums through shared memory, added in order; then bias and store
  __syncthreads();
  float* sums = reinterpret_cast<float*>(smem);  // [WK][WN][kRows][16]
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      sums[((wk * WN + wn) * kRows + j * 8 + 2 * t + (i & 1)) * 16 + g + (i >> 1) * 8] = acc[j][i];
  __syncthreads();
  for (int i = threadIdx.x; i < WN * kRows * 16; i += kInt4Warps * 32) {
    const int c = i % (16 * WN), row = i / (16 * WN), n = blockIdx.x * WN * 16 + c;
    if (row >= rows || n >= a.n) continue;
    float v = 0.0f;
#pragma unroll
    for (int q = 0; q < WK; ++q) v += sums[((q * WN + c / 16) * kRows + row) * 16 + c % 16];
    if (a.bias != nullptr) v += __ldg(a.bias + n);
    const int64_t at = (m0 + row) * a.n + n;
    if (a.out_type == H3_TYPE_F32) reinterpret_cast<float*>(a.out)[at] = v;
    else reinterpret_cast<T*>(a.out)[at] = from_f32<T>(v);
  }
}

template <typename T, typename S, bool ZEROS, int MT, int WN, bool VEC>
int launch_int4(Int4Args& a, cudaStream_t stream) {
  constexpr int kStages = 4;
  auto kern = int4_kernel<T, S, ZEROS, MT, WN, VEC, kStages>;
  // x of all of k where it fits beside the weights' stages and a second CTA, else in chunks
  const int ring = kInt4Warps * kStages * kStageBytes, budget = 110 * 1024 - ring;
  const int all = (a.k + kStageK - 1) / kStageK * kStageK;
  a.chunk = std::max(kStageK, std::min(all, (budget / (8 * MT) - 64) / 2 / kStageK * kStageK));
  const int smem = std::max(ring + 8 * MT * (a.chunk * 2 + 64), (int)sizeof(float) * kInt4Warps * 8 * MT * 16);
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
    cudaGetLastError();
    return H3_ERR_CUDA;
  }
  const dim3 grid((a.n + 16 * WN - 1) / (16 * WN), (unsigned)((a.m + 8 * MT - 1) / (8 * MT)));
  kern<<<grid, kInt4Warps * 32, smem, stream>>>(a);
  return h3host::check_launch();
}

template <typename T, typename S, bool ZEROS>
int launch_int4_shape(Int4Args& a, int sms, cudaStream_t stream) {
  const bool vec = a.k % 32 == 0 && h3host::aligned(a.w, 16);
  if (!vec) return a.m <= 8 ? launch_int4<T, S, ZEROS, 1, 2, false>(a, stream)
                            : launch_int4<T, S, ZEROS, 4, 2, false>(a, stream);
  if (a.m <= 8) return launch_int4<T, S, ZEROS, 1, 2, true>(a, stream);
  if (a.m <= 16) return launch_int4<T, S, ZEROS, 2, 2, true>(a, stream);
  return launch_int4<T, S, ZEROS, 4, 2, true>(a, stream);
}

template <typename T>
int launch_int4_type(Int4Args& a, int scale_type, int sms, cudaStream_t stream) {
  const bool z = a.zeros != nullptr;
  if (scale_type == H3_TYPE_F32)
    return z ? launch_int4_shape<T, float, true>(a, sms, stream) : launch_int4_shape<T, float, false>(a, sms, stream);
  if (scale_type == H3_TYPE_F16)
    return z ? launch_int4_shape<T, __half, true>(a, sms, stream) : launch_int4_shape<T, __half, false>(a, sms, stream);
  return z ? launch_int4_shape<T, __nv_bfloat16, true>(a, sms, stream)
           : launch_int4_shape<T, __nv_bfloat16, false>(a, sms, stream);
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
  if (x == nullptr || w == nullptr || scales == nullptr || out == nullptr || m < 0 ||
      m > 32 * 65535 || k < 1 || n < 1 || x_ld < 0 || (m > 1 && x_ld < k) || k > (1 << 24) ||
      n > (1 << 24) || (group != 32 && group != 64 && group != 128) || !type_ok(scale_type) ||
      (x_type != H3_TYPE_F16 && x_type != H3_TYPE_BF16) ||
      (out_type != H3_TYPE_F32 && out_type != x_type))
    return H3_ERR_INVALID;
  if (m == 0) return H3_OK;
  int dev;
  h3host::DeviceScope scope;
  if (int s = scope.bind(x, &dev)) return s;
  Int4Args a{x, x_ld, m, (int)k, (int)n, w, scales, zeros, bias, out, (int)((k + group - 1) / group),
             (int)((k + 1) / 2), group == 32 ? 0 : group == 64 ? 1 : 2, 0, out_type};
  cudaStream_t st = (cudaStream_t)stream;
  const int sms = h3host::sm_count(dev);
  return x_type == H3_TYPE_F16 ? launch_int4_type<__half>(a, scale_type, sms, st)
                               : launch_int4_type<__nv_bfloat16>(a, scale_type, sms, st);
}
