// Residual update joined with the norms around it:
//   b  = norm_post(branch)                          (none, RMS or LayerNorm)
//   x' = residual_scale * x + gate[l] * b
//   h  = norm_pre(x') * (1 + scale[l]) + shift[l]   (none, RMS or LayerNorm)
// with x' rounded once to the residual's type, and h either rounded once to that type or
// (rotated by ConvRot256 and) quantised per row to INT8.  Statistics, x' and h are held
// in fp32 between the two roundings.
//
// Bound by HBM: x and the branch are read once, x' and h (or the codes) written once; the
// row lives in registers from its load to its last store: eight values a thread, one or two
// rows a CTA at a time, and in rows wider than 8192 values 32 a thread.  What else a row needs is kept off the memory's path: the modulation tables and the
// norms' weights, four times the row's own bytes, are folded into three factors a value
// and stay in registers until a row has another label, and rows to come are fetched by
// cp.async into slots of shared memory that only the fetching thread reads.
//
// 32768 x 3072 fp16 with both norms, gate and h stored (805 MB): 175 us, 0.70 of the measured
// copy rate; with codes of the rotated row instead of h (705 MB) 241 us, 0.45.  Neither is at a
// unit's limit: 49% and 61% of the issue slots are busy at 37% occupancy, and warps wait for
// the next rows, the barriers and the shuffles.  One row at a time and factors read from
// memory, the second took 376 us.
#include "h3_types.cuh"

namespace h3 {

constexpr int kPairThreads = 768;  // most threads of a CTA that takes two rows: 80 registers each
constexpr int kRingSmem = 200 * 1024;  // most shared memory of a CTA's slots

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

// Sums or maxima over the CTA, of one row or of two at once: a tree in each warp, one value
// a warp through shared memory, and the same tree again in every warp.  The trees add in
// one order, whether a row is reduced alone or with another.  `red` has two blocks of 64,
// used in turn: one barrier a call, as a block is written again only after the barrier of
// the call between.  Places without a warp hold zeros from the start.
template <int ROWS>
struct BlockReduce {
  float* red;
  int turn;

  H3_DEV BlockReduce(float* r) : red(r), turn(0) {
    for (int i = threadIdx.x; i < 128; i += blockDim.x) red[i] = 0.0f;
    __syncthreads();
  }
  // value of warp w, row r at [w & 15][w >> 4][r]
  H3_DEV float* next() {
    turn ^= 64;
    return red + turn;
  }
  H3_DEV static int place(int warp) { return (warp & 15) * 4 + (warp >> 4) * 2; }

  H3_DEV void sum(float (&v)[ROWS]) {
    const int lane = threadIdx.x & 31;
    float t;
    if (ROWS == 1) {
      t = v[0] + __shfl_xor_sync(0xffffffffu, v[0], 16);
    } else {  // the lower lanes go on with the first row, the upper ones with the second
      t = lane < 16 ? v[0] : v[ROWS - 1];
      t += __shfl_xor_sync(0xffffffffu, lane < 16 ? v[ROWS - 1] : v[0], 16);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (blockDim.x > 32) {
      float* r = next();
      if ((lane & 15) == 0 && (ROWS == 2 || lane == 0)) r[place(threadIdx.x >> 5) + (lane >> 4)] = t;
      __syncthreads();
      const float* mine = r + (lane & 15) * 4 + (ROWS == 2 ? lane >> 4 : 0);
      t = mine[0] + mine[2];
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    }
    if (ROWS == 1) {
      v[0] = t;
    } else {
      v[0] = __shfl_sync(0xffffffffu, t, 0);
      v[ROWS - 1] = __shfl_sync(0xffffffffu, t, 16);
    }
  }
  // of magnitudes; NAN_WINS: NaN if any value is, else values that are NaN are left out
  template <bool NAN_WINS>
  H3_DEV static float warp_max(float v) {
    float r;
    if (NAN_WINS) asm volatile("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    else asm volatile("redux.sync.max.abs.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
  }
  template <bool NAN_WINS>
  H3_DEV void max(float (&v)[ROWS]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) v[i] = warp_max<NAN_WINS>(v[i]);
    if (blockDim.x == 32) return;
    float* r = next();
    if (lane < ROWS) r[place(threadIdx.x >> 5) + lane] = v[lane == 0 ? 0 : ROWS - 1];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROWS; ++i) v[i] = warp_max<NAN_WINS>(r[lane * 2 + i]);
  }
};

H3_DEV f32x2 shfl2(f32x2 v, int mask) {
  return pk2(__shfl_xor_sync(0xffffffffu, lo2(v), mask), __shfl_xor_sync(0xffffffffu, hi2(v), mask));
}

// The regular 256-point rotation of the 256 values of a warp, v[i] = (value i, value i + 4)
// of lane's eight.  One radix-4 stage takes (x0, x1, x2, x3) to
//   (x0 + x1) + (x2 - x3), (x0 + x1) - (x2 - x3), (x0 - x1) + (x2 + x3), (x2 + x3) - (x0 - x1)
// i.e. y_i = x_i + x_(i^1) + x_(i^2) - x_(i^3).  The first digit of a value's index lies in
// the registers, the second has one bit in the pair and one in the lane, the others are lane
// bits, so they go by shuffles (4.5 a value in all; through shared memory the rotation
// needs four accesses a value and a barrier for each of its two transposes).
H3_DEV void convrot256_warp(f32x2 (&v)[4]) {
  {
    const f32x2 s01 = add2(v[0], v[1]), d01 = sub2(v[0], v[1]);
    const f32x2 s23 = add2(v[2], v[3]), d23 = sub2(v[2], v[3]);
    v[0] = add2(s01, d23); v[1] = sub2(s01, d23);
    v[2] = add2(d01, s23); v[3] = sub2(s23, d01);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float s = lo2(v[i]) + hi2(v[i]);
    const float d = __shfl_xor_sync(0xffffffffu, lo2(v[i]) - hi2(v[i]), 1);
    v[i] = pk2(s + d, s - d);
  }
#pragma unroll
  for (int bit = 2; bit <= 8; bit *= 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 p = shfl2(v[i], bit);
      v[i] = add2(add2(v[i], p), shfl2(sub2(v[i], p), 2 * bit));
    }
  }
  const f32x2 sixteenth = dup2(0.0625f);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = mul2(v[i], sixteenth);
}

// Where value j of a thread's chunk lies in the row.  Eight neighbours where the row allows
// it (VEC: in 16-byte words); rows of a width that is no multiple of eight are dealt value
// by value over the threads, so that a warp's accesses are neighbours.
struct Deal {
  int width, thread_step, value_step, chunk_step;
  H3_DEV int at(int chunk, int j) const {
    return threadIdx.x * thread_step + j * value_step + chunk * chunk_step;
  }
};

// The pairs (value j, value j + 4) of a chunk; values outside the row read as `fill`.
template <bool VEC>
H3_DEV void load_table(const float* t, const Deal& d, int chunk, bool in_row, float fill, f32x2 (&v)[4]) {
  float x[8];
  if constexpr (VEC) {
    if (in_row) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(t + d.at(chunk, 0)));
      const float4 b = __ldg(reinterpret_cast<const float4*>(t + d.at(chunk, 0)) + 1);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = fill;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = d.at(chunk, j) < d.width ? __ldg(t + d.at(chunk, j)) : fill;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pk2(x[i], x[i + 4]);
}

template <typename T, bool VEC>
H3_DEV void load_chunk(const T* row, const Deal& d, int chunk, bool in_row, f32x2 (&v)[4]) {
  float x[8];
  if constexpr (VEC) {
    if (in_row) {
      Raw<T, 8> r;
      r.load(row + d.at(chunk, 0));
      r.unpack(x);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = 0.0f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = d.at(chunk, j) < d.width ? to_f32(row[d.at(chunk, j)]) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pk2(x[i], x[i + 4]);
}

template <typename T, bool VEC>
H3_DEV void store_chunk(T* row, const Deal& d, int chunk, bool in_row, const f32x2 (&v)[4]) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = lo2(v[i]);
    x[i + 4] = hi2(v[i]);
  }
  if constexpr (VEC) {
    if (in_row) {
      Raw<T, 8> r;
      r.pack(x);
      r.store(row + d.at(chunk, 0));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (d.at(chunk, j) < d.width) row[d.at(chunk, j)] = from_f32<T>(x[j]);
  }
}

// What a thread's values of a chunk are multiplied by and shifted by, for one label.
struct Factors {
  f32x2 gate[4];   // gate * post weight
  f32x2 scale[4];  // pre weight * (1 + scale)
  f32x2 shift[4];  // pre bias * (1 + scale) + shift
};

template <bool VEC>
H3_DEV void load_factors(const ResidualNorm& a, const Deal& d, int chunk, bool in_row, int64_t lab, Factors& f) {
  f32x2 t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f.gate[i] = f.scale[i] = dup2(1.0f);
    f.shift[i] = 0;
  }
  if (a.gate != nullptr) load_table<VEC>(a.gate + lab * a.gate_ld, d, chunk, in_row, 0.0f, f.gate);
  if (a.post_weight != nullptr) {
    load_table<VEC>(a.post_weight, d, chunk, in_row, 0.0f, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.gate[i] = mul2(f.gate[i], t[i]);
  }
  if (a.pre_kind == H3_NORM_NONE) return;
  if (a.scale != nullptr) {
    load_table<VEC>(a.scale + lab * a.scale_ld, d, chunk, in_row, 0.0f, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.scale[i] = add2(f.scale[i], t[i]);
  }
  if (a.shift != nullptr) load_table<VEC>(a.shift + lab * a.shift_ld, d, chunk, in_row, 0.0f, f.shift);
  if (a.pre_bias != nullptr) {
    load_table<VEC>(a.pre_bias, d, chunk, in_row, 0.0f, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.shift[i] = fma2(t[i], f.scale[i], f.shift[i]);
  }
  if (a.pre_weight != nullptr) {
    load_table<VEC>(a.pre_weight, d, chunk, in_row, 0.0f, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.scale[i] = mul2(f.scale[i], t[i]);
  }
}

// v += gate * post bias.
template <bool VEC>
H3_DEV void add_post_bias(const ResidualNorm& a, const Deal& d, int chunk, bool in_row, int64_t lab, f32x2 (&v)[4]) {
  f32x2 b[4], g[4] = {dup2(1.0f), dup2(1.0f), dup2(1.0f), dup2(1.0f)};
  load_table<VEC>(a.post_bias, d, chunk, in_row, 0.0f, b);
  if (a.gate != nullptr) load_table<VEC>(a.gate + lab * a.gate_ld, d, chunk, in_row, 0.0f, g);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = fma2(g[i], b[i], v[i]);
}

// (v - mean) * inv of ROWS rows, in place; values outside the row are 0 before and after.
// The variance of LayerNorm is taken around the mean, in a second sum.
template <int ROWS, int NC, bool VEC>
H3_DEV void normalise(f32x2 (&v)[ROWS][NC][4], const ResidualNorm& a, const Deal& d, const bool (&in_row)[NC],
                      int kind, float eps, BlockReduce<ROWS>& reduce) {
  float sum[ROWS];
  if (kind == H3_NORM_LAYER) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      f32x2 t = 0;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) t = add2(t, v[r][c][i]);
      sum[r] = lo2(t) + hi2(t);
    }
    reduce.sum(sum);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const f32x2 mean = dup2(sum[r] * a.inv_width);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x2 m = sub2(v[r][c][i], mean);
          if (VEC) {
            v[r][c][i] = in_row[c] ? m : 0;
          } else {
            v[r][c][i] = pk2(d.at(c, i) < d.width ? lo2(m) : 0.0f, d.at(c, i + 4) < d.width ? hi2(m) : 0.0f);
          }
        }
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    f32x2 t = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) t = fma2(v[r][c][i], v[r][c][i], t);
    sum[r] = lo2(t) + hi2(t);
  }
  reduce.sum(sum);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const f32x2 inv = dup2(rsqrtf(__fmaf_rn(sum[r], a.inv_width, eps)));
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[r][c][i] = mul2(v[r][c][i], inv);
  }
}

// The code of a value of a row that holds infinities or NaN (rare: kept out of line, where
// it costs the other rows no registers).
__device__ __noinline__ uint32_t any_code(float v, float scale) {
  return (uint32_t)(int)quantize_code(v, scale, 0);
}

// h of ROWS rows to their INT8 codes and row scales; rows outside `todo` are not stored.
template <int ROWS, int NC, bool VEC>
H3_DEV void quantise(f32x2 (&v)[ROWS][NC][4], const ResidualNorm& a, const Deal& d, const bool (&in_row)[NC],
                     int64_t row, uint32_t todo, BlockReduce<ROWS>& reduce) {
  float m[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    m[r] = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (a.convrot) convrot256_warp(v[r][c]);  // whole warps lie in the row or none of their lanes
#pragma unroll
      for (int i = 0; i < 4; ++i) m[r] = max_abs2_nan(m[r], lo2(v[r][c][i]), hi2(v[r][c][i]));
    }
  }
  reduce.template max<true>(m);
  bool finite[ROWS], all_finite = true;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    finite[r] = m[r] < __uint_as_float(0x7f800000u);
    all_finite = all_finite && finite[r];
  }
  if (!all_finite) {  // values that are NaN do not count for the scale
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      m[r] = 0.0f;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) m[r] = fmaxf(m[r], fmaxf(fabsf(lo2(v[r][c][i])), fabsf(hi2(v[r][c][i]))));
    }
    reduce.template max<false>(m);
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const float scale = row_scale_from_max(m[r]);
    const float inv = __fdiv_rn(1.0f, scale);
    int8_t* q = a.q + (row + r) * d.width;
    if (!(todo >> r & 1)) continue;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint32_t code[8];
      if (finite[r]) {
        // the correctly rounded quotient (div_by_scale's correction of v * inv), as the library's
        // other quantisers take it: v * inv alone falls to the other side of a border between
        // codes once in about two million values (32768 x 3072 fp16, calls one after the other: 244 us
        // with it alone, 250 so).
        // |v| / scale <= 127 (1 + 2^-23), so no code leaves the range, and the sum with
        // 1.5 * 2^23 rounds to the nearest integer, ties to even, in the low byte
        const f32x2 i2 = dup2(inv), ns = dup2(-scale);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x2 q0 = mul2(v[r][c][i], i2);
          const f32x2 t = add2(fma2(fma2(q0, ns, v[r][c][i]), i2, q0), dup2(12582912.0f));
          code[i] = __float_as_uint(lo2(t));
          code[i + 4] = __float_as_uint(hi2(t));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          code[i] = any_code(lo2(v[r][c][i]), scale);
          code[i + 4] = any_code(hi2(v[r][c][i]), scale);
        }
      }
      if (VEC) {
        uint2 packed;
        packed.x = __byte_perm(__byte_perm(code[0], code[1], 0x0040), __byte_perm(code[2], code[3], 0x0040), 0x5410);
        packed.y = __byte_perm(__byte_perm(code[4], code[5], 0x0040), __byte_perm(code[6], code[7], 0x0040), 0x5410);
        if (in_row[c]) *reinterpret_cast<uint2*>(q + d.at(c, 0)) = packed;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (d.at(c, j) < d.width) q[d.at(c, j)] = (int8_t)code[j];
      }
    }
    if (threadIdx.x == 0) a.row_scale[row + r] = scale;
  }
}

H3_DEV void prefetch_line(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

H3_DEV int64_t row_label(const ResidualNorm& a, int64_t lab) {
  if (lab >= 0 && lab < a.mod_rows) return lab;
  report_error(a.err, H3_ERR_INVALID);
  return 0;
}

// A chunk of fp32 pairs to memory in its type.
template <typename T>
H3_DEV void store_pairs(T* p, const f32x2 (&v)[4]) {
  Raw<T, 8> r;
  float t[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t[i] = lo2(v[i]);
    t[i + 4] = hi2(v[i]);
  }
  r.pack(t);
  r.store(p);
}

// Rows of whole 16-byte words, one chunk a thread, ROWS neighbouring rows at a time: two
// share their reductions, addresses and barriers (a third of all instructions) and cover
// each other's latencies.  Factors stay in registers, row groups are fetched SLOTS - 1 ahead.
template <typename XT, typename BT, bool BRANCH, bool QUANT, int ROWS, int SLOTS>
__global__ void __launch_bounds__(ROWS == 1 ? 1024 : kPairThreads)
    residual_norm_kernel(const __grid_constant__ ResidualNorm a, const __grid_constant__ Deal d) {
  extern __shared__ __align__(16) uint8_t slots[];
  __shared__ float red[128];
  constexpr int kWordsX = sizeof(XT) / 2, kWordsB = BRANCH ? sizeof(BT) / 2 : 0;  // 16-byte words of a chunk
  constexpr int kWords = ROWS * (kWordsX + kWordsB);
  BlockReduce<ROWS> reduce(red);
  const bool in_row[1] = {(int)threadIdx.x * 8 < d.width};

  // a slot: for each row the words of x, then of the branch, each a word a thread side by side
  const uint32_t word = blockDim.x * 16, slot_bytes = word * kWords;
  uint8_t* const mine = slots + threadIdx.x * 16;
  if (!in_row[0]) {  // values behind the row's end: zeros, never written again
#pragma unroll
    for (int i = 0; i < SLOTS * kWords; ++i)
      *reinterpret_cast<uint4*>(mine + i * word) = make_uint4(0, 0, 0, 0);
  }
  const int64_t step = (int64_t)gridDim.x * ROWS, stride = step * d.width;
  const int64_t first = (int64_t)blockIdx.x * ROWS * d.width + threadIdx.x * 8;
  const XT* x_next = reinterpret_cast<const XT*>(a.x) + first;
  const BT* b_next = reinterpret_cast<const BT*>(a.branch) + first;
  int64_t next = (int64_t)blockIdx.x * ROWS;
  const auto fetch = [&](uint32_t offset) {
    if (in_row[0]) {
      const uint32_t dst = (uint32_t)__cvta_generic_to_shared(mine) + offset;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (next + r >= a.rows) break;
#pragma unroll
        for (int w = 0; w < kWordsX; ++w)
          cp_async16(dst + (r * (kWordsX + kWordsB) + w) * word, x_next + r * d.width + w * (16 / sizeof(XT)));
#pragma unroll
        for (int w = 0; w < kWordsB; ++w)
          cp_async16(dst + (r * (kWordsX + kWordsB) + kWordsX + w) * word,
                     b_next + r * d.width + w * (16 / sizeof(BT)));
      }
    }
    next += step;
    x_next += stride;
    if (BRANCH) b_next += stride;
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < SLOTS - 1; ++i) fetch(i * slot_bytes);

  Factors f;
  int held = -1;
  int lab[ROWS], lab_next[ROWS];
  const auto labels_at = [&](int64_t row) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      lab_next[r] = a.labels != nullptr && row + r < a.rows ? __ldg(a.labels + row + r) : 0;
  };
  labels_at((int64_t)blockIdx.x * ROWS);
  uint32_t at = 0;
  int64_t offset = first;  // of this thread's values in x, out, h and q
  for (int64_t row = (int64_t)blockIdx.x * ROWS; row < a.rows; row += step, offset += stride) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) lab[r] = (int)row_label(a, lab_next[r]);
    labels_at(row + step);
    const auto from_slot = [&](auto type, int word0, f32x2 (&v)[4]) {
      using T = decltype(type);
      Raw<T, 8> raw;
      float t[8];
#pragma unroll
      for (int w = 0; w < (int)sizeof(T) / 2; ++w)
        *reinterpret_cast<uint4*>(&raw.w[4 * w]) = *reinterpret_cast<const uint4*>(mine + at + (word0 + w) * word);
      raw.unpack(t);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = pk2(t[i], t[i + 4]);
    };
    // into the slot of the rows before, whose values were used up there
    fetch(at == 0 ? (SLOTS - 1) * slot_bytes : at - slot_bytes);
    cp_async_wait<SLOTS - 1>();
    uint32_t todo = ROWS == 2 && row + 1 < a.rows ? 3 : 1;
    // rows of different labels are stored one after the other, each under its own factors
    do {
      const int label = todo & 1 ? lab[0] : lab[ROWS - 1];
      const uint32_t now = ROWS == 2 && todo == 3 && lab[0] != lab[ROWS - 1] ? 1 : todo;
      todo ^= now;
      if (label != held) {
        load_factors<true>(a, d, 0, in_row[0], label, f);
        held = label;
      }
      f32x2 v[ROWS][1][4];  // the branch, then x', then h
      if constexpr (BRANCH) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r) from_slot(BT(), r * (kWordsX + kWordsB) + kWordsX, v[r][0]);
        if (a.post_kind != H3_NORM_NONE)
          normalise<ROWS, 1, true>(v, a, d, in_row, a.post_kind, a.post_eps, reduce);
        const f32x2 rs = dup2(a.residual_scale);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          f32x2 x[4];
          from_slot(XT(), r * (kWordsX + kWordsB), x);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[r][0][i] = fma2(f.gate[i], v[r][0][i], mul2(x[i], rs));
          if (a.post_bias != nullptr) add_post_bias<true>(a, d, 0, in_row[0], label, v[r][0]);
          if (in_row[0] && (now >> r & 1)) store_pairs(reinterpret_cast<XT*>(a.out) + offset + r * d.width, v[r][0]);
        }
      } else {
#pragma unroll
        for (int r = 0; r < ROWS; ++r) from_slot(XT(), r * kWordsX, v[r][0]);
      }
      if (a.pre_kind == H3_NORM_NONE) continue;
      normalise<ROWS, 1, true>(v, a, d, in_row, a.pre_kind, a.pre_eps, reduce);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[r][0][i] = fma2(v[r][0][i], f.scale[i], f.shift[i]);
        if (!QUANT && in_row[0] && (now >> r & 1))
          store_pairs(reinterpret_cast<XT*>(a.h) + offset + r * d.width, v[r][0]);
      }
      if constexpr (QUANT) quantise<ROWS, 1, true>(v, a, d, in_row, row, now, reduce);
    } while (todo != 0);
    at = at + slot_bytes == SLOTS * slot_bytes ? 0 : at + slot_bytes;
  }
  cp_async_wait<0>();
}

// Wide rows (NC chunks a thread) and rows of any width and alignment (VEC false).  With one
// chunk a thread the factors stay in registers (16384 x 4001 fp32: 355 us, 461 without); the
// CTA's next row is brought into the L2 (340 us).
template <typename XT, typename BT, int NC, bool VEC, bool QUANT>
__global__ void __launch_bounds__(1024) residual_norm_any_kernel(const __grid_constant__ ResidualNorm a,
                                                                 const __grid_constant__ Deal d) {
  __shared__ float red[128];
  BlockReduce<1> reduce(red);
  bool in_row[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) in_row[c] = d.at(c, 0) < d.width;
  Factors f;
  int64_t held = -1;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t lab = row_label(a, a.labels != nullptr ? __ldg(a.labels + row) : 0);
    const int64_t base = row * a.width;
    if (row + gridDim.x < a.rows) {  // the CTA's next row, one line a thread
      const int64_t next = (row + gridDim.x) * a.width;
      for (int i = threadIdx.x * (128 / (int)sizeof(XT)); i < d.width; i += blockDim.x * (128 / (int)sizeof(XT)))
        prefetch_line(reinterpret_cast<const XT*>(a.x) + next + i);
      if (a.branch != nullptr)
        for (int i = threadIdx.x * (128 / (int)sizeof(BT)); i < d.width; i += blockDim.x * (128 / (int)sizeof(BT)))
          prefetch_line(reinterpret_cast<const BT*>(a.branch) + next + i);
    }
    if (NC == 1 && lab != held) {
      load_factors<VEC>(a, d, 0, in_row[0], lab, f);
      held = lab;
    }
    f32x2 v[1][NC][4];  // the branch, then x', then h
    if (a.branch != nullptr) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
        load_chunk<BT, VEC>(reinterpret_cast<const BT*>(a.branch) + base, d, c, in_row[c], v[0][c]);
      if (a.post_kind != H3_NORM_NONE)
        normalise<1, NC, VEC>(v, a, d, in_row, a.post_kind, a.post_eps, reduce);
      const f32x2 rs = dup2(a.residual_scale);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        f32x2 x[4];
        load_chunk<XT, VEC>(reinterpret_cast<const XT*>(a.x) + base, d, c, in_row[c], x);
        if (NC > 1) load_factors<VEC>(a, d, c, in_row[c], lab, f);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[0][c][i] = fma2(f.gate[i], v[0][c][i], mul2(x[i], rs));
        if (a.post_bias != nullptr) add_post_bias<VEC>(a, d, c, in_row[c], lab, v[0][c]);
        store_chunk<XT, VEC>(reinterpret_cast<XT*>(a.out) + base, d, c, in_row[c], v[0][c]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c)
        load_chunk<XT, VEC>(reinterpret_cast<const XT*>(a.x) + base, d, c, in_row[c], v[0][c]);
    }
    if (a.pre_kind == H3_NORM_NONE) continue;
    normalise<1, NC, VEC>(v, a, d, in_row, a.pre_kind, a.pre_eps, reduce);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (NC > 1) load_factors<VEC>(a, d, c, in_row[c], lab, f);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[0][c][i] = fma2(v[0][c][i], f.scale[i], f.shift[i]);
      if (!QUANT) store_chunk<XT, VEC>(reinterpret_cast<XT*>(a.h) + base, d, c, in_row[c], v[0][c]);
    }
    if (QUANT) quantise<1, NC, VEC>(v, a, d, in_row, row, 1, reduce);
  }
}

template <typename XT, typename BT, bool BRANCH, bool QUANT, int ROWS, int SLOTS>
int launch_ring(const ResidualNorm& a, const Deal& d, int threads, int dev, cudaStream_t stream) {
  auto kern = residual_norm_kernel<XT, BT, BRANCH, QUANT, ROWS, SLOTS>;
  const size_t smem = (size_t)SLOTS * ROWS * threads * 8 * (sizeof(XT) + (BRANCH ? sizeof(BT) : 0));
  static std::atomic<bool> allowed[h3host::kMaxDevices];
  if (smem > 40 * 1024 &&  // with the static part, more than a launch may ask for unasked
      !h3host::allow_smem(kern, kRingSmem, dev, allowed))
    return H3_ERR_CUDA;
  // CTAs an SM: what its registers and its shared memory hold
  const int by_regs = 65536 / ((ROWS == 1 ? 64 : 80) * threads), by_smem = (int)(220 * 1024 / (smem + 2048));
  const int ctas = std::max(1, std::min(std::min(by_regs, by_smem), 16));
  const int grid = (int)std::min<int64_t>((a.rows + ROWS - 1) / ROWS, (int64_t)h3host::sm_count(dev) * ctas);
  kern<<<grid, threads, smem, stream>>>(a, d);
  return h3host::check_launch();
}

template <typename XT, typename BT, bool BRANCH, bool QUANT>
int launch_norm_shape(const ResidualNorm& a, bool vec, int dev, cudaStream_t stream) {
  const int width = (int)a.width;
  // 1024 threads of eight values are the most; beyond, 32 a thread.  8192 rows bf16 with eight and
  // with 32: 5376 wide 106 and 121 us, 8192 wide 159 and 156 (but 4096 wide 93 and 81).
  const int nc = width <= 8192 ? 1 : 4;
  const int threads = ((width + 8 * nc - 1) / (8 * nc) + 31) / 32 * 32;
  Deal d{width, 8, 1, 8 * threads};
  if (width % 8 != 0) d = Deal{width, 1, threads, 8 * threads};
  if (nc == 1 && vec) {
    // Two rows at a time where the registers allow it, there are rows for every SM to have
    // several pairs, and three slots of a pair fit: fp16 codes, 32768 x 3072 240 us against 295 one
    // at a time in four slots and 291 in two, 1184 x 3072 18.7 against 20.0 and 19.5, at the border
    // 592 x 3072 12.0 against 11.8 and 11.5 (narrow rows lose there: 592 x 1024 9.0 against 6.1).
    // Else one row, in four slots or two, between which little lies (6144 wide, FP32 branch: 346
    // and 344; but 16384 x 4096 fp32 309 and 265).
    const int64_t pair = 2ll * threads * 8 * (sizeof(XT) + (BRANCH ? sizeof(BT) : 0));
    if (threads <= kPairThreads && a.rows >= 4ll * h3host::sm_count(dev) && 3 * pair <= kRingSmem)
      return launch_ring<XT, BT, BRANCH, QUANT, 2, 3>(a, d, threads, dev, stream);
    if (4 * pair / 2 <= 100 * 1024)
      return launch_ring<XT, BT, BRANCH, QUANT, 1, 4>(a, d, threads, dev, stream);
    return launch_ring<XT, BT, BRANCH, QUANT, 1, 2>(a, d, threads, dev, stream);
  }
  const int ctas = std::min(16, std::max(1, 1024 / threads));
  const int grid = (int)std::min<int64_t>(a.rows, (int64_t)h3host::sm_count(dev) * ctas);
  if (nc == 1) residual_norm_any_kernel<XT, BT, 1, false, QUANT><<<grid, threads, 0, stream>>>(a, d);
  else if (vec) residual_norm_any_kernel<XT, BT, 4, true, QUANT><<<grid, threads, 0, stream>>>(a, d);
  else residual_norm_any_kernel<XT, BT, 4, false, QUANT><<<grid, threads, 0, stream>>>(a, d);
  return h3host::check_launch();
}

template <typename XT, typename BT>
int launch_residual_norm(const ResidualNorm& a, int dev, cudaStream_t stream) {
  bool vec = a.width % 8 == 0;
  for (const void* p : {a.x, a.branch, (const void*)a.out, (const void*)a.h, (const void*)a.q,
                        (const void*)a.gate, (const void*)a.shift, (const void*)a.scale,
                        (const void*)a.post_weight, (const void*)a.post_bias,
                        (const void*)a.pre_weight, (const void*)a.pre_bias})
    vec = vec && h3host::aligned(p, 16);
  if (a.mod_rows > 1) vec = vec && a.gate_ld % 4 == 0 && a.shift_ld % 4 == 0 && a.scale_ld % 4 == 0;
  if constexpr (sizeof(XT) == sizeof(BT))  // without a branch both types are x's
    if (a.branch == nullptr)
      return a.q != nullptr ? launch_norm_shape<XT, BT, false, true>(a, vec, dev, stream)
                            : launch_norm_shape<XT, BT, false, false>(a, vec, dev, stream);
  return a.q != nullptr ? launch_norm_shape<XT, BT, true, true>(a, vec, dev, stream)
                        : launch_norm_shape<XT, BT, true, false>(a, vec, dev, stream);
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
  // every row reads the tables, weights and labels: x' must lie over none of them
  const auto over = [&](const void* p, int64_t n, int64_t ld) {
    return h3host::rows_meet(p, n, width * 4, ld * 4, out, rows * width * (x_type == H3_TYPE_F32 ? 4 : 2));
  };
  if (over(gate, mod_rows, gate_ld) || over(shift, mod_rows, shift_ld) || over(scale, mod_rows, scale_ld) ||
      over(post_weight, 1, 0) || over(post_bias, 1, 0) || over(pre_weight, 1, 0) || over(pre_bias, 1, 0) ||
      h3host::rows_meet(labels, 1, rows * 4, 0, out, rows * width * (x_type == H3_TYPE_F32 ? 4 : 2)))
    return H3_ERR_INVALID;
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
    return launch_residual_norm<float, float>(a, dev, st);
  if (x_type == H3_TYPE_F16 && branch_type == H3_TYPE_F16)
    return launch_residual_norm<__half, __half>(a, dev, st);
  if (x_type == H3_TYPE_F16 && branch_type == H3_TYPE_F32)
    return launch_residual_norm<__half, float>(a, dev, st);
  if (x_type == H3_TYPE_BF16 && branch_type == H3_TYPE_BF16)
    return launch_residual_norm<__nv_bfloat16, __nv_bfloat16>(a, dev, st);
  if (x_type == H3_TYPE_BF16 && branch_type == H3_TYPE_F32)
    return launch_residual_norm<__nv_bfloat16, float>(a, dev, st);
  return H3_ERR_INVALID;
}
