// Per-head RMS norm and rotary positions over several axes, on the q and k heads of a
// projection's output.  Pair p of a head turns by pos[token][axis[p]] * frequency[p]:
//   (v1, v2) <- (v1 cos - v2 sin, v2 cos + v1 sin)
//
// Bound by HBM: every element is read and written once, and the sines and cosines are
// computed in the kernel (a table of them would be read and written too).  They depend on
// the token and the pair alone, so a lane group takes one token and walks over its heads
// with the angles, times the norm's weights, in registers: no barrier anywhere.  A head is
// held by G = 8, 16 or 32 lanes, eight elements (four pairs) each; the sum of squares is a
// shuffle tree over those lanes.  Each lane keeps the heads to come in flight (three steps, 48
// bytes, of a 16-bit type; one step, 32 bytes, of fp32) through cp.async into slots of shared
// memory that it alone reads: held in registers, the same bytes left too few warps an SM to cover the memory's latency (158 against
// 143 us).  32768 tokens of 24 + 24 heads of 128 in fp16, 805 MB: 140 us, 5.7 TB/s, 0.88 of
// the measured copy rate (halves paired: 156 us; 12 + 12 heads in fp32, the same bytes: 201 us,
// halves 143).  Heads of 72, 80 and 96 take the 16 lanes of 128 and its 141 us.
#include "h3_types.cuh"

namespace h3 {

constexpr int kMaxPairs = 128;  // head_dim <= 256
constexpr int kRopeThreads = 256;
// Four CTAs an SM (64 registers a thread) and slots of 64 bytes a lane, one of them being
// used up; three, five or six CTAs and 128 bytes measured up to 10% slower at 32768 tokens of 48 heads.
constexpr int kRopeCtas = 4;
constexpr int kRopeSlotBytes = 64;

struct HeadView {
  const void* in;
  void* out;
  int in_token, in_head, out_token, out_head;  // strides in elements
  int heads;
  const float* weight;
};

// The plan travels by value with the launch, so it has no device buffer whose lifetime
// or stream a caller would have to mind.
struct RopeArgs {
  HeadView q, k;
  int64_t tokens;
  int dim, pairs, axes, pos_kind, norm;
  int parts;  // lane groups that share the heads of a token
  float eps, inv_dim;
  const void* positions;
  double turns[kMaxPairs];      // frequency / (2 pi)
  unsigned char axis[kMaxPairs];
};

// Angles of far positions need more than 24 bits: the turns are reduced to a fraction of
// one in 64 bits, and the sine and cosine of that fraction taken in 32: its rounding moves the
// angle by at most 2 pi 2^-26, one and a half roundings of fp32 and nothing beside one of a 16-bit
// type (fp32 outputs are 5.2e-8 from the definition, with sines of the 64-bit angle 4.2e-8).
H3_DEV void pair_angle(const RopeArgs& a, int64_t token, int axis, double turns, float& c, float& s) {
  const int64_t at = token * a.axes + axis;
  double pos;
  if (a.pos_kind == H3_POS_I32) pos = (double)__ldg(reinterpret_cast<const int32_t*>(a.positions) + at);
  else if (a.pos_kind == H3_POS_I64) pos = (double)__ldg(reinterpret_cast<const long long*>(a.positions) + at);
  else pos = (double)__ldg(reinterpret_cast<const float*>(a.positions) + at);
  const double t = pos * turns;
  sincospif(2.0f * (float)(t - rint(t)), &s, &c);
}

// The eight elements of lane u: four pairs, as v[0..3] = first elements and v[4..7] =
// second elements, packed two floats to a register pair (half the instructions).  VEC:
// whole 16-byte (or 8-byte) pieces, a lane's pairs all turned or none; else one element at
// a time, any alignment and any head_dim.
template <typename T, bool HALF, bool VEC>
struct HeadLane {
  // where first (i < 4) or second element i of the lane lies in the head
  H3_DEV static int element(const RopeArgs& a, int u, int i) {
    const int p = 4 * u + (i & 3);
    if (HALF && p < a.pairs) return i < 4 ? p : p + a.pairs;
    return 2 * p + (i >> 2);  // neighbours, also behind the turned halves
  }
  // the weight of first or second element i
  H3_DEV static float weight(const RopeArgs& a, const float* w, int u, int i) {
    const int e = VEC && HALF && 4 * u >= a.pairs ? 8 * u + i : element(a, u, i);
    return e < a.dim ? __ldg(w + e) : 0.0f;
  }
  // eight values in memory order to pairs and back; behind turned halves the lane is only
  // scaled, so there the order of its elements does not matter
  H3_DEV static void to_pairs(const float (&x)[8], f32x2 (&v)[4]) {
    if (VEC && !HALF) {
      v[0] = pk2(x[0], x[2]); v[1] = pk2(x[4], x[6]);
      v[2] = pk2(x[1], x[3]); v[3] = pk2(x[5], x[7]);
    } else {
      v[0] = pk2(x[0], x[1]); v[1] = pk2(x[2], x[3]);
      v[2] = pk2(x[4], x[5]); v[3] = pk2(x[6], x[7]);
    }
  }
  H3_DEV static void load(const RopeArgs& a, const T* p, int u, f32x2 (&v)[4]) {  // !VEC
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = element(a, u, i);
      x[i] = e < a.dim ? to_f32(p[e]) : 0.0f;
    }
    to_pairs(x, v);
  }
  H3_DEV static void store(const RopeArgs& a, T* p, int u, const f32x2 (&v)[4]) {
    float x[8];
    if (VEC && !HALF) {
      x[0] = lo2(v[0]); x[2] = hi2(v[0]); x[4] = lo2(v[1]); x[6] = hi2(v[1]);
      x[1] = lo2(v[2]); x[3] = hi2(v[2]); x[5] = lo2(v[3]); x[7] = hi2(v[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = lo2(v[i]);
        x[2 * i + 1] = hi2(v[i]);
      }
    }
    if constexpr (VEC) {
      if (HALF && 4 * u < a.pairs) {
        Raw<T, 4> lo, hi;
        lo.pack(x);
        hi.pack(x + 4);
        lo.store(p + 4 * u);
        hi.store(p + a.pairs + 4 * u);
      } else {
        Raw<T, 8> o;
        o.pack(x);
        o.store(p + 8 * u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = element(a, u, i);
        if (e < a.dim) p[e] = from_f32<T>(x[i]);
      }
    }
  }
};

// (v1, v2) -> inv * (x1 cw1 - x2 sw2, x2 cw2 + x1 sw1): the angles of a lane's pairs with
// the norm's weights taken in (sw2 carries the minus).
struct Turn {
  f32x2 cw1[2], sw1[2], cw2[2], sw2[2];
};

template <typename T, bool HALF, bool VEC>
H3_DEV void weigh(const RopeArgs& a, const float* weight, int u, const float (&c)[4],
                  const float (&s)[4], Turn& t) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float w[4] = {1.0f, 1.0f, 1.0f, 1.0f};
    if (a.norm && weight != nullptr) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        w[e] = HeadLane<T, HALF, VEC>::weight(a, weight, u, 2 * i + e);
        w[2 + e] = HeadLane<T, HALF, VEC>::weight(a, weight, u, 4 + 2 * i + e);
      }
    }
    t.cw1[i] = pk2(c[2 * i] * w[0], c[2 * i + 1] * w[1]);
    t.sw1[i] = pk2(s[2 * i] * w[0], s[2 * i + 1] * w[1]);
    t.cw2[i] = pk2(c[2 * i] * w[2], c[2 * i + 1] * w[3]);
    t.sw2[i] = pk2(-s[2 * i] * w[2], -s[2 * i + 1] * w[3]);
  }
}

// Norm and turn of one head; every lane of the warp calls it.
template <bool VEC, int G>
H3_DEV void turn_head(const RopeArgs& a, int u, const Turn& t, f32x2 (&x)[4]) {
  if (a.norm) {
    f32x2 sq = mul2(x[0], x[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) sq = fma2(x[i], x[i], sq);
    float sum = lo2(sq) + hi2(sq);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const f32x2 inv = dup2(rsqrtf(__fmaf_rn(sum, a.inv_dim, a.eps)));
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = mul2(x[i], inv);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2 x1 = x[i], x2 = x[i + 2];
    x[i] = mul2(x1, t.cw1[i]);
    x[i + 2] = mul2(x2, t.cw2[i]);
    // an element that is not turned must not meet an infinite neighbour times 0
    if (VEC ? 4 * u < a.pairs : 4 * u + 2 * i + 1 < a.pairs) {
      x[i] = fma2(x2, t.sw2[i], x[i]);
      x[i + 2] = fma2(x1, t.sw1[i], x[i + 2]);
    } else if (!VEC && 4 * u + 2 * i < a.pairs) {  // the first of the two alone
      x[i] = pk2(__fmaf_rn(lo2(x2), lo2(t.sw2[i]), lo2(x[i])), hi2(x[i]));
      x[i + 2] = pk2(__fmaf_rn(lo2(x1), lo2(t.sw1[i]), lo2(x[i + 2])), hi2(x[i + 2]));
    }
  }
}

// A round of a CTA: one item for each of its lane groups, an item being a token and the
// part of its heads (part, part + parts, ... of q, then of k) that the group takes.
struct Round {
  bool here;
  int64_t token;
  int part;

  H3_DEV Round(const RopeArgs& a, int item, bool live) {
    const int items = (int)a.tokens * a.parts;
    here = item < items && live;
    token = item < items ? item / a.parts : 0;
    part = item < items ? item - (int)token * a.parts : 0;
  }
  H3_DEV int count(const RopeArgs& a, const HeadView& v) const {
    return here ? (v.heads - part + a.parts - 1) / a.parts : 0;
  }
};

H3_DEV void lane_angles(const RopeArgs& a, int64_t token, int u, const double* turns,
                        const unsigned char* axis, float (&c)[4], float (&s)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c[i] = 1.0f;
    s[i] = 0.0f;
    if (4 * u + i < a.pairs) pair_angle(a, token, axis[4 * u + i], turns[4 * u + i], c[i], s[i]);
  }
}

// Vector form.  Loops over rounds, tensors and steps are the same for every lane of the
// CTA, so that every lane makes every step (the shuffles need them all).
template <typename T, bool HALF, int G>
__global__ void __launch_bounds__(kRopeThreads, kRopeCtas)
    rope_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int kGroups = kRopeThreads / G;
  constexpr int kWords = sizeof(T) / 2;             // 16-byte words of a lane's eight values
  constexpr int kSlots = kRopeSlotBytes / (16 * kWords);
  using Lane = HeadLane<T, HALF, true>;
  __shared__ __align__(16) uint4 ring[kSlots][kWords][kRopeThreads];
  // the plan, where lanes can read different entries of it at once
  __shared__ double turns[kMaxPairs];
  __shared__ unsigned char axis[kMaxPairs];
  for (int i = threadIdx.x; i < kMaxPairs; i += kRopeThreads) {
    turns[i] = a.turns[i];
    axis[i] = a.axis[i];
  }
  __syncthreads();
  const int u = threadIdx.x % G, group = threadIdx.x / G;
  const bool live = 8 * u < a.dim, turned = 4 * u < a.pairs;
  const int rounds = ((int)a.tokens * a.parts + kGroups - 1) / kGroups;
  const int tensors = a.k.heads > 0 ? 2 : 1;

  // the fetching side, kSlots - 1 steps ahead
  int f_round = blockIdx.x, f_which = 0, f_left = 0, f_count = 0;
  const T* f_in = nullptr;
  int64_t f_step = 0;
  const auto f_open = [&]() {
    const HeadView& v = f_which ? a.k : a.q;
    const Round r(a, f_round * kGroups + group, live);
    f_left = (v.heads + a.parts - 1) / a.parts;
    f_count = r.count(a, v);
    f_step = (int64_t)a.parts * v.in_head;
    f_in = reinterpret_cast<const T*>(v.in) + r.token * v.in_token + (int64_t)r.part * v.in_head;
  };
  const uint32_t my_ring = (uint32_t)__cvta_generic_to_shared(&ring[0][0][threadIdx.x]);
  const auto fetch = [&](int slot) {
    if (f_round < rounds) {
      if (f_count > 0) {
        const uint32_t dst = my_ring + slot * (uint32_t)sizeof(ring[0]);
        if (HALF && turned) {
          if (sizeof(T) == 2) {
            cp_async8(dst, f_in + 4 * u);
            cp_async8(dst + 8, f_in + a.pairs + 4 * u);
          } else {
            cp_async16(dst, f_in + 4 * u);
            cp_async16(dst + (uint32_t)sizeof(ring[0][0]), f_in + a.pairs + 4 * u);
          }
        } else {
          cp_async16(dst, f_in + 8 * u);
          if (sizeof(T) == 4) cp_async16(dst + (uint32_t)sizeof(ring[0][0]), f_in + 8 * u + 4);
        }
      }
      f_in += f_step;
      --f_count;
      if (--f_left == 0) {
        if (++f_which == tensors) {
          f_which = 0;
          f_round += gridDim.x;
        }
        if (f_round < rounds) f_open();
      }
    }
    cp_async_commit();
  };
  f_open();
#pragma unroll 1
  for (int i = 0; i < kSlots - 1; ++i) fetch(i);

  int slot = 0;
#pragma unroll 1
  for (int round = blockIdx.x; round < rounds; round += gridDim.x) {
    const Round r(a, round * kGroups + group, live);
    float c[4], s[4];
    lane_angles(a, r.token, u, turns, axis, c, s);
#pragma unroll 1
    for (int which = 0; which < tensors; ++which) {
      const HeadView& v = which ? a.k : a.q;
      const int count = r.count(a, v);
      const int steps = (v.heads + a.parts - 1) / a.parts;
      Turn t;
      weigh<T, HALF, true>(a, v.weight, u, c, s, t);
      const int64_t out_step = (int64_t)a.parts * v.out_head;
      T* out = reinterpret_cast<T*>(v.out) + r.token * v.out_token + (int64_t)r.part * v.out_head;
#pragma unroll 2
      for (int h = 0; h < steps; ++h) {
        cp_async_wait<kSlots - 2>();
        f32x2 x[4] = {0, 0, 0, 0};
        if (h < count) {
          Raw<T, 8> raw;
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            const uint4 q = ring[slot][w][threadIdx.x];
            raw.w[4 * w] = q.x; raw.w[4 * w + 1] = q.y; raw.w[4 * w + 2] = q.z; raw.w[4 * w + 3] = q.w;
          }
          float f[8];
          raw.unpack(f);
          Lane::to_pairs(f, x);
        }
        // the slot of the step before: its values were used up there
        fetch((slot + kSlots - 1) % kSlots);
        slot = (slot + 1) % kSlots;
        turn_head<true, G>(a, u, t, x);
        if (h < count) Lane::store(a, out, u, x);
        out += out_step;
      }
    }
  }
  cp_async_wait<0>();
}

// Any alignment, any head_dim: one element at a time.
template <typename T, bool HALF, int G>
__global__ void __launch_bounds__(kRopeThreads, 2)
    rope_scalar_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int kGroups = kRopeThreads / G;
  using Lane = HeadLane<T, HALF, false>;
  const int u = threadIdx.x % G, group = threadIdx.x / G;
  const bool live = 8 * u < a.dim;
  const int rounds = ((int)a.tokens * a.parts + kGroups - 1) / kGroups;
#pragma unroll 1
  for (int round = blockIdx.x; round < rounds; round += gridDim.x) {
    const Round r(a, round * kGroups + group, live);
    float c[4], s[4];
    lane_angles(a, r.token, u, a.turns, a.axis, c, s);
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
      const HeadView& v = which ? a.k : a.q;
      const int count = r.count(a, v);
      const int steps = (v.heads + a.parts - 1) / a.parts;
      Turn t;
      weigh<T, HALF, false>(a, v.weight, u, c, s, t);
      for (int h = 0; h < steps; ++h) {
        const int64_t head = r.part + (int64_t)h * a.parts;
        f32x2 x[4] = {0, 0, 0, 0};
        if (h < count)
          Lane::load(a, reinterpret_cast<const T*>(v.in) + r.token * v.in_token + head * v.in_head, u, x);
        turn_head<false, G>(a, u, t, x);
        if (h < count)
          Lane::store(a, reinterpret_cast<T*>(v.out) + r.token * v.out_token + head * v.out_head, u, x);
      }
    }
  }
}

template <typename T, bool HALF, bool VEC, int G>
int launch_rope(RopeArgs& a, int sms, cudaStream_t stream) {
  // One lane group a token; with fewer tokens than lane groups on the GPU the heads are
  // split too, down to four a group, as the sines of a token cost about three heads.
  constexpr int kGroups = kRopeThreads / G;
  const int heads = std::max(a.q.heads, a.k.heads);
  const int ctas = VEC ? kRopeCtas : 2;
  const int64_t room = (int64_t)sms * ctas * kGroups;
  a.parts = (int)std::min<int64_t>((heads + 3) / 4, std::max<int64_t>(1, room / a.tokens));
  const int64_t rounds = (a.tokens * a.parts + kGroups - 1) / kGroups;
  const int grid = (int)std::min<int64_t>(rounds, (int64_t)sms * ctas);
  if constexpr (VEC) rope_kernel<T, HALF, G><<<grid, kRopeThreads, 0, stream>>>(a);
  else rope_scalar_kernel<T, HALF, G><<<grid, kRopeThreads, 0, stream>>>(a);
  return h3host::check_launch();
}

template <typename T, bool HALF, bool VEC>
int launch_rope_width(RopeArgs& a, int sms, cudaStream_t stream) {
  if (a.dim <= 64) return launch_rope<T, HALF, VEC, 8>(a, sms, stream);
  if (a.dim <= 128) return launch_rope<T, HALF, VEC, 16>(a, sms, stream);
  return launch_rope<T, HALF, VEC, 32>(a, sms, stream);
}

template <typename T>
int launch_rope_type(RopeArgs& a, bool half, int sms, cudaStream_t stream) {
  // whole 16-byte pieces: every head starts on a 16-byte boundary and has a multiple of
  // eight elements and of four turned pairs
  bool vec = a.dim % 8 == 0 && a.pairs % 4 == 0;
  for (const HeadView* v : {&a.q, &a.k}) {
    if (v->heads == 0) continue;
    vec = vec && h3host::aligned(v->in, 16) && h3host::aligned(v->out, 16);
    for (int s : {v->in_token, v->in_head, v->out_token, v->out_head})
      vec = vec && (int64_t)s * (int64_t)sizeof(T) % 16 == 0;
  }
  if (half) return vec ? launch_rope_width<T, true, true>(a, sms, stream)
                       : launch_rope_width<T, true, false>(a, sms, stream);
  return vec ? launch_rope_width<T, false, true>(a, sms, stream)
             : launch_rope_width<T, false, false>(a, sms, stream);
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
      q_heads < 1 || q_heads > 4096 || k_heads < 0 || k_heads > 4096 || head_dim < 2 ||
      head_dim > 2 * kMaxPairs || tokens > (1 << 30) || positions == nullptr || axes < 1 || axes > 255 ||
      turns == nullptr || axis == nullptr || pairs < 1 || 2 * pairs > head_dim ||
      pos_kind < H3_POS_I32 || pos_kind > H3_POS_F32 || type < H3_TYPE_F32 || type > H3_TYPE_BF16)
    return H3_ERR_INVALID;
  // a stride that is never taken may be anything: no range or alignment is asked of it
  if (k == nullptr) k_token = k_head = ko_token = ko_head = 0;
  if (tokens <= 1) q_token = qo_token = k_token = ko_token = 0;
  if (q_heads == 1) q_head = qo_head = 0;
  if (k_heads == 1) k_head = ko_head = 0;
  for (int64_t s : {q_token, q_head, qo_token, qo_head, k_token, k_head, ko_token, ko_head})
    if (s < 0 || s > 0x7fffffff) return H3_ERR_INVALID;
  RopeArgs a;
  a.q = HeadView{q, q_out, (int)q_token, (int)q_head, (int)qo_token, (int)qo_head, (int)q_heads, q_weight};
  a.k = HeadView{k, k_out, (int)k_token, (int)k_head, (int)ko_token, (int)ko_head, (int)k_heads, k_weight};
  a.tokens = tokens;
  a.dim = (int)head_dim;
  a.pairs = (int)pairs;
  a.axes = axes;
  a.pos_kind = pos_kind;
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
  // every head reads its token's positions and the weights: no output may lie over them
  const int64_t size = type == H3_TYPE_F32 ? 4 : 2;
  for (const HeadView* v : {&a.q, &a.k}) {
    const auto over = [&](const void* p, int64_t bytes) {  // over a token's heads, from first to last
      const int64_t heads = size * ((v->heads - 1) * (int64_t)v->out_head + head_dim);
      return p != nullptr && h3host::rows_meet(v->out, tokens, heads, size * v->out_token, p, bytes);
    };
    if (over(positions, tokens * axes * (pos_kind == H3_POS_I64 ? 8 : 4)) || over(q_weight, head_dim * 4) ||
        over(k_weight, head_dim * 4))
      return H3_ERR_INVALID;
  }
  int dev;
  h3host::DeviceScope scope;
  if (int s = scope.bind(q, &dev)) return s;
  cudaStream_t st = (cudaStream_t)stream;
  const int sms = h3host::sm_count(dev);
  if (type == H3_TYPE_F32) return launch_rope_type<float>(a, half != 0, sms, st);
  if (type == H3_TYPE_F16) return launch_rope_type<__half>(a, half != 0, sms, st);
  return launch_rope_type<__nv_bfloat16>(a, half != 0, sms, st);
}
