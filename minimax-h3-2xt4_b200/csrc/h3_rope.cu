// Per-head RMS norm and rotary positions over several axes, on the q and k heads of a
// projection's output.  Pair p of a head turns by pos[token][axis[p]] * frequency[p]:
//   (v1, v2) <- (v1 cos - v2 sin, v2 cos + v1 sin)
//
// Bound by HBM: every element is read and written once, and the sines and cosines are
// computed in the kernel (a table of them would be read and written too).  They depend on
// the token and the pair alone, so a tile is all heads of a few tokens: a CTA computes the
// angles of the tile once into shared memory, one pair a thread, and then streams the
// tile's heads past them.  CTAs are persistent, so that a thread looks its pair's frequency
// up once.  A head is held by G = 8, 16 or 32 lanes, eight elements (four pairs) each, one
// 16-byte load or two of 8 bytes; the sum of squares is a shuffle tree over those lanes.
#include "h3_types.cuh"

namespace h3 {

constexpr int kMaxPairs = 128;  // head_dim <= 256
constexpr int kRopeThreads = 256;

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
  int tile_tokens, tile_heads;  // of one CTA
  uint32_t head_magic;          // ceil(2^32 / tile_heads)
  float eps, inv_dim;
  const void* positions;
  double turns[kMaxPairs];      // frequency / (2 pi)
  unsigned char axis[kMaxPairs];
};

// Angles of far positions need more than 24 bits: the turns are reduced to a fraction of
// one in 64 bits, and the sine and cosine of that fraction taken in 32.
H3_DEV float2 pair_angle(const RopeArgs& a, int64_t token, int axis, double turns) {
  const int64_t at = token * a.axes + axis;
  double pos;
  if (a.pos_kind == H3_POS_I32) pos = (double)__ldg(reinterpret_cast<const int32_t*>(a.positions) + at);
  else if (a.pos_kind == H3_POS_I64) pos = (double)__ldg(reinterpret_cast<const long long*>(a.positions) + at);
  else pos = (double)__ldg(reinterpret_cast<const float*>(a.positions) + at);
  const double t = pos * turns;
  float s, c;
  sincospif(2.0f * (float)(t - rint(t)), &s, &c);
  return make_float2(c, s);
}

// The four pairs of a lane: first elements in v[0..3], second in v[4..7] when the pairs
// are halves apart, (v[2i], v[2i + 1]) otherwise.  VEC: whole 16-byte (or 8-byte) pieces;
// else one element at a time, any alignment and any head_dim.
template <typename T, bool HALF, bool VEC>
struct HeadLane {
  Raw<T, 8> r;        // VEC
  float x[8];         // !VEC

  H3_DEV static int element(const RopeArgs& a, int u, int i) {
    if (!HALF) return 8 * u + i;
    const int p = 4 * u + (i & 3);          // pair p's element i / 4
    if (p < a.pairs) return i < 4 ? p : p + a.pairs;
    return 2 * p + (i >> 2);                // behind the turned elements: neighbours
  }
  H3_DEV void load(const RopeArgs& a, const T* p, int u) {
    if constexpr (VEC) {
      if (HALF && 4 * u < a.pairs) {
        Raw<T, 4> lo, hi;
        lo.load(p + 4 * u);
        hi.load(p + a.pairs + 4 * u);
#pragma unroll
        for (int i = 0; i < Raw<T, 4>::kWords; ++i) {
          r.w[i] = lo.w[i];
          r.w[Raw<T, 4>::kWords + i] = hi.w[i];
        }
      } else {
        r.load(p + 8 * u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = element(a, u, i);
        x[i] = e < a.dim ? to_f32(p[e]) : 0.0f;
      }
    }
  }
  H3_DEV void values(float* v) const {
    if constexpr (VEC) {
      r.unpack(v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = x[i];
    }
  }
  H3_DEV static void store(const RopeArgs& a, T* p, int u, const float* v) {
    if constexpr (VEC) {
      if (HALF && 4 * u < a.pairs) {
        Raw<T, 4> lo, hi;
        lo.pack(v);
        hi.pack(v + 4);
        lo.store(p + 4 * u);
        hi.store(p + a.pairs + 4 * u);
      } else {
        Raw<T, 8> o;
        o.pack(v);
        o.store(p + 8 * u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = element(a, u, i);
        if (e < a.dim) p[e] = from_f32<T>(v[i]);
      }
    }
  }
  // weight of element i of this lane; VEC keeps neighbours behind the turned elements in
  // memory order, so there the index is the memory's
  H3_DEV static int weight_index(const RopeArgs& a, int u, int i) {
    if (VEC && HALF && 4 * u >= a.pairs) return 8 * u + i;
    return element(a, u, i);
  }
};

template <typename T, bool HALF, bool VEC, int G>
__global__ void __launch_bounds__(kRopeThreads, VEC ? 4 : 2)
    rope_kernel(const __grid_constant__ RopeArgs a) {
  // A lane reads its four angles and its eight weights as 16-byte words, the lanes of a
  // group side by side: [buffer][token][pair & 2][lane] and [q, k][half][lane].
  __shared__ __align__(16) float4 turn[2][kRopeThreads / 2 + 64];
  __shared__ __align__(16) float4 weight[2][2][32];
  constexpr int kGroups = kRopeThreads / G;
  constexpr int kAhead = sizeof(T) == 2 ? 4 : 2;  // heads a lane group has in flight, 64 bytes a lane
  using Lane = HeadLane<T, HALF, VEC>;
  const int u = threadIdx.x % G, group = threadIdx.x / G;
  const int quads = (a.pairs + 3) / 4;  // lanes with turned pairs
  const int head0 = blockIdx.y * a.tile_heads;
  const int heads = min(a.tile_heads, a.q.heads + a.k.heads - head0);
  const bool live = 8 * u < a.dim;

  const bool weighted = a.norm && (a.q.weight != nullptr || a.k.weight != nullptr);
  if (weighted) {
    for (int i = threadIdx.x; i < 512; i += kRopeThreads) {
      const float* w = i < 256 ? a.q.weight : a.k.weight;
      const int lane = (i & 255) >> 3, e = Lane::weight_index(a, lane, i & 7);
      reinterpret_cast<float*>(&weight[i >> 8][(i >> 2) & 1][lane])[i & 3] =
          w != nullptr && e < a.dim ? __ldg(w + e) : 1.0f;
    }
  }
  // this thread's pair of the tile's angles
  const int my_tok = threadIdx.x / a.pairs, my_pair = threadIdx.x - my_tok * a.pairs;
  const double my_turns = my_tok < a.tile_tokens ? a.turns[my_pair] : 0.0;
  const int my_axis = my_tok < a.tile_tokens ? a.axis[my_pair] : 0;
  float2* my_slot = reinterpret_cast<float2*>(
      &turn[0][(my_tok * 2 + ((my_pair >> 1) & 1)) * quads + (my_pair >> 2)]) + (my_pair & 1);

  int buffer = 0;
  for (int64_t tile = blockIdx.x; tile * a.tile_tokens < a.tokens; tile += gridDim.x, buffer ^= 1) {
    const int64_t token0 = tile * a.tile_tokens;
    const int tokens = (int)min((int64_t)a.tile_tokens, a.tokens - token0);
    const int items = tokens * a.tile_heads;
    if (my_tok < tokens)
      my_slot[buffer * (sizeof(turn[0]) / sizeof(float2))] =
          pair_angle(a, token0 + my_tok, my_axis, my_turns);
    // one barrier a tile: the buffer written next was last read before this one
    __syncthreads();
    const T* q_in = reinterpret_cast<const T*>(a.q.in) + token0 * a.q.in_token;
    const T* k_in = reinterpret_cast<const T*>(a.k.in) + token0 * a.k.in_token;
    T* q_out = reinterpret_cast<T*>(a.q.out) + token0 * a.q.out_token;
    T* k_out = reinterpret_cast<T*>(a.k.out) + token0 * a.k.out_token;

    // every lane of the CTA makes every step (the shuffles need them all); `head` is -1
    // where there is nothing to do
    for (int base = group; base - group < items; base += kGroups * kAhead) {
      Lane lane[kAhead];
      int tok[kAhead], head[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int it = base + j * kGroups;
        // it / tile_heads: exact, their product is below 2^32; 2^32 itself has no 32-bit form
        tok[j] = a.head_magic != 0 ? (int)__umulhi((uint32_t)it, a.head_magic) : it;
        head[j] = it - tok[j] * a.tile_heads;
        head[j] = it < items && head[j] < heads && live ? head[j] + head0 : -1;
        if (head[j] >= 0) {
          const bool is_k = head[j] >= a.q.heads;
          const T* in = is_k ? k_in : q_in;
          in += (int64_t)tok[j] * (is_k ? a.k.in_token : a.q.in_token) +
                (int64_t)(is_k ? head[j] - a.q.heads : head[j]) * (is_k ? a.k.in_head : a.q.in_head);
          lane[j].load(a, in, u);
        }
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        float v[8];
        const bool is_k = head[j] >= a.q.heads;
        if (head[j] >= 0) {
          lane[j].values(v);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        }
        if (a.norm) {
          float sum = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) sum = __fmaf_rn(v[i], v[i], sum);
#pragma unroll
          for (int o = G / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          const float inv = rsqrtf(__fmaf_rn(sum, a.inv_dim, a.eps));
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] *= inv;
          if (weighted) {
            const float4 w0 = weight[is_k][0][u], w1 = weight[is_k][1][u];
            v[0] *= w0.x; v[1] *= w0.y; v[2] *= w0.z; v[3] *= w0.w;
            v[4] *= w1.x; v[5] *= w1.y; v[6] *= w1.z; v[7] *= w1.w;
          }
        }
        if (head[j] < 0) continue;
        if (u < quads) {
          const float4* t = &turn[buffer][tok[j] * 2 * quads + u];
          const float4 t0 = t[0], t1 = t[quads];
          const float c[4] = {t0.x, t0.z, t1.x, t1.z}, s[4] = {t0.y, t0.w, t1.y, t1.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (!VEC && 4 * u + i >= a.pairs) continue;
            if (VEC && !HALF && 4 * u + i >= a.pairs) continue;
            float& v1 = v[HALF ? i : 2 * i];
            float& v2 = v[HALF ? i + 4 : 2 * i + 1];
            const float r1 = __fmaf_rn(v1, c[i], -(v2 * s[i]));
            v2 = __fmaf_rn(v2, c[i], v1 * s[i]);
            v1 = r1;
          }
        }
        T* out = is_k ? k_out : q_out;
        out += (int64_t)tok[j] * (is_k ? a.k.out_token : a.q.out_token) +
               (int64_t)(is_k ? head[j] - a.q.heads : head[j]) * (is_k ? a.k.out_head : a.q.out_head);
        Lane::store(a, out, u, v);
      }
    }
  }
}

template <typename T, bool HALF, bool VEC, int G>
int launch_rope(RopeArgs& a, int sms, cudaStream_t stream) {
  // A tile is as many tokens as give every thread one angle; with too few tiles for the
  // SMs it shrinks, at last to a part of one token's heads (rounds of the lane groups).
  constexpr int kGroups = kRopeThreads / G;
  const int heads = a.q.heads + a.k.heads;
  int tokens = std::max<int>(1, kRopeThreads / a.pairs);
  tokens = std::min<int>(tokens, 16);
  while (tokens > 1 && (a.tokens + tokens - 1) / tokens < 2 * sms) tokens /= 2;
  a.tile_tokens = tokens;
  a.tile_heads = heads;
  const int64_t tiles = (a.tokens + tokens - 1) / tokens;
  if (tokens == 1 && tiles < sms)
    a.tile_heads = std::min<int>(heads, kGroups * std::max<int>(1, (int)(tiles * heads / ((int64_t)sms * kGroups))));
  const int splits = (heads + a.tile_heads - 1) / a.tile_heads;
  a.head_magic = (uint32_t)(((1ull << 32) + a.tile_heads - 1) / a.tile_heads);
  const int grid = (int)std::min<int64_t>(tiles, (int64_t)sms * (VEC ? 4 : 2));
  rope_kernel<T, HALF, VEC, G><<<dim3(grid, splits), kRopeThreads, 0, stream>>>(a);
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
  // whole 16-byte pieces: every head starts on a 16-byte boundary, is a multiple of eight
  // elements, and halves (if paired so) are multiples of four pairs
  bool vec = a.dim % 8 == 0 && (!half || a.pairs % 4 == 0);
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
      head_dim > 2 * kMaxPairs || positions == nullptr || axes < 1 || axes > 255 ||
      turns == nullptr || axis == nullptr || pairs < 1 || 2 * pairs > head_dim ||
      pos_kind < H3_POS_I32 || pos_kind > H3_POS_F32 || type < H3_TYPE_F32 || type > H3_TYPE_BF16)
    return H3_ERR_INVALID;
  if (k == nullptr) k_token = k_head = ko_token = ko_head = 0;
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
  int dev;
  h3host::DeviceScope scope;
  if (int s = scope.bind(q, &dev)) return s;
  cudaStream_t st = (cudaStream_t)stream;
  const int sms = h3host::sm_count(dev);
  if (type == H3_TYPE_F32) return launch_rope_type<float>(a, half != 0, sms, st);
  if (type == H3_TYPE_F16) return launch_rope_type<__half>(a, half != 0, sms, st);
  return launch_rope_type<__nv_bfloat16>(a, half != 0, sms, st);
}
