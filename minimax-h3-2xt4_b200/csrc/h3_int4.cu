// Few rows times a 4-bit weight with group scales:
//   y[m][n] = sum_g scale[n][g] * sum_{k in g} x[m][k] (code[n][k] - zero[n][g]) + bias[n]
// code k of a row is the low nibble of byte k / 2 for even k, the high one for odd k.
//
// The floor is the weight's bytes, each read once.  What stands between that and a plain
// product is the unpacking (one weight in half a byte) and, for more than a row or two, the
// multiplications.  Both go to where they cost least: a warp takes 16 output columns and
// runs m16n8k16 products with the unpacked weights as the 16-row operand and eight rows of
// x as the other, so a weight is unpacked once for the CTA's rows (8, 16 or 32), two at a
// time, exactly (code - zero is a small integer in either 16-bit type), and the group's scale
// is applied to the fp32 sum of the group.  (tcgen05.mma could take the unpacked weights from tensor memory,
// written there by tcgen05.st; that form has not been built.)
//
// The order of k inside a product does not matter as long as both operands agree and a
// product stays inside a group, so the weights need no layout of their own: lane t of a row's
// four takes the t-th quarter of each group's bytes in one read of 4, 8 or 16 bytes, and x,
// staged in shared memory, is permuted to match the pairs that the unpacking of a 4-byte word
// yields, (0, 4), (1, 5), (2, 6), (3, 7).  Weights come through cp.async, two stages ahead;
// loaded straight into registers, as far ahead as those allow, the same products took 44 us
// against 38 (9 x 5376 x 32256, fp16, groups of 128).
//
// That case reads 92 MB, 14 us at the measured copy rate; the kernel needs 38 us (0.37), a
// single row of 5120 x 25600 in groups of 64 with zeros 29 us (0.38).  No unit is at its limit:
// of the issue slots 50% and 62% are busy, of the ALU 37% and 53%, of the tensor pipe 29% and
// 14%.  One CTA of 14 and 11 working warps an SM (128 registers a thread, the ring) leaves
// too few warps to cover the waits for weights, for fixed latencies and for the math pipe
// between the 51 and 64 instructions for 16 x 32 weights, 18 of them the unpacking.
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
  int scale_type, out_type;
  int wn;             // column tiles of a CTA at a time
  int chunk;          // k of a chunk of staged x, a multiple of kStageK
  int x_vec;          // rows of x start on 16-byte boundaries
};

constexpr int kInt4Warps = 16;
constexpr int kStageK = 256;  // k of one stage of a warp
constexpr int kStages = 3;
constexpr int kInt4Smem = 226 * 1024;
// Bytes of a slot's row: the stage's, and for rows that do not start on 16-byte boundaries one
// more 16-byte word, as the words around a row's part are fetched whole.
template <bool VEC>
constexpr int kSlotRow = kStageK / 2 + (VEC ? 0 : 16);

// (a & MASK) | b in one instruction, which takes one constant and not two.
template <uint32_t MASK>
H3_DEV uint32_t masked_onto(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "n"(MASK), "r"(b));
  return r;
}

template <typename T>
struct Unpack;

// Eight codes of a word as four pairs (code i, code i + 4) of exact integers code - zero.
// A 16-bit float whose mantissa's low bits are the code is a power of two plus the code:
// 1024 + c in fp16 (or 1024 + 16 c for the upper nibble, scaled back in the subtraction) and
// 128 + c in bf16, so one logical operation and one exact fma unpack two codes.  (The method of
// Y. J. Kim, R. Henry, R. Fahim and H. Awadalla, "Who Says Elephants Can't Run: Bringing Large
// Scale MoE Models into Cloud Scale Production", 2022; the constants follow from the formats.)
template <>
struct Unpack<__half> {
  uint32_t low, high;  // -(1024 + zero) and -(64 + zero) in both halves

  // the bits of -1024 and -64, and what one more adds to them
  H3_DEV explicit Unpack(uint32_t zero) : low(0xe400e400u + zero * 0x00010001u), high(0xd400d400u + zero * 0x00100010u) {}
  H3_DEV void operator()(uint32_t w, uint32_t (&p)[4]) const {
    const uint32_t v = w >> 8;
    p[0] = add(masked_onto<0x000f000fu>(w, 0x64006400u), low);
    p[1] = fma(masked_onto<0x00f000f0u>(w, 0x64006400u), high);
    p[2] = add(masked_onto<0x000f000fu>(v, 0x64006400u), low);
    p[3] = fma(masked_onto<0x00f000f0u>(v, 0x64006400u), high);
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
  H3_DEV static void mma0(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {  // onto zeros
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  }
};

template <>
struct Unpack<__nv_bfloat16> {
  uint32_t low;  // -(128 + zero) in both halves

  H3_DEV explicit Unpack(uint32_t zero) : low(0xc300c300u + zero * 0x00010001u) {}
  H3_DEV void operator()(uint32_t w, uint32_t (&p)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      asm("fma.rn.bf16x2 %0, %1, %2, %3;"
          : "=r"(p[i])
          : "r"(masked_onto<0x000f000fu>(w >> (4 * i), 0x43004300u)), "r"(0x3f803f80u), "r"(low));
  }
  H3_DEV static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  H3_DEV static void mma0(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {  // onto zeros
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  }
};

// A scale as it lies in memory (S: 4 bytes, fp32, or 2, fp16 or bf16), to fp32.
H3_DEV float scale_value(uint32_t bits, int) { return __uint_as_float(bits); }
H3_DEV float scale_value(uint16_t bits, int type) {
  return type == H3_TYPE_F16 ? __half2float(__ushort_as_half(bits)) : __uint_as_float((uint32_t)bits << 16);
}

// Barrier of the `warps` warps that share a column tile (id 1 and up: 0 is the CTA's).
H3_DEV void tile_barrier(int id, int warps) {
  if (warps > 1) asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(warps * 32) : "memory");
  else __syncwarp();
}

// A CTA takes MT * 8 rows of x and, in rounds, wn tiles of 16 columns; its 16 warps are wn
// tiles by WK = 16 / wn slices of k (rounded down, at most the stages; every WK-th stage), whose sums are added in order
// through shared memory at the end of a round.  A warp's stages of all rounds are one
// sequence, fetched kStages - 1 ahead.  Where x of all of k fits, it is staged once.
// GB: 32-k blocks of a group.  VEC: rows of packed weights start on 16-byte boundaries (k a
// multiple of 32); else the aligned words around a row's part are fetched and a lane shifts
// its bytes out of them.
template <typename T, typename S, bool ZEROS, int MT, int GB, bool VEC>
__global__ void __launch_bounds__(kInt4Warps * 32, 1) int4_kernel(const __grid_constant__ Int4Args a) {
  constexpr int kRows = 8 * MT;
  constexpr int kGroups = kStageK / 32 / GB;  // groups of a stage
  constexpr int kRowBytes = kSlotRow<VEC>, kStageBytes = 16 * kRowBytes;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int stages = (a.k + kStageK - 1) / kStageK;
  const int WN = a.wn, WK = min(kInt4Warps / WN, stages);
  // warps beyond wn * wk have no slice: they only help to stage x
  const int wn = warp % WN, wk = warp / WN < WK ? warp / WN : stages + WK;
  const int64_t m0 = (int64_t)blockIdx.y * kRows;
  const int rows = (int)min((int64_t)kRows, a.m - m0);
  const int tiles = (a.n + 15) / 16, rounds = (tiles + WN * (int)gridDim.x - 1) / (WN * (int)gridDim.x);
  // staged x: the rows that exist and one of zeros for those that do not, in 16-byte units of
  // the eight values of a word's codes.  At one step the lanes of a row read every GB-th unit,
  // so the units of four neighbours are exchanged by the number of their four, and
  // neighbouring rows lie half the banks apart: no two of eight lanes meet in a bank.
  const int x_pitch = a.chunk * 2 + 64;
  uint8_t* const ring = smem + warp * kStages * kStageBytes;
  uint8_t* const xs = smem + kInt4Warps * kStages * kStageBytes;
  float* const sums = reinterpret_cast<float*>(xs + (rows + 1) * x_pitch);  // [wn][wk][row][16]
  const uint8_t* x_row[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) x_row[j] = xs + min(j * 8 + g, rows) * x_pitch;
  int x_unit[4];  // of this lane at step i of 128 k
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int u = GB == 4 ? 4 * t + i : GB == 2 ? 8 * (i >> 1) + 2 * t + (i & 1) : 4 * i + t;
    x_unit[i] = ((u & ~3) | ((u ^ (u >> 2)) & 3)) * 16;
  }

  // A stage in its slot: 16 rows of 128 bytes, the 16-byte words of a row exchanged so that
  // the rows that one read of a quarter touches at once fill all banks.
  const auto exchanged = [](int row) { return GB == 4 ? (row & 1) << 2 : GB == 2 ? (row & 3) << 1 : row & 7; };
  const int w_unit = GB == 4 ? t : GB == 2 ? t >> 1 : 0, w_byte = !VEC || GB == 4 ? 0 : GB == 2 ? (t & 1) * 8 : t * 4;

  // the fetching side: stages wk, wk + WK, ... of this warp's tile of every round; rows
  // behind the last column are read as the last.  Behind a row's end a slot keeps any codes:
  // x is 0 there, and so are the scales.
  int f_round = 0, f_stage = wk, f_slot = 0;
  const uint8_t* f_src = nullptr;
  const auto f_open = [&]() {
    const int n0 = ((f_round * (int)gridDim.x + (int)blockIdx.x) * WN + wn) * 16;
    f_src = a.w + (int64_t)min(n0, a.n - 1) * a.pitch;
  };
  const auto fetch = [&]() {
    if (f_round < rounds && f_stage < stages) {
      const int n0 = ((f_round * (int)gridDim.x + (int)blockIdx.x) * WN + wn) * 16;
      const int last = max(min(15, a.n - 1 - n0), 0);  // row of the tile
      uint8_t* dst = ring + f_slot * kStageBytes;
      if (VEC) {
        const int byte = f_stage * (kStageK / 2) + (lane & 7) * 16;
        if (byte < a.pitch) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = i * 4 + (lane >> 3);
            cp_async16((uint32_t)__cvta_generic_to_shared(dst + row * kRowBytes + (((lane & 7) ^ exchanged(row)) << 4)),
                       f_src + (int64_t)min(row, last) * a.pitch + byte);
          }
        }
      } else {
        const uint8_t* const end = a.w + (int64_t)a.n * a.pitch;
        const int left = min(kStageK / 2, a.pitch - f_stage * (kStageK / 2));  // bytes of the part
#pragma unroll 1
        for (int i = lane; i < 16 * 9; i += 32) {
          const int row = i / 9, word = i - row * 9;
          const uint8_t* src = f_src + (int64_t)min(row, last) * a.pitch + f_stage * (kStageK / 2);
          const uint8_t* p = src - ((uintptr_t)src & 15) + word * 16;
          uint8_t* to = dst + row * kRowBytes + word * 16;
          if (p >= src + left) continue;
          if (p >= a.w && p + 16 <= end) {
            cp_async16((uint32_t)__cvta_generic_to_shared(to), p);
          } else {  // the words over the tensor's own ends
            for (int e = 0; e < 16; ++e)
              if (p + e >= a.w && p + e < end) to[e] = p[e];
          }
        }
      }
      f_stage += WK;
      if (f_stage >= stages) {
        f_stage = wk;
        ++f_round;
        f_open();
      }
      f_slot = f_slot + 1 == kStages ? 0 : f_slot + 1;
    }
    cp_async_commit();
  };
  f_open();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch();

  // x of a chunk, zeros behind its columns; a unit's eight values in the order 0 4 1 5 2 6 3 7
  const auto stage_x = [&](int k0) {
    const int units = a.chunk / 8, total = (rows + 1) * units;
#pragma unroll 4
    for (int i = threadIdx.x; i < total; i += kInt4Warps * 32) {
      {
        const int row = i / units, u = i - row * units, k = k0 + u * 8;
        const T* src = reinterpret_cast<const T*>(a.x) + (m0 + row) * a.x_ld;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row < rows && k < a.k) {
          if (a.x_vec && k + 8 <= a.k) {
            v = __ldg(reinterpret_cast<const uint4*>(src + k));
          } else {
            uint32_t h[4] = {0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (k + e < a.k) h[e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(src + k)[e] << (16 * (e & 1));
            v = make_uint4(h[0], h[1], h[2], h[3]);
          }
        }
        const uint4 o = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                                   __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
        *reinterpret_cast<uint4*>(xs + row * x_pitch + ((u & ~3) | ((u ^ (u >> 2)) & 3)) * 16) = o;
      }
    }
  };

  const bool once = a.chunk >= a.k;
  int slot = 0;
  for (int round = 0; round < rounds; ++round) {
    const int n0 = ((round * (int)gridDim.x + (int)blockIdx.x) * WN + wn) * 16;
    float acc[MT][4];
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;

    // scales and zeros of the stage to come; a scale of 0 behind the last group
    S scale[2][kGroups];
    uint8_t zero[2][kGroups];
    const int64_t group0[2] = {(int64_t)min(n0 + g, a.n - 1) * a.groups, (int64_t)min(n0 + g + 8, a.n - 1) * a.groups};
    const auto look = [&](int stage) {
      const int first = stage * kGroups, left = a.groups - first;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int q = 0; q < kGroups; ++q) {
          scale[r][q] = q < left ? __ldg(reinterpret_cast<const S*>(a.scales) + group0[r] + first + q) : (S)0;
          if (ZEROS) zero[r][q] = q < left ? __ldg(a.zeros + group0[r] + first + q) : (uint8_t)0;
        }
    };
    // where the rows g and g + 8 start in their first words
    int skew[2] = {0, 0};
    if (!VEC) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
        skew[r] = (int)((uintptr_t)(a.w + (int64_t)min(n0 + g + 8 * r, a.n - 1) * a.pitch) & 15);
    }
    int s = wk;
    look(s);
    for (int k0 = 0; k0 < a.k; k0 += a.chunk) {
      if (!once || round == 0) {
        if (!once) __syncthreads();
        stage_x(k0);
        __syncthreads();
      }
      const int end = min(stages, (k0 + a.chunk) / kStageK);
#pragma unroll 1
      for (; s < end; s += WK) {
        S now[2][kGroups];
        uint32_t offset[2][kGroups];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int q = 0; q < kGroups; ++q) {
            now[r][q] = scale[r][q];
            offset[r][q] = ZEROS ? zero[r][q] : 8;
          }
        look(s + WK);
        cp_async_wait<kStages - 2>();
        __syncwarp();
        const uint8_t* w_row = ring + slot * kStageBytes + g * kRowBytes + w_byte;
        const int x_at = (s * kStageK - k0) * 2;
#pragma unroll
        for (int q = 0; q < kGroups; ++q) {
          uint32_t w[2][GB];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if (!VEC) {
              const uint8_t* p = w_row + r * 8 * kRowBytes + skew[r] + (q * 4 + t) * 4 * GB;
              const uint32_t* at = reinterpret_cast<const uint32_t*>(p - ((uintptr_t)p & 3));
              const int shift = ((uintptr_t)p & 3) * 8;
              uint32_t low = at[0];
#pragma unroll
              for (int i = 0; i < GB; ++i) {
                const uint32_t high = at[i + 1];
                w[r][i] = __funnelshift_r(low, high, shift);
                low = high;
              }
              continue;
            }
            // rows g and g + 8 are exchanged alike
            const uint8_t* p = w_row + r * 8 * kRowBytes + (((q * GB + w_unit) ^ exchanged(g)) << 4);
            if (GB == 4) {
              const uint4 v = *reinterpret_cast<const uint4*>(p);
              w[r][0] = v.x; w[r][1 % GB] = v.y; w[r][2 % GB] = v.z; w[r][3 % GB] = v.w;
            } else if (GB == 2) {
              const uint2 v = *reinterpret_cast<const uint2*>(p);
              w[r][0] = v.x; w[r][1 % GB] = v.y;
            } else {
              w[r][0] = *reinterpret_cast<const uint32_t*>(p);
            }
          }
          const Unpack<T> u0(offset[0][q]), u1(offset[1][q]);
          float part[MT][4];
#pragma unroll
          for (int i = 0; i < GB; ++i) {
            const int block = q * GB + i;
            uint32_t p0[4], p1[4];
            u0(w[0][i], p0);
            u1(w[1][i], p1);
            const uint32_t first[4] = {p0[0], p1[0], p0[1], p1[1]}, second[4] = {p0[2], p1[2], p0[3], p1[3]};
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              const uint4 xv =
                  *reinterpret_cast<const uint4*>(x_row[j] + x_at + x_unit[block & 3] + (block >> 2) * 256);
              if (i == 0) Unpack<T>::mma0(part[j], first, xv.x, xv.y);
              else Unpack<T>::mma(part[j], first, xv.x, xv.y);
              Unpack<T>::mma(part[j], second, xv.z, xv.w);
            }
          }
          const float f0 = scale_value(now[0][q], a.scale_type), f1 = scale_value(now[1][q], a.scale_type);
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            acc[j][0] = __fmaf_rn(f0, part[j][0], acc[j][0]);
            acc[j][1] = __fmaf_rn(f0, part[j][1], acc[j][1]);
            acc[j][2] = __fmaf_rn(f1, part[j][2], acc[j][2]);
            acc[j][3] = __fmaf_rn(f1, part[j][3], acc[j][3]);
          }
        }
        __syncwarp();
        fetch();  // into the slot of the stage before
        slot = slot + 1 == kStages ? 0 : slot + 1;
      }
    }

    // the slices' sums through shared memory, added in order; then bias and store.  Only the
    // warps of one tile wait for one another.
    if (wk < WK) {
      float* const tile = sums + wn * WK * rows * 16;
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = j * 8 + 2 * t + (i & 1);
          if (row < rows) tile[(wk * rows + row) * 16 + g + (i >> 1) * 8] = acc[j][i];
        }
      tile_barrier(1 + wn, WK);
      for (int i = wk * 32 + lane; i < rows * 16; i += WK * 32) {
        const int n = n0 + (i & 15), row = i >> 4;
        if (n >= a.n) continue;
        float v = 0.0f;
        for (int q = 0; q < WK; ++q) v += tile[q * rows * 16 + i];
        if (a.bias != nullptr) v += __ldg(a.bias + n);
        const int64_t at = (m0 + row) * a.n + n;
        if (a.out_type == H3_TYPE_F32) reinterpret_cast<float*>(a.out)[at] = v;
        else reinterpret_cast<T*>(a.out)[at] = from_f32<T>(v);
      }
      tile_barrier(1 + wn, WK);
    }
  }
  cp_async_wait<0>();
}

template <typename T, typename S, bool ZEROS, int MT, int GB, bool VEC>
int launch_int4(Int4Args& a, int dev, cudaStream_t stream) {
  auto kern = int4_kernel<T, S, ZEROS, MT, GB, VEC>;
  // Column tiles at a time.  The busiest SM's time in stages: its warps' work, which about 12
  // warps saturate, or the longest chain of one warp; and for each round the joining of the
  // slices (1 x 5120 x 25600: 28.4 us as 11 tiles without slices, which the rule takes, 28.7 as
  // 12, 34.8 as 16, 31.7 as 4 tiles of 4 slices in 3 rounds, 52.5 as 8 of 2 in 2, 44.0 as 1 of
  // 16 in 11; 9 x 5376 x 32256: 38.0 as 14, 38.7 as 16, 47.6 as 4, 45.3 as 8, 85.2 as 12 in 2).
  const int stages = (a.k + kStageK - 1) / kStageK, tiles = (a.n + 15) / 16;
  const int blocks_m = (int)((a.m + 8 * MT - 1) / (8 * MT));
  const int ctas = std::max(1, h3host::sm_count(dev) / blocks_m);
  float best = 0.0f;
  for (int wn = 1; wn <= kInt4Warps; ++wn) {
    const int wk = std::min(kInt4Warps / wn, stages);
    const float rounds = (float)((tiles + wn * ctas - 1) / (wn * ctas));
    const float work = rounds * (float)wn * (float)stages / 12.0f, chain = rounds * (float)((stages + wk - 1) / wk);
    const float cost = std::max(work, chain) + rounds * (wk > 1 ? 1.5f : 0.3f);
    if (wn == 1 || cost < best) {
      best = cost;
      a.wn = wn;
    }
  }
  // x of all of k where it fits beside the weights' stages and the sums, else in chunks
  const int rows = (int)std::min<int64_t>(8 * MT, a.m);
  const int fixed = kInt4Warps * (kStages * 16 * kSlotRow<VEC> + rows * 16 * (int)sizeof(float));
  const int all = stages * kStageK, room = (kInt4Smem - fixed) / (rows + 1) - 64;
  a.chunk = room / 2 / kStageK * kStageK;
  if (a.chunk >= all) a.chunk = all;
  else if (const int slices = std::min(kInt4Warps / a.wn, stages) * kStageK; a.chunk >= slices)
    a.chunk -= a.chunk % slices;  // as many stages for every slice of k
  const int smem = fixed + (rows + 1) * (a.chunk * 2 + 64);
  static std::atomic<bool> allowed[h3host::kMaxDevices];
  if (!h3host::allow_smem(kern, kInt4Smem, dev, allowed)) return H3_ERR_CUDA;
  const dim3 grid(std::min(ctas, (tiles + a.wn - 1) / a.wn), blocks_m);
  kern<<<grid, kInt4Warps * 32, smem, stream>>>(a);
  return h3host::check_launch();
}

template <typename T, typename S, bool ZEROS, int GB>
int launch_int4_shape(Int4Args& a, int dev, cudaStream_t stream) {
  const bool vec = a.k % 32 == 0 && h3host::aligned(a.w, 16);
  if (a.m <= 8) return vec ? launch_int4<T, S, ZEROS, 1, GB, true>(a, dev, stream)
                           : launch_int4<T, S, ZEROS, 1, GB, false>(a, dev, stream);
  // 16 rows a CTA, or 32 where all of their x fits (32 x 12800 x 5120: 60 us as two blocks
  // of 16 rows, 88 as one of 32 with two and a half times the chunks of x).  The border is
  // rough: 32 x 1152 x 12800 takes 17 us as one block and would take 14 as two, 17 rows of
  // 5120 x 25600 take 87 as two and would take 66 as one, of 2816 x 25600 44 as two and 38 as one.
  const int64_t rows = std::min<int64_t>(a.m, 32), x32 = (rows + 1) * (2 * (int64_t)a.k + 512 + 64);
  if (a.m <= 16 || x32 + kInt4Warps * (kStages * 16 * (vec ? kSlotRow<true> : kSlotRow<false>) + rows * 64) > kInt4Smem)
    return vec ? launch_int4<T, S, ZEROS, 2, GB, true>(a, dev, stream)
               : launch_int4<T, S, ZEROS, 2, GB, false>(a, dev, stream);
  return vec ? launch_int4<T, S, ZEROS, 4, GB, true>(a, dev, stream)
             : launch_int4<T, S, ZEROS, 4, GB, false>(a, dev, stream);
}

template <typename T, typename S, bool ZEROS>
int launch_int4_group(Int4Args& a, int group, int dev, cudaStream_t stream) {
  if (group == 32) return launch_int4_shape<T, S, ZEROS, 1>(a, dev, stream);
  if (group == 64) return launch_int4_shape<T, S, ZEROS, 2>(a, dev, stream);
  return launch_int4_shape<T, S, ZEROS, 4>(a, dev, stream);
}

template <typename T>
int launch_int4_type(Int4Args& a, int group, int dev, cudaStream_t stream) {
  const bool z = a.zeros != nullptr;
  if (a.scale_type == H3_TYPE_F32)
    return z ? launch_int4_group<T, uint32_t, true>(a, group, dev, stream)
             : launch_int4_group<T, uint32_t, false>(a, group, dev, stream);
  return z ? launch_int4_group<T, uint16_t, true>(a, group, dev, stream)
           : launch_int4_group<T, uint16_t, false>(a, group, dev, stream);
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
      m > 16 * 65535 || k < 1 || n < 1 || x_ld < 0 || (m > 1 && x_ld < k) || k > (1 << 24) ||
      n > (1 << 24) || (group != 32 && group != 64 && group != 128) || !type_ok(scale_type) ||
      (x_type != H3_TYPE_F16 && x_type != H3_TYPE_BF16) ||
      (out_type != H3_TYPE_F32 && out_type != x_type))
    return H3_ERR_INVALID;
  if (m == 0) return H3_OK;
  int dev;
  h3host::DeviceScope scope;
  if (int s = scope.bind(x, &dev)) return s;
  Int4Args a{x, x_ld, m, (int)k, (int)n, w, scales, zeros, bias, out, (int)((k + group - 1) / group),
             (int)((k + 1) / 2), scale_type, out_type, 0, 0,
             h3host::aligned(x, 16) && (m == 1 || x_ld % 8 == 0)};
  cudaStream_t st = (cudaStream_t)stream;
  return x_type == H3_TYPE_F16 ? launch_int4_type<__half>(a, group, dev, st)
                               : launch_int4_type<__nv_bfloat16>(a, group, dev, st);
}
