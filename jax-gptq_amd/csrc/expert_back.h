// The transposed product, the gradient of the activations: a workgroup computes 32, 64 or 128 rows x 256 input features
// of one expert, the contraction runs over the output channels n in stages, cut into parts where the tiles are few.
//
//   y[p, k] = sum_n (x[p, n] s[G(k), n]) (o + c[k, n]) - sum_n (x[p, n] s[G(k), n]) (o + z[G(k), n])
//
// The scale varies along the contraction, so it goes to the activations: a = x s in fp32, as two bf16 parts, each rounded
// to nearest (fp32 activations: all 24 bits in three), which meet the exact codes in as many products; the second sum is
// taken in fp32 over the very values that were multiplied.  What two parts leave out is 2^-18 of a term at most, far below
// the rounding of a 16-bit result; one part of 8 or 11 bits would not be.  The second sum is taken from the first every
// BACK_CLOSE channels.
// Bound by the matrix cores, two products per 16-bit operand pair, and by the instructions that make the parts: a
// wavefront owns 32 or 64 rows x 128 features (one group of 128, or two or four smaller ones), so that the parts of its
// rows are used for four column blocks.  Rows, codes and tables travel to LDS without passing a register, several
// stages deep, one barrier per stage, as in the untransposed tiles.
// Measured: 16384 rows of 8 experts, 4096 x 11008, bf16: 2720 us, 543 TFLOP/s of the 598 that two products each leave;
// 4096 rows on 4096 x 4096, fp16: 293 us (469); 64 rows: 46 us, where 75 MB of weights and tables take 15.  Parts that are
// cut off instead of rounded (2^-15 of a term, always towards zero) took 2645, 295 and 48.5 us; with groups of 32, where
// the parts are made once per group, 577 instead of 661 us for 2000 rows.
#pragma once
#include "expert_tile.h"

namespace xqmm {

// rows padded with zeros to whole stages, where they do not come that way
template <typename U>
__global__ __launch_bounds__(256) void pad_rows_kernel(const U *__restrict__ x, int64_t N, int64_t Np,
                                                       U *__restrict__ out) {
  const int64_t row = blockIdx.x;
  for (int64_t n = threadIdx.x; n < Np; n += 256) out[row * Np + n] = n < N ? x[row * N + n] : U(0);
}
// 16-bit tables as fp32
static __global__ __launch_bounds__(256) void widen_tables_kernel(const char *__restrict__ zero,
                                                           const char *__restrict__ scale, int dtype, int64_t n,
                                                           float *__restrict__ out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    out[i] = table_value(zero, dtype, i);
    out[n + i] = table_value(scale, dtype, i);
  }
}

constexpr int BACK_BN = 256;
// Channels after which the second sum is taken from the first.  With gradients of one sign both grow by a hundred times
// what their difference does, so that over all channels their rounding is what is left of it.  Largest error against the
// size of the results for a gradient of ones, 11008 channels, fp16 rows, 4 bits: 1.6e-3 without, 2.9e-4 / 1.5e-4 / 5.6e-5
// every 512 / 256 / 128; fp32 rows 2.8e-4, 1.2e-5 / 6.8e-6 / 5.0e-6.  It costs 16384 bf16 rows on 4096 x 11008 2 to 4 %
// (2527, then 2574 / 2596 / 2635 us); fp32 rows gain (526, then 474 / 481 / 486 us for 4096 rows on 4096 x 4096).
constexpr int BACK_CLOSE = 128;
// A contraction is cut into at most four parts of at least eight stages (six or eight parts, or of four stages, are no
// faster: what the tiles gain their sums' way through memory costs).
constexpr int BACK_MOST = 4, BACK_MIN_STAGES = 8;

// Rows of a tile, by the rows of an expert on average.  The instructions that make the operands of codes are shared by
// its rows, so a tall tile is the faster the fuller it is.  Measured with 32 / 64 / 128 rows, us a call:
//   8 experts 4096 x 4096, fp16:   8 rows each 46 68 78,  60: 75 78 87,  125: 146 112 139,  200: 180 149 154,
//                                  375: 324 246 242,  512: 368 305 280
//   64 experts 2048 x 1424, bf16:  10 rows each 62 94 140,  31: 89 97 141,  64: 142 146 146,  256: 390 380 412
//   8 experts 4096 x 4096, fp32:   8 rows each 58 62 111,  40: 109 68 114,  162: 218 216 211,  512: 494 481 476
enum BackRows { BACK_32, BACK_64, BACK_128 };
static inline BackRows back_rows(int64_t P, int E) {
  const int64_t rows = P / E;
  return rows <= 32 ? BACK_32 : (rows <= 256 ? BACK_64 : BACK_128);
}

struct BackLayout {
  BackRows rows;
  int slots, most;              // workgroups that run at a time; parts of the contraction: see Split
  bool pad, widen;
  int64_t Np, tables;           // row pitch in elements; table elements of all experts
  size_t tables_at, parts_at, bytes;
};
static inline BackLayout back_layout(int64_t x_rows, int64_t P, int64_t R, int64_t N, int bits, int64_t group,
                                     int E, int x_dtype, int zs_dtype) {
  BackLayout l;
  const int64_t K = bits == 4 ? 2 * R : R, size = x_dtype == GPTQ_HIP_F32 ? 4 : 2;
  l.Np = round_up64(N, 64);
  l.pad = l.Np != N;
  l.widen = zs_dtype != GPTQ_HIP_F32;
  l.tables = (int64_t)E * (group ? K / group : 1) * N;
  l.tables_at = l.pad ? (size_t)round_up64(x_rows * l.Np * size, 256) : 0;
  l.parts_at = l.tables_at + (l.widen ? (size_t)round_up64(2 * l.tables * 4, 256) : 0);
  l.rows = back_rows(P, E);
  l.slots = (x_dtype == GPTQ_HIP_F32 ? 512 : 1024) / (l.rows == BACK_128 ? 2 : 1);
  const int64_t stages = l.Np * size / 128;
  l.most = (int)(stages / BACK_MIN_STAGES < BACK_MOST ? stages / BACK_MIN_STAGES : BACK_MOST);
  if (l.most < 1) l.most = 1;
  const int BM = l.rows == BACK_128 ? 128 : (l.rows == BACK_64 ? 64 : 32);
  l.bytes = l.parts_at + (size_t)unit_bound(P, E, BM, ceil_div64(K, BACK_BN), l.slots, l.most) * BM * BACK_BN * 4;
  return l;
}

struct BackArgs {
  ExpertArgs a;
  const char *x;                // rows of whole stages
  const float *zero, *scale;
  int64_t row_bytes;
  int stages, slots, most;
  float *parts;                 // sums of parts
};

// {bf16(a), bf16(b)}, rounded to nearest
__device__ __forceinline__ uint32_t nearest2(float a, float b) {
  typedef float float2v __attribute__((ext_vector_type(2)));
  typedef __bf16 bfloat2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v){a, b}, bfloat2));
}

// NG: groups a wavefront's 128 features lie in; the tile's rows are WM times RB blocks of 32, a wavefront has RB of them
template <int XT, int BITS, bool ALIGNED, int NG, int WM, int RB> struct BackShape {
  static constexpr int WAVES = 2 * WM, THREADS = 64 * WAVES, BM = 32 * RB * WM, BN = BACK_BN;
  static constexpr int BK = XT == GPTQ_HIP_F32 ? 32 : 64;           // channels of a stage: 128 bytes of a row
  static constexpr int STEPS = BK / 32;
  static constexpr int PARTS = XT == GPTQ_HIP_F32 ? 3 : 2;
  static constexpr int ROWS = BITS == 4 ? BN / 2 : BN;              // packed rows of the tile
  static constexpr int TROWS = 2 * NG;                              // table rows of the tile
  static constexpr int A = BM * 128, B = ROWS * BK, Z = TROWS * 256;
  static constexpr int STAGE = A + B + 2 * Z;
  static constexpr int STAGES = 3 * STAGE <= 40 * 1024 * WM ? 3 : 2;     // wavefronts of eight such tiles' rows share a CU
  static constexpr int LDS = STAGES * STAGE;
  static constexpr int AI = A / 1024 / WAVES, BI = B / 1024 / WAVES, ZI = 2 * TROWS / WAVES;
  static constexpr int LOADS = AI + BI + ZI;
};

template <int XT, int BITS, bool ALIGNED, int NG, int WM, int RB>
__global__ __launch_bounds__(128 * WM, XT == GPTQ_HIP_F32 ? 1 : 2) void back_kernel(BackArgs t) {
  using T = BackShape<XT, BITS, ALIGNED, NG, WM, RB>;
  using O = Op<GPTQ_HIP_BF16>;
  typedef __attribute__((address_space(3))) char lds_char;
  constexpr bool CONVERT = XT == GPTQ_HIP_F32 || BITS == 8;         // codes as c itself, else as 128 + c
  constexpr float OFFSET = CONVERT ? 0.f : 128.f;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const ExpertArgs &a = t.a;
  const int lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int64_t N = a.C, K = BITS == 4 ? 2 * a.R : a.R;
  const bool f32 = a.out_dtype == GPTQ_HIP_F32;

  const Unit unit = find_unit<4>(a.offsets, a.E, (int)a.P, T::BM, (uint32_t)((K + T::BN - 1) / T::BN), t.slots, t.most);
  const Item &tile = unit.item;
  if (tile.rows <= 0) return;
  const int64_t k0 = (int64_t)tile.col * T::BN;
  if (tile.expert == a.E) {                            // rows of nowhere
    if (unit.part > 0) return;
    for (int i = threadIdx.x; i < tile.rows * T::BN; i += T::THREADS) {
      const int64_t k = k0 + i % T::BN;
      if (k < K) store_out<XT>(a.out, f32, (int64_t)(tile.row0 + i / T::BN) * K + k, 0.f);
    }
    return;
  }

  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char *)lds;
  const int64_t tables = a.group ? K / a.group : 1;
  const uint8_t *packed = a.packed + (int64_t)tile.expert * a.R * N;
  const int64_t r0 = BITS == 4 ? k0 / 2 : k0;

  const char *arow[T::AI];
#pragma unroll
  for (int j = 0; j < T::AI; ++j) {
    int m = 8 * (T::AI * wave + j) + (lane >> 3);
    m = m < tile.rows ? m : tile.rows - 1;             // rows past the last repeat it and are not stored
    arow[j] = t.x + x_row_of(a.order, a.top_k, a.T, tile.row0 + m) * t.row_bytes + ((lane & 7) ^ (lane >> 3)) * 16;
  }
  constexpr int CH = T::BK / 16;                       // 16-byte chunks of a packed row in a stage
  const uint8_t *brow[T::BI];
#pragma unroll
  for (int j = 0; j < T::BI; ++j) {
    int64_t r = r0 + (T::BI * wave + j) * (64 / CH) + lane / CH;
    r = r < a.R ? r : a.R - 1;
    brow[j] = packed + r * N;
  }
  // (rows of 64 bytes: chunks lie turned by every fourth row, so that reads of 8 neighbouring rows meet all banks)
  auto turn = [](int row) -> int { return CH == 4 ? (row >> 2) & 3 : 0; };
  const int bcol = 16 * ((lane % CH) ^ turn(lane / CH));
  const float *trow[T::ZI];
#pragma unroll
  for (int j = 0; j < T::ZI; ++j) {
    const int i = T::ZI * wave + j, which = i / T::TROWS, g = i % T::TROWS;
    int64_t row = 0;
    if (a.group) {
      row = (k0 + g * (128 / NG)) / a.group;
      row = row < tables ? row : tables - 1;
    }
    trow[j] = (which ? t.scale : t.zero) + ((int64_t)tile.expert * tables + row) * N;
  }
  u32x4 breg[ALIGNED ? 1 : T::BI];

  auto issue = [&](int stage, int slot) __attribute__((always_inline)) {
    const uint32_t base = lds0 + slot * T::STAGE;
    const int64_t n0 = (int64_t)stage * T::BK;
#pragma unroll
    for (int j = 0; j < T::AI; ++j)
      to_lds_16(arow[j] + (int64_t)stage * 128, base + (T::AI * wave + j) * 1024);
#pragma unroll
    for (int j = 0; j < T::ZI; ++j) {
      int64_t n = n0 + lane % T::BK;
      n = n < N ? n : N - 1;                           // (past N the activations are zero)
      to_lds_4(trow[j] + n, base + T::A + T::B + (T::ZI * wave + j) * 256);
    }
#pragma unroll
    for (int j = 0; j < T::BI; ++j) {
      int64_t n = n0 + bcol;
      if constexpr (ALIGNED) {
        n = n < N ? n : 0;
        to_lds_16(brow[j] + n, base + T::A + (T::BI * wave + j) * 1024);
      } else {
        breg[j] = load_end16(brow[j], n, N);
      }
    }
  };
  auto land = [&](int slot) __attribute__((always_inline)) {
    if constexpr (!ALIGNED) {
#pragma unroll
      for (int j = 0; j < T::BI; ++j)
        *reinterpret_cast<u32x4 *>(lds + slot * T::STAGE + T::A + (T::BI * wave + j) * 1024 + lane * 16) = breg[j];
    }
  };

  // 32 x 32 products over 16 channels: row (column) l32, 8 channels a lane; sums lie with column l32, rows
  // 8 (r / 4) + 4 hi + r % 4.  A lane's packed row gives it two columns at 4 bits (low and high codes), one at 8.
  constexpr int CB = BITS == 4 ? 2 : 1;
  f32x16 acc[RB][4];                                     // [row block][column block]
  float sub[NG][RB];
#pragma unroll
  for (int i = 0; i < RB; ++i) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][c][r] = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) sub[g][i] = 0.f;
  }

  // Channels 32 u + 16 hi .. + 15 of a stage are the lane's in two products w: 16 bytes of a packed row.
  auto step = [&](const char *base, int u, int w) __attribute__((always_inline)) {
    const int n = 32 * u + 16 * hi + 8 * w;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float z[8], s[8];
      const char *zp = base + T::A + T::B + (wn * NG + g) * 256 + n * 4;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const f32x4 zv = *reinterpret_cast<const f32x4 *>(zp + 16 * v);
        const f32x4 sv = *reinterpret_cast<const f32x4 *>(zp + T::Z + 16 * v);
#pragma unroll
        for (int i = 0; i < 4; ++i) { z[4 * v + i] = zv[i] + OFFSET; s[4 * v + i] = sv[i]; }
      }
      u32x4 x[RB][T::PARTS];
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const char *row = base + (wm * 32 * RB + 32 * i + l32) * 128;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {                // two channels at a time, of 4 (fp32) or 8 in 16 bytes
          u32x4 q;
          if (XT == GPTQ_HIP_F32) q = *reinterpret_cast<const u32x4 *>(row + ((n / 4 + e / 4) ^ (l32 & 7)) * 16);
          else q = *reinterpret_cast<const u32x4 *>(row + ((n / 8) ^ (l32 & 7)) * 16);
          float p[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t word = XT == GPTQ_HIP_F32 ? q[(e + k) & 3] : q[e / 2];
            if (XT == GPTQ_HIP_F32) {
              p[k] = __builtin_bit_cast(float, word) * s[e + k];
            } else if (XT == GPTQ_HIP_BF16) {
              p[k] = __builtin_bit_cast(float, k ? word & 0xFFFF0000u : word << 16) * s[e + k];
            } else {                                    // (conversion and product in one instruction)
              const uint16_t h = (uint16_t)(k ? word >> 16 : word);
              p[k] = fmaf((float)__builtin_bit_cast(_Float16, h), s[e + k], 0.f);
            }
          }
          if constexpr (T::PARTS == 2) {                // rounded to nearest, both of them; the sum is of their values
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint32_t both = nearest2(p[0], p[1]);
              x[i][c][e / 2] = both;
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float v = __builtin_bit_cast(float, k ? both & 0xFFFF0000u : both << 16);
                sub[g][i] = fmaf(v, z[e + k], sub[g][i]);
                p[k] -= v;
              }
            }
          } else {
            uint32_t part[2][3];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              sub[g][i] = fmaf(p[k], z[e + k], sub[g][i]);
              three_parts(p[k], part[k]);
            }
#pragma unroll
            for (int c = 0; c < T::PARTS; ++c) x[i][c][e / 2] = upper_halves(part[0][c], part[1][c]);
          }
        }
      }
      // blocks of 32 packed rows with columns in this group; a block of 4-bit codes and groups of 32 columns lies in two
      // groups, each takes its half of the lanes
      constexpr int RBS = 4 / CB, HALF_BLOCK = NG > RBS;
#pragma unroll
      for (int b = HALF_BLOCK ? g / 2 : g * RBS / NG; b < (HALF_BLOCK ? g / 2 + 1 : (g + 1) * RBS / NG); ++b) {
        const int row = wn * (T::ROWS / 2) + 32 * b + l32;
        const uint2 d2 = *reinterpret_cast<const uint2 *>(
            base + T::A + row * T::BK + (((n / 16) ^ turn(row)) * 16) + 8 * w);
        u32x4 op[CB];
        const uint32_t bias = opaque(0x43004300u);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t d = j < 2 ? d2.x : d2.y;
          const int q = 2 * (j & 1);
          if constexpr (CONVERT && BITS == 4) {
            const uint32_t lo = d & 0x0F0F0F0Fu, up = (d >> 4) & 0x0F0F0F0Fu;
            op[0][j] = Codes<XT, BITS>::pair_f32(Codes<XT, BITS>::byte_f32(lo, q), Codes<XT, BITS>::byte_f32(lo, q + 1));
            op[CB - 1][j] = Codes<XT, BITS>::pair_f32(Codes<XT, BITS>::byte_f32(up, q), Codes<XT, BITS>::byte_f32(up, q + 1));
          } else if constexpr (CONVERT) {
            op[0][j] = Codes<XT, BITS>::pair_f32(Codes<XT, BITS>::byte_f32(d, q), Codes<XT, BITS>::byte_f32(d, q + 1));
          } else {
            const uint32_t p = __builtin_amdgcn_perm(0u, d, q ? 0x0C030C02u : 0x0C010C00u);
            op[0][j] = (p & 0x000F000Fu) | bias;
            op[CB - 1][j] = ((p >> 4) & 0x000F000Fu) | bias;
          }
        }
        if (HALF_BLOCK) {
          const uint32_t keep = (l32 >> 4) == (g & 1) ? 0xFFFFFFFFu : 0u;
#pragma unroll
          for (int c = 0; c < CB; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) op[c][j] &= keep;
        }
#pragma unroll
        for (int c = 0; c < CB; ++c)
#pragma unroll
          for (int i = 0; i < RB; ++i)
#pragma unroll
            for (int p = 0; p < T::PARTS; ++p) acc[i][b * CB + c] = O::mma32(x[i][p], op[c], acc[i][b * CB + c]);
      }
      // (one group's parts at a time: with those of the next made early the registers do not suffice)
      if (NG > 1) __builtin_amdgcn_sched_barrier(0);
    }
  };

  // The second sums leave the first: one product each.  A lane's sum lies with row l32, over its half of the channels, in
  // three bf16 parts against -1.
  auto close = [&]() __attribute__((always_inline)) {
    constexpr int RBS = 4 / CB, HALF_BLOCK = NG > RBS;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const uint32_t keep = !HALF_BLOCK || (l32 >> 4) == (g & 1) ? 0xFFFFFFFFu : 0u;
      const u32x4 minus = {0xBF80BF80u & keep, 0x0000BF80u & keep, 0u, 0u};
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        uint32_t part[3];
        three_parts(sub[g][i], part);
        sub[g][i] = 0.f;
        const u32x4 sum = {upper_halves(part[0], part[1]), upper_halves(part[2], 0u), 0u, 0u};
#pragma unroll
        for (int c = HALF_BLOCK ? g / 2 * CB : g * 4 / NG; c < (HALF_BLOCK ? (g / 2 + 1) * CB : (g + 1) * 4 / NG); ++c)
          acc[i][c] = O::mma32(sum, minus, acc[i][c]);
      }
    }
  };

  constexpr int AHEAD = T::STAGES - 1;
  const int first = (int)((int64_t)t.stages * unit.part / unit.parts);
  const int past = (int)((int64_t)t.stages * (unit.part + 1) / unit.parts);
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) {
    issue(first + s < past ? first + s : past - 1, s);
    land(s);
  }
  int slot = 0, into = AHEAD;
  for (int s = first; s < past; ++s) {
    wait_and_meet<ALIGNED ? (AHEAD - 1) * T::LOADS : 0>();
    issue(s + AHEAD < past ? s + AHEAD : past - 1, into);
    const char *base = lds + slot * T::STAGE;
#pragma unroll
    for (int h = 0; h < 2 * T::STEPS; ++h) step(base, h / 2, h % 2);
    if ((s + 1 - first) % (BACK_CLOSE / T::BK) == 0 || s + 1 == past) close();
    land(into);
    slot = slot + 1 == T::STAGES ? 0 : slot + 1;
    into = into + 1 == T::STAGES ? 0 : into + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // no load may reach LDS after this workgroup's end

  if (unit.parts > 1) {
    f32x4 *to = reinterpret_cast<f32x4 *>(t.parts) + (int64_t)unit.slot * (T::BM * T::BN / 4) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (wm * 32 * RB + 32 * i + 8 * j >= tile.rows) continue;        // (rows past the last)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          to[((i * 4 + c) * 4 + j) * T::THREADS] =
              f32x4{acc[i][c][4 * j], acc[i][c][4 * j + 1], acc[i][c][4 * j + 2], acc[i][c][4 * j + 3]};
      }
    return;
  }
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int b = 0; b < 4 / CB; ++b) {
        const int m = wm * 32 * RB + 32 * i + 8 * (r / 4) + 4 * hi + r % 4;
        const int64_t k = k0 + wn * 128 + CB * (32 * b + l32);
        if (m >= tile.rows || k >= K) continue;
        const int64_t at = (int64_t)(tile.row0 + m) * K + k;
        if constexpr (CB == 2) store2<XT>(a.out, f32, at, acc[i][2 * b][r], acc[i][2 * b + 1][r]);
        else store_out<XT>(a.out, f32, at, acc[i][b][r]);
      }
}

// The tiles that were cut, added up part by part: blockIdx.y takes a quarter of a block of 32 rows of each wavefront's,
// and one of its pairs of columns' blocks.
template <int XT, int BITS, int WM, int RB> __global__ __launch_bounds__(128 * WM) void back_join_kernel(BackArgs t) {
  constexpr int CB = BITS == 4 ? 2 : 1, BM = 32 * RB * WM;
  const ExpertArgs &a = t.a;
  const int64_t K = BITS == 4 ? 2 * a.R : a.R;
  const uint32_t cols = (uint32_t)((K + BACK_BN - 1) / BACK_BN);
  Tiles tiles(a.offsets, a.E, (int)a.P, BM);
  const Split s = split_items(tiles.total * cols, t.slots, t.most);
  if (s.parts < 2 || blockIdx.x >= s.rem) return;
  const Item tile = tiles.at<4>(s.full + blockIdx.x, cols);
  const int i = blockIdx.y >> 3, c0 = blockIdx.y >> 1 & 2, j = blockIdx.y & 3;
  const int lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5, wave = threadIdx.x >> 6;
  const int m0 = (wave >> 1) * 32 * RB + 32 * i + 8 * j + 4 * hi;
  if (tile.rows <= m0 - 4 * hi || tile.expert == a.E) return;
  const bool f32 = a.out_dtype == GPTQ_HIP_F32;
  const f32x4 *from = reinterpret_cast<const f32x4 *>(t.parts) + (int64_t)blockIdx.x * (BM * BACK_BN / 4) + threadIdx.x;
  f32x4 w[BACK_MOST][2];
#pragma unroll
  for (int p = 0; p < BACK_MOST; ++p)
#pragma unroll
    for (int c = 0; c < 2; ++c)                        // (parts that there are not: the last once more, left out below)
      w[p][c] = from[(int64_t)min(p, s.parts - 1) * s.rem * (BM * BACK_BN / 4) + ((i * 4 + c0 + c) * 4 + j) * 128 * WM];
#pragma unroll
  for (int p = 1; p < BACK_MOST; ++p)
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (p < s.parts) w[0][c] += w[p][c];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (m0 + r >= tile.rows) continue;
#pragma unroll
    for (int b = 0; b < 2 / CB; ++b) {
      const int64_t k = (int64_t)tile.col * BACK_BN + (wave & 1) * 128 + CB * (32 * (c0 / CB + b) + l32);
      if (k >= K) continue;
      const int64_t at = (int64_t)(tile.row0 + m0 + r) * K + k;
      if constexpr (CB == 2) store2<XT>(a.out, f32, at, w[0][0][r], w[0][1][r]);
      else store_out<XT>(a.out, f32, at, w[0][b][r]);
    }
  }
}

template <int XT, int BITS, bool ALIGNED, int NG, int WM, int RB> static int back_one(hipStream_t s, const BackArgs &t) {
  using T = BackShape<XT, BITS, ALIGNED, NG, WM, RB>;
  const int64_t K = BITS == 4 ? 2 * t.a.R : t.a.R;
  const int64_t cols = ceil_div64(K, T::BN), parts = unit_bound(t.a.P, t.a.E, T::BM, cols, t.slots, t.most);
  const unsigned blocks = item_grid(t.a.P, t.a.E, T::BM, cols, T::THREADS, parts);
  if (!blocks) return GPTQ_HIP_EINVAL;
  if (!gptq_raise_lds_limit((const void *)back_kernel<XT, BITS, ALIGNED, NG, WM, RB>, T::LDS)) return GPTQ_HIP_ELAUNCH;
  back_kernel<XT, BITS, ALIGNED, NG, WM, RB><<<blocks, T::THREADS, T::LDS, s>>>(t);
  GPTQ_CHECK_LAUNCH();
  if (parts) {
    back_join_kernel<XT, BITS, WM, RB><<<dim3((unsigned)(parts / 2), 8 * RB), T::THREADS, 0, s>>>(t);
    GPTQ_CHECK_LAUNCH();
  }
  return GPTQ_HIP_OK;
}
template <int XT, int BITS, bool ALIGNED, int WM, int RB> static int back_groups(hipStream_t s, const BackArgs &t) {
  if (t.a.group % 128 == 0) return back_one<XT, BITS, ALIGNED, 1, WM, RB>(s, t);
  return t.a.group % 64 == 0 ? back_one<XT, BITS, ALIGNED, 2, WM, RB>(s, t)
                             : back_one<XT, BITS, ALIGNED, 4, WM, RB>(s, t);
}
template <int XT, int BITS, bool ALIGNED> static int back_shape(hipStream_t s, const BackArgs &t, BackRows rows) {
  if (rows == BACK_32) return back_groups<XT, BITS, ALIGNED, 1, 1>(s, t);
  return rows == BACK_64 ? back_groups<XT, BITS, ALIGNED, 1, 2>(s, t) : back_groups<XT, BITS, ALIGNED, 2, 2>(s, t);
}

template <int XT> static int back_launch(hipStream_t s, const ExpertArgs &a, void *ws) {
  const BackLayout l = back_layout(a.T, a.P, a.R, a.C, a.bits, a.group, a.E, a.x_dtype, a.zs_dtype);
  constexpr int SZ = XT == GPTQ_HIP_F32 ? 4 : 2;
  BackArgs t = {a, (const char *)a.x, (const float *)a.zero, (const float *)a.scale, l.Np * SZ,
                (int)(l.Np * SZ / 128), l.slots, l.most, (float *)((char *)ws + l.parts_at)};
  if (l.pad) {
    typedef typename std::conditional<SZ == 4, uint32_t, uint16_t>::type U;
    pad_rows_kernel<U><<<(unsigned)a.T, 256, 0, s>>>((const U *)a.x, a.C, l.Np, (U *)ws);
    GPTQ_CHECK_LAUNCH();
    t.x = (const char *)ws;
  }
  if (l.widen) {
    float *f = (float *)((char *)ws + l.tables_at);
    const int64_t blocks = ceil_div64(l.tables, 256);
    widen_tables_kernel<<<(unsigned)(blocks < 65536 ? blocks : 65536), 256, 0, s>>>(
        (const char *)a.zero, (const char *)a.scale, a.zs_dtype, l.tables, f);
    GPTQ_CHECK_LAUNCH();
    t.zero = f;
    t.scale = f + l.tables;
  }
  if (a.C % 16 == 0 && (uintptr_t)a.packed % 16 == 0)
    return a.bits == 4 ? back_shape<XT, 4, true>(s, t, l.rows) : back_shape<XT, 8, true>(s, t, l.rows);
  return a.bits == 4 ? back_shape<XT, 4, false>(s, t, l.rows) : back_shape<XT, 8, false>(s, t, l.rows);
}

}  // namespace xqmm
