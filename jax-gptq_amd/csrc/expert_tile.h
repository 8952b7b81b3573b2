// Many rows per expert: a workgroup computes a tile of one expert's outputs, 32 or 64 rows x 256 channels, K in stages
// of 64.  Where the tiles are few, K is cut: in two halves side by side in a workgroup of twice the wavefronts, or in
// parts of their own, which a second kernel adds up.
//
//   y[p, n] = sum_G s[G, n] (sum_{k in G} x[p, k] (o + c[k, n]) - (o + z[G, n]) sum_{k in G} x[p, k])
//
// Bound by the matrix cores and the instructions that turn codes into their operands (many rows), by the bytes of the
// weights (few).  Everything a stage needs goes from memory to LDS without passing a register, three or four stages
// deep: the activations of the tile's rows, the packed codes (they stay packed in LDS), the group's scales and zeros
// and the rows' sums.  One barrier per stage: wavefronts wait for their own loads of stage s, meet, and issue the loads
// of a later stage into the buffer that everybody has finished with.  Each wavefront owns 64 (or 32) x 64 outputs: its
// operands of codes are built in registers and used for two (one) blocks of 32 rows.  fp32 sums of a group are scaled
// into a second set of accumulators, so codes stay exact 16-bit operands whatever the scales are.
// The zero point's term is one product more per group: sum and -(o + z) are fp32 numbers in three bf16 parts each, whose
// six largest products (the rest is below 2^-24 of the term) are six of the sixteen features of a 32 x 32 product.  It
// takes the place of an instruction for every sum, which the vector units have less time for than the matrix cores.
// Measured: 8192 rows of 8 experts on 4096 x 11008, bf16: 851 to 888 us, 830 to 870 TFLOP/s of the 1196 that a large
// library product of plain bf16 matrices reaches.  The matrix cores are busy 44 % of the cycles at the 1.9 to 2.0 GHz
// that the chip keeps up under it; the loads alone, without a product, take 530 us (18 TB/s from L2).  8192 rows on
// 4096 x 4096 fp16: 355 us (773); fp32: 969 us (284, three products each).
// A first kernel writes the activations once more, in the order of the operands (fp32: as three bf16 parts), padded to
// whole stages, and the sums of every row over the part of its group up to the end of each stage, as such an operand.
#pragma once
#include "expert_common.h"
#include <math.h>

namespace xqmm {

constexpr int TILE_BK = 64;
constexpr int TILE_LONG = 512;            // a sum is closed after 512 features at most, without groups and within long
                                          // ones: short sums keep the offset of the codes from costing precision

// 16 or 4 bytes per lane from memory to LDS at dst (the wavefront's) + 16 or 4 * lane.  Inline assembly: the compiler
// knows nothing of the LDS write and adds no waits of its own; the waits are explicit, ahead of the barriers.  (m0 is
// reserved, which the compiler remarks; nothing else in these kernels uses it.)
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void to_lds_16(const void *src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(dst), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void to_lds_4(const void *src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(dst), "v"(src) : "memory", "m0");
}
// the same from a base that all lanes share plus a lane's 32-bit offset
__device__ __forceinline__ void to_lds_16(const void *base, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(dst), "v"(off), "s"(base) : "memory", "m0");
}
template <int VM> __device__ __forceinline__ void wait_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(VM) : "memory");
}

// parts of a contraction at most, stages of one at least, workgroups that run at a time at most
constexpr int TILE_MOST = 4, TILE_MIN_STAGES = 8, TILE_SLOTS = 512;
constexpr int TILE_BN = 256;
static inline int tile_rows(int shape) { return shape == TILE_32x256 ? 32 : 64; }
// groups that are no multiple of a stage are closed after every k-step
static inline bool tile_half(int64_t group) { return group % 64 != 0; }
// stages after which a sum is closed: those of a group, or the largest part of them that TILE_LONG holds.  (65536 features
// in one group, random bf16 rows, 4 bits: largest error 4.3e-4 of the results' size for the whole of it, 1.0e-5 by 512;
// K can be cut within the group, too: 300 rows of 8 experts on 8192 x 4096, a group for each channel, 99 -> 57 us.)
static inline int tile_close(int64_t group) {
  if (tile_half(group)) return 1;
  const int most = TILE_LONG / TILE_BK, stages = group ? (int)(group / TILE_BK) : most;
  int close = stages < most ? stages : most;
  while (stages % close) --close;
  return close;
}

// layout of the workspace
struct Staged {
  int64_t Kp;              // K padded to whole stages
  int64_t row_bytes;       // of the staged activations: parts * Kp * 2
  int64_t per_row;         // sums of a row, 16 bytes each: one per stage, or per k-step where groups are odd multiples of 32
  int most;                // parts of the contraction: see Split
  size_t sums_at, parts_at, bytes;
};
static inline Staged staged_layout(int64_t x_rows, int64_t P, int64_t K, int64_t N, int64_t group, int E, int x_dtype,
                                   int shape) {
  const bool half = tile_half(group);
  Staged l;
  l.Kp = round_up64(K, TILE_BK);
  l.row_bytes = (x_dtype == GPTQ_HIP_F32 ? 3 : 1) * l.Kp * 2;
  l.per_row = l.Kp / (half ? 32 : 64);
  l.sums_at = (size_t)round_up64(x_rows * l.row_bytes, 256);
  l.parts_at = (size_t)round_up64(l.sums_at + (x_rows * l.per_row) * 16, 256);
  const int64_t stages = l.Kp / TILE_BK, pieces = ceil_div64(stages, tile_close(group));
  const int64_t most = pieces < stages / TILE_MIN_STAGES ? pieces : stages / TILE_MIN_STAGES;
  const int BM = tile_rows(shape), BN = TILE_BN;
  // Whether to cut at all is settled here, by the tiles that P rows come to when their experts are drawn at random: the
  // second kernel costs 2 to 5 us also where it finds nothing to add up (8 experts on 4096 x 4096, whole / always cut:
  // 1300 rows, 0.7 of a round, 84 / 90 us; 2000 rows, 1.1 rounds, 128 / 108; 64 experts on 2048 x 1424, 640 rows: 41 / 44).
  const double busy = E * (1.0 - exp(-(double)P / E)), items = ((double)P / BM + busy / 2) * ceil_div64(N, BN);
  const int slots = shape == TILE_64x256_K2 ? TILE_SLOTS / 2 : TILE_SLOTS;
  const bool pays = items - slots * floor(items / slots) <= 0.5 * slots;
  l.most = (int)(most < 1 || !pays ? 1 : (most < TILE_MOST ? most : TILE_MOST));
  l.bytes = l.parts_at + (size_t)unit_bound(P, E, BM, ceil_div64(N, BN), TILE_SLOTS, l.most) * BM * BN * 4;
  return l;
}

// v in three bf16 parts
__device__ __forceinline__ void three_parts(float v, uint32_t *part) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    part[i] = __builtin_bit_cast(uint32_t, v);
    v -= __builtin_bit_cast(float, part[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint32_t upper_halves(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}
// features 0 .. 7 of the zero point's product: parts 1 2 3 1 2 1 of the sum against 1 1 1 2 2 3 of the factor
__device__ __forceinline__ u32x4 sum_operand(float v) {
  uint32_t p[3];
  three_parts(v, p);
  return u32x4{upper_halves(p[0], p[1]), upper_halves(p[2], p[0]), upper_halves(p[1], p[0]), 0u};
}
__device__ __forceinline__ u32x4 factor_operand(float v) {
  uint32_t p[3];
  three_parts(v, p);
  return u32x4{upper_halves(p[0], p[0]), upper_halves(p[0], p[1]), upper_halves(p[1], p[2]), 0u};
}

// One workgroup per row of x.
template <int XT, bool DEALT>
__global__ __launch_bounds__(1024) void stage_rows_kernel(const void *__restrict__ x, int64_t K, int64_t Kp,
                                                         int64_t per_row, int64_t row_bytes, int half, int per,
                                                         char *__restrict__ rows, u32x4 *__restrict__ sums) {
  extern __shared__ float seg[];                      // sums of the row's stages (or k-steps)
  constexpr int SZ = XT == GPTQ_HIP_F32 ? 4 : 2, WORDS = SZ / 2;
  const int64_t row = blockIdx.x;
  const char *src = (const char *)x + row * K * SZ;
  char *dst = rows + row * row_bytes;
  // (the rounded-up trip count keeps whole wavefronts together for the shuffles)
  for (int64_t c = threadIdx.x; c < (Kp / 8 + 63) / 64 * 64; c += blockDim.x) {
    const int64_t k = 8 * c;
    u32x4 v[WORDS];
#pragma unroll
    for (int w = 0; w < WORDS; ++w) v[w] = u32x4{0, 0, 0, 0};
    if (k + 8 <= K) {
#pragma unroll
      for (int w = 0; w < WORDS; ++w) v[w] = load16(src + k * SZ + 16 * w);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (k + i < K) {
          if (SZ == 4) v[(i / 4) % WORDS][i & 3] = ((const uint32_t *)src)[k + i];
          else v[0][i / 2] |= (uint32_t)((const uint16_t *)src)[k + i] << (16 * (i & 1));
        }
      }
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float e;
      if (XT == GPTQ_HIP_F32) {
        const uint32_t w = v[(i / 4) % WORDS][i & 3];       // (a bit cast of the element itself reads element 0)
        e = __builtin_bit_cast(float, w);
      } else {
        const uint32_t h = (v[0][i / 2] >> (16 * (i & 1))) & 0xFFFFu;
        e = XT == GPTQ_HIP_BF16 ? __builtin_bit_cast(float, h << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
      }
      s += e;
    }
    if (k < Kp) {
      if constexpr (XT == GPTQ_HIP_F32) {
        u32x4 part[3];
        parts3(v[0], v[1], part);
#pragma unroll
        for (int p = 0; p < 3; ++p)
          *reinterpret_cast<u32x4 *>(dst + p * Kp * 2 + k * 2) = DEALT ? deal(part[p]) : part[p];
      } else {
        *reinterpret_cast<u32x4 *>(dst + k * 2) = DEALT ? deal(v[0]) : v[0];
      }
    }
    s += __shfl_xor(s, 1);
    s += __shfl_xor(s, 2);
    if (!half) s += __shfl_xor(s, 4);
    const int lanes = half ? 4 : 8;
    if (k < Kp && c % lanes == 0) seg[c / lanes] = s;
  }
  __syncthreads();
  if (half) {
    for (int64_t i = threadIdx.x; i < per_row; i += blockDim.x) sums[row * per_row + i] = sum_operand(seg[i]);
  } else {
    // running sums inside each piece of `per` stages: what its last stage holds is the piece's
    for (int64_t i0 = (int64_t)threadIdx.x * per; i0 < per_row; i0 += (int64_t)blockDim.x * per) {
      float s = 0.f;
      for (int64_t i = i0; i < i0 + per && i < per_row; ++i) {
        s += seg[i];
        sums[row * per_row + i] = sum_operand(s);
      }
    }
  }
}

struct TileArgs {
  ExpertArgs a;
  const char *rows;           // staged activations
  const u32x4 *sums;
  int64_t row_bytes, Kp, per_row;
  int stages;                 // Kp / 64
  int close;                  // stages of a piece of the sum
  int grouped, most;
  float *parts;               // sums of parts
};

// ZL: how tables lie in LDS: 4 or 2 bytes an element as they are in memory, 0: operands that start or end anywhere,
// whose codes and tables pass through registers (tables converted to fp32).
// A wavefront owns 16 RBW rows x 64 channels; four cover the tile, WK such sets take a part of K each.
template <int XT, int BITS, int ZL, bool HALF, int RBW, int WK> struct TileShape {
  static constexpr int SET = 4, WAVES = SET * WK, THREADS = 64 * WAVES, BM = 16 * RBW, BN = TILE_BN;
  static constexpr int PARTS = Op<XT>::PARTS;
  static constexpr int BROWS = BITS == 4 ? 32 : 64;       // packed rows of a part's stage
  static constexpr int HN = HALF ? 2 : 1;
  // one part's rows, codes, zeros and scales (of a group), sums; then all parts'
  static constexpr int AP = PARTS * BM * 128, BP = BROWS * BN, ZP = 2 * BN * 4, SP = 1024;
  static constexpr int A = WK * AP, B = WK * BP, Z = WK * HN * ZP, S = WK * HN * SP;
  // a stage's rows and codes, and its tables, in rings of their own: rows and codes are in registers half a stage before
  // the tables are needed, so their place is free one stage earlier
  static constexpr int DATA = A + B, TABLE = Z + S, STAGE = DATA + TABLE;
  // up to four stages; workgroups of four wavefronts leave room for a second one on the CU where that takes no more
  // than a stage
  static constexpr int ROOM = (WAVES == 4 && 2 * STAGE + TABLE <= 80 * 1024 ? 80 * 1024 : 160 * 1024) - TABLE;
  static constexpr int STAGES = 4 * STAGE <= ROOM ? 4 : (3 * STAGE <= ROOM ? 3 : 2);
  static constexpr int LDS = STAGES * STAGE + TABLE;
  static constexpr int SLOTS = WAVES == 4 && LDS <= 80 * 1024 ? TILE_SLOTS : TILE_SLOTS / 2;   // that run at a time
  // loads of a wavefront per stage
  static constexpr int AI = A / 1024 / WAVES, BI = B / 1024 / WAVES;
  static constexpr int SI = WK * HN, TI = WK * HN * (BN / 128), ITEMS = SI + TI;
  static constexpr int MI = (ITEMS + WAVES - 1) / WAVES;
  static constexpr int LOADS = AI + BI + MI;
  static_assert(A % (1024 * WAVES) == 0 && B % (1024 * WAVES) == 0 && LDS <= 160 * 1024, "whole loads");
  static_assert(RBW % 2 == 0 && (WK == 1 || (WK - 1) * SET * RBW * 4 * 1024 <= LDS), "partial tiles fit");
};

template <int XT, int BITS, int ZL, bool HALF, int RBW, int WK>
__global__ __launch_bounds__(256 * WK, 2) void tile_kernel(TileArgs t) {
  using T = TileShape<XT, BITS, ZL, HALF, RBW, WK>;
  using C = Codes<XT, BITS>;
  using O = Op<XT>;
  typedef __attribute__((address_space(3))) char lds_char;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const ExpertArgs &a = t.a;
  const int lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = wave / T::SET, wn = wave % T::SET;
  const int64_t N = a.C;
  const bool f32 = a.out_dtype == GPTQ_HIP_F32;

  const Unit unit = find_unit<4>(a.offsets, a.E, (int)a.P, T::BM, (uint32_t)((N + T::BN - 1) / T::BN), T::SLOTS, t.most);
  const Item &tile = unit.item;
  if (tile.rows <= 0) return;
  const int64_t n0 = (int64_t)tile.col * T::BN;
  if (tile.expert == a.E) {                            // rows of nowhere
    if (unit.part > 0) return;
    for (int i = threadIdx.x; i < tile.rows * T::BN; i += T::THREADS) {
      const int64_t n = n0 + i % T::BN;
      if (n < N) store_out<XT>(a.out, f32, (int64_t)(tile.row0 + i / T::BN) * N + n, 0.f);
    }
    return;
  }

  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char *)lds;
  const uint8_t *packed = a.packed + (int64_t)tile.expert * a.R * N;
  constexpr int ZB = ZL ? ZL : 4;
  const int64_t tables = t.grouped ? (BITS == 4 ? 2 * a.R : a.R) / a.group : 1;
  const int zsize = a.zs_dtype == GPTQ_HIP_F32 ? 4 : 2;
  const char *zero = (const char *)a.zero + (int64_t)tile.expert * tables * N * zsize;
  const char *scale = (const char *)a.scale + (int64_t)tile.expert * tables * N * zsize;
  // the workgroup's stages of K, and set p's: p * span .. of them; cuts lie between pieces
  const int pieces = (t.stages + t.close - 1) / t.close;
  const int begin = pieces * unit.part / unit.parts * t.close;
  const int end = min(pieces * (unit.part + 1) / unit.parts * t.close, t.stages);
  const int span = WK == 1 ? end - begin : ((end - begin + WK - 1) / WK + t.close - 1) / t.close * t.close;
  auto stage_of = [&](int p, int s) -> int {           // (past the end: the last once more, not multiplied)
    const int st = begin + p * span + s;
    return st < end ? st : end - 1;
  };

  // sources of this lane's loads.  The 16-byte chunks of a row of activations lie turned by the row's number, those of
  // codes by their lane group, so that the reads of a wavefront meet all banks.
  auto row_base = [&](int m) -> int64_t {
    m = m < tile.rows ? m : tile.rows - 1;             // rows past the last repeat it and are not stored
    return x_row_of(a.order, a.top_k, a.T, tile.row0 + m);
  };
  const char *arow[T::AI];
#pragma unroll
  for (int j = 0; j < T::AI; ++j)
    arow[j] = t.rows + row_base(8 * ((wave * T::AI + j) % (T::BM / 8)) + (lane >> 3)) * t.row_bytes +
              ((lane & 7) ^ (lane >> 3)) * 16;
  const u32x4 *srow[T::MI];
#pragma unroll
  for (int j = 0; j < T::MI; ++j) {
    const int it = (wave + T::WAVES * j) % T::ITEMS;
    srow[j] = t.sums;
    if (it < T::SI) srow[j] = t.sums + row_base(lane) * t.per_row;
  }
  auto table_row = [&](int st, int h) -> int64_t {
    if (!t.grouped) return 0;
    const uint32_t unit = HALF ? 2u * st + h : (uint32_t)st;
    const uint32_t per = (uint32_t)a.group / (HALF ? 32u : 64u);
    const int64_t r = unit / per;
    return r < tables ? r : tables - 1;
  };
  // lane group that reads packed row r of a stage
  auto reader = [](int r) -> int { return BITS == 4 ? (r >> 2) & 3 : (r >> 3) & 3; };
  constexpr int CH = T::BN / 16;                       // chunks of a row of codes
  constexpr int TABLE_REGS = WK * T::HN * 2 * T::BN / T::THREADS;
  u32x4 breg[ZL ? 1 : T::BI];
  float zreg[ZL ? 1 : TABLE_REGS];
  // this lane's packed rows and channels in a stage, as offsets from its first row; in the last stage rows past K are
  // replaced by the last (any code: the activations are zero there)
  int brow[T::BI], bcol[T::BI];
  uint32_t boff[T::BI], bend[T::BI];
#pragma unroll
  for (int j = 0; j < T::BI; ++j) {
    const int at = (wave * T::BI + j) % (T::BP / 1024) * (64 / CH) + lane / CH, g = reader(at);
    brow[j] = at;
    bcol[j] = 16 * ((lane % CH) ^ (4 * g));
    const int64_t n = n0 + bcol[j] < N ? n0 + bcol[j] : 0, left = a.R - (int64_t)(t.stages - 1) * T::BROWS;
    boff[j] = (uint32_t)(brow[j] * N + n);
    bend[j] = (uint32_t)((brow[j] < left ? brow[j] : left - 1) * N + n);
  }
  // and its channels in a row of the tables: zeros, then scales, 1 KB each
  const int64_t tn = n0 + (ZB == 4 ? 4 * lane : 8 * (lane % (T::BN / 8)));
  const uint32_t toff = (uint32_t)((tn < N ? tn : 0) * ZB);

  auto issue = [&](int s, int slot, int table) __attribute__((always_inline)) {
    const uint32_t base = lds0 + slot * T::DATA, tbase = lds0 + T::STAGES * T::DATA + table * T::TABLE;
#pragma unroll
    for (int j = 0; j < T::AI; ++j) {
      const int i = wave * T::AI + j, p = i / (T::AP / 1024), q = i % (T::AP / 1024) / (T::BM / 8);
      to_lds_16(arow[j] + q * t.Kp * 2 + (int64_t)stage_of(p, s) * 128, base + i * 1024);
    }
#pragma unroll
    for (int j = 0; j < T::BI; ++j) {
      const int i = wave * T::BI + j, st = stage_of(i / (T::BP / 1024), s);
      if constexpr (ZL) {
        to_lds_16(packed + (int64_t)st * T::BROWS * N, st + 1 < t.stages ? boff[j] : bend[j], base + T::A + i * 1024);
      } else {
        int64_t r = (int64_t)st * T::BROWS + brow[j];
        r = r < a.R ? r : a.R - 1;
        breg[j] = load_end16(packed + r * N, n0 + bcol[j], N);
      }
    }
#pragma unroll
    for (int j = 0; j < T::MI; ++j) {
      const int it = (wave + T::WAVES * j) % T::ITEMS;   // (more wavefronts than items: the same bytes twice)
      if (it < T::SI) {
        const int h = it % T::HN, st = stage_of(it / T::HN, s);
        to_lds_16(srow[j] + (HALF ? 2 * st + h : st), tbase + T::Z + it * 1024);
      } else if constexpr (ZL != 0) {
        const int i = it - T::SI, q = i / (T::BN / 128);
        const int64_t row = table_row(stage_of(q / T::HN, s), q % T::HN) * N * ZB;
        to_lds_16((i & 1 ? scale : zero) + row, toff, tbase + i * 1024);
      }
    }
    if constexpr (!ZL) {
#pragma unroll
      for (int j = 0; j < TABLE_REGS; ++j) {
        const int i = threadIdx.x + j * T::THREADS, which = i / T::BN & 1, q = i / (2 * T::BN);
        int64_t n = n0 + i % T::BN;
        n = n < N ? n : N - 1;
        zreg[j] = table_value(which ? scale : zero, a.zs_dtype,
                              table_row(stage_of(q / T::HN, s), q % T::HN) * N + n);
      }
    }
  };
  auto land = [&](int slot, int table) __attribute__((always_inline)) {      // what passed through registers
    if constexpr (!ZL) {
      char *base = lds + slot * T::DATA;
#pragma unroll
      for (int j = 0; j < T::BI; ++j)
        *reinterpret_cast<u32x4 *>(base + T::A + (wave * T::BI + j) * 1024 + lane * 16) = breg[j];
#pragma unroll
      for (int j = 0; j < TABLE_REGS; ++j)
        *reinterpret_cast<float *>(lds + T::STAGES * T::DATA + table * T::TABLE + (threadIdx.x + j * T::THREADS) * 4) =
            zreg[j];
    }
  };

  // 32 x 32 products over 16 features: row (column) l32, features 8 hi .. + 7; sums lie with column l32, rows
  // 8 (r / 4) + 4 hi + r % 4.  Column block c of a wavefront's 64 channels: channel 4 (l32 % 16) + 2 (l32 / 16) + c, so
  // that a dword of codes serves two lanes and a lane's two channels are neighbours.
  constexpr int RB = RBW / 2;
  const int mycol = 4 * (l32 & 15) + 2 * (l32 >> 4);
  const uint32_t sel[2] = {C::select(2 * (l32 >> 4)), C::select(2 * (l32 >> 4) + 1)};
  f32x16 out[RB][2], acc[RB][2];                        // [row block][column block]
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int r = 0; r < 16; ++r) out[i][c][r] = acc[i][c][r] = 0.f;

  auto table_pair = [&](const char *p, float *v) __attribute__((always_inline)) {       // of this lane's two channels
    const int col = wn * 64 + mycol;
    if constexpr (ZB == 4) {
      const float2 w = *reinterpret_cast<const float2 *>(p + col * 4);
      v[0] = w.x;
      v[1] = w.y;
    } else {
      const uint32_t w = *reinterpret_cast<const uint32_t *>(p + col * 2);
      const bool bf = a.zs_dtype == GPTQ_HIP_BF16;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t h = (w >> (16 * c)) & 0xFFFFu;
        v[c] = bf ? __builtin_bit_cast(float, h << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
      }
    }
  };
  // the zero point's term of a group (features 8 .. 15 of that product are zero on the codes' side)
  auto correct = [&](int table, int h) __attribute__((always_inline)) {
    const char *base = lds + T::STAGES * T::DATA + table * T::TABLE;
    float z[2];
    table_pair(base + (part * T::HN + h) * T::ZP, z);
    u32x4 f[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) f[c] = factor_operand(hi ? 0.f : -(z[c] + C::OFFSET));
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      const u32x4 sum = *reinterpret_cast<const u32x4 *>(base + T::Z + (part * T::HN + h) * T::SP +
                                                         (32 * i + l32) * 16);
#pragma unroll
      for (int c = 0; c < 2; ++c) acc[i][c] = Op<GPTQ_HIP_BF16>::mma32(sum, f[c], acc[i][c]);
    }
  };
  auto close = [&](int table, int h) __attribute__((always_inline)) {
    float s[2];
    table_pair(lds + T::STAGES * T::DATA + table * T::TABLE + (part * T::HN + h) * T::ZP + T::BN * 4, s);
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) out[i][c][r] = fmaf(s[c], acc[i][c][r], out[i][c][r]);
  };
  struct Step {                                         // operands of 32 features: rows, and codes as they are
    u32x4 x[2][RB][T::PARTS];
    uint32_t r[2][C::ROWS];
  };
  // where this lane reads: rows (by k-step and product), codes (by product); the two k-steps of a stage are read at
  // different times, so each has its own addresses, moved on with the ring
  int xat[2][2], rat[2][2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks)
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const int g = 2 * v + hi, chunk = (wn * 4 + ((l32 & 15) >> 2)) ^ (4 * g);
      xat[ks][v] = part * T::AP + (l32) * 128 + (((4 * ks + g) ^ (l32 & 7)) * 16);
      rat[ks][v] = T::A + part * T::BP + C::ROWS * g * T::BN + chunk * 16 + (l32 & 3) * 4;
    }
  auto fetch = [&](Step &f, int ks) __attribute__((always_inline)) {
#pragma unroll
    for (int v = 0; v < 2; ++v) {
#pragma unroll
      for (int i = 0; i < C::ROWS; ++i)
        f.r[v][i] =
            *reinterpret_cast<const uint32_t *>(lds + rat[ks][v] + ((BITS == 4 ? 16 : 32) * ks + i) * T::BN);
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int p = 0; p < T::PARTS; ++p)
          f.x[v][i][p] = *reinterpret_cast<const u32x4 *>(lds + xat[ks][v] + p * T::BM * 128 + 32 * i * 128);
    }
  };
  auto move_on = [&](int ks, int by) __attribute__((always_inline)) {
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      xat[ks][v] += by;
      rat[ks][v] += by;
    }
  };
  auto multiply = [&](Step &f, bool fresh) __attribute__((always_inline)) {
    f32x16 none;
#pragma unroll
    for (int r = 0; r < 16; ++r) none[r] = 0.f;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const u32x4 w = C::operand(f.r[v], sel[c]);
#pragma unroll
        for (int i = 0; i < RB; ++i)
#pragma unroll
          for (int p = 0; p < T::PARTS; ++p)
            acc[i][c] = O::mma32(f.x[v][i][p], w, fresh && v == 0 && p == 0 ? none : acc[i][c]);
      }
  };

  // The operands of a k-step are fetched from LDS while the one before is multiplied; the second half of a stage
  // starts with the barrier that publishes the next stage and frees this one's rows and codes.
  // (fp32: two sets of operands do not fit the registers, a k-step's are fetched when the one before is done.)
  constexpr bool EARLY = T::PARTS == 1;
  constexpr int NS = T::STAGES;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    issue(s, s, s);
    land(s, s);
  }
  wait_and_meet<ZL ? (NS - 1) * T::LOADS : 0>();
  Step f0, f1;
  fetch(f0, 0);
  int slot = 0, table = 0, fresh_table = NS;
  auto stage = [&](int s, bool fresh, bool last) __attribute__((always_inline)) {
    const bool live = WK == 1 || begin + part * span + s < end;
    const int by = slot + 1 == NS ? -(NS - 1) * T::DATA : T::DATA;
    move_on(0, by);
    if (EARLY) fetch(f1, 1);
    const bool ends = !HALF && live && (last || begin + part * span + s + 1 == end);
    if (live) {
      multiply(f0, HALF || fresh);
      if constexpr (HALF) {
        correct(table, 0);
        close(table, 0);
      }
    }
    if (ends) correct(table, 0);
    if (!EARLY) fetch(f1, 1);
    move_on(1, by);
    wait_and_meet<ZL ? (NS - 2) * T::LOADS : 0>();
    issue(s + NS, slot, fresh_table);
    const int next = slot + 1 == NS ? 0 : slot + 1;
    if (EARLY) fetch(f0, 0);
    if (live) {
      multiply(f1, HALF);
      if constexpr (HALF) {
        correct(table, 1);
        close(table, 1);
      }
    }
    if (ends) close(table, 0);
    if (!EARLY) fetch(f0, 0);
    land(slot, fresh_table);
    slot = next;
    table = table == NS ? 0 : table + 1;
    fresh_table = fresh_table == NS ? 0 : fresh_table + 1;
  };
  if constexpr (HALF) {
    for (int s = 0; s < span; ++s) stage(s, true, true);
  } else {
    for (int s = 0; s < span;) {
      stage(s, true, t.close == 1);
      ++s;
      for (int j = 2; j <= t.close && s < span; ++j, ++s) stage(s, false, j == t.close);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // no load may reach LDS after this workgroup's end

  if constexpr (WK > 1) {                               // the other parts hand their sums to the first
    f32x4 *red = reinterpret_cast<f32x4 *>(lds) + wave % T::SET * RB * 8 * 64 + lane;
    __syncthreads();
    if (part > 0) {
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            red[((part - 1) * T::SET * RB * 8 + (i * 2 + c) * 4 + j) * 64] =
                f32x4{out[i][c][4 * j], out[i][c][4 * j + 1], out[i][c][4 * j + 2], out[i][c][4 * j + 3]};
    }
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int p = 0; p < WK - 1; ++p) {
            const f32x4 v = red[(p * T::SET * RB * 8 + (i * 2 + c) * 4 + j) * 64];
#pragma unroll
            for (int r = 0; r < 4; ++r) out[i][c][4 * j + r] += v[r];
          }
  }

  if (unit.parts > 1) {
    f32x4 *to = reinterpret_cast<f32x4 *>(t.parts) + (int64_t)unit.slot * (T::BM * T::BN / 4) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          to[((i * 2 + c) * 4 + j) * (T::SET * 64)] =
              f32x4{out[i][c][4 * j], out[i][c][4 * j + 1], out[i][c][4 * j + 2], out[i][c][4 * j + 3]};
    return;
  }
  const int64_t n = n0 + wn * 64 + mycol;
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int m = 32 * i + 8 * (r / 4) + 4 * hi + r % 4;
      if (m >= tile.rows || n >= N) continue;
      const int64_t at = (int64_t)(tile.row0 + m) * N + n;
      if (n + 1 < N) store2<XT>(a.out, f32, at, out[i][0][r], out[i][1][r]);
      else store_out<XT>(a.out, f32, at, out[i][0][r]);
    }
}

// The tiles that were cut, added up part by part; blockIdx.y takes a quarter of a block of 32 rows.
template <int XT, int RBW> __global__ __launch_bounds__(256) void tile_join_kernel(TileArgs t, uint32_t slots) {
  constexpr int BM = 16 * RBW, BN = TILE_BN;
  const ExpertArgs &a = t.a;
  const uint32_t cols = (uint32_t)((a.C + BN - 1) / BN);
  Tiles tiles(a.offsets, a.E, (int)a.P, BM);
  const Split s = split_items(tiles.total * cols, slots, t.most);
  if (s.parts < 2 || blockIdx.x >= s.rem) return;
  const Item tile = tiles.at<4>(s.full + blockIdx.x, cols);
  if (tile.rows <= 0 || tile.expert == a.E) return;
  const int lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5, wave = threadIdx.x >> 6;
  const int i = blockIdx.y >> 2, j = blockIdx.y & 3, m0 = 32 * i + 8 * j + 4 * hi;
  const int64_t n = (int64_t)tile.col * BN + wave * 64 + 4 * (l32 & 15) + 2 * (l32 >> 4);
  const bool f32 = a.out_dtype == GPTQ_HIP_F32;
  if (n >= a.C || 32 * i + 8 * j >= tile.rows) return;
  const f32x4 *from = reinterpret_cast<const f32x4 *>(t.parts) + (int64_t)blockIdx.x * (BM * BN / 4) + threadIdx.x;
  f32x4 w[TILE_MOST][2];
#pragma unroll
  for (int p = 0; p < TILE_MOST; ++p)
#pragma unroll
    for (int c = 0; c < 2; ++c)                        // (parts that there are not: the last once more, left out below)
      w[p][c] = from[(int64_t)min(p, s.parts - 1) * s.rem * (BM * BN / 4) + ((i * 2 + c) * 4 + j) * 256];
#pragma unroll
  for (int p = 1; p < TILE_MOST; ++p)
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (p < s.parts) w[0][c] += w[p][c];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (m0 + r >= tile.rows) continue;
    const int64_t at = (int64_t)(tile.row0 + m0 + r) * a.C + n;
    if (n + 1 < a.C) store2<XT>(a.out, f32, at, w[0][0][r], w[0][1][r]);
    else store_out<XT>(a.out, f32, at, w[0][0][r]);
  }
}

template <int XT, int BITS, int ZL, bool HALF, int RBW, int WK>
static int tile_one(hipStream_t s, const TileArgs &t) {
  using T = TileShape<XT, BITS, ZL, HALF, RBW, WK>;
  const void *kernel = (const void *)tile_kernel<XT, BITS, ZL, HALF, RBW, WK>;
  const int64_t cols = ceil_div64(t.a.C, T::BN), parts = unit_bound(t.a.P, t.a.E, T::BM, cols, T::SLOTS, t.most);
  const unsigned blocks = item_grid(t.a.P, t.a.E, T::BM, cols, T::THREADS, parts);
  if (!blocks) return GPTQ_HIP_EINVAL;
  if (!gptq_raise_lds_limit(kernel, T::LDS)) return GPTQ_HIP_ELAUNCH;
  tile_kernel<XT, BITS, ZL, HALF, RBW, WK><<<blocks, T::THREADS, T::LDS, s>>>(t);
  GPTQ_CHECK_LAUNCH();
  if (parts) {
    tile_join_kernel<XT, RBW><<<dim3((unsigned)(parts / 2), 2 * RBW), 256, 0, s>>>(t, T::SLOTS);
    GPTQ_CHECK_LAUNCH();
  }
  return GPTQ_HIP_OK;
}
template <int XT, int BITS, int RBW, int WK>
static int tile_tables(hipStream_t s, const TileArgs &t, bool half, int zl) {
  if (half) {
    if (zl == 4) return tile_one<XT, BITS, 4, true, RBW, WK>(s, t);
    if (zl == 2) return tile_one<XT, BITS, 2, true, RBW, WK>(s, t);
    return tile_one<XT, BITS, 0, true, RBW, WK>(s, t);
  }
  if (zl == 4) return tile_one<XT, BITS, 4, false, RBW, WK>(s, t);
  if (zl == 2) return tile_one<XT, BITS, 2, false, RBW, WK>(s, t);
  return tile_one<XT, BITS, 0, false, RBW, WK>(s, t);
}
template <int XT, int BITS> static int tile_shape(hipStream_t s, const TileArgs &t, int shape, bool half, int zl) {
  if (shape == TILE_32x256) return tile_tables<XT, BITS, 2, 1>(s, t, half, zl);
  if constexpr (XT == GPTQ_HIP_F32) {                   // (three operands of 64 rows fill the registers and LDS)
    return GPTQ_HIP_EINVAL;
  } else {
    if (shape == TILE_64x256_K2) return tile_tables<XT, BITS, 4, 2>(s, t, half, zl);
    return tile_tables<XT, BITS, 4, 1>(s, t, half, zl);
  }
}

template <int XT> static int tile_launch(hipStream_t s, const ExpertArgs &a, int shape, void *ws) {
  const int64_t K = a.bits == 4 ? 2 * a.R : a.R;
  const bool half = tile_half(a.group);
  const int close = tile_close(a.group);
  const Staged l = staged_layout(a.T, a.P, K, a.C, a.group, a.E, a.x_dtype, shape);
  char *rows = (char *)ws;
  u32x4 *sums = (u32x4 *)((char *)ws + l.sums_at);
  // (few rows leave most of the chip idle: a whole workgroup of 1024 for each; 300 rows of 11008: 7.7 -> 5.3 us)
  const int threads = a.T <= 1024 ? 1024 : 256;
  if (a.bits == 4 && Codes<XT, 4>::DEALT)
    stage_rows_kernel<XT, true><<<(unsigned)a.T, threads, l.per_row * 4, s>>>(a.x, K, l.Kp, l.per_row, l.row_bytes,
                                                                              half, close, rows, sums);
  else
    stage_rows_kernel<XT, false><<<(unsigned)a.T, threads, l.per_row * 4, s>>>(a.x, K, l.Kp, l.per_row, l.row_bytes,
                                                                               half, close, rows, sums);
  GPTQ_CHECK_LAUNCH();
  const TileArgs t = {a, rows, sums, l.row_bytes, l.Kp, l.per_row, (int)(l.Kp / TILE_BK), close,
                      a.group != 0, l.most, (float *)((char *)ws + l.parts_at)};
  const bool aligned = a.C % 16 == 0 && (uintptr_t)a.packed % 16 == 0 && (uintptr_t)a.zero % 16 == 0 &&
                       (uintptr_t)a.scale % 16 == 0;
  const int zl = !aligned ? 0 : (a.zs_dtype == GPTQ_HIP_F32 ? 4 : 2);
  return a.bits == 4 ? tile_shape<XT, 4>(s, t, shape, half, zl) : tile_shape<XT, 8>(s, t, shape, half, zl);
}

}  // namespace xqmm
