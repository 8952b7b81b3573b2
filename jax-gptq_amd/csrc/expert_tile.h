// Many rows per expert: a workgroup computes BM x 256 outputs of one expert (BM = 128 or 64), K in stages of 64.
//
//   y[p, n] = sum_G s[G, n] (sum_{k in G} x[p, k] (o + c[k, n]) - (o + z[G, n]) sum_{k in G} x[p, k])
//
// Bound by the matrix cores and the instructions that turn codes into their operands.  Everything a stage needs goes
// from memory to LDS without passing a register, four stages deep: the activations of the tile's rows (16 KB at
// BM = 128), the packed codes (8 KB; they stay packed in LDS), the group's scales and zeros and the rows' sums.  One
// barrier per stage: wavefronts wait for their own loads of stage s, meet, and issue the loads of stage s + 3 into the
// buffer that everybody has finished with.  Each wavefront owns 64 x 64 outputs: its four operands of codes are built
// in registers and used for four row blocks.  fp32 sums of a group are scaled into a second set of accumulators, so
// codes stay exact 16-bit operands whatever the scales are.
// A first kernel writes the activations once more, in the order of the operands (fp32: as three bf16 parts), padded to
// whole stages, and the sums of every row over the part of its group up to the end of each stage.
#pragma once
#include "expert_common.h"

namespace xqmm {

constexpr int TILE_BK = 64, TILE_BN = 256, TILE_STAGES = 4;
constexpr int TILE_LONG = 512;            // without groups a sum is closed every 512 features all the same: short sums
                                          // keep the offset of the codes from costing precision

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
template <int VM> __device__ __forceinline__ void wait_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(VM) : "memory");
}

// layout of the workspace
struct Staged {
  int64_t Kp;              // K padded to whole stages
  int64_t row_bytes;       // of the staged activations: parts * Kp * 2
  int64_t per_row;         // sums of a row: one per stage, or per k-step where groups are odd multiples of 32
  size_t sums_at, bytes;
};
static inline Staged staged_layout(int64_t x_rows, int64_t K, int x_dtype, bool half) {
  Staged l;
  l.Kp = round_up64(K, TILE_BK);
  l.row_bytes = (x_dtype == GPTQ_HIP_F32 ? 3 : 1) * l.Kp * 2;
  l.per_row = l.Kp / (half ? 32 : 64);
  l.sums_at = (size_t)round_up64(x_rows * l.row_bytes, 256);
  l.bytes = l.sums_at + (size_t)round_up64(x_rows * l.per_row * 4, 256);
  return l;
}

// One workgroup per row of x.
template <int XT, bool DEALT>
__global__ __launch_bounds__(256) void stage_rows_kernel(const void *__restrict__ x, int64_t K, int64_t Kp,
                                                         int64_t per_row, int64_t row_bytes, int half, int group,
                                                         char *__restrict__ rows, float *__restrict__ sums) {
  extern __shared__ float seg[];                      // sums of the row's stages (or k-steps)
  constexpr int SZ = XT == GPTQ_HIP_F32 ? 4 : 2, WORDS = SZ / 2;
  const int64_t row = blockIdx.x;
  const char *src = (const char *)x + row * K * SZ;
  char *dst = rows + row * row_bytes;
  // (the rounded-up trip count keeps whole wavefronts together for the shuffles)
  for (int64_t c = threadIdx.x; c < (Kp / 8 + 255) / 256 * 256; c += 256) {
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
        for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4 *>(dst + p * Kp * 2 + k * 2) = part[p];
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
    for (int64_t i = threadIdx.x; i < per_row; i += 256) sums[row * per_row + i] = seg[i];
  } else {
    // running sums inside each group: what its last stage holds is the group's
    const int per = group / 64;
    for (int64_t i0 = (int64_t)threadIdx.x * per; i0 < per_row; i0 += 256 * per) {
      float s = 0.f;
      for (int64_t i = i0; i < i0 + per && i < per_row; ++i) {
        s += seg[i];
        sums[row * per_row + i] = s;
      }
    }
  }
}

struct TileArgs {
  ExpertArgs a;
  const char *rows;           // staged activations
  const float *sums;
  int64_t row_bytes, Kp, per_row;
  int stages;                 // Kp / 64
  int close;                  // stages of a group (or of a piece of the sum)
  int grouped;
};

// ZL: how tables lie in LDS: 4 or 2 bytes an element as they are in memory, 0: operands that start or end anywhere,
// whose codes and tables pass through registers (tables converted to fp32)
template <int XT, int BITS, int ZL, bool HALF, int WM>
struct TileShape {
  static constexpr int WAVES = 4 * WM, THREADS = 64 * WAVES, BM = 64 * WM;
  static constexpr int PARTS = Op<XT>::PARTS;
  static constexpr int BROWS = BITS == 4 ? 32 : 64;       // packed rows of a stage
  static constexpr int HN = HALF ? 2 : 1;
  static constexpr int A = PARTS * BM * 128, B = BROWS * 256, Z = HN * 1024, S = HN * BM * 4;
  static constexpr int STAGE = A + B + 2 * Z + S;
  static constexpr int STAGES = 4 * STAGE <= 160 * 1024 ? 4 : (3 * STAGE <= 160 * 1024 ? 3 : 2);
  static constexpr int LDS = STAGES * STAGE;
  // loads of a wavefront per stage
  static constexpr int AI = 2 * PARTS, BI = BROWS / 4 / WAVES;
  static constexpr int SUMS = HN * WM, ITEMS = SUMS + 2 * HN;        // sums by 64 rows, zeros, scales
  static constexpr int MI = (ITEMS + WAVES - 1) / WAVES;
  static constexpr int LOADS = AI + BI + MI;
};

template <int XT, int BITS, int ZL, bool HALF, int WM>
__global__ __launch_bounds__(256 * WM, 2) void tile_kernel(TileArgs t) {
  using T = TileShape<XT, BITS, ZL, HALF, WM>;
  using C = Codes<XT, BITS>;
  using O = Op<XT>;
  typedef __attribute__((address_space(3))) char lds_char;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const ExpertArgs &a = t.a;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  const int64_t N = a.C;
  const bool f32 = a.out_dtype == GPTQ_HIP_F32;

  // Which tile.  Workgroups go round the eight XCDs; each XCD takes a run of the list (panels of four column tiles, row
  // tile by row tile), so what runs on it at a time shares rows and weights in its L2.
  const int row_tiles = count_tiles(a.offsets, a.E, (int)a.P, T::BM);
  const int cols = (int)((N + TILE_BN - 1) / TILE_BN);
  const int64_t total = (int64_t)row_tiles * cols, run = (total + 7) / 8;
  const int64_t pos = blockIdx.x >> 3, item = (blockIdx.x & 7) * run + pos;
  if (pos >= run || item >= total) return;
  const int panel = (int)(item / ((int64_t)row_tiles * 4));
  const int rest = (int)(item - (int64_t)panel * row_tiles * 4);
  const int width = cols - 4 * panel < 4 ? cols - 4 * panel : 4;
  const int64_t n0 = (int64_t)(4 * panel + rest % width) * TILE_BN;
  const Tile tile = find_tile(a.offsets, a.E, (int)a.P, T::BM, rest / width);
  if (tile.rows <= 0) return;
  if (tile.expert == a.E) {                            // rows of nowhere
    for (int i = threadIdx.x; i < tile.rows * TILE_BN; i += T::THREADS) {
      const int64_t n = n0 + i % TILE_BN;
      if (n < N) store_out<XT>(a.out, f32, (int64_t)(tile.row0 + i / TILE_BN) * N + n, 0.f);
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

  // sources of this lane's loads
  const char *arow[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    int m = 8 * (2 * wave + j) + (lane >> 3);
    m = m < tile.rows ? m : tile.rows - 1;             // rows past the last repeat it and are not stored
    arow[j] = t.rows + x_row_of(a.order, a.top_k, a.T, tile.row0 + m) * t.row_bytes + ((lane & 7) ^ (lane >> 3)) * 16;
  }
  const float *srow = nullptr;
  {
    const int sums_item = wave % T::ITEMS % WM;        // the 64 rows whose sums this wavefront may load
    int m = 64 * sums_item + lane;
    m = m < tile.rows ? m : tile.rows - 1;
    srow = t.sums + x_row_of(a.order, a.top_k, a.T, tile.row0 + m) * t.per_row;
  }
  auto table_row = [&](int stage, int h) -> int64_t {
    if (!t.grouped) return 0;
    const uint32_t unit = HALF ? 2u * stage + h : (uint32_t)stage;
    const uint32_t per = HALF ? (uint32_t)(a.group / 32) : (uint32_t)t.close;
    const int64_t r = unit / per;
    return r < tables ? r : tables - 1;
  };
  u32x4 breg[ZL ? 1 : T::BI];
  float zreg[ZL ? 1 : 2 * T::HN * TILE_BN / T::THREADS];

  auto issue = [&](int stage, int slot) __attribute__((always_inline)) {
    const uint32_t base = lds0 + slot * T::STAGE;
#pragma unroll
    for (int p = 0; p < T::PARTS; ++p)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        to_lds_16(arow[j] + p * t.Kp * 2 + (int64_t)stage * 128, base + p * T::BM * 128 + (2 * wave + j) * 1024);
#pragma unroll
    for (int j = 0; j < T::BI; ++j) {
      const int i = wave * T::BI + j, row = 4 * i + (lane >> 4);
      const int turn = BITS == 4 ? (i & 3) : ((i >> 1) & 3);
      int64_t r = (int64_t)stage * T::BROWS + row;
      r = r < a.R ? r : a.R - 1;                       // (past K: any code, the activations are zero)
      const int chunk = (lane & 15) ^ (4 * turn);
      int64_t n = n0 + 16 * chunk;
      if constexpr (ZL) {
        n = n < N ? n : 0;
        to_lds_16(packed + r * N + n, base + T::A + i * 1024);
      } else {
        breg[j] = load_end16(packed + r * N, n, N);
      }
    }
#pragma unroll
    for (int j = 0; j < T::MI; ++j) {
      const int it = (wave + T::WAVES * j) % T::ITEMS;   // (more wavefronts than items: the same bytes twice)
      if (it < T::SUMS) {
        // 64 rows: it % WM, half it / WM
        const int h = it / WM;
        const float *s = srow;
        if (T::MI > 1 || T::ITEMS > T::WAVES) {
          int m = 64 * (it % WM) + lane;
          m = m < tile.rows ? m : tile.rows - 1;
          s = t.sums + x_row_of(a.order, a.top_k, a.T, tile.row0 + m) * t.per_row;
        }
        to_lds_4(s + (HALF ? 2 * stage + h : stage), base + T::A + T::B + 2 * T::Z + (h * T::BM + 64 * (it % WM)) * 4);
      } else if constexpr (ZL != 0) {
        const int which = (it - T::SUMS) / T::HN, h = (it - T::SUMS) % T::HN;
        const char *src = which ? scale : zero;
        int64_t n = ZB == 4 ? n0 + 4 * lane : n0 + 8 * (lane & 31);
        n = n < N ? n : 0;
        to_lds_16(src + (table_row(stage, h) * N + n) * ZB, base + T::A + T::B + which * T::Z + h * 1024);
      }
    }
    if constexpr (!ZL) {
#pragma unroll
      for (int j = 0; j < 2 * T::HN * TILE_BN / T::THREADS; ++j) {
        const int i = threadIdx.x + j * T::THREADS, which = i / (T::HN * TILE_BN), h = i / TILE_BN % T::HN;
        int64_t n = n0 + i % TILE_BN;
        n = n < N ? n : N - 1;
        zreg[j] = table_value(which ? scale : zero, a.zs_dtype, table_row(stage, h) * N + n);
      }
    }
  };
  auto land = [&](int slot) __attribute__((always_inline)) {      // what passed through registers
    if constexpr (!ZL) {
      char *base = lds + slot * T::STAGE;
#pragma unroll
      for (int j = 0; j < T::BI; ++j)
        *reinterpret_cast<u32x4 *>(base + T::A + (wave * T::BI + j) * 1024 + lane * 16) = breg[j];
#pragma unroll
      for (int j = 0; j < 2 * T::HN * TILE_BN / T::THREADS; ++j) {
        const int i = threadIdx.x + j * T::THREADS, which = i / (T::HN * TILE_BN), h = i / TILE_BN % T::HN;
        *reinterpret_cast<float *>(base + T::A + T::B + which * T::Z + h * 1024 + (i % TILE_BN) * 4) = zreg[j];
      }
    }
  };

  f32x4 out[4][4], acc[4][4];                           // [row block][byte of the codes]
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) out[i][q] = acc[i][q] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto close = [&](const char *base, int h) __attribute__((always_inline)) {
    const char *zp = base + T::A + T::B + h * 1024;
    float z[4], s[4];
    const int col = wn * 64 + 4 * l16;
    if constexpr (ZB == 4) {
      const f32x4 zv = *reinterpret_cast<const f32x4 *>(zp + col * 4);
      const f32x4 sv = *reinterpret_cast<const f32x4 *>(zp + T::Z + col * 4);
#pragma unroll
      for (int q = 0; q < 4; ++q) { z[q] = zv[q]; s[q] = sv[q]; }
    } else {
      const bool bf = a.zs_dtype == GPTQ_HIP_BF16;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t zh = *reinterpret_cast<const uint16_t *>(zp + (col + q) * 2);
        const uint32_t sh = *reinterpret_cast<const uint16_t *>(zp + T::Z + (col + q) * 2);
        z[q] = bf ? __builtin_bit_cast(float, zh << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)zh);
        s[q] = bf ? __builtin_bit_cast(float, sh << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)sh);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 sum = *reinterpret_cast<const f32x4 *>(base + T::A + T::B + 2 * T::Z +
                                                         (h * T::BM + wm * 64 + 16 * i + 4 * g4) * 4);
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          out[i][q][r] = fmaf(s[q], fmaf(-(z[q] + C::OFFSET), sum[r], acc[i][q][r]), out[i][q][r]);
    }
  };
  auto step = [&](const char *base, int ks, bool fresh) __attribute__((always_inline)) {
    u32x4 x[4][T::PARTS];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int p = 0; p < T::PARTS; ++p)
        x[i][p] = *reinterpret_cast<const u32x4 *>(base + p * T::BM * 128 + (wm * 64 + 16 * i + l16) * 128 +
                                                   (((4 * ks + g4) ^ (l16 & 7)) * 16));
    uint32_t r[C::ROWS];
    const int chunk = (wn * 4 + (l16 >> 2)) ^ (4 * g4);
#pragma unroll
    for (int i = 0; i < C::ROWS; ++i)
      r[i] = *reinterpret_cast<const uint32_t *>(base + T::A + ((BITS == 4 ? 16 : 32) * ks + C::ROWS * g4 + i) * 256 +
                                                 chunk * 16 + (l16 & 3) * 4);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const u32x4 w = C::operand(r, q);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int p = 0; p < T::PARTS; ++p)
          acc[i][q] = O::mma(x[i][p], w, fresh && p == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[i][q]);
    }
  };

  // stages past the last load it again: every stage then has the same number of loads in flight
  constexpr int AHEAD = T::STAGES - 1;
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) {
    issue(s < t.stages ? s : t.stages - 1, s);
    land(s);
  }
  int in_group = 0, slot = 0, into = AHEAD;
  for (int s = 0; s < t.stages; ++s) {
    wait_and_meet<ZL ? (AHEAD - 1) * T::LOADS : 0>();
    issue(s + AHEAD < t.stages ? s + AHEAD : t.stages - 1, into);
    const char *base = lds + slot * T::STAGE;
    if constexpr (HALF) {
      step(base, 0, true);
      close(base, 0);
      step(base, 1, true);
      close(base, 1);
    } else {
      if (in_group == 0) step(base, 0, true);
      else step(base, 0, false);
      step(base, 1, false);
      if (++in_group == t.close || s + 1 == t.stages) {
        close(base, 0);
        in_group = 0;
      }
    }
    land(into);
    slot = slot + 1 == T::STAGES ? 0 : slot + 1;
    into = into + 1 == T::STAGES ? 0 : into + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // no load may reach LDS after this workgroup's end

#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = wm * 64 + 16 * i + 4 * g4 + r;
      if (m >= tile.rows) continue;
      const int64_t n = n0 + wn * 64 + 4 * l16, at = (int64_t)(tile.row0 + m) * N + n;
      if (n + 4 <= N) {
        store4<XT>(a.out, f32, at, out[i][0][r], out[i][1][r], out[i][2][r], out[i][3][r]);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n + q < N) store_out<XT>(a.out, f32, at + q, out[i][q][r]);
      }
    }
}

template <int XT, int BITS, int ZL, bool HALF, int WM> static int tile_one(hipStream_t s, const TileArgs &t) {
  using T = TileShape<XT, BITS, ZL, HALF, WM>;
  const int64_t blocks = round_up64(tile_bound(t.a.P, t.a.E, T::BM) * ceil_div64(t.a.C, TILE_BN), 8);
  if (blocks * T::THREADS >= (int64_t)1 << 32) return GPTQ_HIP_EINVAL;
  if (!gptq_raise_lds_limit((const void *)tile_kernel<XT, BITS, ZL, HALF, WM>, T::LDS)) return GPTQ_HIP_ELAUNCH;
  tile_kernel<XT, BITS, ZL, HALF, WM><<<(unsigned)blocks, T::THREADS, T::LDS, s>>>(t);
  GPTQ_CHECK_LAUNCH();
  return GPTQ_HIP_OK;
}
template <int XT, int BITS, int WM> static int tile_tables(hipStream_t s, const TileArgs &t, bool half, int zl) {
  if (half) {
    if (zl == 4) return tile_one<XT, BITS, 4, true, WM>(s, t);
    if (zl == 2) return tile_one<XT, BITS, 2, true, WM>(s, t);
    return tile_one<XT, BITS, 0, true, WM>(s, t);
  }
  if (zl == 4) return tile_one<XT, BITS, 4, false, WM>(s, t);
  if (zl == 2) return tile_one<XT, BITS, 2, false, WM>(s, t);
  return tile_one<XT, BITS, 0, false, WM>(s, t);
}

// groups that are no multiple of a stage are closed after every k-step
static inline bool tile_half(int64_t group) { return group % 64 != 0; }

template <int XT> static int tile_launch(hipStream_t s, const ExpertArgs &a, int row_blocks, void *ws) {
  const int64_t K = a.bits == 4 ? 2 * a.R : a.R;
  const bool half = tile_half(a.group);
  const Staged l = staged_layout(a.T, K, a.x_dtype, half);
  const int group = a.group ? (int)a.group : TILE_LONG;
  char *rows = (char *)ws;
  float *sums = (float *)((char *)ws + l.sums_at);
  if (a.bits == 4 && Codes<XT, 4>::DEALT)
    stage_rows_kernel<XT, true><<<(unsigned)a.T, 256, l.per_row * 4, s>>>(a.x, K, l.Kp, l.per_row, l.row_bytes, half,
                                                                          group, rows, sums);
  else
    stage_rows_kernel<XT, false><<<(unsigned)a.T, 256, l.per_row * 4, s>>>(a.x, K, l.Kp, l.per_row, l.row_bytes, half,
                                                                           group, rows, sums);
  GPTQ_CHECK_LAUNCH();
  const TileArgs t = {a, rows, sums, l.row_bytes, l.Kp, l.per_row, (int)(l.Kp / TILE_BK), group / 64, a.group != 0};
  const bool aligned = a.C % 16 == 0 && (uintptr_t)a.packed % 16 == 0 && (uintptr_t)a.zero % 16 == 0 &&
                       (uintptr_t)a.scale % 16 == 0;
  const int zl = !aligned ? 0 : (a.zs_dtype == GPTQ_HIP_F32 ? 4 : 2);
  if constexpr (XT != GPTQ_HIP_F32) {
    if (row_blocks == 8) return a.bits == 4 ? tile_tables<XT, 4, 2>(s, t, half, zl) : tile_tables<XT, 8, 2>(s, t, half, zl);
  }
  return a.bits == 4 ? tile_tables<XT, 4, 1>(s, t, half, zl) : tile_tables<XT, 8, 1>(s, t, half, zl);
}

}  // namespace xqmm
