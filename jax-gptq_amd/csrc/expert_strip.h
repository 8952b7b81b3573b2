// Few rows per expert: y[p, n] for 16 rows of one expert and a strip of 16 CW channels, over all of K.
//
//   y[p, n] = sum_G s[G, n] (sum_{k in G} x[p, k] (o + c[k, n]) - (o + z[G, n]) sum_{k in G} x[p, k])
//
// Bound by the weights' bytes (every expert that any row picked is read once from HBM as long as its rows fit one
// tile).  Each of the eight wavefronts takes every eighth unit of 32 KS input features and multiplies all rows of the
// tile with the whole strip (sixteen wavefronts, for the calls that have few workgroups, are a quarter slower): nothing
// is shared while K runs, so there is no barrier, and a wavefront has the next units' loads (weights, tables,
// activations) in flight while it multiplies one.  A workgroup covers K by itself, so no partial result leaves it: no
// workspace, no counter, no second launch.
// Measured: 1 token of 2 experts on 4096 x 11008, 4 bits, groups of 128, 14.4 us a call for 48 MB of codes and tables
// (3.3 TB/s, of which the start and end of the launch take 4 to 5 us; a copy runs at 5.2); 12 tokens of 4 of 64 experts
// on 2048 x 1424, groups of 64, 17.5 us for 63 MB.
// Codes enter the matrix cores exactly; the group's sum of activations comes from one more product against ones; the
// scale and the zero point (with the codes' offset) are applied to the fp32 sums group by group.
// In a k-step of 32 features lane (l16, g) owns features 8 g .. 8 g + 7; it loads CW consecutive bytes of a packed row;
// byte q of all lanes' rows is channel CW l16 + q: product tile q.  Weights go to registers as they are needed there;
// the activations of 16 rows, which as operands would be 16-byte pieces of 16 places, go to LDS in whole lines.
#pragma once
#include "expert_tile.h"
#include <math.h>

namespace xqmm {

constexpr int STRIP_WAVES = 8;

// DMA: the rows' features travel through LDS (16-byte aligned rows); else through registers.
template <int XT, int BITS, int ZT, int KS, int CW, bool DMA> struct Strip {
  using C = Codes<XT, BITS>;
  using O = Op<XT>;
  static constexpr int ZB = ZT == GPTQ_HIP_F32 ? 4 : 2; // bytes of a table's element
  static constexpr int SPAN = 32 * KS;                  // input features of a unit, all in one group
  static constexpr int DW = CW / 4;                     // dwords of a packed row
  static constexpr int XW = XT == GPTQ_HIP_F32 ? 2 : 1; // 16-byte words of 8 activations
  static constexpr int ZD = CW * ZB / 4;                // dwords of a lane's channels in one table row
  struct Unit {
    uint32_t w[KS][DW][C::ROWS];
    uint32_t z[ZD], s[ZD];
    u32x4 x[DMA ? 1 : KS][XW];
  };
  // a unit's 16 rows in LDS, a wavefront's own: 16-byte chunks of a row lie turned by its number, so that the reads of
  // 8 neighbouring lanes (rows) meet all banks
  static constexpr int SZ = XT == GPTQ_HIP_F32 ? 4 : 2, CPR = SPAN * SZ / 16, PIECE = 16 * SPAN * SZ;
  static __device__ __forceinline__ int turn(int row) { return CPR >= 8 ? row & 7 : (row >> 2) & 3; }
  struct Ctx {
    const uint8_t *w;             // packed row 0 of the expert (the same for all lanes, as all pointers but x)
    const char *zero, *scale;     // table row 0
    const char *x;                // the lane's row of x, at the lane group's first feature
    const char *row[PIECE / 1024];   // DMA: the rows whose chunks the lane fetches, at those chunks
    int64_t K, R, N;
    uint32_t col, at_w, at_z;     // the lane's first channel; its bytes past `w` and past the tables' rows
    uint32_t magic;               // unit -> table row: 0 (all channels), 1 (a row each), else floor(2^32 / units a row) + 1
    int g4;
  };

  // the rows' features of a unit on their way to LDS; the loads of the unit's weights come behind them
  // (What this wavefront read from there has arrived: with the wait the loads cannot overtake it.)
  static __device__ __forceinline__ void send_rows(const Ctx &c, int unit, uint32_t lds) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < PIECE / 1024; ++i) to_lds_16(c.row[i] + (int64_t)unit * SPAN * SZ, lds + i * 1024);
  }
  // TAIL: the unit may reach past K.  Activations from there are zero, the other loads are kept inside.
  template <bool TAIL> static __device__ __forceinline__ void load_weights(Unit &u, const Ctx &c, int unit) {
    const uint8_t *wu = c.w + (int64_t)unit * (BITS == 4 ? SPAN / 2 : SPAN) * c.N;
#pragma unroll
    for (int t = 0; t < KS; ++t) {
#pragma unroll
      for (int i = 0; i < C::ROWS; ++i) {
        const uint8_t *p;
        if (TAIL) {
          int64_t r = (int64_t)unit * (BITS == 4 ? SPAN / 2 : SPAN) + (BITS == 4 ? 16 : 32) * t + C::ROWS * c.g4 + i;
          r = r < c.R ? r : c.R - 1;
          p = c.w + r * c.N + c.col;
        } else {
          p = wu + (int64_t)((BITS == 4 ? 16 : 32) * t + i) * c.N + c.at_w;
        }
        if (CW == 4) {
          u.w[t][0][i] = reinterpret_cast<const U32u *>(p)->v;
        } else {
          const U64u v = *reinterpret_cast<const U64u *>(p);
#pragma unroll
          for (int d = 0; d < DW; ++d) u.w[t][d][i] = v.v[d];
        }
      }
    }
    const uint32_t row = c.magic < 2 ? c.magic * (uint32_t)unit : __umulhi((uint32_t)unit, c.magic);
    const char *zp = c.zero + (int64_t)row * c.N * ZB + c.at_z, *sp = c.scale + (int64_t)row * c.N * ZB + c.at_z;
    if (ZD == 2) {
      const U64u a = *reinterpret_cast<const U64u *>(zp), b = *reinterpret_cast<const U64u *>(sp);
#pragma unroll
      for (int d = 0; d < 2; ++d) { u.z[d] = a.v[d]; u.s[d] = b.v[d]; }
    } else {
#pragma unroll
      for (int d4 = 0; d4 < ZD / 4; ++d4) {
        const u32x4 a = load16(zp + 16 * d4), b = load16(sp + 16 * d4);
#pragma unroll
        for (int d = 0; d < 4; ++d) { u.z[4 * d4 + d] = a[d]; u.s[4 * d4 + d] = b[d]; }
      }
    }
  }
  template <bool TAIL> static __device__ __forceinline__ void load_rows(u32x4 (*x)[XW], const Ctx &c, int unit) {
    const char *xu = c.x + (int64_t)unit * SPAN * SZ;
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      const int64_t k = (int64_t)unit * SPAN + 32 * t + 8 * c.g4;
      if (!TAIL || k + 8 <= c.K) {
#pragma unroll
        for (int v = 0; v < XW; ++v) x[t][v] = load16(xu + 32 * t * SZ + 16 * v);
      } else {
#pragma unroll
        for (int v = 0; v < XW; ++v) {
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            uint32_t word = 0;
            if (SZ == 4) {
              if (k + 4 * v + d < c.K) word = ((const uint32_t *)xu)[32 * t + 4 * v + d];
            } else {
              const uint16_t *p = (const uint16_t *)xu + 32 * t;
              if (k + 2 * d < c.K) word = p[2 * d];
              if (k + 2 * d + 1 < c.K) word |= (uint32_t)p[2 * d + 1] << 16;
            }
            x[t][v][d] = word;
          }
        }
      }
    }
  }
  // A unit's features from LDS.  They have arrived: a load of the unit's weights, issued behind them, has (naming its
  // register makes the compiler wait for it, and loads return in order).
  static __device__ __forceinline__ void read_rows(u32x4 (*x)[XW], const Unit &u, const Ctx &c, const char *lds, int l16) {
    asm volatile("" : : "v"(u.w[KS - 1][DW - 1][C::ROWS - 1]) : "memory");
#pragma unroll
    for (int t = 0; t < KS; ++t)
#pragma unroll
      for (int v = 0; v < XW; ++v) {
        const int chunk = (4 * t + c.g4) * XW + v;
        x[t][v] = *reinterpret_cast<const u32x4 *>(lds + l16 * SPAN * SZ + (chunk ^ turn(l16)) * 16);
      }
  }

  // the lane's channels of a table row in fp32
  static __device__ __forceinline__ void table(const uint32_t *raw, float *v) {
#pragma unroll
    for (int q = 0; q < CW; ++q) {
      if (ZB == 4) {
        v[q] = __builtin_bit_cast(float, raw[q]);
      } else {
        const uint32_t h = (raw[q / 2] >> (16 * (q & 1))) & 0xFFFFu;
        v[q] = ZT == GPTQ_HIP_BF16 ? __builtin_bit_cast(float, h << 16)
                                   : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
      }
    }
  }

  static __device__ __forceinline__ void multiply(const Unit &u, u32x4 (*x)[XW], const Ctx &c, f32x4 out[CW]) {
    u32x4 a[KS][O::PARTS];
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    const u32x4 ones = {O::ONE, O::ONE, O::ONE, O::ONE};
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      if constexpr (XT == GPTQ_HIP_F32) parts3(x[t][0], x[t][XW - 1], a[t]);
      else a[t][0] = x[t][0];
#pragma unroll
      for (int p = 0; p < O::PARTS; ++p) {
        if (C::DEALT) a[t][p] = deal(a[t][p]);
        sum = O::mma(a[t][p], ones, sum);
      }
    }
    float z[CW], s[CW];
    table(u.z, z);
    table(u.s, s);
#pragma unroll
    for (int q = 0; q < CW; ++q) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        const u32x4 w = C::operand(u.w[t][q / 4], C::select(q & 3));
#pragma unroll
        for (int p = 0; p < O::PARTS; ++p) acc = O::mma(a[t][p], w, acc);
      }
      const float zq = -(z[q] + C::OFFSET), sq = s[q];
#pragma unroll
      for (int r = 0; r < 4; ++r) out[q][r] = fmaf(sq, fmaf(zq, sum[r], acc[r]), out[q][r]);
    }
  }
};

template <int XT, int BITS, int ZT, int KS, int CW, bool DMA>
__global__ __launch_bounds__(STRIP_WAVES * 64) void strip_kernel(ExpertArgs a) {
  using S = Strip<XT, BITS, ZT, KS, CW, DMA>;
  constexpr int ZB = S::ZB;
  // register sets and pieces of LDS that the units of a wavefront go round
  constexpr int D = KS == 1 ? 3 : 2;
  constexpr int ROWS_LDS = DMA ? STRIP_WAVES * D * S::PIECE : 0, RED_LDS = STRIP_WAVES / 2 * CW * 1024;
  typedef __attribute__((address_space(3))) char lds_char;
  __shared__ __attribute__((aligned(16))) char lds[ROWS_LDS > RED_LDS ? ROWS_LDS : RED_LDS];
  const int lane = threadIdx.x & 63, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t N = a.C, K = BITS == 4 ? 2 * a.R : a.R;
  const Item tile = find_item<0>(a.offsets, a.E, (int)a.P, 16, (uint32_t)((N + 16 * CW - 1) / (16 * CW)));
  if (tile.rows <= 0) return;
  // (the last strip ends where N does; what it shares with the one before it is computed twice, to the same bits)
  const int64_t n0 = (int64_t)tile.col * 16 * CW + 16 * CW <= N ? (int64_t)tile.col * 16 * CW : N - 16 * CW;
  const bool f32 = a.out_dtype == GPTQ_HIP_F32;
  if (tile.expert == a.E) {                            // rows of nowhere
    for (int i = threadIdx.x; i < tile.rows * 16 * CW; i += STRIP_WAVES * 64) {
      const int64_t n = n0 + i % (16 * CW);
      store_out<XT>(a.out, f32, (int64_t)(tile.row0 + i / (16 * CW)) * N + n, 0.f);
    }
    return;
  }
  typename S::Ctx c;
  c.K = K;
  c.R = a.R;
  c.N = N;
  const int64_t tables = a.group ? K / a.group : 1;
  const uint32_t per = a.group ? (uint32_t)(a.group / S::SPAN) : 0u;
  c.magic = per < 2 ? per : 0xFFFFFFFFu / per + 1u;    // (exact: a unit's number times `per` stays far below 2^32)
  c.g4 = lane >> 4;
  const int64_t col = n0 + CW * l16;
  c.w = a.packed + (int64_t)tile.expert * a.R * N;
  c.zero = (const char *)a.zero + (int64_t)tile.expert * tables * N * ZB;
  c.scale = (const char *)a.scale + (int64_t)tile.expert * tables * N * ZB;
  c.col = (uint32_t)col;
  c.at_w = (uint32_t)(S::C::ROWS * c.g4 * N + col);
  c.at_z = (uint32_t)(col * ZB);
  auto row_of = [&](int m) -> const char * {
    m = m < tile.rows ? m : tile.rows - 1;             // rows past the last repeat it and are not stored
    return (const char *)a.x + x_row_of(a.order, a.top_k, a.T, tile.row0 + m) * K * S::SZ;
  };
  const uint32_t piece0 = (uint32_t)(uintptr_t)(lds_char *)lds + wave * D * S::PIECE;
  if (DMA) {
#pragma unroll
    for (int i = 0; i < S::PIECE / 1024; ++i) {
      const int row = i * (64 / S::CPR) + lane / S::CPR;
      c.row[i] = row_of(row) + ((lane % S::CPR) ^ S::turn(row)) * 16;
    }
  }
  c.x = row_of(l16) + 8 * c.g4 * S::SZ;

  f32x4 out[CW];
#pragma unroll
  for (int q = 0; q < CW; ++q) out[q] = f32x4{0.f, 0.f, 0.f, 0.f};

  // units wave, wave + STRIP_WAVES, ...; the one that K ends in (no groups then) by itself
  const int whole = (int)(K / S::SPAN);
  const int mine = whole > wave ? (whole - wave + STRIP_WAVES - 1) / STRIP_WAVES : 0;
  if (mine > 0) {
    typename S::Unit ring[D];
    // (past the end: the last unit once more, not multiplied)
    auto load = [&](int d, int i) __attribute__((always_inline)) {
      const int unit = wave + STRIP_WAVES * (i < mine ? i : mine - 1);
      if constexpr (DMA) S::send_rows(c, unit, piece0 + d * S::PIECE);
      S::template load_weights<false>(ring[d], c, unit);
      if constexpr (!DMA) S::template load_rows<false>(ring[d].x, c, unit);
    };
#pragma unroll
    for (int d = 0; d + 1 < D; ++d) load(d, d);
    for (int i = 0; i < mine; i += D) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        load((d + D - 1) % D, i + d + D - 1);
        if (i + d < mine) {
          if constexpr (DMA) {
            u32x4 x[KS][S::XW];
            S::read_rows(x, ring[d], c, lds + (wave * D + d) * S::PIECE, l16);
            S::multiply(ring[d], x, c, out);
          } else {
            S::multiply(ring[d], ring[d].x, c, out);
          }
        }
      }
    }
    if (DMA) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // (the last loads reach LDS before it is used again)
  }
  if (K % S::SPAN && whole % STRIP_WAVES == wave) {
    typename S::Unit u;
    u32x4 x[KS][S::XW];
    S::template load_weights<true>(u, c, whole);
    S::template load_rows<true>(x, c, whole);
    S::multiply(u, x, c, out);
  }

  // the partial tiles: the upper half of the wavefronts hand theirs to the lower, whose sums are then added up
  f32x4 *red = reinterpret_cast<f32x4 *>(lds);
  __syncthreads();
  if (wave >= STRIP_WAVES / 2) {
#pragma unroll
    for (int q = 0; q < CW; ++q) red[((wave - STRIP_WAVES / 2) * CW + q) * 64 + lane] = out[q];
  }
  __syncthreads();
  if (wave < STRIP_WAVES / 2) {
#pragma unroll
    for (int q = 0; q < CW; ++q) red[(wave * CW + q) * 64 + lane] += out[q];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < CW * 64; i += STRIP_WAVES * 64) {
    const int l = i & 63, q = i >> 6;
    f32x4 v = red[i];
#pragma unroll
    for (int w = 1; w < STRIP_WAVES / 2; ++w) v += red[w * CW * 64 + i];
    const int64_t n = n0 + CW * (l & 15) + q;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = 4 * (l >> 4) + r;
      if (m < tile.rows) store_out<XT>(a.out, f32, (int64_t)(tile.row0 + m) * N + n, v[r]);
    }
  }
}

template <int XT, int CW, bool DMA>
static int strip_tables(hipStream_t s, const ExpertArgs &a, int ks) {
  const unsigned grid = item_grid(a.P, a.E, 16, ceil_div64(a.C, 16 * CW), STRIP_WAVES * 64);
  if (!grid) return GPTQ_HIP_EINVAL;
#define GPTQ_STRIP(B, S)                                                                                          \
  if (a.bits == B && ks == S) {                                                                                   \
    if (a.zs_dtype == GPTQ_HIP_F32)                                                                               \
      strip_kernel<XT, B, GPTQ_HIP_F32, S, CW, DMA><<<grid, STRIP_WAVES * 64, 0, s>>>(a);                        \
    else if (a.zs_dtype == GPTQ_HIP_F16)                                                                          \
      strip_kernel<XT, B, GPTQ_HIP_F16, S, CW, DMA><<<grid, STRIP_WAVES * 64, 0, s>>>(a);                        \
    else                                                                                                          \
      strip_kernel<XT, B, GPTQ_HIP_BF16, S, CW, DMA><<<grid, STRIP_WAVES * 64, 0, s>>>(a);                       \
  }
  GPTQ_STRIP(4, 2) GPTQ_STRIP(4, 1) GPTQ_STRIP(8, 2) GPTQ_STRIP(8, 1)
#undef GPTQ_STRIP
  GPTQ_CHECK_LAUNCH();
  return GPTQ_HIP_OK;
}

template <int XT> static int strip_launch(hipStream_t s, const ExpertArgs &a) {
  const int64_t K = a.bits == 4 ? 2 * a.R : a.R;
  // 64 features lie in one group, or 32; units of 128 keep one workgroup on a CU where two fit and are no faster
  const int ks = a.group % 64 == 0 ? 2 : 1;
  if ((uintptr_t)a.x % 16 || K * (XT == GPTQ_HIP_F32 ? 4 : 2) % 16) return strip_tables<XT, 8, false>(s, a, ks);
  // Strips of 64 channels: two neighbours share the lines of memory they begin and end in, on the same XCD; more
  // workgroups, less for each (8 experts 11008 x 4096, one token: 20 us, in strips of 128 channels 29; 64 experts
  // 2048 x 1424, 32 tokens of 2: 19 against 22).  Strips of 128 read the activations half as often, which decides where
  // they take one round of workgroups on the 256 CUs (11008 x 4096, 16 tokens of 2: 45 against 61 us).
  const double busy = a.E * (1.0 - exp(-(double)a.P / a.E)), strips = busy * ceil_div64(a.C, 128);
  const bool wide = strips > 128 && strips <= 256 && a.P < 8 * a.E;
  return wide ? strip_tables<XT, 8, true>(s, a, ks) : strip_tables<XT, 4, true>(s, a, ks);
}

}  // namespace xqmm
