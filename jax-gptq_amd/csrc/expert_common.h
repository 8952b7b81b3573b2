// Device parts the experts' product kernels share: operand types, codes as matrix-core operands, the tile of a workgroup.
#pragma once
#include "expert_qmm.h"
#include <type_traits>

namespace xqmm {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef __bf16 bfloat8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// loads of 4, 8, 16 bytes at any address that fits the element type
struct __attribute__((packed, aligned(1))) U32u { uint32_t v; };
struct __attribute__((packed, aligned(1))) U64u { uint32_t v[2]; };
struct __attribute__((packed, aligned(2))) U128u { uint32_t v[4]; };
__device__ __forceinline__ u32x4 load16(const void *p) {
  const U128u r = *reinterpret_cast<const U128u *>(p);
  return u32x4{r.v[0], r.v[1], r.v[2], r.v[3]};
}

__device__ __forceinline__ u32x4 load16u(const uint8_t *p) {
  struct __attribute__((packed, aligned(1))) U128b { uint32_t v[4]; };
  const U128b r = *reinterpret_cast<const U128b *>(p);
  return u32x4{r.v[0], r.v[1], r.v[2], r.v[3]};
}
// bytes n .. n + 15 of a row of N >= 16; past the row's end any bytes of it (its last 16, moved into place)
__device__ __forceinline__ u32x4 load_end16(const uint8_t *row, int64_t n, int64_t N) {
  if (n + 16 <= N) return load16u(row + n);
  const int64_t over = n - (N - 16);
  const u32x4 v = load16u(row + N - 16);
  uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
  const int sh = (int)(over < 16 ? over : 15) * 8;
  if (sh >= 64) {
    lo = hi >> (sh - 64);
    hi = 0;
  } else if (sh > 0) {
    lo = lo >> sh | hi << (64 - sh);
    hi >>= sh;
  }
  return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}
// one value of a scale or zero table
__device__ __forceinline__ float table_value(const char *p, int dtype, int64_t i) {
  if (dtype == GPTQ_HIP_F32) return ((const float *)p)[i];
  if (dtype == GPTQ_HIP_F16) return __half2float(((const __half *)p)[i]);
  return __bfloat162float(((const __hip_bfloat16 *)p)[i]);
}

// Operand types of the matrix cores for activations of type XT: fp16 as they are, bf16 as they are, fp32 as three
// bf16 parts (truncated: 3 x 8 bits are all 24, so the parts add up to the value exactly).
// Codes are exact in either: a 4-bit code sits in the mantissa under the exponent of 64 (fp16: 64 + c) or 128 (bf16:
// 128 + c), and the offset leaves with the zero point; 8-bit codes, and codes against fp32 parts, where the offset
// would cost bits of the sum, become c itself.  (The bits of a code are also the subnormal fp16 c 2^-24, one
// instruction less.  Single products of it are exact; sums of 32 to 512 with random rows come out up to 8e-6 of their
// size off, those with 16 c 2^-24 3e-7 to 9e-7, with c 2e-7 to 9e-7, with 64 + c, its 64 sum x taken off, 2e-6 to 1e-5.)
template <int XT> struct Op;
template <> struct Op<GPTQ_HIP_F16> {
  static constexpr int PARTS = 1;
  static constexpr uint32_t ONE = 0x3C003C00u;
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  }
};
template <> struct Op<GPTQ_HIP_BF16> {
  static constexpr int PARTS = 1;
  static constexpr uint32_t ONE = 0x3F803F80u;
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bfloat8, a), __builtin_bit_cast(bfloat8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bfloat8, a), __builtin_bit_cast(bfloat8, b), c, 0, 0, 0);
  }
};
template <> struct Op<GPTQ_HIP_F32> : Op<GPTQ_HIP_BF16> {
  static constexpr int PARTS = 3;
};

// A constant in a vector register, unknown to the compiler: "mask, then or" is one instruction then.  With both
// constants in sight it is two, since an instruction reads one scalar register at most.
__device__ __forceinline__ uint32_t opaque(uint32_t v) {
  asm("" : "+v"(v));
  return v;
}

// Packed rows that a lane holds for 8 input features, and how one byte of each becomes a B operand: 4 packed rows of
// 4-bit codes, 8 of 8-bit codes.
template <int XT, int BITS> struct Codes {
  static constexpr int ROWS = BITS == 4 ? 4 : 8;
  static constexpr bool CONVERT = XT == GPTQ_HIP_F32 || (XT == GPTQ_HIP_BF16 && BITS == 8);
  static constexpr float OFFSET = (CONVERT || BITS == 8) ? 0.f : (XT == GPTQ_HIP_BF16 ? 128.f : 64.f);
  // features in the order 0 2 1 3 4 6 5 7 (4-bit codes taken pairwise from two rows): the activations are dealt alike
  static constexpr bool DEALT = BITS == 4;

  static __device__ __forceinline__ uint32_t pair_f32(float a, float b) {      // {bf16(a), bf16(b)}, exact here
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
  }
  static __device__ __forceinline__ float byte_f32(uint32_t w, int q) { return (float)((w >> (8 * q)) & 255u); }

  // the byte permutation that takes byte q (0 .. 3) of two rows into the halves of a word
  static __device__ __forceinline__ uint32_t select(int q) { return 0x0C040C00u + 0x00010001u * (uint32_t)q; }
  // B operand of the selected byte of the dwords r[0 .. ROWS - 1]
  static __device__ __forceinline__ u32x4 operand(const uint32_t *r, uint32_t sel) {
    u32x4 b;
    if (BITS == 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t p = __builtin_amdgcn_perm(r[2 * i + 1], r[2 * i], sel);
        if (CONVERT) {
          b[i] = pair_f32(byte_f32(p, 0), byte_f32(p, 2));
        } else {
          const half2 v = __builtin_bit_cast(half2, p | 0x64006400u) - half2{(_Float16)1024.f, (_Float16)1024.f};
          b[i] = __builtin_bit_cast(uint32_t, v);
        }
      }
    } else {
      const uint32_t bias = opaque(XT == GPTQ_HIP_BF16 ? 0x43004300u : 0x54005400u);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t p = __builtin_amdgcn_perm(r[2 * i + 1], r[2 * i], sel);
        if (CONVERT) {
          const uint32_t lo = p & 0x000F000Fu, hi = (p >> 4) & 0x000F000Fu;
          b[2 * i] = pair_f32(byte_f32(lo, 0), byte_f32(lo, 2));
          b[2 * i + 1] = pair_f32(byte_f32(hi, 0), byte_f32(hi, 2));
        } else if (XT == GPTQ_HIP_BF16) {
          b[2 * i] = (p & 0x000F000Fu) | bias;
          b[2 * i + 1] = ((p >> 4) & 0x000F000Fu) | bias;
        } else {
          b[2 * i] = ((p << 4) & 0x00F000F0u) | bias;
          b[2 * i + 1] = (p & 0x00F000F0u) | bias;
        }
      }
    }
    return b;
  }
};

// 8 activations in natural order -> the order of Codes::DEALT
__device__ __forceinline__ u32x4 deal(u32x4 a) {
  return u32x4{__builtin_amdgcn_perm(a[1], a[0], 0x05040100u), __builtin_amdgcn_perm(a[1], a[0], 0x07060302u),
               __builtin_amdgcn_perm(a[3], a[2], 0x05040100u), __builtin_amdgcn_perm(a[3], a[2], 0x07060302u)};
}

// 8 fp32 values -> three operands of bf16 parts
__device__ __forceinline__ void parts3(const u32x4 &lo4, const u32x4 &hi4, u32x4 *out) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w[2] = {i < 2 ? lo4[2 * i] : hi4[2 * i - 4], i < 2 ? lo4[2 * i + 1] : hi4[2 * i - 3]};
    uint32_t part[3][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float v = __builtin_bit_cast(float, w[j]);
      part[0][j] = w[j];
      const float r1 = v - __builtin_bit_cast(float, w[j] & 0xFFFF0000u);
      part[1][j] = __builtin_bit_cast(uint32_t, r1);
      const float r2 = r1 - __builtin_bit_cast(float, part[1][j] & 0xFFFF0000u);
      part[2][j] = __builtin_bit_cast(uint32_t, r2);
    }
#pragma unroll
    for (int p = 0; p < 3; ++p) out[p][i] = __builtin_amdgcn_perm(part[p][1], part[p][0], 0x07060302u);
  }
}

// Which rows and columns a workgroup owns.  Tiles of H rows are counted expert by expert (the rows of nowhere as one
// more) and each comes with `cols` columns; PANEL columns at a time (0: all), all tiles of them, make the list of items.
// The counts come from a scan over the experts, 64 at a time; every wavefront does it for itself.
struct Item {
  int expert, row0, rows, col;        // rows == 0: nothing to do
};
struct Tiles {
  const int *__restrict__ offsets;
  int E, P, H, lo, hi, n, scan;
  uint32_t total;

  __device__ __forceinline__ int count(int e, int &l, int &h) const {
    l = h = 0;
    if (e <= E) {                       // (whatever the offsets say, no row outside 0 .. P - 1)
      l = min(max(offsets[e], 0), P);
      h = e < E ? min(max(offsets[e + 1], l), P) : P;
    }
    return (h - l + H - 1) / H;
  }
  __device__ __forceinline__ void load(int e0) {
    const int lane = threadIdx.x & 63;
    n = scan = count(e0 + lane, lo, hi);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(scan, d);
      if (lane >= d) scan += up;
    }
  }
  __device__ __forceinline__ Tiles(const int *offsets_, int E_, int P_, int H_)
      : offsets(offsets_), E(E_), P(P_), H(H_) {
    load(0);
    int all = __shfl(scan, 63);
    if (E >= 64) {
      int more = 0, l, h;
      for (int e = 64 + (threadIdx.x & 63); e <= E; e += 64) more += count(e, l, h);
#pragma unroll
      for (int d = 32; d; d >>= 1) more += __shfl_xor(more, d);
      all += more;
    }
    total = (uint32_t)__builtin_amdgcn_readfirstlane(all);
  }
  template <int PANEL> __device__ __forceinline__ Item at(uint32_t item, uint32_t cols) {
    const uint32_t panel = PANEL ? item / (total * PANEL) : 0u, rest = item - panel * total * PANEL;
    const uint32_t left = cols - PANEL * panel, width = PANEL && left > (uint32_t)PANEL ? (uint32_t)PANEL : left;
    const int tile = (int)(rest / width), col = (int)(PANEL * panel + rest % width);
    int before = 0;
    for (int e0 = 0;; e0 += 64) {
      if (e0 > 0) load(e0);
      const uint64_t past = __ballot(before + scan > tile);
      if (past) {
        const int who = __ffsll((unsigned long long)past) - 1;
        const int first = before + __shfl(scan - n, who);
        const int l = __shfl(lo, who), h = __shfl(hi, who), row0 = l + (tile - first) * H;
        const int rows = h - row0 < H ? h - row0 : H;
        return {__builtin_amdgcn_readfirstlane(e0 + who), __builtin_amdgcn_readfirstlane(row0),
                __builtin_amdgcn_readfirstlane(rows), col};
      }
      before += __shfl(scan, 63);
      if (e0 + 64 > E) return {0, 0, 0, 0};
    }
  }
};
// Workgroups go round the eight XCDs; each XCD takes a run of the list, so what runs on it at a time shares rows and
// weights (and lines that two neighbouring strips begin in) in its L2.
template <int PANEL>
__device__ __forceinline__ Item find_item(const int *__restrict__ offsets, int E, int P, int H, uint32_t cols) {
  Tiles tiles(offsets, E, P, H);
  const uint32_t items = tiles.total * cols, run = (items + 7) / 8;
  const uint32_t pos = blockIdx.x >> 3, item = (blockIdx.x & 7) * run + pos;
  if (pos >= run || item >= items) return {0, 0, 0, 0};
  return tiles.at<PANEL>(item, cols);
}
// The same where the items of the last, incomplete round are cut into parts: `slots` workgroups run at a time, so what
// is left over after whole rounds of them leaves the chip nearly idle, and as many parts of the contraction as fit fill
// it.  A second kernel adds the parts up, in order.
struct Split {
  uint32_t full, rem;                 // items in whole rounds, and after them
  int parts;                          // of each of those
};
__device__ __forceinline__ Split split_items(uint32_t items, uint32_t slots, int most) {
  Split s;
  s.full = items / slots * slots;
  s.rem = items - s.full;
  s.parts = s.rem ? (int)(slots / s.rem) : 1;
  if (s.parts > most) s.parts = most;
  return s;
}
struct Unit {
  Item item;
  int part, parts, slot;              // slot: of the part's sums
};
template <int PANEL>
__device__ __forceinline__ Unit find_unit(const int *__restrict__ offsets, int E, int P, int H, uint32_t cols,
                                          uint32_t slots, int most) {
  Tiles tiles(offsets, E, P, H);
  const uint32_t items = tiles.total * cols;
  const Split s = split_items(items, slots, most);
  const uint32_t whole = s.parts == 1 ? items : s.full;          // items that stay in one piece, a run for each XCD
  const uint32_t run = (whole + 7) / 8;
  if (blockIdx.x < 8 * run) {
    const uint32_t item = (blockIdx.x & 7) * run + (blockIdx.x >> 3);
    if (item >= whole) return {{0, 0, 0, 0}, 0, 1, 0};
    return {tiles.at<PANEL>(item, cols), 0, 1, 0};
  }
  if (s.parts == 1) return {{0, 0, 0, 0}, 0, 1, 0};
  const uint32_t u = blockIdx.x - s.full;
  if (u >= s.rem * (uint32_t)s.parts) return {{0, 0, 0, 0}, 0, 1, 0};
  return {tiles.at<PANEL>(s.full + u % s.rem, cols), (int)(u / s.rem), s.parts, (int)u};
}
// tiles there can be
static inline int64_t tile_bound(int64_t P, int E, int H) { return P / H + (P < E + 1 ? P : E + 1); }
// workgroups of `threads` for all items there can be, and `parts` more; 0: too many for a launch
static inline unsigned item_grid(int64_t P, int E, int H, int64_t cols, int threads, int64_t parts = 0) {
  const int64_t blocks = round_up64(tile_bound(P, E, H) * cols, 8) + parts;
  return blocks * threads >= (int64_t)1 << 32 ? 0u : (unsigned)blocks;
}
// parts of items there can be, of which each keeps its sums (in at most `slots` places)
static inline int64_t unit_bound(int64_t P, int E, int H, int64_t cols, int64_t slots, int most) {
  const int64_t items = tile_bound(P, E, H) * cols;
  return most < 2 ? 0 : (items * most < slots ? items * most : slots);
}

// the row of x that row p reads
__device__ __forceinline__ int64_t x_row_of(const int *__restrict__ order, int top_k, int64_t T, int64_t p) {
  if (!order) return p;
  const uint32_t t = (uint32_t)order[p] / (uint32_t)top_k;
  return (int64_t)t < T ? t : T - 1;
}

template <int XT> struct Elem { typedef __half type; };
template <> struct Elem<GPTQ_HIP_BF16> { typedef __hip_bfloat16 type; };
template <> struct Elem<GPTQ_HIP_F32> { typedef float type; };

template <int XT>
__device__ __forceinline__ void store_out(void *out, bool f32, int64_t i, float v) {
  if (f32) ((float *)out)[i] = v;
  else ((typename Elem<XT>::type *)out)[i] = from_f32<typename Elem<XT>::type>(v);
}

// two neighbours of a row
template <int XT> __device__ __forceinline__ void store2(void *out, bool f32, int64_t i, float a, float b) {
  typedef typename Elem<XT>::type E;
  if (f32) {
    struct __attribute__((packed, aligned(4))) F2 { float v[2]; };
    *reinterpret_cast<F2 *>((float *)out + i) = F2{{a, b}};
  } else {
    struct __attribute__((packed, aligned(sizeof(E)))) E2 { E v[2]; };
    *reinterpret_cast<E2 *>((E *)out + i) = E2{{from_f32<E>(a), from_f32<E>(b)}};
  }
}

}  // namespace xqmm
