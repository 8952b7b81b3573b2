// Rows of every expert times its packed matrix.
//
// E matrices W[e] [K, N], packed along K as for the single matrix (4 bits: byte [j, n] holds rows 2 j and 2 j + 1; 8
// bits: one row a byte), with zero / scale [E, N] or, for groups of g input features, [E, K / g, N]:
//   y[p, n]  = sum_k x[p, k] (c[k, n] - z[G(k), n]) s[G(k), n]      (transposed: x[p, n] summed over n)
// Row p belongs to the expert e with offsets[e] <= p < offsets[e + 1]; rows from offsets[E] on are zero.  The row of x
// is p itself or, with `order`, the token order[p] / top_k.
#include "expert_back.h"

namespace {

// the expert of row p (E: none), by bisection
__device__ __forceinline__ int expert_of(const int *__restrict__ offsets, int E, int64_t p) {
  int lo = 0, hi = E;                       // offsets[lo] <= p is kept
  if (p >= offsets[E]) return E;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= p) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int64_t x_row(const int *__restrict__ order, int top_k, int64_t T, int64_t p) {
  if (!order) return p;
  const int64_t t = order[p] / top_k;
  return t < 0 ? 0 : (t < T ? t : T - 1);
}

template <int BITS>
__device__ __forceinline__ float code_at(const uint8_t *__restrict__ w, int64_t C, int64_t k, int64_t n) {
  if (BITS == 8) return (float)w[k * C + n];
  const uint8_t b = w[(k >> 1) * C + n];
  return (float)((k & 1) ? b >> 4 : b & 15);
}

// One thread per output.  The shapes that no tiled kernel takes: groups that are no multiple of 32 features.
template <typename TX, typename TO, typename TZ, int BITS>
__global__ __launch_bounds__(256) void simple_fwd_kernel(ExpertArgs a) {
  const int64_t p = blockIdx.x;
  const int64_t n = (int64_t)blockIdx.y * 256 + threadIdx.x;
  if (n >= a.C) return;
  const int e = expert_of(a.offsets, a.E, p);
  TO *out = (TO *)a.out + p * a.C + n;
  if (e == a.E) {
    *out = from_f32<TO>(0.f);
    return;
  }
  const int64_t K = BITS == 4 ? 2 * a.R : a.R, g = a.group ? a.group : K, tables = a.group ? K / a.group : 1;
  const TX *x = (const TX *)a.x + x_row(a.order, a.top_k, a.T, p) * K;
  const uint8_t *w = a.packed + (int64_t)e * a.R * a.C;
  const TZ *zero = (const TZ *)a.zero + (int64_t)e * tables * a.C + n;
  const TZ *scale = (const TZ *)a.scale + (int64_t)e * tables * a.C + n;
  float total = 0.f;
  const int64_t run = a.group ? a.group : 128;       // a long sum is made of short ones
  for (int64_t k0 = 0; k0 < K; k0 += run) {
    const float z = to_f32(zero[k0 / g * a.C]);
    const int64_t k1 = k0 + run < K ? k0 + run : K;
    float sum = 0.f;
    for (int64_t k = k0; k < k1; ++k) sum = fmaf(to_f32(x[k]), code_at<BITS>(w, a.C, k, n) - z, sum);
    total = fmaf(sum, to_f32(scale[k0 / g * a.C]), total);
  }
  *out = from_f32<TO>(total);
}

// One wavefront per output column of the transposed product (a row of W).
template <typename TX, typename TO, typename TZ, int BITS>
__global__ __launch_bounds__(256) void simple_bwd_kernel(ExpertArgs a) {
  const int64_t p = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int64_t K = BITS == 4 ? 2 * a.R : a.R, k = (int64_t)blockIdx.y * 4 + (threadIdx.x >> 6);
  if (k >= K) return;
  const int e = expert_of(a.offsets, a.E, p);
  TO *out = (TO *)a.out + p * K + k;
  if (e == a.E) {
    if (lane == 0) *out = from_f32<TO>(0.f);
    return;
  }
  const int64_t g = a.group ? a.group : K, tables = a.group ? K / a.group : 1;
  const TX *x = (const TX *)a.x + x_row(a.order, a.top_k, a.T, p) * a.C;
  const uint8_t *w = a.packed + (int64_t)e * a.R * a.C;
  const TZ *zero = (const TZ *)a.zero + ((int64_t)e * tables + k / g) * a.C;
  const TZ *scale = (const TZ *)a.scale + ((int64_t)e * tables + k / g) * a.C;
  float sum = 0.f;
  for (int64_t n = lane; n < a.C; n += 64)
    sum = fmaf(to_f32(x[n]) * to_f32(scale[n]), code_at<BITS>(w, a.C, k, n) - to_f32(zero[n]), sum);
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) *out = from_f32<TO>(sum);
}

template <typename TX, typename TO, typename TZ, int BITS>
static int simple_launch(hipStream_t s, const ExpertArgs &a) {
  const int64_t K = BITS == 4 ? 2 * a.R : a.R;
  if (a.transpose)
    simple_bwd_kernel<TX, TO, TZ, BITS><<<dim3((unsigned)a.P, (unsigned)ceil_div64(K, 4)), 256, 0, s>>>(a);
  else
    simple_fwd_kernel<TX, TO, TZ, BITS><<<dim3((unsigned)a.P, (unsigned)ceil_div64(a.C, 256)), 256, 0, s>>>(a);
  GPTQ_CHECK_LAUNCH();
  return GPTQ_HIP_OK;
}
template <typename TX, typename TO>
static int simple_tables(hipStream_t s, const ExpertArgs &a) {
  if (a.zs_dtype == GPTQ_HIP_F32)
    return a.bits == 4 ? simple_launch<TX, TO, float, 4>(s, a) : simple_launch<TX, TO, float, 8>(s, a);
  if (a.zs_dtype == GPTQ_HIP_F16)
    return a.bits == 4 ? simple_launch<TX, TO, __half, 4>(s, a) : simple_launch<TX, TO, __half, 8>(s, a);
  return a.bits == 4 ? simple_launch<TX, TO, __hip_bfloat16, 4>(s, a)
                     : simple_launch<TX, TO, __hip_bfloat16, 8>(s, a);
}
static int simple_run(hipStream_t s, const ExpertArgs &a) {
  if (a.x_dtype == GPTQ_HIP_F32) return simple_tables<float, float>(s, a);
  if (a.x_dtype == GPTQ_HIP_F16)
    return a.out_dtype == GPTQ_HIP_F32 ? simple_tables<__half, float>(s, a) : simple_tables<__half, __half>(s, a);
  return a.out_dtype == GPTQ_HIP_F32 ? simple_tables<__hip_bfloat16, float>(s, a)
                                     : simple_tables<__hip_bfloat16, __hip_bfloat16>(s, a);
}

static bool float_type(int dt) { return dt == GPTQ_HIP_F32 || dt == GPTQ_HIP_F16 || dt == GPTQ_HIP_BF16; }

static int strip_run(hipStream_t s, const ExpertArgs &a) {
  if (a.x_dtype == GPTQ_HIP_F32) return expert_strip_f32(s, a);
  return a.x_dtype == GPTQ_HIP_F16 ? expert_strip_f16(s, a) : expert_strip_bf16(s, a);
}

static int tile_run(hipStream_t s, const ExpertArgs &a, int shape, void *ws) {
  if (a.x_dtype == GPTQ_HIP_F32) return expert_tile_f32(s, a, shape, ws);
  return a.x_dtype == GPTQ_HIP_F16 ? expert_tile_f16(s, a, shape, ws) : expert_tile_bf16(s, a, shape, ws);
}

static int back_run(hipStream_t s, const ExpertArgs &a, void *ws) {
  if (a.x_dtype == GPTQ_HIP_F32) return expert_back_f32(s, a, ws);
  return a.x_dtype == GPTQ_HIP_F16 ? expert_back_f16(s, a, ws) : expert_back_bf16(s, a, ws);
}

// Which kernel a product runs on.
struct Choice {
  enum Kind { SIMPLE, STRIP, TILE, BACK } kind;
  int shape;                // TILE_*
};
// By the rows of an expert, on average, and by whether tiles of 256 channels, one row of them per expert, fill the 256
// CUs (`wide`).  Each kernel costs nearly the same for 1 row as for all that its tile holds, so a taller tile pays once the
// rows fill half of it or so; where there are few columns of tiles, strips last longer, and two halves of K in a workgroup
// beat parts in two.  Measured, us a call (strip / 32 x 256 / 64 x 256 / 64 x 256 in halves of K):
//   8 experts 4096 x 11008 (wide):  8 rows each 40 61 76 86,  15: 47 61 77 -,  20: 70 62 76 -,  37: - 90 78 91,
//                                   80: - 127 129 138,  162: - 222 179 209
//   64 experts 2048 x 1424 (wide):  5 rows each 27 41 50 58,  15: 36 40 49 -,  31: - 54 52 62,  64: - 75 74 91
//   8 experts 11008 x 4096:  8 rows each 41 58 73 71,  15: 48 58 74 -,  25: 72 69 76 75,  37: - 93 79 111,  50: - 117 80 113,
//                            80: - 153 134 124,  125: - 179 194 167,  162: - 234 203 225
// fp32 rows are three operands, for which 64 rows are too many (strip / 32 x 256 / 64 x 256):
//   8 experts 4096 x 4096:  8 rows each 32 51 285,  20: 57 51 301,  40: 81 77 306,  162: - 187 387,  512: - 483 1012
static Choice choose(int64_t P, int E, int64_t C, int64_t group, int x_dtype, int transpose) {
  if ((group && group % 32) || C < 16) return {Choice::SIMPLE, 0};
  if (transpose) return {Choice::BACK, 0};
  const int64_t rows = P / E;
  const bool wide = (P < E ? P : E) * ceil_div64(C, 256) >= 256, fp32 = x_dtype == GPTQ_HIP_F32;
  if (C >= 128 && rows <= (wide || fp32 ? 15 : 24)) return {Choice::STRIP, 0};
  if (fp32 || rows <= (wide ? 31 : 24)) return {Choice::TILE, TILE_32x256};
  return {Choice::TILE, !wide && rows > 56 && rows <= 128 ? TILE_64x256_K2 : TILE_64x256};
}

// the sizes that the product takes
static bool sizes_fit(int64_t x_rows, int64_t rows, int64_t R, int64_t C, int bits, int64_t group, int E) {
  if ((bits != 4 && bits != 8) || E < 1 || E > 1024 || R < 1 || C < 1 || x_rows < 0 || rows < 0) return false;
  const int64_t lim = (int64_t)1 << 30;
  // (the plain kernels have one workgroup of 256 threads per row and four output columns in a grid dimension)
  if (rows >= (int64_t)1 << 24 || R > lim || C > (int64_t)1 << 20 || x_rows > lim) return false;
  const int64_t K = bits == 4 ? 2 * R : R;
  return K <= 262140 && group >= 0 && !(group && (K % group || (bits == 4 && group % 2)));
}

// GPTQ_HIP_OK, or why the product is refused
static int check_args(const ExpertArgs &a) {
  if (a.bits != 4 && a.bits != 8) return GPTQ_HIP_EINVAL;
  if (!float_type(a.x_dtype) || !float_type(a.out_dtype) || !float_type(a.zs_dtype)) return GPTQ_HIP_EDTYPE;
  if (a.out_dtype != a.x_dtype && a.out_dtype != GPTQ_HIP_F32) return GPTQ_HIP_EDTYPE;
  if (!sizes_fit(a.T, a.P, a.R, a.C, a.bits, a.group, a.E) || a.top_k < 1) return GPTQ_HIP_EINVAL;
  if (a.order ? a.P != a.T * a.top_k : a.P != a.T) return GPTQ_HIP_EINVAL;
  if (a.P == 0) return GPTQ_HIP_OK;
  if (!a.x || !a.offsets || !a.packed || !a.zero || !a.scale || !a.out) return GPTQ_HIP_EINVAL;
  return GPTQ_HIP_OK;
}

}  // namespace

extern "C" {

size_t gptq_hip_expert_qmatmul_workspace_bytes(int64_t x_rows, int64_t rows, int64_t R, int64_t C, int bits,
                                               int64_t group_size, int n_experts, int x_dtype, int zs_dtype,
                                               int transpose_b) {
  if (!sizes_fit(x_rows, rows, R, C, bits, group_size, n_experts) || rows == 0 || x_rows == 0) return 0;
  if (!float_type(x_dtype) || !float_type(zs_dtype)) return 0;
  const Choice c = choose(rows, n_experts, C, group_size, x_dtype, transpose_b);
  if (c.kind == Choice::TILE)
    return xqmm::staged_layout(x_rows, rows, bits == 4 ? 2 * R : R, C, group_size, n_experts, x_dtype, c.shape).bytes;
  if (c.kind == Choice::BACK)
    return xqmm::back_layout(x_rows, rows, R, C, bits, group_size, n_experts, x_dtype, zs_dtype).bytes;
  return 0;
}

int gptq_hip_expert_qmatmul(void *stream, const void *x, int x_dtype, int64_t x_rows, const int32_t *order, int top_k,
                            int64_t rows, const int32_t *offsets, int n_experts, const uint8_t *packed, int64_t R,
                            int64_t C, const void *zero, const void *scale, int zs_dtype, int64_t group_size, int bits,
                            int transpose_b, void *out, int out_dtype, void *ws, size_t ws_bytes) {
  const ExpertArgs a = {x, packed, zero, scale, out, order, offsets, x_rows, rows, R, C, group_size, top_k, n_experts,
                        bits, x_dtype, zs_dtype, out_dtype, transpose_b ? 1 : 0};
  if (int rc = check_args(a)) return rc;
  if (a.P == 0) return GPTQ_HIP_OK;
  hipStream_t s = as_stream(stream);
  const Choice c = choose(a.P, a.E, a.C, a.group, a.x_dtype, a.transpose);
  if (c.kind == Choice::STRIP) return strip_run(s, a);
  const size_t need = gptq_hip_expert_qmatmul_workspace_bytes(a.T, a.P, a.R, a.C, a.bits, a.group, a.E, a.x_dtype,
                                                              a.zs_dtype, a.transpose);
  if (need && (!ws || ws_bytes < need)) return GPTQ_HIP_EWORKSPACE;
  if (need && (uintptr_t)ws % 16) return GPTQ_HIP_EINVAL;
  if (c.kind == Choice::TILE) return tile_run(s, a, c.shape, ws);
  if (c.kind == Choice::BACK && (uintptr_t)a.x % 16 == 0) return back_run(s, a, ws);
  return simple_run(s, a);
}

}  // extern "C"
