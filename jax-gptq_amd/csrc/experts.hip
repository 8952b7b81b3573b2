// Tokens sorted by expert and back: the order of the (token, choice) pairs, copies of the tokens' rows in that order,
// the weighted sum of the experts' rows at their tokens, and the gradients of both.
//
// T tokens with k choices each make P = T k pairs, pair i = t k + j.  `order` lists the pairs by expert, ties in
// order of the pair; `position` is its inverse; `offsets[e]` is where expert e's rows begin, offsets[E] where the
// rows of pairs that go nowhere (an id outside 0 .. E - 1) begin.  All sums run in a fixed order, so equal calls give
// equal bits.
#include "common.h"

namespace {

constexpr int MAX_EXPERTS = 1024;
constexpr int SORT_CHUNK = 4096;       // pairs of one workgroup where there are several
constexpr int SORT_MAX_GROUPS = 256;   // each of them reads the counts of all
constexpr int SORT_LDS_WORDS = 11264;  // counters of a workgroup: one per wavefront and bucket

// bucket of a pair: its expert, or E for an id that names none (compared in 64 bits: 2^32 is not expert 0)
template <typename ID>
__device__ __forceinline__ int bucket_of(ID id, int E) {
  return (id >= 0 && (int64_t)id < (int64_t)E) ? (int)id : E;
}

static inline int sort_waves(int64_t pairs, int E) {
  int64_t w = ceil_div64(pairs, 64);
  w = w < 1 ? 1 : (w > 16 ? 16 : w);
  const int fit = SORT_LDS_WORDS / (E + 1);
  return (int)(w < fit ? w : fit);
}
static inline int64_t sort_chunk(int64_t P) {
  const int64_t c = round_up64(ceil_div64(P, SORT_MAX_GROUPS), 1024);
  return c > SORT_CHUNK ? c : SORT_CHUNK;
}

// Pairs of every bucket in each chunk.
template <typename ID>
__global__ __launch_bounds__(1024) void sort_count_kernel(const ID *__restrict__ ids, int64_t P, int64_t chunk, int E,
                                                          int *__restrict__ counts) {
  extern __shared__ int hist[];
  for (int b = threadIdx.x; b <= E; b += blockDim.x) hist[b] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * chunk;
  const int64_t hi = lo + chunk < P ? lo + chunk : P;
  for (int64_t i = lo + threadIdx.x; i < hi; i += blockDim.x) atomicAdd(&hist[bucket_of(ids[i], E)], 1);
  __syncthreads();
  for (int b = threadIdx.x; b <= E; b += blockDim.x) counts[(int64_t)blockIdx.x * (E + 1) + b] = hist[b];
}

// A stable counting sort.  Each wavefront owns a run of its workgroup's chunk and counts it; the counters, read bucket
// by bucket and wavefront by wavefront, then hold where each wavefront's first pair of each bucket goes.  The second
// walk takes 64 pairs at a time: the lanes that share a bucket are found with one ballot per bit of the bucket number,
// a lane's rank is the number of such lanes before it, and the first of them moves the counter on.
// `counts` (several chunks): the pairs of every bucket in every chunk, from sort_count_kernel.
// Bound by latency: ids come in, two passes over LDS counters, scattered stores of 4 bytes.  48 pairs: 3.0 us; 262144 pairs
// of 128 experts: 2.4 us for the counts and 11.6 us for this kernel, whose 64 workgroups each add up all chunks' counts.
template <typename ID>
__global__ __launch_bounds__(1024) void sort_kernel(const ID *__restrict__ ids, int64_t P, int64_t chunk, int E,
                                                    const int *__restrict__ counts, int n_chunks,
                                                    int *__restrict__ order, int *__restrict__ position,
                                                    int *__restrict__ offsets) {
  extern __shared__ int hist[];          // [wavefronts][E + 1], then two more rows where there are several chunks
  __shared__ int wave_sum[16];
  const int waves = blockDim.x >> 6, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int nb = E + 1;
  int *all = hist + waves * nb, *before = all + nb;      // pairs of every bucket in all chunks and in those before
  for (int i = threadIdx.x; i < (counts ? waves + 2 : waves) * nb; i += blockDim.x) hist[i] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * chunk;
  const int64_t hi = lo + chunk < P ? lo + chunk : P;
  const int64_t per = ((hi - lo + waves - 1) / waves + 63) / 64 * 64;
  const int64_t wlo = lo + w * per < hi ? lo + w * per : hi;
  const int64_t whi = wlo + per < hi ? wlo + per : hi;
  int *mine = hist + w * nb;
  for (int64_t i = wlo + lane; i < whi; i += 64) atomicAdd(&mine[bucket_of(ids[i], E)], 1);
  if (counts) {
    for (int i = threadIdx.x; i < n_chunks * nb; i += blockDim.x) {
      const int v = counts[i], b = i % nb;
      if (v) {
        atomicAdd(&all[b], v);
        if (i / nb < (int)blockIdx.x) atomicAdd(&before[b], v);
      }
    }
  }
  __syncthreads();

  // thread t: `each` consecutive buckets, their totals summed, scanned over the workgroup
  const int each = (nb + (int)blockDim.x - 1) / (int)blockDim.x;
  const int b0 = threadIdx.x * each < nb ? threadIdx.x * each : nb;
  const int b1 = b0 + each < nb ? b0 + each : nb;
  int total = 0;
  for (int b = b0; b < b1; ++b) {
    if (counts) total += all[b];
    else for (int v = 0; v < waves; ++v) total += hist[v * nb + b];
  }
  int scan = total;
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(scan, d);
    if (lane >= d) scan += up;
  }
  if (lane == 63) wave_sum[w] = scan;
  __syncthreads();
  int base = scan - total;
  for (int v = 0; v < w; ++v) base += wave_sum[v];
  for (int b = b0; b < b1; ++b) {
    if (blockIdx.x == 0) offsets[b] = base;      // bucket E: where the rows of nowhere begin
    int at = counts ? base + before[b] : base;
    for (int v = 0; v < waves; ++v) {
      const int n = hist[v * nb + b];
      hist[v * nb + b] = at;
      at += n;
    }
    base = counts ? base + all[b] : at;
  }
  __syncthreads();

  int bits = 0;
  while ((1 << bits) < nb) ++bits;
  for (int64_t i0 = wlo; i0 < whi; i0 += 64) {
    const int64_t i = i0 + lane;
    const bool have = i < whi;
    const int b = have ? bucket_of(ids[i], E) : -1;
    uint64_t same = __ballot(have);
    for (int t = 0; t < bits; ++t) {
      const uint64_t set = __ballot((b >> t) & 1);
      same &= ((b >> t) & 1) ? set : ~set;
    }
    if (have) {                                  // (lanes without a pair took part in the ballots only)
      const int rank = __popcll(same & ((1ull << lane) - 1));
      const int first = __ffsll((unsigned long long)same) - 1;
      int at = 0;
      if (lane == first) at = atomicAdd(&mine[b], __popcll(same));
      at = __shfl(at, first) + rank;
      order[at] = (int)i;
      position[i] = at;
    }
  }
}

// ------------------------------------------------------------------------------------- rows
// 16 bytes at any address that fits the element type (rows of odd lengths begin anywhere)
template <typename T> struct Vec {
  static constexpr int N = 16 / sizeof(T);
  struct __attribute__((packed, aligned(sizeof(T)))) Raw { T v[N]; };
  static __device__ __forceinline__ Raw load(const T *p) { return *reinterpret_cast<const Raw *>(p); }
  static __device__ __forceinline__ void store(T *p, const Raw &r) { *reinterpret_cast<Raw *>(p) = r; }
};

// copies of the tokens' rows: each row is read once and written to its k places.  Bound by the stores: 8192 rows of 4096
// bf16 to two places each, 201 MB in 63 us (3.2 TB/s; stores alone run at 2.3 to 2.6 TB/s here).
template <typename T>
__global__ __launch_bounds__(256) void gather_kernel(const T *__restrict__ x, int top_k, int64_t K,
                                                     const int *__restrict__ position,
                                                     const int *__restrict__ offsets, int E, int64_t P,
                                                     T *__restrict__ out) {
  using V = Vec<T>;
  constexpr int EACH = 2;                          // pieces of a thread: both are loaded before either is stored
  const int64_t t = blockIdx.x;
  const int live = offsets[E];
  int64_t c[EACH];
  typename V::Raw r[EACH], zero;
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
    c[u] = (((int64_t)blockIdx.y * EACH + u) * 256 + threadIdx.x) * V::N;
    if (c[u] + V::N <= K) {
      r[u] = V::load(x + t * K + c[u]);
    } else {
      for (int i = 0; i < V::N; ++i) r[u].v[i] = c[u] + i < K ? x[t * K + c[u] + i] : from_f32<T>(0.f);
    }
  }
  for (int i = 0; i < V::N; ++i) zero.v[i] = from_f32<T>(0.f);
  for (int j = 0; j < top_k; ++j) {
    const int64_t p = position[t * top_k + j];
    if (p < 0 || p >= P) continue;
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      const typename V::Raw &s = p < live ? r[u] : zero;
      if (c[u] + V::N <= K) {
        V::store(out + p * K + c[u], s);
      } else {
        for (int i = 0; c[u] + i < K; ++i) out[p * K + c[u] + i] = s.v[i];
      }
    }
  }
}

template <typename TW>
__device__ __forceinline__ float weight_at(const TW *w, int64_t i) { return w ? to_f32(w[i]) : 1.f; }

// out[t] = sum_j w[t, j] y[position[t, j]], fp32 in order of j, rounded once; pairs that go nowhere are not read.  Bound by
// the loads: 4096 tokens of 4 rows of 4096 bf16, 168 MB in 38 us (4.4 TB/s).
template <typename T, typename TO, typename TW>
__global__ __launch_bounds__(256) void combine_kernel(const T *__restrict__ y, int top_k, int64_t N,
                                                      const int *__restrict__ position,
                                                      const int *__restrict__ offsets, int E, int64_t P,
                                                      const TW *__restrict__ weights, TO *__restrict__ out) {
  using V = Vec<T>;
  const int64_t t = blockIdx.x;
  const int64_t c = ((int64_t)blockIdx.y * 256 + threadIdx.x) * V::N;
  if (c >= N) return;
  const int64_t live = offsets[E] < P ? offsets[E] : P;
  const bool whole = c + V::N <= N;
  float acc[V::N];
  for (int i = 0; i < V::N; ++i) acc[i] = 0.f;
  if (whole) {
    // four rows' loads in flight; a pair that goes nowhere reads row 0 in its place, which is left out of the sum
    for (int j0 = 0; j0 < top_k; j0 += 4) {
      typename V::Raw r[4];
      bool in[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t p = j0 + j < top_k ? position[t * top_k + j0 + j] : -1;
        in[j] = p >= 0 && p < live;
        r[j] = V::load(y + (in[j] ? p : 0) * N + c);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!in[j]) continue;
        const float w = weight_at(weights, t * top_k + j0 + j);
        for (int i = 0; i < V::N; ++i) acc[i] = fmaf(w, to_f32(r[j].v[i]), acc[i]);
      }
    }
  } else {
    for (int j = 0; j < top_k; ++j) {
      const int64_t p = position[t * top_k + j];
      if (p < 0 || p >= live) continue;
      const float w = weight_at(weights, t * top_k + j);
      for (int i = 0; c + i < N; ++i) acc[i] = fmaf(w, to_f32(y[p * N + c + i]), acc[i]);
    }
  }
  if (whole) {
    struct __attribute__((packed, aligned(sizeof(TO)))) Raw { TO v[V::N]; } r;
    for (int i = 0; i < V::N; ++i) r.v[i] = from_f32<TO>(acc[i]);
    *reinterpret_cast<Raw *>(out + t * N + c) = r;
  } else {
    for (int i = 0; i < V::N && c + i < N; ++i) out[t * N + c + i] = from_f32<TO>(acc[i]);
  }
}

// dy[p] = w[t, j] g[t] and dw[t, j] = <g[t], y[p]>, one workgroup per token; zero for pairs that go nowhere.  y and dy pass
// once, g stays in L2: 4096 tokens of 4 rows of 4096 bf16, 302 MB in 60 us (5.0 TB/s, what a copy reaches).
template <typename T, typename TW>
__global__ __launch_bounds__(256) void combine_grad_kernel(const T *__restrict__ y, const T *__restrict__ g, int top_k,
                                                           int64_t N, const int *__restrict__ position,
                                                           const int *__restrict__ offsets, int E, int64_t P,
                                                           const TW *__restrict__ weights, T *__restrict__ dy,
                                                           TW *__restrict__ dw) {
  using V = Vec<T>;
  __shared__ float part[4];
  const int64_t t = blockIdx.x;
  const int64_t live = offsets[E] < P ? offsets[E] : P;
  for (int j = 0; j < top_k; ++j) {
    const int64_t p = position[t * top_k + j];
    const bool in = p >= 0 && p < P, alive = in && p < live;
    const float w = alive ? weight_at(weights, t * top_k + j) : 0.f;
    float dot = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V::N; c < N && in; c += 256 * V::N) {
      if (c + V::N <= N) {
        typename V::Raw d;
        for (int i = 0; i < V::N; ++i) d.v[i] = from_f32<T>(0.f);
        if (alive) {
          const typename V::Raw a = V::load(g + t * N + c);
          if (dw) {
            const typename V::Raw b = V::load(y + p * N + c);
            for (int i = 0; i < V::N; ++i) dot = fmaf(to_f32(a.v[i]), to_f32(b.v[i]), dot);
          }
          for (int i = 0; i < V::N; ++i) d.v[i] = from_f32<T>(w * to_f32(a.v[i]));
        }
        if (dy) V::store(dy + p * N + c, d);
      } else {
        for (int64_t i = c; i < N; ++i) {
          const float a = alive ? to_f32(g[t * N + i]) : 0.f;
          if (dw && alive) dot = fmaf(a, to_f32(y[p * N + i]), dot);
          if (dy) dy[p * N + i] = from_f32<T>(alive ? w * a : 0.f);
        }
      }
    }
    if (dw) {
      for (int d = 32; d; d >>= 1) dot += __shfl_xor(dot, d);
      if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = dot;
      __syncthreads();
      if (threadIdx.x == 0) dw[t * top_k + j] = from_f32<TW>((part[0] + part[1]) + (part[2] + part[3]));
      __syncthreads();
    }
  }
}

// ------------------------------------------------------------------------------------- dispatch
static bool float_type(int dt) { return dt == GPTQ_HIP_F32 || dt == GPTQ_HIP_F16 || dt == GPTQ_HIP_BF16; }

// shapes every row operator takes; `width` elements a row
static int check_rows(int64_t T, int top_k, int64_t width, int E) {
  if (T < 0 || top_k < 1 || width < 0 || E < 1 || E > MAX_EXPERTS) return GPTQ_HIP_EINVAL;
  // (a launch has one workgroup of 256 threads per token, and fewer than 2^32 threads)
  if (T >= (int64_t)1 << 24 || T * top_k > (int64_t)1 << 30 || width > (int64_t)1 << 25) return GPTQ_HIP_EINVAL;
  return GPTQ_HIP_OK;
}
template <typename T> static dim3 row_grid(int64_t rows, int64_t width, int each) {
  return dim3((unsigned)rows, (unsigned)ceil_div64(width, each * 256 * (16 / (int64_t)sizeof(T))));
}

template <typename T, typename TO, typename TW>
static int combine_launch(hipStream_t s, const void *y, int64_t T_, int top_k, int64_t N, const int *position,
                          const int *offsets, int E, const void *weights, void *out) {
  const dim3 grid = row_grid<T>(T_, N, 1);
  combine_kernel<T, TO, TW><<<grid, 256, 0, s>>>((const T *)y, top_k, N, position, offsets, E, T_ * top_k,
                                                 (const TW *)weights, (TO *)out);
  GPTQ_CHECK_LAUNCH();
  return GPTQ_HIP_OK;
}
template <typename T, typename TO>
static int combine_weights(hipStream_t s, const void *y, int64_t T_, int top_k, int64_t N, const int *position,
                           const int *offsets, int E, const void *weights, int w_dtype, void *out) {
  if (!weights || w_dtype == GPTQ_HIP_F32)
    return combine_launch<T, TO, float>(s, y, T_, top_k, N, position, offsets, E, weights, out);
  if (w_dtype == GPTQ_HIP_F16)
    return combine_launch<T, TO, __half>(s, y, T_, top_k, N, position, offsets, E, weights, out);
  return combine_launch<T, TO, __hip_bfloat16>(s, y, T_, top_k, N, position, offsets, E, weights, out);
}
template <typename T, typename TW>
static int grad_launch(hipStream_t s, const void *y, const void *g, int64_t T_, int top_k, int64_t N,
                       const int *position, const int *offsets, int E, const void *weights, void *dy, void *dw) {
  combine_grad_kernel<T, TW><<<dim3((unsigned)T_), 256, 0, s>>>((const T *)y, (const T *)g, top_k, N, position,
                                                                offsets, E, T_ * top_k, (const TW *)weights, (T *)dy,
                                                                (TW *)dw);
  GPTQ_CHECK_LAUNCH();
  return GPTQ_HIP_OK;
}
template <typename T>
static int grad_weights(hipStream_t s, const void *y, const void *g, int64_t T_, int top_k, int64_t N,
                        const int *position, const int *offsets, int E, const void *weights, int w_dtype, void *dy,
                        void *dw) {
  if (w_dtype == GPTQ_HIP_F32)
    return grad_launch<T, float>(s, y, g, T_, top_k, N, position, offsets, E, weights, dy, dw);
  if (w_dtype == GPTQ_HIP_F16)
    return grad_launch<T, __half>(s, y, g, T_, top_k, N, position, offsets, E, weights, dy, dw);
  return grad_launch<T, __hip_bfloat16>(s, y, g, T_, top_k, N, position, offsets, E, weights, dy, dw);
}

template <typename ID>
static int sort_launch(hipStream_t s, const void *ids, int64_t P, int E, int *order, int *position, int *offsets,
                       int *counts) {
  const ID *p = (const ID *)ids;
  const int64_t chunk = sort_chunk(P);
  if (P <= chunk) {
    const int waves = sort_waves(P, E);
    sort_kernel<ID><<<1, waves * 64, (size_t)waves * (E + 1) * 4, s>>>(p, P, chunk, E, nullptr, 1, order, position,
                                                                       offsets);
    GPTQ_CHECK_LAUNCH();
    return GPTQ_HIP_OK;
  }
  const int n = (int)ceil_div64(P, chunk), waves = sort_waves(chunk, E);
  sort_count_kernel<ID><<<n, 1024, (size_t)(E + 1) * 4, s>>>(p, P, chunk, E, counts);
  GPTQ_CHECK_LAUNCH();
  sort_kernel<ID><<<n, waves * 64, (size_t)(waves + 2) * (E + 1) * 4, s>>>(p, P, chunk, E, counts, n, order, position,
                                                                     offsets);
  GPTQ_CHECK_LAUNCH();
  return GPTQ_HIP_OK;
}

}  // namespace

extern "C" {

size_t gptq_hip_expert_sort_workspace_bytes(int64_t pairs, int n_experts) {
  if (pairs <= 0 || pairs > (int64_t)1 << 30 || n_experts < 1 || n_experts > MAX_EXPERTS) return 0;
  const int64_t chunk = sort_chunk(pairs);
  return pairs <= chunk ? 0 : (size_t)ceil_div64(pairs, chunk) * (n_experts + 1) * 4;
}

int gptq_hip_expert_sort(void *stream, const void *ids, int id_bytes, int64_t pairs, int n_experts, int32_t *order,
                         int32_t *position, int32_t *offsets, void *ws, size_t ws_bytes) {
  if (pairs < 0 || pairs > (int64_t)1 << 30 || n_experts < 1 || n_experts > MAX_EXPERTS || !offsets)
    return GPTQ_HIP_EINVAL;
  if (id_bytes != 4 && id_bytes != 8) return GPTQ_HIP_EDTYPE;
  if (pairs > 0 && (!ids || !order || !position)) return GPTQ_HIP_EINVAL;
  if (ws_bytes < gptq_hip_expert_sort_workspace_bytes(pairs, n_experts)) return GPTQ_HIP_EWORKSPACE;
  if (gptq_hip_expert_sort_workspace_bytes(pairs, n_experts) > 0 && !ws) return GPTQ_HIP_EWORKSPACE;
  hipStream_t s = as_stream(stream);
  return id_bytes == 4 ? sort_launch<int32_t>(s, ids, pairs, n_experts, order, position, offsets, (int *)ws)
                       : sort_launch<int64_t>(s, ids, pairs, n_experts, order, position, offsets, (int *)ws);
}

int gptq_hip_expert_gather(void *stream, const void *x, int dtype, int64_t tokens, int top_k, int64_t K,
                           const int32_t *position, const int32_t *offsets, int n_experts, void *out) {
  if (int rc = check_rows(tokens, top_k, K, n_experts)) return rc;
  if (!float_type(dtype)) return GPTQ_HIP_EDTYPE;
  if (tokens == 0 || K == 0) return GPTQ_HIP_OK;
  if (!x || !position || !offsets || !out) return GPTQ_HIP_EINVAL;
  hipStream_t s = as_stream(stream);
  const int64_t P = tokens * top_k;
  if (dtype == GPTQ_HIP_F32) {
    const dim3 grid = row_grid<float>(tokens, K, 2);
    gather_kernel<float><<<grid, 256, 0, s>>>((const float *)x, top_k, K, position, offsets, n_experts, P,
                                              (float *)out);
  } else {                                        // 16-bit rows are copied as they are
    const dim3 grid = row_grid<__half>(tokens, K, 2);
    gather_kernel<__half><<<grid, 256, 0, s>>>((const __half *)x, top_k, K, position, offsets, n_experts, P,
                                               (__half *)out);
  }
  GPTQ_CHECK_LAUNCH();
  return GPTQ_HIP_OK;
}

int gptq_hip_expert_combine(void *stream, const void *y, int y_dtype, int64_t tokens, int top_k, int64_t N,
                            const int32_t *position, const int32_t *offsets, int n_experts, const void *weights,
                            int w_dtype, void *out, int out_dtype) {
  if (int rc = check_rows(tokens, top_k, N, n_experts)) return rc;
  if (!float_type(y_dtype) || !float_type(out_dtype) || (weights && !float_type(w_dtype))) return GPTQ_HIP_EDTYPE;
  if (out_dtype != y_dtype && y_dtype != GPTQ_HIP_F32) return GPTQ_HIP_EDTYPE;
  if (tokens == 0 || N == 0) return GPTQ_HIP_OK;
  if (!y || !position || !offsets || !out) return GPTQ_HIP_EINVAL;
  hipStream_t s = as_stream(stream);
#define GPTQ_COMBINE(T, TO) \
  return combine_weights<T, TO>(s, y, tokens, top_k, N, position, offsets, n_experts, weights, w_dtype, out)
  if (y_dtype == GPTQ_HIP_F16) GPTQ_COMBINE(__half, __half);
  if (y_dtype == GPTQ_HIP_BF16) GPTQ_COMBINE(__hip_bfloat16, __hip_bfloat16);
  if (out_dtype == GPTQ_HIP_F32) GPTQ_COMBINE(float, float);
  if (out_dtype == GPTQ_HIP_F16) GPTQ_COMBINE(float, __half);
  GPTQ_COMBINE(float, __hip_bfloat16);
#undef GPTQ_COMBINE
}

int gptq_hip_expert_combine_grad(void *stream, const void *y, const void *g, int dtype, int64_t tokens, int top_k,
                                 int64_t N, const int32_t *position, const int32_t *offsets, int n_experts,
                                 const void *weights, int w_dtype, void *dy, void *dw) {
  if (int rc = check_rows(tokens, top_k, N, n_experts)) return rc;
  if (!float_type(dtype) || !float_type(w_dtype)) return GPTQ_HIP_EDTYPE;
  if (tokens == 0 || (!dy && !dw)) return GPTQ_HIP_OK;
  if (!position || !offsets || (N > 0 && (!g || (dw && !y)))) return GPTQ_HIP_EINVAL;
  hipStream_t s = as_stream(stream);
#define GPTQ_GRAD(T) \
  return grad_weights<T>(s, y, g, tokens, top_k, N, position, offsets, n_experts, weights, w_dtype, dy, dw)
  if (dtype == GPTQ_HIP_F16) GPTQ_GRAD(__half);
  if (dtype == GPTQ_HIP_BF16) GPTQ_GRAD(__hip_bfloat16);
  GPTQ_GRAD(float);
#undef GPTQ_GRAD
}

}  // extern "C"
