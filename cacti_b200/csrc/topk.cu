// The largest K logits of each row, sorted, and the row's log of the sum of its exponentials: what a teacher's forward pass
// hands to the distillation loss instead of its whole logits tensor.
//
// No counterpart in the reference (its arg-max, src/librarium/llama.rs:546, is the case K = 1).  Order: larger values first,
// equal values (+0 equals -0) by ascending index, NaN above +inf.  Floats are compared through an order-preserving map
// to unsigned keys.
#include "common.cuh"

namespace cb {

constexpr int kTopkMaxK = 256;
constexpr int64_t kTopkMaxVocab = 1 << 18;
constexpr int kTopkThreads = 256;

__device__ __forceinline__ unsigned order_key(float v) {
  if (v != v) return 0xffffffffu;
  const unsigned b = __float_as_uint(v == 0.f ? 0.f : v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One CTA a row: the K-th largest key by bisection on counts, then the entries above it (at most K - 1, ranked by
// counting) and the first entries equal to it in index order.
template <typename T>
__global__ void __launch_bounds__(kTopkThreads)
logits_topk_kernel(T* __restrict__ values, int* __restrict__ indices, float* __restrict__ lse, const T* __restrict__ L,
                   int64_t rows, int V, int K, double inv_temp) {
  __shared__ float s_red[33];
  __shared__ unsigned s_key[kTopkMaxK];
  __shared__ int s_pos[kTopkMaxK];
  __shared__ int s_n, s_ties, s_warp[kTopkThreads / 32];
  const int t = threadIdx.x;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* x = L + row * V;
    unsigned lo = 0u, hi = 0xffffffffu;                         // the largest key with at least K entries at or above it
    while (lo < hi) {
      const unsigned mid = lo + (hi - lo) / 2 + 1;
      float n = 0.f;                                            // counts below 2^24 are exact in f32
      for (int j = t; j < V; j += blockDim.x) n += order_key(Elem<T>::to_f32(x[j])) >= mid ? 1.f : 0.f;
      if (block_reduce<SumOp>(n, s_red) >= (float)K) lo = mid;
      else hi = mid - 1;
    }
    if (t == 0) { s_n = 0; s_ties = 0; }
    __syncthreads();
    for (int j = t; j < V; j += blockDim.x) {
      const unsigned key = order_key(Elem<T>::to_f32(x[j]));
      if (key > lo) { const int at = atomicAdd(&s_n, 1); s_key[at] = key; s_pos[at] = j; }
    }
    __syncthreads();
    const int n = s_n;
    if (t < n) {
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += s_key[i] > s_key[t] || (s_key[i] == s_key[t] && s_pos[i] < s_pos[t]);
      values[row * K + rank] = x[s_pos[t]];
      indices[row * K + rank] = s_pos[t];
    }
    for (int j0 = 0; j0 < V && s_ties < K - n; j0 += blockDim.x) {
      const int j = j0 + t;
      const bool tie = j < V && order_key(Elem<T>::to_f32(x[j])) == lo;
      const unsigned b = __ballot_sync(0xffffffffu, tie);
      if ((t & 31) == 0) s_warp[t >> 5] = __popc(b);
      __syncthreads();
      int at = n + s_ties + __popc(b & ((1u << (t & 31)) - 1u));
      int total = 0;
      for (int i = 0; i < (int)(blockDim.x >> 5); ++i) { if (i < (t >> 5)) at += s_warp[i]; total += s_warp[i]; }
      if (tie && at < K) { values[row * K + at] = x[j]; indices[row * K + at] = j; }
      __syncthreads();
      if (t == 0) s_ties += total;
      __syncthreads();
    }
    if (lse) {
      float m = -INFINITY;
      for (int j = t; j < V; j += blockDim.x) m = fmaxf(m, Elem<T>::to_f32(x[j]));
      m = block_reduce<MaxOp>(m, s_red);
      if (isinf(m)) m = 0.f;                                    // no inf - inf: the sum is then 0 or inf
      const float c = (float)(inv_temp * 1.4426950408889634);
      float z = 0.f;
      for (int j = t; j < V; j += blockDim.x) z += exp2f_approx((Elem<T>::to_f32(x[j]) - m) * c);
      z = block_reduce<SumOp>(z, s_red);
      if (t == 0) lse[row] = (float)(log((double)z) + inv_temp * (double)m);
    }
    __syncthreads();
  }
}

template <typename T>
static int launch_topk(uint64_t values, uint64_t indices, uint64_t lse, uint64_t logits, int64_t rows, int64_t vocab, int64_t k,
                       double inv_temp, cudaStream_t st) {
  const int64_t cap = (int64_t)kNumSMs * 8;
  logits_topk_kernel<T><<<(unsigned)(rows < cap ? rows : cap), kTopkThreads, 0, st>>>(
      reinterpret_cast<T*>(values), reinterpret_cast<int*>(indices), reinterpret_cast<float*>(lse),
      reinterpret_cast<const T*>(logits), rows, (int)vocab, (int)k, inv_temp);
  return check_launch();
}

}  // namespace cb

extern "C" {
int cacti_b200_logits_topk(cacti_b200_dptr values, cacti_b200_dptr indices, cacti_b200_dptr lse, cacti_b200_dptr logits,
                           int64_t rows, int64_t vocab, int64_t k, float temperature, int dtype, cacti_b200_stream stream) {
  using namespace cb;
  if (rows < 0 || vocab < 0 || k < 0) return CACTI_B200_ERR_INVALID_VALUE;
  if (!(temperature >= 1e-4f && temperature <= 1e4f)) return CACTI_B200_ERR_INVALID_VALUE;
  if (dtype != CACTI_B200_R_32F && dtype != CACTI_B200_R_16F && dtype != CACTI_B200_R_16BF) return CACTI_B200_ERR_DTYPE;
  if (vocab > kTopkMaxVocab || k > kTopkMaxK || k < 1 || k > vocab || rows > 0x7fffffffLL) return CACTI_B200_ERR_SHAPE;
  if (rows == 0) return CACTI_B200_OK;
  const int es = dtype == CACTI_B200_R_32F ? 4 : 2;
  if (!values || !indices || !logits || values % es || logits % es || (indices & 3) || (lse & 3)) return CACTI_B200_ERR_INVALID_VALUE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dispatch_dtype(dtype, [&](auto tag) -> int {
    return launch_topk<decltype(tag)>(values, indices, lse, logits, rows, vocab, k, 1.0 / (double)temperature, st);
  });
}
}
