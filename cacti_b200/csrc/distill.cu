// Distillation from a teacher's listed logits: loss and student gradient in one call.
//
// No counterpart in the reference; it stands where softmax_nll stands in a training step (src/librarium/llama.rs:542-545),
// with a row's target given by K (index, logit) pairs of a teacher instead of one index.  With c = 1 / temperature:
//   q = softmax(c x) over the whole row;  p_k = softmax of the listed c z, or exp(c z_k - lse) when the teacher's log of
//   its sum of exponentials is given; then r = max(0, 1 - sum p) is the mass of all unlisted positions together.
//   loss = sum_k p_k (log p_k - log q_{t_k}) + r (log r - log sum_{unlisted} q)
//   dloss/dx_j = c (P q_j - [j listed] p_j - [j unlisted] r q_j / sum_{unlisted} q),  P = sum p + r
// The unlisted sum is formed from the unlisted exponentials themselves, never as total minus listed: in a trained student
// the listed part is nearly everything.  What belongs to a listed entry or to a row is kept in double (a few hundred
// operations a row): the loss is a difference of nearly equal logarithms, and r is what a sum near one leaves.
#include "common.cuh"
#include <type_traits>

namespace cb {

constexpr int kDistillMaxK = 256;
constexpr int64_t kDistillMaxVocab = 1 << 18;
constexpr int kDistillThreads = 256;

struct DistillParams {
  const void* t_values;          // teacher logits [rows, k] in t_dtype
  const void* t_indices;         // [rows, k] int32 or uint16
  const float* t_lse;            // [rows] or null: renormalise over the list
  const float* w_rows;           // [rows] or null
  float* loss_rows;              // [rows] or null
  unsigned* status;              // u32 or null
  double inv_temp;
  float w_scalar;
  int64_t rows;
  int vocab, k;
  int t_dtype, idx_dtype, beta;
};

__device__ __forceinline__ double teacher_value(const DistillParams& p, int64_t i) {
  if (p.t_dtype == CACTI_B200_R_32F) return (double)reinterpret_cast<const float*>(p.t_values)[i];
  if (p.t_dtype == CACTI_B200_R_16F) return (double)__half2float(reinterpret_cast<const __half*>(p.t_values)[i]);
  return (double)__bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.t_values)[i]);
}
// -1: unused slot; -2: outside the vocabulary.  65535 marks an unused slot of a uint16 list where it is no index.
__device__ __forceinline__ int teacher_index(const DistillParams& p, int64_t i) {
  if (p.idx_dtype == CACTI_B200_R_32I) {
    const int v = reinterpret_cast<const int*>(p.t_indices)[i];
    return v >= 0 && v < p.vocab ? v : (v == -1 ? -1 : -2);
  }
  const int v = reinterpret_cast<const uint16_t*>(p.t_indices)[i];
  return v < p.vocab ? v : (v == 65535 ? -1 : -2);
}

__device__ __forceinline__ double block_sum_f64(double v, double* smem) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[w] = v;
  __syncthreads();
  double r = 0.;
  for (int i = 0; i < nw; ++i) r += smem[i];
  return r;
}

// One CTA a row, the row read three times from memory (the later times from L2).  Thread t < k owns slot t of the list; a
// bitmap in shared memory says which positions are listed.
template <typename T, bool BWD>
__global__ void __launch_bounds__(kDistillThreads)
distill_rows_kernel(T* __restrict__ dL, const T* __restrict__ L, const DistillParams p) {
  extern __shared__ unsigned bitmap[];
  __shared__ int s_idx[kDistillMaxK];
  __shared__ float s_red[33];
  __shared__ double s_redd[32];
  const int words = (p.vocab + 31) / 32, V = p.vocab;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float w = p.w_rows ? p.w_rows[row] : p.w_scalar;
    const T* x = L + row * V;
    T* d = BWD ? dL + row * V : nullptr;
    if (w == 0.f) {                                             // not read: loss 0, gradient 0
      if (threadIdx.x == 0 && p.loss_rows) p.loss_rows[row] = 0.f;
      if (BWD && !p.beta) for (int j = threadIdx.x; j < V; j += blockDim.x) d[j] = Elem<T>::from_f32(0.f);
      continue;
    }
    for (int i = threadIdx.x; i < words; i += blockDim.x) bitmap[i] = 0u;
    const int t = threadIdx.x;
    int idx = t < p.k ? teacher_index(p, row * p.k + t) : -1;
    if (t < kDistillMaxK) s_idx[t] = idx;
    __syncthreads();
    bool bad = idx == -2;
    if (idx >= 0) for (int j = 0; j < t; ++j) if (s_idx[j] == idx) { bad = true; break; }
    if (bad) idx = -1;
    const bool row_bad = __syncthreads_or(bad) != 0;
    double zs = -INFINITY;
    float xk = 0.f;
    if (idx >= 0) {
      zs = p.inv_temp * teacher_value(p, row * p.k + t);
      xk = Elem<T>::to_f32(x[idx]);
      atomicOr(bitmap + (idx >> 5), 1u << (idx & 31));
    }
    // the list's probabilities
    double pk = 0., lse_t;
    if (p.t_lse) {
      lse_t = (double)p.t_lse[row];
    } else {
      double zm = zs;                                           // maximum: through the float reduction would round it
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) { const double v = __shfl_xor_sync(0xffffffffu, zm, o); zm = v > zm || v != v ? v : zm; }
      __syncthreads();
      if ((t & 31) == 0) s_redd[t >> 5] = zm;
      __syncthreads();
      for (int i = 0; i < (int)(blockDim.x >> 5); ++i) zm = s_redd[i] > zm || s_redd[i] != s_redd[i] ? s_redd[i] : zm;
      lse_t = zm + log(block_sum_f64(zs == -INFINITY ? 0. : exp(zs - zm), s_redd));
    }
    if (zs != -INFINITY) pk = exp(zs - lse_t);
    const double psum = block_sum_f64(pk, s_redd);
    const double ent = block_sum_f64(pk != 0. ? pk * (zs - lse_t) : 0., s_redd);
    const int listed = (int)block_sum_f64(idx >= 0 ? 1. : 0., s_redd);
    // the student's row: maximum, then the sums over listed and unlisted positions
    float m = -INFINITY;
    for (int j = t; j < V; j += blockDim.x) m = fmaxf(m, Elem<T>::to_f32(x[j]));
    m = block_reduce<MaxOp>(m, s_red);
    // differences to the maximum, so that a row of values like the type's lowest loses nothing
    const double px = block_sum_f64(pk != 0. ? pk * ((double)xk - (double)m) : 0., s_redd);
    const float c = (float)(p.inv_temp * 1.4426950408889634);    // exponentials are 2^((x - m) c)
    float zr = 0.f;
    for (int j = t; j < V; j += blockDim.x)
      if (!((bitmap[j >> 5] >> (j & 31)) & 1u)) zr += exp2f_approx((Elem<T>::to_f32(x[j]) - m) * c);
    const float ek = idx >= 0 ? exp2f_approx((xk - m) * c) : 0.f;
    const double rest = block_sum_f64((double)zr, s_redd), all = rest + block_sum_f64((double)ek, s_redd);
    double r = p.t_lse && listed && listed < V ? 1. - psum : 0.;
    if (r < 0.) r = 0.;
    const double mass = psum + r;
    if (t == 0) {
      if (row_bad && p.status) atomicMax(p.status, (unsigned)CACTI_B200_ERR_INDEX_RANGE);
      if (p.loss_rows) {
        double loss = mass != 0. ? ent - p.inv_temp * px + psum * log(all) : 0.;
        if (r > 0.) loss += r * (log(r) - log(rest) + log(all));
        p.loss_rows[row] = row_bad ? __int_as_float(0x7fc00000) : (float)loss;
      }
    }
    if (BWD) {
      const double wc = (double)w * p.inv_temp;
      const float g_all = mass != 0. ? (float)(wc * mass / all) : 0.f;
      const float g_rest = mass != 0. ? (float)(wc * (mass / all - (r > 0. && rest > 0. ? r / rest : 0.))) : 0.f;
      for (int j = t; j < V; j += blockDim.x) {
        if ((bitmap[j >> 5] >> (j & 31)) & 1u) continue;
        const float v = exp2f_approx((Elem<T>::to_f32(x[j]) - m) * c) * g_rest;
        d[j] = p.beta ? Elem<T>::from_f32(Elem<T>::to_f32(d[j]) + round_to<T>(v)) : Elem<T>::from_f32(v);
      }
      if (idx >= 0) {
        const float v = ek * g_all - (float)(wc * pk);
        d[idx] = p.beta ? Elem<T>::from_f32(Elem<T>::to_f32(d[idx]) + round_to<T>(v)) : Elem<T>::from_f32(v);
      }
    }
    __syncthreads();
  }
}

// loss_sum = sum_i w_i loss_i in a fixed order: 1024 strided partial sums, then a tree.  Rows of weight 0 add nothing.
__global__ void __launch_bounds__(1024)
distill_loss_sum_kernel(float* __restrict__ loss_sum, const float* __restrict__ loss_rows, const float* __restrict__ w_rows,
                        float w_scalar, int64_t rows) {
  __shared__ double sm[1024];
  double acc = 0.;
  dependent_wait();
  for (int64_t i = threadIdx.x; i < rows; i += 1024) acc += (double)(w_rows ? w_rows[i] : w_scalar) * (double)loss_rows[i];
  sm[threadIdx.x] = acc;
  __syncthreads();
  for (int s = 512; s > 0; s >>= 1) {
    if ((int)threadIdx.x < s) sm[threadIdx.x] += sm[threadIdx.x + s];
    __syncthreads();
  }
  if (threadIdx.x == 0) *loss_sum = (float)sm[0];
}

template <typename T>
static int launch_distill(uint64_t dl, uint64_t l, const DistillParams& p, cudaStream_t st) {
  const size_t smem = (size_t)((p.vocab + 31) / 32) * 4;
  const int64_t cap = (int64_t)kNumSMs * 8;
  const unsigned grid = (unsigned)(p.rows < cap ? p.rows : cap);
  T* dL = reinterpret_cast<T*>(dl);
  const T* L = reinterpret_cast<const T*>(l);
  if (dl) distill_rows_kernel<T, true><<<grid, kDistillThreads, smem, st>>>(dL, L, p);
  else distill_rows_kernel<T, false><<<grid, kDistillThreads, smem, st>>>(dL, L, p);
  return check_launch();
}

}  // namespace cb

extern "C" {
size_t cacti_b200_distill_topk_workspace_bytes(int64_t rows) { return rows > 0 ? (size_t)rows * sizeof(float) + 256 : 256; }

int cacti_b200_distill_topk_fwd_bwd(cacti_b200_dptr loss_sum, cacti_b200_dptr loss_rows, cacti_b200_dptr dlogits,
                                    cacti_b200_dptr logits, cacti_b200_dptr t_values, int t_dtype, cacti_b200_dptr t_indices,
                                    int index_dtype, cacti_b200_dptr t_lse, int64_t k, float temperature,
                                    cacti_b200_dptr w_rows, float w_scalar, int64_t rows, int64_t vocab, int dtype,
                                    int beta_dlogits, cacti_b200_dptr status, cacti_b200_dptr workspace, size_t workspace_bytes,
                                    cacti_b200_stream stream) {
  using namespace cb;
  if (rows < 0 || vocab < 0 || k < 0 || (beta_dlogits & ~1)) return CACTI_B200_ERR_INVALID_VALUE;
  if (!(temperature >= 1e-4f && temperature <= 1e4f)) return CACTI_B200_ERR_INVALID_VALUE;
  if (index_dtype != CACTI_B200_R_32I && index_dtype != CACTI_B200_R_16U) return CACTI_B200_ERR_DTYPE;
  const int dts[2] = {dtype, t_dtype};
  for (int d : dts)
    if (d != CACTI_B200_R_32F && d != CACTI_B200_R_16F && d != CACTI_B200_R_16BF) return CACTI_B200_ERR_DTYPE;
  if (vocab > kDistillMaxVocab || k > kDistillMaxK || k < 1) return CACTI_B200_ERR_SHAPE;
  if ((loss_sum & 3) || (loss_rows & 3) || (t_lse & 3) || (w_rows & 3) || (status & 3)) return CACTI_B200_ERR_INVALID_VALUE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (rows == 0 || vocab == 0) return CACTI_B200_OK;
  if (rows > 0x7fffffffLL) return CACTI_B200_ERR_SHAPE;
  if (!logits || !t_values || !t_indices) return CACTI_B200_ERR_INVALID_VALUE;
  const int es = dtype == CACTI_B200_R_32F ? 4 : 2, ts = t_dtype == CACTI_B200_R_32F ? 4 : 2;
  const int is = index_dtype == CACTI_B200_R_32I ? 4 : 2;
  if (logits % es || dlogits % es || t_values % ts || t_indices % is) return CACTI_B200_ERR_INVALID_VALUE;
  float* lrows = reinterpret_cast<float*>(loss_rows);
  if (loss_sum && !lrows) {
    if (!workspace || (workspace & 3) || workspace_bytes < cacti_b200_distill_topk_workspace_bytes(rows))
      return CACTI_B200_ERR_WORKSPACE;
    lrows = reinterpret_cast<float*>(workspace);
  }
  DistillParams p;
  p.t_values = reinterpret_cast<const void*>(t_values); p.t_indices = reinterpret_cast<const void*>(t_indices);
  p.t_lse = reinterpret_cast<const float*>(t_lse); p.w_rows = reinterpret_cast<const float*>(w_rows);
  p.loss_rows = lrows; p.status = reinterpret_cast<unsigned*>(status);
  p.inv_temp = 1.0 / (double)temperature; p.w_scalar = w_scalar;
  p.rows = rows; p.vocab = (int)vocab; p.k = (int)k;
  p.t_dtype = t_dtype; p.idx_dtype = index_dtype; p.beta = beta_dlogits;
  int rc = dispatch_dtype(dtype, [&](auto tag) -> int { return launch_distill<decltype(tag)>(dlogits, logits, p, st); });
  if (rc) return rc;
  if (loss_sum) {
    launch_dependent(distill_loss_sum_kernel, 1u, 1024u, st, reinterpret_cast<float*>(loss_sum), (const float*)lrows,
                     p.w_rows, w_scalar, rows);
    return check_launch();
  }
  return CACTI_B200_OK;
}
}
