// Gated feed-forward block: h = silu(x Wg^T) * (x Wu^T) in one kernel, and its adjoint.
//
// Stands beside the separate path (two matmuls, src/librarium/llama.rs:522-525, and swiglu, :526-527).  With s = sigmoid(g):
//   g = x Wg^T, u = x Wu^T, h = g s u
//   dg = dh u s (1 + g (1 - s)),  du = dh g s;  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
// g and u stay in f32 up to h's one rounding (the thunk chain rounds them, and every primitive after them, to 16 bits).
// For the backward pass they are kept as rounded to 16 bits; dg and du are rounded to 16 bits to be operands of the tensor
// cores, a relative error of half a step on each term of sums over hundreds of terms, as for any stored activation gradient.
#include "common.cuh"
#include <type_traits>

namespace cb {

constexpr int kFfnTile = 64, kFfnK = 16;

// silu and its derivative from one sigmoid
__device__ __forceinline__ float sigmoid_f32(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }

// One 64 x 64 tile of h: 256 threads, 4 x 4 outputs each of g and of u; f32 multiply-adds.
template <typename T>
__global__ void __launch_bounds__(256)
gated_ffn_simple_kernel(T* __restrict__ H, T* __restrict__ G, T* __restrict__ U, const T* __restrict__ X,
                        const T* __restrict__ Wg, const T* __restrict__ Wu, int64_t tokens, int64_t D, int64_t F) {
  __shared__ float sx[kFfnK][kFfnTile + 1], sg[kFfnK][kFfnTile + 1], su[kFfnK][kFfnTile + 1];
  const int64_t m0 = (int64_t)blockIdx.y * kFfnTile, n0 = (int64_t)blockIdx.x * kFfnTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float g[4][4] = {}, u[4][4] = {};
  for (int64_t k0 = 0; k0 < D; k0 += kFfnK) {
    for (int i = threadIdx.x; i < kFfnTile * kFfnK; i += 256) {
      const int r = i / kFfnK, k = i % kFfnK;
      const bool kin = k0 + k < D;
      sx[k][r] = kin && m0 + r < tokens ? Elem<T>::to_f32(X[(m0 + r) * D + k0 + k]) : 0.f;
      sg[k][r] = kin && n0 + r < F ? Elem<T>::to_f32(Wg[(n0 + r) * D + k0 + k]) : 0.f;
      su[k][r] = kin && n0 + r < F ? Elem<T>::to_f32(Wu[(n0 + r) * D + k0 + k]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kFfnK; ++k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          g[i][j] = fmaf(sx[k][ty * 4 + i], sg[k][tx * 4 + j], g[i][j]);
          u[i][j] = fmaf(sx[k][ty * 4 + i], su[k][tx * 4 + j], u[i][j]);
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = m0 + ty * 4 + i, c = n0 + tx * 4 + j;
      if (r >= tokens || c >= F) continue;
      H[r * F + c] = Elem<T>::from_f32(g[i][j] * sigmoid_f32(g[i][j]) * u[i][j]);
      if (G) { G[r * F + c] = Elem<T>::from_f32(g[i][j]); U[r * F + c] = Elem<T>::from_f32(u[i][j]); }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
gated_ffn_adjoint_kernel(T* __restrict__ dG, T* __restrict__ dU, const T* __restrict__ dH, const T* __restrict__ G,
                         const T* __restrict__ U, int64_t n, int64_t F) {
  // dG and dU are the two halves of rows of 2 F
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t o = i + i / F * F;
    const float g = Elem<T>::to_f32(G[i]), u = Elem<T>::to_f32(U[i]), dh = Elem<T>::to_f32(dH[i]);
    const float s = sigmoid_f32(g);
    dG[o] = Elem<T>::from_f32(dh * u * (s * (1.f + g * (1.f - s))));
    dU[o] = Elem<T>::from_f32(dh * (g * s));
  }
}

static size_t ffn_align(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace cb

extern "C" {
size_t cacti_b200_gated_ffn_fwd_workspace_bytes(int64_t tokens, int64_t d_model, int64_t d_ffn, int aligned) {
  (void)tokens; (void)d_model; (void)d_ffn; (void)aligned;
  return 256;
}

int cacti_b200_gated_ffn_fwd(cacti_b200_dptr h, cacti_b200_dptr gate, cacti_b200_dptr up, cacti_b200_dptr x,
                             cacti_b200_dptr w_gate, cacti_b200_dptr w_up, int64_t tokens, int64_t d_model, int64_t d_ffn,
                             int dtype, cacti_b200_dptr workspace, size_t workspace_bytes, cacti_b200_stream stream) {
  using namespace cb;
  (void)workspace; (void)workspace_bytes;
  if (tokens < 0 || d_model < 0 || d_ffn < 0) return CACTI_B200_ERR_INVALID_VALUE;
  if (dtype != CACTI_B200_R_16F && dtype != CACTI_B200_R_16BF) return CACTI_B200_ERR_DTYPE;
  if (tokens > 0x3fffffffLL || d_model > 0x3fffffffLL || d_ffn > 0x3fffffffLL || d_model == 0 || d_ffn == 0) return CACTI_B200_ERR_SHAPE;
  if (tokens == 0) return CACTI_B200_OK;
  if (!h || !x || !w_gate || !w_up || !gate != !up) return CACTI_B200_ERR_INVALID_VALUE;
  if ((h | gate | up | x | w_gate | w_up) & 1) return CACTI_B200_ERR_INVALID_VALUE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)((d_ffn + kFfnTile - 1) / kFfnTile), (unsigned)((tokens + kFfnTile - 1) / kFfnTile));
  if (grid.y > 65535u) return CACTI_B200_ERR_SHAPE;
  auto go = [&](auto tag) -> int {
    using T = decltype(tag);
    gated_ffn_simple_kernel<T><<<grid, 256, 0, st>>>(reinterpret_cast<T*>(h), reinterpret_cast<T*>(gate), reinterpret_cast<T*>(up),
                                                      reinterpret_cast<const T*>(x), reinterpret_cast<const T*>(w_gate),
                                                      reinterpret_cast<const T*>(w_up), tokens, d_model, d_ffn);
    return check_launch();
  };
  return dtype == CACTI_B200_R_16F ? go(__half{}) : go(__nv_bfloat16{});
}

size_t cacti_b200_gated_ffn_bwd_workspace_bytes(int64_t tokens, int64_t d_model, int64_t d_ffn, int aligned) {
  (void)aligned;
  if (tokens < 0 || d_model < 0 || d_ffn < 0) return 0;
  const size_t a = cacti_b200_gemm_workspace_bytes(tokens, d_model, 2 * d_ffn, 1, 1);
  const size_t b = cacti_b200_gemm_workspace_bytes(d_ffn, d_model, tokens, 1, 1);
  return cb::ffn_align((size_t)tokens * d_ffn * 4) + cb::ffn_align((size_t)d_ffn * d_model * 4) + (a > b ? a : b) + 256;
}

int cacti_b200_gated_ffn_bwd(cacti_b200_dptr dx, cacti_b200_dptr dw_gate, cacti_b200_dptr dw_up, cacti_b200_dptr dh,
                             cacti_b200_dptr x, cacti_b200_dptr w_gate, cacti_b200_dptr w_up, cacti_b200_dptr gate,
                             cacti_b200_dptr up, int64_t tokens, int64_t d_model, int64_t d_ffn, int dtype, int beta_dx,
                             int beta_dw, cacti_b200_dptr workspace, size_t workspace_bytes, cacti_b200_stream stream) {
  using namespace cb;
  if (tokens < 0 || d_model < 0 || d_ffn < 0 || ((beta_dx | beta_dw) & ~1)) return CACTI_B200_ERR_INVALID_VALUE;
  if (dtype != CACTI_B200_R_16F && dtype != CACTI_B200_R_16BF) return CACTI_B200_ERR_DTYPE;
  if (tokens > 0x3fffffffLL || d_model > 0x3fffffffLL || d_ffn > 0x3fffffffLL || d_model == 0 || d_ffn == 0) return CACTI_B200_ERR_SHAPE;
  if (!dw_gate || !dw_up) return CACTI_B200_ERR_INVALID_VALUE;
  if (tokens > 0 && (!dx || !dh || !x || !w_gate || !w_up || !gate || !up)) return CACTI_B200_ERR_INVALID_VALUE;
  if ((dx | dw_gate | dw_up | dh | x | w_gate | w_up | gate | up) & 1) return CACTI_B200_ERR_INVALID_VALUE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (tokens == 0) {                                            // an empty sum: the weight gradients are zero
    if (!beta_dw)
      for (uint64_t w : {dw_gate, dw_up})
        if (cudaMemsetAsync(reinterpret_cast<void*>(w), 0, (size_t)d_ffn * d_model * 2, st) != cudaSuccess) return check_launch();
    return CACTI_B200_OK;
  }
  if (!workspace || (workspace & 255) || workspace_bytes < cacti_b200_gated_ffn_bwd_workspace_bytes(tokens, d_model, d_ffn, 0))
    return CACTI_B200_ERR_WORKSPACE;
  // [dg | du] as rows of 2 d_ffn and [w_gate; w_up] one below the other: dx is one product over 2 d_ffn, rounded once
  const size_t part = ffn_align((size_t)tokens * d_ffn * 4), wpart = ffn_align((size_t)d_ffn * d_model * 4);
  const uint64_t dg = workspace, du = dg + (uint64_t)d_ffn * 2, wcat = workspace + part, ws = wcat + wpart;
  const size_t wsb = workspace_bytes - part - wpart, wb = (size_t)d_ffn * d_model * 2;
  if (cudaMemcpyAsync(reinterpret_cast<void*>(wcat), reinterpret_cast<const void*>(w_gate), wb, cudaMemcpyDeviceToDevice, st) != cudaSuccess ||
      cudaMemcpyAsync(reinterpret_cast<void*>(wcat + wb), reinterpret_cast<const void*>(w_up), wb, cudaMemcpyDeviceToDevice, st) != cudaSuccess)
    return check_launch();
  const int64_t n = tokens * d_ffn;
  const int64_t want = (n + 255) / 256, cap = (int64_t)kNumSMs * 32;
  auto go = [&](auto tag) -> int {
    using T = decltype(tag);
    gated_ffn_adjoint_kernel<T><<<(unsigned)(want < cap ? want : cap), 256, 0, st>>>(
        reinterpret_cast<T*>(dg), reinterpret_cast<T*>(du), reinterpret_cast<const T*>(dh), reinterpret_cast<const T*>(gate),
        reinterpret_cast<const T*>(up), n, d_ffn);
    return check_launch();
  };
  int rc = dtype == CACTI_B200_R_16F ? go(__half{}) : go(__nv_bfloat16{});
  const float one = 1.f, zero = 0.f;
  const float *bx = beta_dx ? &one : &zero, *bw = beta_dw ? &one : &zero;
  const int64_t f2 = 2 * d_ffn;
  if (!rc) rc = cacti_b200_gemm(dx, dg, wcat, tokens, d_model, f2, f2, d_model, d_model, 0, 0, &one, bx, dtype, ws, wsb, stream);
  if (!rc) rc = cacti_b200_gemm(dw_gate, dg, x, d_ffn, d_model, tokens, f2, d_model, d_model, 1, 0, &one, bw, dtype, ws, wsb, stream);
  if (!rc) rc = cacti_b200_gemm(dw_up, du, x, d_ffn, d_model, tokens, f2, d_model, d_model, 1, 0, &one, bw, dtype, ws, wsb, stream);
  return rc;
}
}
