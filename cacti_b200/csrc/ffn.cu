// Gated feed-forward block: h = silu(x Wg^T) * (x Wu^T) in one kernel, and its adjoint.
//
// Stands beside the separate path (two matmuls, src/librarium/llama.rs:522-525, and swiglu, :526-527).  With s = sigmoid(g):
//   g = x Wg^T, u = x Wu^T, h = g s u
//   dg = dh u s (1 + g (1 - s)),  du = dh g s;  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
// g and u stay in f32 up to h's one rounding (the thunk chain rounds them, and every primitive after them, to 16 bits).
// For the backward pass they are kept as rounded to 16 bits; dg and du are rounded to 16 bits to be operands of the tensor
// cores, a relative error of half a step on each term of sums over hundreds of terms, as for any stored activation gradient.
//
// Forward: the matmul kernels' structure (TMA ring -> tcgen05.mma -> TMEM, epilogue warps on the previous tile) with a
// B tile that is half gate rows and half up rows, so that the two sums of an output element sit in one TMEM lane, a
// fixed number of columns apart, and the epilogue forms h without an exchange.  In the two-SM form the halves are what the two
// CTAs of a pair load anyway: the leader the gate rows, the peer the up rows.
// Backward: one element-wise pass (dg, du), then one launch for all three products: its tiles are those of dx (contraction
// over the gate part and then the up part, one accumulator, one rounding) followed by those of dWg and dWu.
//
// The tile walk is static: no global counter, so calls may overlap on any streams and graphs.
#include "gemm_common.cuh"

namespace cb {

struct FfnMaps { CUtensorMap a[2], b[3], c[3]; };

// silu's sigmoid, f32 with the fast exponential and division: relative error below 2^-20 for |g| < 30, far below the 16-bit
// rounding that follows; g = -inf gives s = 0.
__device__ __forceinline__ float sigmoid_f32(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }

// ---- forward ------------------------------------------------------------------------------------------------------
struct FfnFwdParams {
  int M, N, nkb;                 // tokens, d_ffn, k-blocks
  int tiles_m, tiles_n, group_m;
  uint32_t idesc;
  int out_tma;                   // outputs are written with TMA stores
  int a_rows;                    // rows of the x box (a multiple of 8)
};

__device__ __forceinline__ void ffn_decode(int tile, int tiles_m, int tiles_n, int group_m, int& tm, int& tn) {
  const int per_group = group_m * tiles_n;
  const int grp = tile / per_group, in = tile - grp * per_group;
  const int m0 = grp * group_m;
  const int gm = tiles_m - m0 < group_m ? tiles_m - m0 : group_m;
  tn = in / gm;
  tm = m0 + (in - tn * gm);
}

// Copy a [32 rows][64 columns] swizzled staging buffer to an output whose rows TMA cannot address: a warp writes one row at
// a time, consecutive lanes consecutive elements.
template <typename T>
__device__ __forceinline__ void ffn_store_rows(const unsigned char* buf, T* __restrict__ out, int row0, int M, int col0, int N, int lane) {
#pragma unroll 1
  for (int r = 0; r < 32; ++r) {
    if (row0 + r >= M) break;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int c = half * 32 + lane;
      if (col0 + c < N)
        out[(long long)(row0 + r) * N + col0 + c] = *reinterpret_cast<const T*>(buf + r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2);
    }
  }
}

// Epilogue of one accumulator for one warp: TMEM lanes [q*32, +32), columns [acc * 2 HALF, +HALF) hold g and the next HALF u of
// output columns tn * HALF ...; h (and g, u when SAVE) leave through swizzled staging, 64 columns a trip.
template <typename T, int HALF, bool SAVE>
__device__ __forceinline__ void ffn_epilogue(const FfnFwdParams& p, const FfnMaps& maps, T* __restrict__ H, T* __restrict__ G, T* __restrict__ U,
                                             uint32_t tmem_base, int acc, int row0, int tn, int q, int lane,
                                             unsigned char* mybuf, uint32_t tempty_addr) {
  constexpr int TRIPS = HALF / 64;
#pragma unroll 1
  for (int c = 0; c < TRIPS; ++c) {
    const int col0 = tn * HALF + c * 64;
    const uint32_t t0 = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * 2 * HALF + c * 64);
    uint32_t g[2][32], u[2][32];
    tc_ld32(t0, g[0]);
    tc_ld32(t0 + HALF, u[0]);
    tc_ld32(t0 + 32, g[1]);
    tc_ld32(t0 + HALF + 32, u[1]);
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // the staging has been read
    tc_ld_wait();
    if (c == TRIPS - 1) {                                 // the accumulator is free
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty_addr);
    } else {
      __syncwarp();
    }
    if (col0 < p.N) {                                     // warp-uniform
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float g8[8], u8[8], h8[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            g8[i] = __uint_as_float(g[hh][k * 8 + i]);
            u8[i] = __uint_as_float(u[hh][k * 8 + i]);
            h8[i] = g8[i] * sigmoid_f32(g8[i]) * u8[i];
          }
          const int off = lane * 128 + (((hh * 4 + k) ^ (lane & 7)) << 4);
          *reinterpret_cast<uint4*>(mybuf + off) = pack<T>(h8);
          if (SAVE) {
            *reinterpret_cast<uint4*>(mybuf + 4096 + off) = pack<T>(g8);
            *reinterpret_cast<uint4*>(mybuf + 8192 + off) = pack<T>(u8);
          }
        }
      }
      if (p.out_tma) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          tma_store_4d(&maps.c[0], mybuf, col0, row0, 0, 0);
          if (SAVE) {
            tma_store_4d(&maps.c[1], mybuf + 4096, col0, row0, 0, 0);
            tma_store_4d(&maps.c[2], mybuf + 8192, col0, row0, 0, 0);
          }
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      } else {
        __syncwarp();
        ffn_store_rows(mybuf, H, row0, p.M, col0, p.N, lane);
        if (SAVE) {
          ffn_store_rows(mybuf + 4096, G, row0, p.M, col0, p.N, lane);
          ffn_store_rows(mybuf + 8192, U, row0, p.M, col0, p.N, lane);
        }
        __syncwarp();
      }
    }
  }
}

// Shared memory behind the operand stages: barriers, then per epilogue warp one staging buffer for each output.
constexpr uint32_t kFfnStageBytes = 32768;                // both forms: 128 rows of x and 128 rows of weights, 64 deep
template <bool SAVE> constexpr int ffn_fwd_stages() { return SAVE ? 5 : 6; }
template <bool SAVE> constexpr size_t ffn_fwd_smem() {
  return (size_t)ffn_fwd_stages<SAVE>() * kFfnStageBytes + 1024 + 1024 + 4 * (SAVE ? 12288 : 4096);
}

// PAIR: a cluster of two CTAs computes 256 tokens x 128 columns of h (a 256 x 256 accumulator).
// Otherwise one CTA computes 128 tokens x 64 columns (a 128 x 128 accumulator): for few tokens, where the block is bound
// by reading the weights and 64-column tiles spread them over twice as many SMs.
template <typename T, bool PAIR, bool SAVE>
__device__ __forceinline__ void ffn_fwd_body(const FfnMaps& maps, T* __restrict__ H, T* __restrict__ G, T* __restrict__ U, const FfnFwdParams& p) {
  constexpr int HALF = PAIR ? 128 : 64, STAGES = ffn_fwd_stages<SAVE>(), TM = PAIR ? 256 : 128;
  constexpr uint32_t A_BYTES = kBM * kBK * 2, STAGE_BYTES = kFfnStageBytes;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + (size_t)STAGES * STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  unsigned char* cstage = tiles + (size_t)STAGES * STAGE_BYTES + 1024;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0;
  const int worker = PAIR ? blockIdx.x >> 1 : blockIdx.x, nworkers = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int total = p.tiles_m * p.tiles_n;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(tfull + a, 1); mbar_init(tempty + a, PAIR ? 8 : 4); }
    mbar_fence_init();
  }
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();               // the peer's barriers are initialised before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer (both CTAs of a pair) ----------------
    int s = 0; unsigned ph = 0;
    bool ok = true;
    const uint32_t bytes = PAIR ? 2 * STAGE_BYTES : (uint32_t)p.a_rows * kBK * 2 + STAGE_BYTES - A_BYTES;
    for (int tile = worker; ok && tile < total; tile += nworkers) {
      int tm, tn;
      ffn_decode(tile, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
      for (int kb = 0; kb < p.nkb; ++kb) {
        if (!mbar_wait_bounded(empty + s, ph ^ 1, kDevErrGemmTimeout)) { ok = false; break; }
        unsigned char* sa = tiles + (size_t)s * STAGE_BYTES;
        unsigned char* sb = sa + A_BYTES;
        if (rank == 0) mbar_expect_tx(full + s, bytes);
        if (PAIR) {
          const uint32_t fb = map_to_rank(smem_u32(full + s), 0);
          tma_load_4d_pair(sa, &maps.a[0], fb, kb * kBK, tm * TM + (int)rank * kBM, 0, 0);
          tma_load_4d_pair(sb, &maps.b[rank], fb, kb * kBK, tn * HALF, 0, 0);
        } else {
          tma_load_4d(sa, &maps.a[0], full + s, kb * kBK, tm * TM, 0, 0);
          tma_load_4d(sb, &maps.b[0], full + s, kb * kBK, tn * HALF, 0, 0);
          tma_load_4d(sb + 8192, &maps.b[1], full + s, kb * kBK, tn * HALF, 0, 0);
        }
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
    }
    // the leader's last commits still arrive on this CTA's empty barriers: wait for them before leaving
    if (PAIR)
      for (int i = 0; ok && i < STAGES; ++i) {
        ok = mbar_wait_bounded(empty + s, ph ^ 1, kDevErrGemmTimeout);
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ---------------- MMA issuer (a pair's leader) ----------------
    int s = 0; unsigned ph = 0;
    int local = 0;
    bool ok = true;
    for (int tile = worker; ok && tile < total; tile += nworkers, ++local) {
      const int acc = local & 1;
      if (!mbar_wait_bounded(tempty + acc, (unsigned)((local >> 1) & 1) ^ 1, kDevErrGemmTimeout)) break;
      tc_fence_after();
      const uint32_t tacc = tmem_base + (uint32_t)(acc * 2 * HALF);
      for (int kb = 0; kb < p.nkb; ++kb) {
        if (!mbar_wait_bounded(full + s, ph, kDevErrGemmTimeout)) { ok = false; break; }
        tc_fence_after();
        const uint32_t sa = smem_u32(tiles + (size_t)s * STAGE_BYTES), sb = sa + A_BYTES;
#pragma unroll
        for (int k4 = 0; k4 < kBK / 16; ++k4) {
          const uint64_t da = make_desc(sa + k4 * 32, 1, 64), db = make_desc(sb + k4 * 32, 1, 64);
          if (PAIR) tc_mma_f16_pair(tacc, da, db, p.idesc, (kb || k4) ? 1u : 0u);
          else tc_mma_f16(tacc, da, db, p.idesc, (kb || k4) ? 1u : 0u);
        }
        if (PAIR) tc_commit_pair(empty + s);
        else tc_commit(empty + s);              // stage free once these MMAs have read it
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
      if (!ok) break;
      if (PAIR) tc_commit_pair(tfull + acc);
      else tc_commit(tfull + acc);              // accumulator complete
    }
  } else if (warp >= 2) {
    // ---------------- epilogue (each CTA on its own 128 rows) ----------------
    const int q = warp & 3;                     // TMEM lane quarter this warp may read
    int local = 0;
    for (int tile = worker; tile < total; tile += nworkers, ++local) {
      int tm, tn;
      ffn_decode(tile, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
      const int acc = local & 1;
      // all 32 lanes leave together: a wait that ran out on some lanes only must not split the warp before tcgen05.ld
      if (!mbar_wait_bounded_warp(tfull + acc, (unsigned)((local >> 1) & 1), kDevErrGemmTimeout)) break;
      tc_fence_after();
      const uint32_t te = PAIR ? map_to_rank(smem_u32(tempty + acc), 0) : smem_u32(tempty + acc);
      ffn_epilogue<T, HALF, SAVE>(p, maps, H, G, U, tmem_base, acc, tm * TM + (int)rank * kBM + q * 32, tn, q, lane,
                                  cstage + (size_t)(warp - 2) * (SAVE ? 12288 : 4096), te);
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();                 // both CTAs have finished reading TMEM and signalling each other
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  }
}

template <typename T, bool SAVE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1)
ffn_fwd_pair_kernel(const __grid_constant__ FfnMaps maps, T* __restrict__ H, T* __restrict__ G, T* __restrict__ U, const FfnFwdParams p) {
  ffn_fwd_body<T, true, SAVE>(maps, H, G, U, p);
}
template <typename T, bool SAVE>
__global__ void __launch_bounds__(kGemmThreads, 1)
ffn_fwd_kernel(const __grid_constant__ FfnMaps maps, T* __restrict__ H, T* __restrict__ G, T* __restrict__ U, const FfnFwdParams p) {
  ffn_fwd_body<T, false, SAVE>(maps, H, G, U, p);
}

// A packed matrix as an operand; repacked into the workspace when TMA cannot address it.
static int ffn_operand(Operand& o, uint64_t ptr, int64_t rows, int64_t cols, uint64_t ws, size_t ws_bytes, size_t& off, cudaStream_t st) {
  o = Operand{ptr, rows, cols, cols, 0, 0, 0, 0};
  if (tma_ok(o, 1, 1)) return CACTI_B200_OK;
  const size_t need = packed_bytes(rows, cols, 1);
  if (!ws || (ws & 255) || off + need > ws_bytes) return CACTI_B200_ERR_WORKSPACE;
  const int rc = repack_operand(o, 1, 1, ws + off, st);
  off += need;
  return rc;
}

static bool ffn_rows_aligned(uint64_t ptr, int64_t cols) { return ((ptr | (uint64_t)(cols * 2)) & 15) == 0; }

static uint32_t ffn_idesc(bool bf16, int a_mn, int b_mn, int n, int m) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <typename T>
static int ffn_fwd_run(uint64_t h, uint64_t gate, uint64_t up, uint64_t x, uint64_t wg, uint64_t wu, int64_t tokens, int64_t D,
                       int64_t F, uint64_t ws, size_t ws_bytes, cudaStream_t st) {
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  Operand ox, og, ou;
  size_t off = 0;
  int rc = ffn_operand(ox, x, tokens, D, ws, ws_bytes, off, st);
  if (!rc) rc = ffn_operand(og, wg, F, D, ws, ws_bytes, off, st);
  if (!rc) rc = ffn_operand(ou, wu, F, D, ws, ws_bytes, off, st);
  if (rc) return rc;
  const bool save = gate != 0, pair = tokens > kBM;
  const int tm = pair ? 256 : 128, half = pair ? 128 : 64;
  FfnFwdParams p;
  p.M = (int)tokens; p.N = (int)F; p.nkb = (int)((D + kBK - 1) / kBK);
  p.tiles_m = (int)((tokens + tm - 1) / tm); p.tiles_n = (int)((F + half - 1) / half);
  p.group_m = p.tiles_m < 8 ? p.tiles_m : 8;               // 2048 rows of x stay in L2 while the weight panels stream
  p.idesc = ffn_idesc(bf16, 0, 0, 2 * half, tm);
  p.a_rows = pair || tokens >= 128 ? 128 : (int)((tokens + 7) / 8 * 8);
  p.out_tma = ffn_rows_aligned(h, F) && (!save || (ffn_rows_aligned(gate, F) && ffn_rows_aligned(up, F)));
  FfnMaps maps;
  rc = encode_operand(&maps.a[0], ox, 1, 1, 64, p.a_rows, bf16);
  if (!rc) rc = encode_operand(&maps.b[0], og, 1, 1, 64, half, bf16);
  if (!rc) rc = encode_operand(&maps.b[1], ou, 1, 1, 64, half, bf16);
  maps.a[1] = maps.a[0]; maps.b[2] = maps.b[0];
  for (int i = 0; i < 3; ++i) {
    maps.c[i] = maps.a[0];
    const uint64_t ptr = i == 0 ? h : i == 1 ? gate : up;
    if (!rc && p.out_tma && ptr) rc = encode_operand(&maps.c[i], Operand{ptr, tokens, F, F, 0, 0, 0, 0}, 1, 1, 64, 32, bf16);
  }
  if (rc) return rc;
  T *H = reinterpret_cast<T*>(h), *G = reinterpret_cast<T*>(gate), *U = reinterpret_cast<T*>(up);
  const long long total = (long long)p.tiles_m * p.tiles_n;
  if (total > 0x3fffffffLL) return CACTI_B200_ERR_SHAPE;
  const long long cap = pair ? kNumSMs / 2 : kNumSMs, workers = total < cap ? total : cap;
#define CB_FFN(KERN_, SAVE_, GRID_)                                                               \
  do {                                                                                            \
    auto kern = KERN_<T, SAVE_>;                                                                  \
    static bool attr_set[kMaxDevices] = {};                                                       \
    ensure_dynamic_smem(kern, ffn_fwd_smem<SAVE_>(), attr_set);                                   \
    kern<<<(unsigned)(GRID_), kGemmThreads, ffn_fwd_smem<SAVE_>(), st>>>(maps, H, G, U, p);       \
  } while (0)
  if (pair) { if (save) CB_FFN(ffn_fwd_pair_kernel, true, 2 * workers); else CB_FFN(ffn_fwd_pair_kernel, false, 2 * workers); }
  else { if (save) CB_FFN(ffn_fwd_kernel, true, workers); else CB_FFN(ffn_fwd_kernel, false, workers); }
#undef CB_FFN
  return check_launch();
}

// ---- backward -----------------------------------------------------------------------------------------------------
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
  if (tokens < 0 || d_model < 0 || d_ffn < 0) return 0;
  if (aligned && d_model % 8 == 0) return 256;
  return cb::packed_bytes(tokens, d_model, 1) + 2 * cb::packed_bytes(d_ffn, d_model, 1) + 256;
}

int cacti_b200_gated_ffn_fwd(cacti_b200_dptr h, cacti_b200_dptr gate, cacti_b200_dptr up, cacti_b200_dptr x,
                             cacti_b200_dptr w_gate, cacti_b200_dptr w_up, int64_t tokens, int64_t d_model, int64_t d_ffn,
                             int dtype, cacti_b200_dptr workspace, size_t workspace_bytes, cacti_b200_stream stream) {
  using namespace cb;
  if (tokens < 0 || d_model < 0 || d_ffn < 0) return CACTI_B200_ERR_INVALID_VALUE;
  if (dtype != CACTI_B200_R_16F && dtype != CACTI_B200_R_16BF) return CACTI_B200_ERR_DTYPE;
  if (tokens > 0x3fffffffLL || d_model > 0x3fffffffLL || d_ffn > 0x3fffffffLL || d_model == 0 || d_ffn == 0) return CACTI_B200_ERR_SHAPE;
  if (tokens == 0) return CACTI_B200_OK;
  if (!h || !x || !w_gate || !w_up || !gate != !up) return CACTI_B200_ERR_INVALID_VALUE;
  if ((h | gate | up | x | w_gate | w_up) & 1) return CACTI_B200_ERR_INVALID_VALUE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == CACTI_B200_R_16F)
    return ffn_fwd_run<__half>(h, gate, up, x, w_gate, w_up, tokens, d_model, d_ffn, workspace, workspace_bytes, st);
  return ffn_fwd_run<__nv_bfloat16>(h, gate, up, x, w_gate, w_up, tokens, d_model, d_ffn, workspace, workspace_bytes, st);
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
