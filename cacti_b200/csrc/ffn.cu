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
// Calls may overlap on any streams and graphs: the forward's tile walk is static, the backward's draws its items from a
// counter in the call's own workspace.  The backward's items differ in length (2 F and T deep), and their contractions are so long
// that workers on a static walk drift apart and no longer share operand panels in L2: at 16384 x 3200 x 8640, sustained, the
// static walk took 3.58 ms against 2.94 ms.
//
// Bound: the tensor cores, 4 T D F operations forward and 8 T D F backward, at the measured
// cuBLAS rate (1.67 PFLOP/s burst, 1.40 sustained under the power cap).  16384 x 3200 x 8640 f16 in a loop at the power cap, which differs
// from card to card: forward 1.29 to 1.43 ms without the projections kept (1.27 to 1.40 PFLOP/s), 1.36 to 1.52 ms with them (0.57 GB more
// written); backward 2.92 to 3.38 ms (1.07 to 1.24 PFLOP/s), of which the adjoint pass is 1.4 GB and 215 us.  2048 tokens: 381 to 418 us.
// The separate operators (matmuls and swiglu) in the same run and graphs: 16384 tokens 1645 us forward (this file 1505) and 3446 us
// backward (3364); 2048 tokens 224 (196) and 488 (409); 333 tokens 62 (55) and 171 (125).
// Tensor pipes are active 87 percent of the cycles forward and 85 percent backward at 2048 tokens.
#include "gemm_common.cuh"
#include <utility>

namespace cb {

struct FfnMaps { CUtensorMap a[2], b[3], c[3], ak[2]; };

// silu's sigmoid, f32 with the fast exponential and division.  By their documented bounds its relative error is at most
// (5 + 1.2 |g|) 2^-23 for negative g (2^-20 at -3, 2^-17.6 at -30) and 2^-20 for positive g: far below the 16-bit rounding that
// follows.  g = -inf gives s = 0.
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
// Otherwise one CTA computes 128 tokens x 64 columns (a 128 x 128 accumulator): for few tokens, where the block is bound by reading
// the weights and 64-column tiles spread them over twice as many SMs (the rule is in ffn_fwd_run).
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

static bool ffn_rows_aligned(uint64_t ptr, int64_t cols) { return ((ptr | (uint64_t)(cols * 2)) & 15) == 0; }

// ---- forward, one token -------------------------------------------------------------------------------------------------
// Bound by reading the weights once.  A warp takes an output column at a time: its gate row and its up row in 16-byte vectors,
// eight loads ahead, against the token in shared memory (f32, so that it is converted once); sums in f32, joined over the lanes in a
// fixed order.  3200 x 8640 f16: 18.7 us = 5.9 TB/s, 0.91 of the measured copy rate; the tensor-core kernel takes 22.1 us.  For two
// tokens it is the other way round (22.7 against 22.1 us): the multiply-adds no longer hide.
constexpr int kFfnVecElems = 24576;                            // the token has to fit
template <typename T>
__global__ void __launch_bounds__(512, 2)
ffn_fwd_vec_kernel(T* __restrict__ H, T* __restrict__ G, T* __restrict__ U, const T* __restrict__ X, const T* __restrict__ Wg,
                   const T* __restrict__ Wu, int D, int F) {
  extern __shared__ float sx[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nvec = D / 8;
  for (int i = threadIdx.x; i < D; i += 512) sx[i] = Elem<T>::to_f32(X[i]);
  __syncthreads();
  for (int f = blockIdx.x * 16 + warp; f < F; f += gridDim.x * 16) {
    const uint4* wg = reinterpret_cast<const uint4*>(Wg + (long long)f * D);
    const uint4* wu = reinterpret_cast<const uint4*>(Wu + (long long)f * D);
    float g = 0.f, u = 0.f;
    auto take = [&](const uint4& a, const uint4& b, int v) {
      float ga[8], ub[8];
      unpack<T>(a, ga);
      unpack<T>(b, ub);
      const float4 x0 = *reinterpret_cast<const float4*>(sx + v * 8), x1 = *reinterpret_cast<const float4*>(sx + v * 8 + 4);
      const float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) { g = fmaf(ga[e], x[e], g); u = fmaf(ub[e], x[e], u); }
    };
    int v = lane;
#pragma unroll 1
    for (; v + 96 < nvec; v += 128) {
      uint4 a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { a[i] = ld_stream(wg + v + 32 * i); b[i] = ld_stream(wu + v + 32 * i); }
#pragma unroll
      for (int i = 0; i < 4; ++i) take(a[i], b[i], v + 32 * i);
    }
#pragma unroll 1
    for (; v < nvec; v += 32) take(ld_stream(wg + v), ld_stream(wu + v), v);
    g = warp_reduce<SumOp>(g);
    u = warp_reduce<SumOp>(u);
    if (lane == 0) {
      H[f] = Elem<T>::from_f32(g * sigmoid_f32(g) * u);
      if (G) { G[f] = Elem<T>::from_f32(g); U[f] = Elem<T>::from_f32(u); }
    }
  }
}

// Up to three packed matrices [rows][cols] to rows of cols_pad (a multiple of 64) with zeros behind the data, for operands that TMA
// cannot address.  One 16-byte vector a thread: five aligned 4-byte loads, shifted where the row starts at an odd element.
struct FfnPack { const unsigned char* src[3]; uint4* dst[3]; unsigned first[4]; unsigned rows[3]; };   // first: vector counts, running
__global__ void __launch_bounds__(256) ffn_pack_kernel(const FfnPack p, unsigned cols, unsigned vpr /* vectors per padded row */) {
  const unsigned i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= p.first[3]) return;
  const int m = i >= p.first[2] ? 2 : i >= p.first[1] ? 1 : 0;
  const unsigned v = i - p.first[m], row = v / vpr, c = (v - row * vpr) * 8;
  const uint64_t begin = reinterpret_cast<uint64_t>(p.src[m]), end = begin + (uint64_t)p.rows[m] * cols * 2;
  const uint64_t a = begin + ((uint64_t)row * cols + c) * 2, base = a & ~3ull;
  uint32_t o[4] = {0, 0, 0, 0};
  if (c + 8 <= cols && base >= begin && base + 20 <= end) {
    const uint32_t* s = reinterpret_cast<const uint32_t*>(base);
    uint32_t w[5];
#pragma unroll
    for (int k = 0; k < 5; ++k) w[k] = __ldg(s + k);
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = (a & 2) ? __funnelshift_r(w[k], w[k + 1], 16) : w[k];
  } else {                                                      // a row's end, the matrix's ends
    for (unsigned k = 0; k < 8; ++k)
      if (c + k < cols) o[k >> 1] |= (uint32_t)reinterpret_cast<const unsigned short*>(a)[k] << (16 * (k & 1));
  }
  p.dst[m][v] = make_uint4(o[0], o[1], o[2], o[3]);
}

// Packed matrices as operands; those that TMA cannot address are repacked into the workspace, in one launch.
static int ffn_operands(Operand (&o)[3], const uint64_t (&ptr)[3], const int64_t (&rows)[3], int64_t cols, uint64_t ws, size_t ws_bytes,
                        size_t off, cudaStream_t st) {
  FfnPack p{};
  const int64_t cp = packed_cols(cols), vpr = cp / 8;
  unsigned n = 0;
  for (int i = 0; i < 3; ++i) {
    o[i] = Operand{ptr[i], rows[i], cols, cols, 0, 0, 0, 0};
    p.first[i] = n;
    if (tma_ok(o[i], 1, 1)) continue;
    const size_t need = packed_bytes(rows[i], cols, 1);
    if (!ws || (ws & 255) || off + need > ws_bytes) return CACTI_B200_ERR_WORKSPACE;
    p.src[i] = reinterpret_cast<const unsigned char*>(ptr[i]);
    p.dst[i] = reinterpret_cast<uint4*>(ws + off);
    p.rows[i] = (unsigned)rows[i];
    n += (unsigned)(rows[i] * vpr);
    o[i].ptr = ws + off; o[i].ld = cp; o[i].map_cols = cp;
    off += need;
  }
  p.first[3] = n;
  if (!n) return CACTI_B200_OK;
  ffn_pack_kernel<<<(n + 255) / 256, 256, 0, st>>>(p, (unsigned)cols, (unsigned)vpr);
  return check_launch();
}

// No output shares bytes with an input or with another output.
template <int NO, int NI> static bool ffn_separate(const Span (&out)[NO], const Span (&in)[NI]) {
  for (int o = 0; o < NO; ++o) {
    for (int i = 0; i < NI; ++i) if (overlap(out[o], in[i])) return false;
    for (int i = 0; i < o; ++i) if (overlap(out[o], out[i])) return false;
  }
  return true;
}

// Sizes whose tile, k-block and vector counts fit 32-bit indices, one operand at a time.
static bool ffn_sizes_ok(int64_t tokens, int64_t D, int64_t F) {
  constexpr int64_t kMax = 1 << 24, kElems = 1LL << 34;
  return D > 0 && F > 0 && tokens <= kMax && D <= kMax && F <= kMax && tokens * (F + 64) < kElems && tokens * D < kElems && F * D < kElems;
}
// The repacking launch numbers the vectors of all the operands that it copies in 32 bits: three operands near the bound above, copies of
// 64 GiB and more together, do not fit and are refused.
static bool ffn_pack_ok(const uint64_t (&ptr)[3], const int64_t (&rows)[3], int64_t cols) {
  int64_t n = 0;
  for (int i = 0; i < 3; ++i)
    if (!ffn_rows_aligned(ptr[i], cols)) n += rows[i] * (packed_cols(cols) / 8);
  return n <= 0xffffffffLL - 256;                               // whole blocks of 256 threads
}


static uint32_t ffn_idesc(bool bf16, int a_mn, int b_mn, int n, int m) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <typename T>
static int ffn_fwd_run(uint64_t h, uint64_t gate, uint64_t up, uint64_t x, uint64_t wg, uint64_t wu, int64_t tokens, int64_t D,
                       int64_t F, uint64_t ws, size_t ws_bytes, cudaStream_t st) {
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  if (tokens == 1 && D <= kFfnVecElems && ffn_rows_aligned(wg, D) && ffn_rows_aligned(wu, D)) {
    auto kern = ffn_fwd_vec_kernel<T>;
    static bool attr_set[kMaxDevices] = {};
    ensure_dynamic_smem(kern, kFfnVecElems * sizeof(float), attr_set);
    const int64_t blocks = (F + 15) / 16;
    kern<<<(unsigned)(blocks < 2 * kNumSMs ? blocks : 2 * kNumSMs), 512, (size_t)D * sizeof(float), st>>>(
        reinterpret_cast<T*>(h), reinterpret_cast<T*>(gate), reinterpret_cast<T*>(up), reinterpret_cast<const T*>(x),
        reinterpret_cast<const T*>(wg), reinterpret_cast<const T*>(wu), (int)D, (int)F);
    return check_launch();
  }
  Operand op[3];
  int rc = ffn_operands(op, {x, wg, wu}, {tokens, F, F}, D, ws, ws_bytes, 0, st);
  if (rc) return rc;
  // Two-SM tiles of 256 tokens x 128 columns, or one-SM tiles of 128 x 64, whichever needs less time: waves of the persistent grid
  // times a tile's cost per wave.  The costs are the matmul kernels' (gemm.cu): 0.93 of 256 columns against 1.3 of 128; measured here
  // at 333 x 1160 x 3080: one-SM 147 tiles in one wave 13.5 us, two-SM 50 tiles 17.5 us; at 2048 x 3200 x 8640: 250 us against 187 us.
  auto waves = [](int64_t tiles, int64_t workers) { return (double)((tiles + workers - 1) / workers); };
  const double cost2 = waves((tokens + 255) / 256 * ((F + 127) / 128), kNumSMs / 2) * 256 * 0.93;
  const double cost1 = waves((tokens + 127) / 128 * ((F + 63) / 64), kNumSMs) * 128 * 1.3;
  const bool save = gate != 0, pair = tokens > kBM && cost2 <= cost1;
  const int tm = pair ? 256 : 128, half = pair ? 128 : 64;
  FfnFwdParams p;
  p.M = (int)tokens; p.N = (int)F; p.nkb = (int)((D + kBK - 1) / kBK);
  p.tiles_m = (int)((tokens + tm - 1) / tm); p.tiles_n = (int)((F + half - 1) / half);
  p.group_m = p.tiles_m < 8 ? p.tiles_m : 8;               // 2048 rows of x stay in L2 while the weight panels stream
  p.idesc = ffn_idesc(bf16, 0, 0, 2 * half, tm);
  p.a_rows = pair || tokens >= 128 ? 128 : (int)((tokens + 7) / 8 * 8);
  p.out_tma = ffn_rows_aligned(h, F) && (!save || (ffn_rows_aligned(gate, F) && ffn_rows_aligned(up, F)));
  FfnMaps maps;
  rc = encode_operand(&maps.a[0], op[0], 1, 1, 64, p.a_rows, bf16);
  if (!rc) rc = encode_operand(&maps.b[0], op[1], 1, 1, 64, half, bf16);
  if (!rc) rc = encode_operand(&maps.b[1], op[2], 1, 1, 64, half, bf16);
  maps.a[1] = maps.ak[0] = maps.ak[1] = maps.a[0]; maps.b[2] = maps.b[0];
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
// dg and du, rows zero-padded from F to Fp = a multiple of 64 elements, so that no box of the products is partly out of range.
// One 16-byte vector of each a thread and trip; VEC: the inputs' rows are 16-byte aligned.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
ffn_adjoint_kernel(T* __restrict__ dG, T* __restrict__ dU, const T* __restrict__ dH, const T* __restrict__ G,
                   const T* __restrict__ U, unsigned nvec, unsigned F, unsigned vpr /* vectors per padded row */,
                   unsigned* __restrict__ next) {
  if (blockIdx.x == 0 && threadIdx.x == 0) *next = 0;           // the item counter of the products that follow
  for (unsigned i = blockIdx.x * blockDim.x + threadIdx.x; i < nvec; i += gridDim.x * blockDim.x) {
    const unsigned row = i / vpr, c = (i - row * vpr) * 8;
    float g[8], u[8], d[8];
    const long long src = (long long)row * F + c;
    if (VEC) {
      const bool in = c < F;
      const uint4 z = make_uint4(0, 0, 0, 0);
      unpack<T>(in ? ld_stream(G + src) : z, g);
      unpack<T>(in ? ld_stream(U + src) : z, u);
      unpack<T>(in ? ld_stream(dH + src) : z, d);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = c + e < F;
        g[e] = in ? Elem<T>::to_f32(G[src + e]) : 0.f;
        u[e] = in ? Elem<T>::to_f32(U[src + e]) : 0.f;
        d[e] = in ? Elem<T>::to_f32(dH[src + e]) : 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float s = sigmoid_f32(g[e]);
      const float dg = d[e] * u[e] * (s * (1.f + g[e] * (1.f - s)));
      u[e] = d[e] * (g[e] * s);
      g[e] = dg;
    }
    reinterpret_cast<uint4*>(dG)[i] = pack<T>(g);
    reinterpret_cast<uint4*>(dU)[i] = pack<T>(u);
  }
}

// The products of the adjoint.  pr[0]: dx, contraction over `parts` = 2 operand pairs of nkb k-blocks, cut into `splits`
// ranges; pr[1]: dWg and, `tiles` further on, dWu.
struct FfnProduct { GemmParams g; int nkb, tiles; };
struct FfnBwdParams {
  FfnProduct pr[2];
  int splits;                    // ranges of dx's contraction; 1: none, else partial sums go to `part`
  float* part;                   // [splits][M][N] f32
  int nx, total;                 // items of dx (tiles * splits), all items
  unsigned* next;                // items drawn so far beyond the workers' first ones
};

struct FfnItem { int prod, part, tm, tn, kb0, kb1, split; };
__device__ __forceinline__ FfnItem ffn_item(const FfnBwdParams& p, int t) {
  FfnItem it;
  it.split = 0; it.part = 0;
  if (t < p.nx) {
    it.prod = 0;
    const int tiles = p.pr[0].tiles, nk = 2 * p.pr[0].nkb;
    it.split = t / tiles;                // neighbours in time share a range of the contraction, and so operand panels
    t -= it.split * tiles;
    it.kb0 = (int)((long long)nk * it.split / p.splits);
    it.kb1 = (int)((long long)nk * (it.split + 1) / p.splits);
  } else {
    it.prod = 1;
    t -= p.nx;
    it.part = t / p.pr[1].tiles;
    t -= it.part * p.pr[1].tiles;
    it.kb0 = 0; it.kb1 = p.pr[1].nkb;
  }
  const GemmParams& g = p.pr[it.prod].g;
  ffn_decode(t, g.tiles_m, g.tiles_n, g.group_m, it.tm, it.tn);
  return it;
}

// Epilogues by rows: 64 accumulator columns at a time to f32 staging (one thread a row, 16-byte chunks placed by row so that neither
// side conflicts), then one row at a time to memory, consecutive lanes consecutive columns.  emit(row, column, value).
template <int BN, typename F>
__device__ __forceinline__ void ffn_tile_rows(int M, int N, uint32_t tmem_base, int acc, int row0, int tn, int q, int lane, unsigned char* mybuf,
                                              uint32_t tempty_addr, F&& emit) {
#pragma unroll 1
  for (int c = 0; c < BN / 64; ++c) {
    const int col0 = tn * BN + c * 64;
    if (col0 >= N) break;                // warp-uniform
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      uint32_t v[32];
      tc_ld32(tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + c * 64 + hh * 32), v);
      tc_ld_wait();
#pragma unroll
      for (int k = 0; k < 8; ++k)
        *reinterpret_cast<uint4*>(mybuf + lane * 256 + (((hh * 8 + k) ^ (lane & 15)) << 4)) = make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    }
    __syncwarp();
#pragma unroll 4
    for (int r = 0; r < 32; ++r) {
      if (row0 + r < M) {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int j = hh * 32 + lane;
          if (col0 + j < N)
            emit(row0 + r, col0 + j, *reinterpret_cast<const float*>(mybuf + r * 256 + (((j >> 2) ^ (r & 15)) << 4) + (j & 3) * 4));
        }
      }
    }
    __syncwarp();
  }
  // the staging's next writer may be a TMA load (the old values of an accumulating tile): after these ordinary accesses
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive_cluster(tempty_addr);
}

// The two-SM matmul kernel over the items of all three products.  A is dg / du, stored [tokens][Fp]: K-major for dx, MN-major
// for the weight gradients; B is MN-major throughout (weights [F][D], x [tokens][D]).
template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1)
ffn_bwd_kernel(const __grid_constant__ FfnMaps maps, T* __restrict__ dX, T* __restrict__ dWg, T* __restrict__ dWu,
               const __grid_constant__ FfnBwdParams p) {
  constexpr int BN = 256, HB = 128, STAGES = 6;
  constexpr uint32_t A_BYTES = kBM * kBK * 2, STAGE_BYTES = kFfnStageBytes;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + (size_t)STAGES * STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* cbar = tempty + 2;                  // one per epilogue warp: old C boxes have arrived
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(cbar + 4);
  SchedSmem* sched = reinterpret_cast<SchedSmem*>(tmem_slot + 4);
  unsigned char* cstage = tiles + (size_t)STAGES * STAGE_BYTES + 1024;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int worker = blockIdx.x >> 1, nworkers = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(tfull + a, 1); mbar_init(tempty + a, 8); }
    for (int w = 0; w < 4; ++w) mbar_init(cbar + w, 1);
    // schedule ring: in the leader read by the MMA thread and four epilogue warps (empty), in the peer by the producer
    // thread and four epilogue warps, which report to the leader's empty_peer
    for (int i = 0; i < kSchedDepth; ++i) { mbar_init(sched->full + i, 1); mbar_init(sched->empty + i, 5); mbar_init(sched->empty_peer + i, 5); }
    mbar_fence_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                           // the peer's barriers are initialised before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // the leader's barriers on which the peer CTA's consumers report their reads of the schedule ring
  const uint32_t leader_empty_peer0 = map_to_rank(smem_u32(sched->empty_peer), 0);

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    int s = 0; unsigned ph = 0;
    bool ok = true;
    const uint32_t full0 = map_to_rank(smem_u32(full), 0);
    unsigned sn = 0;
    int t = worker, nxt = -1;                   // the grid never has more workers than items
    for (;;) {
      if (rank == 0) {
        if (!sched_publish<true>(sched, sn, t)) { ok = false; break; }
        if (t < 0) break;
        const unsigned drawn = (unsigned)nworkers + atomicAdd(p.next, 1u);     // in flight while this item's loads are issued
        nxt = drawn < (unsigned)p.total ? (int)drawn : -1;
      } else {
        t = sched_take<true>(sched, sn, true, leader_empty_peer0);
        if (t < 0) { ok = t == -1; break; }
      }
      const FfnItem it = ffn_item(p, t);
      const FfnProduct& pr = p.pr[it.prod];
      // a last column tile with at most 128 columns runs as an N = 128 MMA: each CTA then supplies 64 rows of B
      const int hb = (pr.g.N - it.tn * BN <= HB) ? HB / 2 : HB;
      const int m0 = it.tm * 256 + (int)rank * kBM, n0 = it.tn * BN + (int)rank * hb;
      // one run of k-blocks of one operand pair (dx: the gate part, then the up part)
      auto run = [&](auto a_mn, const CUtensorMap* ma, const CUtensorMap* mb, int kb0, int kb1) {
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait_bounded(empty + s, ph ^ 1, kDevErrGemmTimeout)) { ok = false; return; }
          unsigned char* sa = tiles + (size_t)s * STAGE_BYTES;
          unsigned char* sb = sa + A_BYTES;
          const uint32_t fb = full0 + (uint32_t)s * 8u;
          if (rank == 0) mbar_expect_tx(full + s, 2 * STAGE_BYTES);
          if (a_mn) {
            tma_load_4d_pair(sa, ma, fb, m0, kb * kBK, 0, 0);
            tma_load_4d_pair(sa + 8192, ma, fb, m0 + 64, kb * kBK, 0, 0);
          } else {
            tma_load_4d_pair(sa, ma, fb, kb * kBK, m0, 0, 0);
          }
          tma_load_4d_pair(sb, mb, fb, n0, kb * kBK, 0, 0);
          tma_load_4d_pair(sb + 8192, mb, fb, n0 + 64, kb * kBK, 0, 0);
          if (++s == STAGES) { s = 0; ph ^= 1; }
        }
      };
      if (it.prod) {
        run(std::true_type{}, &maps.a[it.part], &maps.b[2], it.kb0, it.kb1);
      } else {
        const int mid = it.kb1 < pr.nkb ? it.kb1 : pr.nkb;
        run(std::false_type{}, &maps.ak[0], &maps.b[0], it.kb0, mid);
        if (ok) run(std::false_type{}, &maps.ak[1], &maps.b[1], it.kb0 > pr.nkb ? it.kb0 - pr.nkb : 0, it.kb1 - pr.nkb);
      }
      if (!ok) break;
      t = nxt;
    }
    // the leader's last commits still arrive on this CTA's empty barriers: wait for them before leaving
    for (int i = 0; ok && i < STAGES; ++i) {
      ok = mbar_wait_bounded(empty + s, ph ^ 1, kDevErrGemmTimeout);
      if (++s == STAGES) { s = 0; ph ^= 1; }
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ---------------- MMA issuer (leader CTA) ----------------
    int s = 0; unsigned ph = 0;
    int local = 0;
    bool ok = true;
    const uint32_t sa0 = smem_u32(tiles);
    const uint64_t desc_a[2] = {make_desc(sa0, 1, 64), make_desc(sa0, 512, 64)};      // K-major (dx), MN-major
    const uint64_t desc_b = make_desc(sa0 + A_BYTES, 512, 64);
    unsigned sn = 0;
    for (;; ++local) {
      const int t = sched_take<false>(sched, sn, true, 0);
      if (t < 0) break;
      const FfnItem it = ffn_item(p, t);
      const FfnProduct& pr = p.pr[it.prod];
      const uint32_t idesc = (pr.g.N - it.tn * BN <= HB) ? idesc_with_n(pr.g.idesc, HB) : pr.g.idesc;      // see the producer
      const int acc = local & 1;
      if (!mbar_wait_bounded(tempty + acc, (unsigned)((local >> 1) & 1) ^ 1, kDevErrGemmTimeout)) break;
      tc_fence_after();
      const uint32_t tacc = tmem_base + (uint32_t)acc * BN;
      auto run = [&](auto a_mn) {
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          if (!mbar_wait_bounded(full + s, ph, kDevErrGemmTimeout)) { ok = false; return; }
          tc_fence_after();
          // the address field of a descriptor counts 16 bytes: stages and k steps are additions to it
          const uint64_t da = desc_a[a_mn ? 1 : 0] + (uint64_t)(s * (STAGE_BYTES / 16)), db = desc_b + (uint64_t)(s * (STAGE_BYTES / 16));
#pragma unroll
          for (int k4 = 0; k4 < kBK / 16; ++k4)
            tc_mma_f16_pair(tacc, da + k4 * (a_mn ? 128 : 2), db + k4 * 128, idesc, (kb > it.kb0 || k4) ? 1u : 0u);
          tc_commit_pair(empty + s);
          if (++s == STAGES) { s = 0; ph ^= 1; }
        }
      };
      if (it.prod) run(std::true_type{});
      else run(std::false_type{});
      if (!ok) break;
      tc_commit_pair(tfull + acc);
    }
  } else if (warp >= 2) {
    // ---------------- epilogue (both CTAs, each on its own 128 rows) ----------------
    const int q = warp & 3;
    int local = 0;
    unsigned cpar = 0;                          // phase of this warp's old-C barrier
    unsigned sn = 0;
    for (;; ++local) {
      const int t = rank == 0 ? sched_take_warp<false>(sched, sn, lane, 0) : sched_take_warp<true>(sched, sn, lane, leader_empty_peer0);
      if (t < 0) break;
      const FfnItem it = ffn_item(p, t);
      const int acc = local & 1;
      if (!mbar_wait_bounded_warp(tfull + acc, (unsigned)((local >> 1) & 1), kDevErrGemmTimeout)) break;
      tc_fence_after();
      const int row0 = it.tm * 256 + (int)rank * kBM + q * 32;
      const uint32_t te = map_to_rank(smem_u32(tempty + acc), 0);
      const GemmParams& g = p.pr[it.prod].g;
      unsigned char* stage = cstage + (size_t)(warp - 2) * 8192;
      T* out = it.prod == 0 ? dX : it.part ? dWu : dWg;
      if ((it.prod == 0 && p.splits > 1) || !g.c_tma) {
        // a range's partial sums, or a result whose rows TMA cannot address
        float* part = it.prod == 0 && p.splits > 1 ? p.part + (long long)it.split * g.M * g.N : nullptr;
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");     // the staging has been read
        __syncwarp();
        ffn_tile_rows<BN>(g.M, g.N, tmem_base, acc, row0, it.tn, q, lane, stage, te, [&](int r, int j, float v) {
          const long long at = (long long)r * g.N + j;
          if (part) __stcg(part + at, v);
          else out[at] = Elem<T>::from_f32(g.beta != 0.f ? v + Elem<T>::to_f32(out[at]) : v);
        });
      } else {
        epilogue_tile<T, BN>(g, maps.c[it.prod + it.part], out, tmem_base, acc, row0, it.tn, 0, 0, q, lane, stage, te, cbar + (warp - 2), cpar);
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                           // both CTAs have finished reading TMEM and signalling each other
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  }
}
constexpr size_t kFfnBwdSmem = (size_t)6 * kFfnStageBytes + 1024 + 1024 + 4 * 8192;

// dx = T(sum of the ranges' partial sums in order + beta * old)
template <typename T>
__global__ void __launch_bounds__(256)
ffn_join_kernel(T* __restrict__ out, const float* __restrict__ part, long long n, int splits, int beta) {
  dependent_wait();
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
    float v = 0.f;
    for (int s = 0; s < splits; ++s) v += __ldcg(part + (long long)s * n + i);
    if (beta) v += Elem<T>::to_f32(out[i]);
    out[i] = Elem<T>::from_f32(v);
  }
}

// What a backward call does, from its sizes alone.
struct FfnBwdPlan { int64_t Fp; size_t dpart, part; int tiles_x, tiles_w, nkb_x, nkb_w, splits, workers; };
static FfnBwdPlan ffn_bwd_plan(int64_t T, int64_t D, int64_t F) {
  FfnBwdPlan b;
  b.Fp = packed_cols(F);
  b.dpart = ((size_t)T * b.Fp * 2 + 255) / 256 * 256;
  const int64_t tn = (D + 255) / 256;
  const int64_t tx = (T + 255) / 256 * tn, tw = (F + 255) / 256 * tn;
  b.tiles_x = (int)tx; b.tiles_w = (int)tw;
  b.nkb_x = (int)(b.Fp / kBK); b.nkb_w = (int)((T + kBK - 1) / kBK);
  const int64_t W = kNumSMs / 2;
  // dx's contraction is cut when one of its tiles would last longer than a worker's share of all the work (few tokens:
  // few tiles, each 2 F deep); ranges of at least 8 k-blocks
  const int64_t work = tx * 2 * b.nkb_x + 2 * tw * b.nkb_w, share = (work + W - 1) / W;
  int64_t s = (2 * b.nkb_x + share - 1) / share;
  if (s > 2 * b.nkb_x / 8) s = 2 * b.nkb_x / 8;
  if (s > 16) s = 16;
  if (s < 1) s = 1;
  b.splits = (int)s;
  b.part = s > 1 ? ((size_t)s * T * D * 4 + 255) / 256 * 256 : 0;
  const int64_t items = tx * s + 2 * tw;
  b.workers = (int)(items < W ? items : W);
  return b;
}

static int ffn_result(FfnProduct& pr, CUtensorMap* map, uint64_t c, int64_t M, int64_t N, int a_mn, int nkb, int beta, bool bf16) {
  GemmParams& g = pr.g;
  g = GemmParams{};
  g.M = (int)M; g.N = (int)N;
  g.nb_inner = g.nb_outer = 1;
  g.tiles_m = (int)((M + 255) / 256); g.tiles_n = (int)((N + 255) / 256);
  g.ldc = N; g.alpha = 1.f; g.beta = beta ? 1.f : 0.f;
  g.idesc = ffn_idesc(bf16, a_mn, 1, 256, 256);
  const uint64_t all = c | (uint64_t)(N * 2);
  g.c_align = (all & 15) == 0 ? 16 : (all & 7) == 0 ? 8 : (all & 3) == 0 ? 4 : 2;
  g.group_m = g.tiles_m < 8 ? g.tiles_m : 8;
  pr.nkb = nkb; pr.tiles = g.tiles_m * g.tiles_n;
  g.c_tma = (all & 15) == 0;
  return g.c_tma ? encode_operand(map, Operand{c, M, N, N, 0, 0, 0, 0}, 1, 1, 64, 32, bf16) : CACTI_B200_OK;
}

template <typename T>
static int ffn_bwd_run(uint64_t dx, uint64_t dwg, uint64_t dwu, uint64_t dh, uint64_t x, uint64_t wg, uint64_t wu, uint64_t gate,
                       uint64_t up, int64_t tokens, int64_t D, int64_t F, int beta_dx, int beta_dw, uint64_t ws, size_t ws_bytes,
                       cudaStream_t st) {
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  const FfnBwdPlan b = ffn_bwd_plan(tokens, D, F);
  // workspace: item counter | dg | du | dx's partial sums | repacked operands
  const uint64_t dg = ws + 256;
  unsigned* counter = reinterpret_cast<unsigned*>(ws);
  size_t off = 256 + 2 * b.dpart + b.part;
  if (!ws || (ws & 255) || ws_bytes < off) return CACTI_B200_ERR_WORKSPACE;
  Operand op[3];
  for (const auto& [ptr, rows] : {std::pair<uint64_t, int64_t>{x, tokens}, {wg, F}, {wu, F}}) {     // before anything is launched
    if (!ffn_rows_aligned(ptr, D)) off += packed_bytes(rows, D, 1);
  }
  if (ws_bytes < off) return CACTI_B200_ERR_WORKSPACE;
  const uint64_t tok = 2ull * tokens * D, act = 2ull * tokens * F, wts = 2ull * F * D;
  if (!ffn_separate({{dx, tok}, {dwg, wts}, {dwu, wts}}, {{dh, act}, {x, tok}, {wg, wts}, {wu, wts}, {gate, act}, {up, act}}))
    return CACTI_B200_ERR_INVALID_VALUE;
  off = 256 + 2 * b.dpart + b.part;
  const unsigned vpr = (unsigned)(b.Fp / 8), nvec = (unsigned)(tokens * vpr);
  const unsigned want = (nvec + 255) / 256, cap = kNumSMs * 32;
  const bool vec = ffn_rows_aligned(dh, F) && ffn_rows_aligned(gate, F) && ffn_rows_aligned(up, F);
  auto adj = vec ? ffn_adjoint_kernel<T, true> : ffn_adjoint_kernel<T, false>;
  adj<<<want < cap ? want : cap, 256, 0, st>>>(reinterpret_cast<T*>(dg), reinterpret_cast<T*>(dg + b.dpart),
                                               reinterpret_cast<const T*>(dh), reinterpret_cast<const T*>(gate),
                                               reinterpret_cast<const T*>(up), nvec, (unsigned)F, vpr, counter);
  int rc = check_launch();
  if (!rc) rc = ffn_operands(op, {x, wg, wu}, {tokens, F, F}, D, ws, ws_bytes, off, st);
  if (rc) return rc;
  FfnMaps maps;
  for (int i = 0; i < 2 && !rc; ++i) {
    const Operand o{dg + i * b.dpart, tokens, b.Fp, b.Fp, 0, 0, 0, 0};
    rc = encode_operand(&maps.a[i], o, 1, 1, 64, 64, bf16);
    if (!rc) rc = encode_operand(&maps.ak[i], o, 1, 1, 64, kBM, bf16);
  }
  if (!rc) rc = encode_operand(&maps.b[0], op[1], 1, 1, 64, 64, bf16);
  if (!rc) rc = encode_operand(&maps.b[1], op[2], 1, 1, 64, 64, bf16);
  if (!rc) rc = encode_operand(&maps.b[2], op[0], 1, 1, 64, 64, bf16);
  if (rc) return rc;
  for (auto& m : maps.c) m = maps.a[0];
  FfnBwdParams p;
  rc = ffn_result(p.pr[0], &maps.c[0], dx, tokens, D, 0, b.nkb_x, beta_dx, bf16);
  if (!rc) rc = ffn_result(p.pr[1], &maps.c[1], dwg, F, D, 1, b.nkb_w, beta_dw, bf16);
  if (rc) return rc;
  FfnProduct up_pr;                             // the up half differs from the gate half in its result's map and alignment only
  rc = ffn_result(up_pr, &maps.c[2], dwu, F, D, 1, b.nkb_w, beta_dw, bf16);
  if (rc) return rc;
  if (up_pr.g.c_align < p.pr[1].g.c_align) p.pr[1].g.c_align = up_pr.g.c_align;
  p.pr[1].g.c_tma &= up_pr.g.c_tma;
  p.splits = b.splits;
  p.part = reinterpret_cast<float*>(dg + 2 * b.dpart);
  p.nx = b.tiles_x * b.splits;
  p.total = p.nx + 2 * b.tiles_w;
  p.next = counter;
  auto kern = ffn_bwd_kernel<T>;
  static bool attr_set[kMaxDevices] = {};
  ensure_dynamic_smem(kern, kFfnBwdSmem, attr_set);
  kern<<<(unsigned)(2 * b.workers), kGemmThreads, kFfnBwdSmem, st>>>(maps, reinterpret_cast<T*>(dx), reinterpret_cast<T*>(dwg),
                                                                     reinterpret_cast<T*>(dwu), p);
  rc = check_launch();
  if (!rc && b.splits > 1) {
    const long long n = (long long)tokens * D, blocks = (n + 255) / 256;
    launch_dependent(ffn_join_kernel<T>, (unsigned)(blocks < kNumSMs * 8 ? blocks : kNumSMs * 8), 256u, st, reinterpret_cast<T*>(dx),
                     (const float*)p.part, n, b.splits, beta_dx);
    rc = check_launch();
  }
  return rc;
}

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
  if (!ffn_sizes_ok(tokens, d_model, d_ffn)) return CACTI_B200_ERR_SHAPE;
  if (tokens == 0) return CACTI_B200_OK;
  if (!h || !x || !w_gate || !w_up || !gate != !up) return CACTI_B200_ERR_INVALID_VALUE;
  if ((h | gate | up | x | w_gate | w_up) & 1) return CACTI_B200_ERR_INVALID_VALUE;
  if (!ffn_pack_ok({x, w_gate, w_up}, {tokens, d_ffn, d_ffn}, d_model)) return CACTI_B200_ERR_SHAPE;
  const uint64_t act = 2ull * tokens * d_ffn, wts = 2ull * d_ffn * d_model;
  if (!ffn_separate({{h, act}, {gate, act}, {up, act}}, {{x, 2ull * tokens * d_model}, {w_gate, wts}, {w_up, wts}}))
    return CACTI_B200_ERR_INVALID_VALUE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == CACTI_B200_R_16F)
    return ffn_fwd_run<__half>(h, gate, up, x, w_gate, w_up, tokens, d_model, d_ffn, workspace, workspace_bytes, st);
  return ffn_fwd_run<__nv_bfloat16>(h, gate, up, x, w_gate, w_up, tokens, d_model, d_ffn, workspace, workspace_bytes, st);
}

size_t cacti_b200_gated_ffn_bwd_workspace_bytes(int64_t tokens, int64_t d_model, int64_t d_ffn, int aligned) {
  if (tokens < 0 || d_model < 0 || d_ffn < 0) return 0;
  if (tokens == 0 || d_model == 0 || d_ffn == 0) return 256;
  const cb::FfnBwdPlan b = cb::ffn_bwd_plan(tokens, d_model, d_ffn);
  size_t n = 2 * b.dpart + b.part + 256;
  if (!aligned || d_model % 8) n += cb::packed_bytes(tokens, d_model, 1) + 2 * cb::packed_bytes(d_ffn, d_model, 1);
  return n;
}

int cacti_b200_gated_ffn_bwd(cacti_b200_dptr dx, cacti_b200_dptr dw_gate, cacti_b200_dptr dw_up, cacti_b200_dptr dh,
                             cacti_b200_dptr x, cacti_b200_dptr w_gate, cacti_b200_dptr w_up, cacti_b200_dptr gate,
                             cacti_b200_dptr up, int64_t tokens, int64_t d_model, int64_t d_ffn, int dtype, int beta_dx,
                             int beta_dw, cacti_b200_dptr workspace, size_t workspace_bytes, cacti_b200_stream stream) {
  using namespace cb;
  if (tokens < 0 || d_model < 0 || d_ffn < 0 || ((beta_dx | beta_dw) & ~1)) return CACTI_B200_ERR_INVALID_VALUE;
  if (dtype != CACTI_B200_R_16F && dtype != CACTI_B200_R_16BF) return CACTI_B200_ERR_DTYPE;
  if (!ffn_sizes_ok(tokens, d_model, d_ffn)) return CACTI_B200_ERR_SHAPE;
  if (!dw_gate || !dw_up) return CACTI_B200_ERR_INVALID_VALUE;
  if (tokens > 0 && (!dx || !dh || !x || !w_gate || !w_up || !gate || !up)) return CACTI_B200_ERR_INVALID_VALUE;
  if ((dx | dw_gate | dw_up | dh | x | w_gate | w_up | gate | up) & 1) return CACTI_B200_ERR_INVALID_VALUE;
  if (!ffn_pack_ok({x, w_gate, w_up}, {tokens, d_ffn, d_ffn}, d_model)) return CACTI_B200_ERR_SHAPE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (tokens == 0) {                                            // an empty sum: the weight gradients are zero
    if (!beta_dw)
      for (uint64_t w : {dw_gate, dw_up})
        if (cudaMemsetAsync(reinterpret_cast<void*>(w), 0, (size_t)d_ffn * d_model * 2, st) != cudaSuccess) return check_launch();
    return CACTI_B200_OK;
  }
  if (dtype == CACTI_B200_R_16F)
    return ffn_bwd_run<__half>(dx, dw_gate, dw_up, dh, x, w_gate, w_up, gate, up, tokens, d_model, d_ffn, beta_dx, beta_dw, workspace,
                               workspace_bytes, st);
  return ffn_bwd_run<__nv_bfloat16>(dx, dw_gate, dw_up, dh, x, w_gate, w_up, gate, up, tokens, d_model, d_ffn, beta_dx, beta_dw,
                                    workspace, workspace_bytes, st);
}
}
