// What the tensor-core matmul kernels share: parameters, tile order, the epilogue, two-SM (cta_group::2) helpers, operand
// descriptions, their tensor maps and the repacking of operands that TMA cannot address.
#pragma once
#include "tc_common.cuh"
#include <atomic>
#include <type_traits>

namespace cb {

constexpr int kBM = 128, kBK = 64;
constexpr int kGemmThreads = 192;

struct GemmParams {
  int M, N, K;
  int nb_inner, nb_outer;                 // block grid: j (inner) and i (outer)
  int tiles_m, tiles_n;
  int a_j, a_i, b_j, b_i;                 // 1: operand has that block dimension, 0: broadcast
  long long ldc, c_stride_inner, c_stride_outer;
  float alpha, beta;
  uint32_t idesc;
  int c_align;                            // bytes every output row chunk is aligned to: 16, 8, 4 or 2
  int c_tma;                              // 1: C is written with TMA stores from a swizzled staging buffer
  int group_m;                            // tile rasterisation: m-tiles per group (L2 reuse of the B panel)
  int tri, diag;                          // triangular-structure hint (CACTI_B200_TRI_*) and its diagonal offset
  // k-split schedule of the two-SM kernel (see WorkIter); sk_tiles == 0: every tile is computed whole
  long long sk_tiles, sk_units;           // tiles [0, sk_tiles) are shared out in k-blocks: sk_units = sk_tiles * k-blocks
  float* sk_part;                         // [workers][2 CTAs][256 columns][128 rows] f32 partial accumulators
  int sk_slot;                            // which row of g_sk_flags this launch signals through
  int dyn;                                // 1: tiles beyond a worker's first come from g_tile_next[sk_slot] (dynamic schedule)
};

enum { kItemFull = 0, kItemContrib = 1, kItemOwner = 2 };
constexpr unsigned kDevErrGemmSplitTimeout = 4u;
constexpr size_t kSkPartFloats = 256 * 128;         // per (worker, CTA of the pair)
__device__ __forceinline__ unsigned long long global_timer_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Lane 0 polls the flag (acquire) for at most about a second; the whole warp gets the same answer.
__device__ __forceinline__ bool sk_wait_flag(const unsigned* flag, int lane) {
  unsigned ok = 1;
  if (lane == 0) {
    ok = 0;
    const unsigned long long t0 = global_timer_ns();
    for (unsigned it = 1;; ++it) {
      unsigned v;
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(flag) : "memory");
      if (v) { ok = 1; break; }
      __nanosleep(100);
      if ((it & 255u) == 0 && global_timer_ns() - t0 > 1000000000ull) break;
    }
    if (!ok) atomicMax(&g_dev_error, kDevErrGemmSplitTimeout);
  }
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

// What the epilogue does with one accumulator (two-SM kernel).
struct SkEpi {
  int kind;                 // kItemFull: normal epilogue; kItemContrib: store the accumulator; kItemOwner: add, then normal
  float* my_part;           // contribution: this CTA's slot
  unsigned* my_flags;       // contribution: this CTA's four flags (one per epilogue warp)
  const float* part0;       // owner: slot of the first contributor (the next worker), same CTA rank; next worker 2 slots on
  unsigned* flags0;         // owner: flags of the first contributor; next worker 8 words on
  int ncontrib;
};

// Tile order inside one block: groups of `group_m` m-tiles; inside a group the m index runs fastest, so
// the CTAs that run at the same time share a few B (weight) panels and a bounded set of A rows in L2.
__device__ __forceinline__ void decode_tile(long long tile, long long tiles_per_block, const GemmParams& p, int& blk,
                                            int& tm, int& tn) {
  blk = (int)(tile / tiles_per_block);
  const int r = (int)(tile - (long long)blk * tiles_per_block);
  const int per_group = p.group_m * p.tiles_n;
  const int grp = r / per_group, in = r - grp * per_group;
  const int m0 = grp * p.group_m;
  const int gm = p.tiles_m - m0 < p.group_m ? p.tiles_m - m0 : p.group_m;
  tn = in / gm;
  tm = m0 + (in - tn * gm);
  // With a triangular hint the work of a tile depends on tm; rotating tm by the block index makes the tiles a
  // CTA meets (tile, tile + grid, ...) run through all row positions instead of a few residues.
  if (p.tri) tm = (tm + blk) % p.tiles_m;
}

// Instruction descriptor with the N extent replaced (edge tiles issue narrower MMAs instead of multiplying zeros).
__device__ __forceinline__ uint32_t idesc_with_n(uint32_t idesc, int n) {
  return (idesc & ~(0x3Fu << 17)) | ((uint32_t)(n >> 3) << 17);
}

// Triangular hints, per output tile whose rows are [row0, row0 + rows) and whose first column is col0.
//   C_LOWER: only C[r, c] with c <= r + diag is wanted; a tile wholly beyond that is skipped (not written).
//   A_LOWER: op(A)[r, k] == 0 for k > r + diag; k-blocks wholly beyond the tile's last row are skipped.
//   A_UPPER: op(A)[r, k] == 0 for k < r - diag; k-blocks wholly before the tile's first row are skipped.
// Skipped products are exact zeros, so the result is bit-identical to the full computation.
__device__ __forceinline__ bool tile_skipped(const GemmParams& p, int row0, int rows, int col0) {
  return p.tri == CACTI_B200_TRI_C_LOWER && (long long)col0 > (long long)row0 + rows - 1 + p.diag;
}
__device__ __forceinline__ void k_block_range(const GemmParams& p, int row0, int rows, int nkb, int& kb0, int& kb1) {
  kb0 = 0; kb1 = nkb;
  if (p.tri == CACTI_B200_TRI_A_LOWER) {
    const long long last = (long long)row0 + rows - 1 + p.diag;
    const long long e = last < 0 ? 1 : last / kBK + 1;
    kb1 = e < 1 ? 1 : (e < nkb ? (int)e : nkb);
  } else if (p.tri == CACTI_B200_TRI_A_UPPER) {
    const long long first = (long long)row0 - p.diag;
    const long long b = first < 0 ? 0 : first / kBK;
    kb0 = b > nkb - 1 ? nkb - 1 : (int)b;
  }
}

// Epilogue of one accumulator for one warp: TMEM lanes [q*32, q*32+32) x BN columns of accumulator `acc` become
// rows row0 .. row0+31 of the output tile whose first column is tn * BN.  `tempty_addr` is the shared::cluster
// address of the barrier that frees the accumulator: the warp arrives on it once, as soon as its last
// tcgen05.ld has completed.  `cbar` / `cpar`: this warp's barrier and phase for the TMA loads that bring the old
// C boxes into the staging buffers when beta != 0 (Accumulate mode, src/thunk/mod.rs:347-351).
template <typename T, int BN>
__device__ __forceinline__ void epilogue_tile(const GemmParams& p, const CUtensorMap& tmC, T* __restrict__ C,
                                              uint32_t tmem_base, int acc, int row0, int tn, int bj, int bi, int q, int lane,
                                              unsigned char* mybuf, uint32_t tempty_addr, uint64_t* cbar, unsigned& cpar,
                                              const SkEpi sk = SkEpi{}) {
  const int prow = q * 32 + lane;             // this thread's row inside its CTA's 128 rows (partial-slot index)
  if (sk.kind == kItemContrib) {
    // this CTA's piece of a tile another worker owns: accumulator -> f32 slot (column-major, so a warp's stores of
    // one column are 128 contiguous bytes), then the flag
#pragma unroll 1
    for (int c = 0; c < BN / 64; ++c) {
      if (tn * BN + c * 64 >= p.N) break;
      uint32_t v[2][32];
      tc_ld32(tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + c * 64), v[0]);
      tc_ld32(tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + c * 64 + 32), v[1]);
      tc_ld_wait();
      float* dst = sk.my_part + (size_t)(c * 64) * kBM + prow;
#pragma unroll
      for (int i = 0; i < 64; ++i) __stcg(dst + (size_t)i * kBM, __uint_as_float(v[i >> 5][i & 31]));
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive_cluster(tempty_addr);
    __threadfence();
    __syncwarp();
    if (lane == 0) asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(sk.my_flags + q), "r"(1u) : "memory");
    return;
  }
  if (sk.kind == kItemOwner) {
    // the contributions were computed first by their workers; a wait that runs out is recorded and the tile is
    // finished with what is there (the device error word tells the caller the result is void)
    for (int ci = 0; ci < sk.ncontrib; ++ci) sk_wait_flag(sk.flags0 + ci * 8 + q, lane);
  }
  if (p.c_tma) {
    // TMEM -> registers -> swizzled shared staging -> TMA store (clips rows/columns past M, N)
    // 128 accumulator columns per trip: four tcgen05.ld in flight, one wait, two 64-column TMA stores
    const bool scale = p.alpha != 1.f;
    const bool accum = p.beta != 0.f;
    constexpr int TRIPS = (BN + 127) / 128;
#pragma unroll 1
    for (int c = 0; c < TRIPS; ++c) {
      const int col0 = tn * BN + c * 128;
      if (col0 >= p.N) break;               // warp-uniform
      const int ncols = BN - c * 128 < 128 ? BN - c * 128 : 128;      // columns of this tile in this trip (128 or 64)
      uint32_t v[4][32];
#pragma unroll
      for (int hh = 0; hh < 4; ++hh)
        if (hh * 32 < ncols)
          tc_ld32(tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + c * 128 + hh * 32), v[hh]);
      // both staging buffers must have been read by the stores of the previous trip
      if (lane == 0) {
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        if (accum) {
          // old C: the same boxes the stores below write, into the same (swizzled) places of the staging buffers;
          // rows and columns past M, N arrive as zeros and are clipped again by the store
          const bool two = col0 + 64 < p.N && ncols > 64;
          mbar_expect_tx(cbar, two ? 8192u : 4096u);
          tma_load_4d(mybuf, &tmC, cbar, col0, row0, bj, bi);
          if (two) tma_load_4d(mybuf + 4096, &tmC, cbar, col0 + 64, row0, bj, bi);
        }
      }
      tc_ld_wait();
      if (c == TRIPS - 1 || col0 + 128 >= p.N) {         // last trip of this tile: the accumulator is free
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(tempty_addr);
      } else {
        __syncwarp();
      }
      if (sk.kind == kItemOwner) {                       // + the other workers' pieces, in increasing k
        for (int ci = 0; ci < sk.ncontrib; ++ci) {
          const float* src = sk.part0 + (size_t)ci * 2 * kSkPartFloats + (size_t)(c * 128) * kBM + prow;
#pragma unroll
          for (int hh = 0; hh < 4; ++hh) {
            if (hh * 32 < ncols && col0 + hh * 32 < p.N) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                v[hh][i] = __float_as_uint(__uint_as_float(v[hh][i]) + __ldcg(src + (size_t)(hh * 32 + i) * kBM));
            }
          }
        }
      }
      if (accum) {
        // the warp decides together: a wait that ran out leaves the tile unwritten (device error word set)
        const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(cbar, cpar, kDevErrGemmTimeout));
        cpar ^= 1u;
        if (!ok) return;
      }
#pragma unroll
      for (int hb = 0; hb < 2; ++hb) {
        if (hb * 64 >= ncols) break;
        unsigned char* buf = mybuf + hb * 4096;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float t8[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float a = __uint_as_float(v[hb * 2 + hh][g * 8 + i]);
              t8[i] = scale ? p.alpha * a : a;
            }
            const int chunk = hh * 4 + g;       // 16-byte chunk inside the 128-byte row
            uint4* slot = reinterpret_cast<uint4*>(buf + lane * 128 + ((chunk ^ (lane & 7)) << 4));
            if (accum && (hb == 0 || col0 + 64 < p.N)) {
              float o8[8];
              unpack<T>(*slot, o8);
#pragma unroll
              for (int i = 0; i < 8; ++i) t8[i] = fmaf(p.beta, o8[i], t8[i]);
            }
            *slot = pack<T>(t8);
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        tma_store_4d(&tmC, mybuf, col0, row0, bj, bi);
        if (col0 + 64 < p.N && ncols > 64) tma_store_4d(&tmC, mybuf + 4096, col0 + 64, row0, bj, bi);
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    }
    if (sk.kind == kItemOwner && lane == 0)
      for (int ci = 0; ci < sk.ncontrib; ++ci) sk.flags0[ci * 8 + q] = 0;       // ready for the next launch
    return;                                   // the accumulator was released inside the loop
  }
  const int row = row0 + lane;
  T* crow = C + (long long)bi * p.c_stride_outer + (long long)bj * p.c_stride_inner + (long long)row * p.ldc;
#pragma unroll 1
  for (int c = 0; c < BN / 32; ++c) {
    const int col0 = tn * BN + c * 32;
    if (col0 >= p.N) break;               // warp-uniform
    uint32_t v[32];
    tc_ld32(tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + c * 32), v);
    tc_ld_wait();
    if (sk.kind == kItemOwner) {
      for (int ci = 0; ci < sk.ncontrib; ++ci) {
        const float* src = sk.part0 + (size_t)ci * 2 * kSkPartFloats + (size_t)(c * 32) * kBM + prow;
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) + __ldcg(src + (size_t)i * kBM));
      }
    }
    if (row < p.M) {
      float f[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) f[i] = p.alpha * __uint_as_float(v[i]);
      const int nvalid = p.N - col0 < 32 ? p.N - col0 : 32;
      T* out = crow + col0;
      if (p.beta != 0.f) {
#pragma unroll
        for (int i = 0; i < 32; ++i) if (i < nvalid) f[i] = fmaf(p.beta, Elem<T>::to_f32(out[i]), f[i]);
      }
      if (nvalid == 32 && p.c_align >= 16) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float t8[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) t8[i] = f[g * 8 + i];
          *reinterpret_cast<uint4*>(out + g * 8) = pack<T>(t8);
        }
      } else if (p.c_align >= 8) {
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          if (g * 4 + 4 <= nvalid) {
            uint2 w;
            if constexpr (std::is_same<T, __half>::value) {
              __half2 a = __floats2half2_rn(f[g * 4], f[g * 4 + 1]), b = __floats2half2_rn(f[g * 4 + 2], f[g * 4 + 3]);
              w.x = *reinterpret_cast<uint32_t*>(&a); w.y = *reinterpret_cast<uint32_t*>(&b);
            } else {
              __nv_bfloat162 a = __floats2bfloat162_rn(f[g * 4], f[g * 4 + 1]), b = __floats2bfloat162_rn(f[g * 4 + 2], f[g * 4 + 3]);
              w.x = *reinterpret_cast<uint32_t*>(&a); w.y = *reinterpret_cast<uint32_t*>(&b);
            }
            *reinterpret_cast<uint2*>(out + g * 4) = w;
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) if (g * 4 + i < nvalid) out[g * 4 + i] = Elem<T>::from_f32(f[g * 4 + i]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) if (i < nvalid) out[i] = Elem<T>::from_f32(f[i]);
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive_cluster(tempty_addr);
  if (sk.kind == kItemOwner && lane == 0)
    for (int ci = 0; ci < sk.ncontrib; ++ci) sk.flags0[ci * 8 + q] = 0;
}

__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void tma_load_4d_pair(void* dst, const CUtensorMap* map, uint32_t bar_addr, int c0, int c1, int c2,
                                                 int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(bar_addr), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tc_commit_pair(uint64_t* bar) {       // arrives on `bar` in both CTAs of the pair
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(smem_u32(bar)), "h"((unsigned short)3)
               : "memory");
}
__device__ __forceinline__ void tc_mma_f16_pair(uint32_t tmem_c, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_c), "l"(da), "l"(db), "r"(idesc), "r"(accum)
      : "memory");
}

// Ring through which the thread that draws a dynamic schedule's tiles hands them to the other roles.
constexpr int kSchedDepth = 4;
struct SchedSmem {
  uint64_t full[kSchedDepth];          // an entry has been published (1 arrival: the scheduling thread)
  uint64_t empty[kSchedDepth];         // this CTA's consumers have read it
  uint64_t empty_peer[kSchedDepth];    // two-SM kernel, leader only: the peer CTA's consumers have read theirs
  int ring[kSchedDepth];
};

__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, unsigned parity) {   // acquire at cluster scope
  unsigned ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(g_mbar_suspend_ns) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_bounded_cluster(uint64_t* bar, unsigned parity, unsigned err_code) {
  for (unsigned it = 0; it < kMbarPolls; ++it)
    if (mbar_try_wait_cluster(bar, parity)) return true;
  atomicMax(&g_dev_error, err_code);
  return false;
}
// Consumer side of the ring for one thread (n: entries read so far).  Returns the tile, -1 at the end of the walk, -2
// when the wait ran out.  `arrive`: this thread reports the read (one thread per consuming warp does).
// CLUSTER: the entry was written by the other CTA of the pair, and the read is reported to that CTA's barrier.
template <bool CLUSTER>
__device__ __forceinline__ int sched_take(SchedSmem* sm, unsigned& n, bool arrive, uint32_t leader_empty_peer0) {
  const int sl = (int)(n % kSchedDepth);
  const unsigned ph = (n / kSchedDepth) & 1u;
  const bool ok = CLUSTER ? mbar_wait_bounded_cluster(sm->full + sl, ph, kDevErrGemmTimeout)
                          : mbar_wait_bounded(sm->full + sl, ph, kDevErrGemmTimeout);
  if (!ok) return -2;
  const int tile = *reinterpret_cast<volatile int*>(&sm->ring[sl]);
  if (arrive) {
    if (CLUSTER) mbar_arrive_cluster(leader_empty_peer0 + (uint32_t)sl * 8u);
    else mbar_arrive(sm->empty + sl);
  }
  ++n;
  return tile;
}
// The same for a whole warp (all lanes get the tile; lane 0 reports the read after every lane has it).
template <bool CLUSTER>
__device__ __forceinline__ int sched_take_warp(SchedSmem* sm, unsigned& n, int lane, uint32_t leader_empty_peer0) {
  const int sl = (int)(n % kSchedDepth);
  const unsigned ph = (n / kSchedDepth) & 1u;
  const bool ok = CLUSTER ? mbar_wait_bounded_cluster(sm->full + sl, ph, kDevErrGemmTimeout)
                          : mbar_wait_bounded(sm->full + sl, ph, kDevErrGemmTimeout);
  if (!__all_sync(0xffffffffu, ok)) return -2;
  const int tile = *reinterpret_cast<volatile int*>(&sm->ring[sl]);
  __syncwarp();
  if (lane == 0) {
    if (CLUSTER) mbar_arrive_cluster(leader_empty_peer0 + (uint32_t)sl * 8u);
    else mbar_arrive(sm->empty + sl);
  }
  ++n;
  return tile;
}
// Scheduling thread: publish `tile` (or -1) as entry n.  PAIR: also into the peer CTA's ring.
template <bool PAIR>
__device__ __forceinline__ bool sched_publish(SchedSmem* sm, unsigned& n, int tile) {
  const int sl = (int)(n % kSchedDepth);
  const unsigned ph = (n / kSchedDepth) & 1u;
  if (!mbar_wait_bounded(sm->empty + sl, ph ^ 1u, kDevErrGemmTimeout)) return false;
  if (PAIR && !mbar_wait_bounded_cluster(sm->empty_peer + sl, ph ^ 1u, kDevErrGemmTimeout)) return false;
  sm->ring[sl] = tile;
  mbar_arrive(sm->full + sl);                                  // release: the entry is visible to who sees the arrival
  if (PAIR) {
    uint32_t peer_ring, peer_full;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer_ring) : "r"(smem_u32(&sm->ring[sl])), "r"(1u));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer_full) : "r"(smem_u32(sm->full + sl)), "r"(1u));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_ring), "r"((uint32_t)tile) : "memory");
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(peer_full) : "memory");
  }
  ++n;
  return true;
}
// Repack blocks [nbo][nbi] of a stored matrix [rows x cols] (leading dimension ld, block strides so/si)
// into a dense [nbo*nbi][rows][cols_pad] buffer, zero-filling the padding columns.  One thread per unit of
// UNIT bytes (8 when every row start is 8-byte aligned and cols % 4 == 0, else 4 or 2); consecutive threads
// take consecutive units of a row, so both sides are coalesced.
template <typename U>
__global__ void __launch_bounds__(256)
pack_blocks_kernel(U* __restrict__ dst, const U* __restrict__ src, unsigned rows, unsigned upr_src /* units per source row */,
                   unsigned upr_dst, long long ld_units, unsigned nbi, long long so_units, long long si_units,
                   long long total_units) {
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total_units; i += (long long)gridDim.x * blockDim.x) {
    const long long t = i / upr_dst;                      // destination row
    const unsigned c = (unsigned)(i - t * upr_dst);
    const unsigned blk = (unsigned)(t / rows);
    const unsigned r = (unsigned)(t - (long long)blk * rows);
    const unsigned bo = blk / nbi, bi = blk - bo * nbi;
    U v{};
    if (c < upr_src) v = src[bo * so_units + bi * si_units + (long long)r * ld_units + c];
    dst[i] = v;
  }
}

// One operand as stored: `rows` x `cols` elements, cols contiguous, leading dimension ld, block strides.
struct Operand {
  uint64_t ptr; long long rows, cols, ld, stride_inner, stride_outer; int has_j, has_i;
  long long map_cols = 0;     // inner extent given to the tensor map (0: cols); > cols for zero-padded repacked operands
};

static bool tma_ok(const Operand& o, int nbi, int nbo) {
  if (o.ptr & 15) return false;
  if ((o.ld * 2) & 15) return false;
  if (o.has_j && nbi > 1 && ((o.stride_inner * 2) & 15)) return false;
  if (o.has_i && nbo > 1 && ((o.stride_outer * 2) & 15)) return false;
  return true;
}

static int encode_operand(CUtensorMap* map, const Operand& o, int nbi, int nbo, int box_inner, int box_outer, bool bf16) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return CACTI_B200_ERR_LAUNCH;
  const cuuint64_t dj = (o.has_j && nbi > 1) ? (cuuint64_t)nbi : 1, di = (o.has_i && nbo > 1) ? (cuuint64_t)nbo : 1;
  cuuint64_t dims[4] = {(cuuint64_t)(o.map_cols ? o.map_cols : o.cols), (cuuint64_t)o.rows, dj, di};
  const cuuint64_t row_bytes = (cuuint64_t)o.ld * 2;
  const cuuint64_t dflt = row_bytes * (cuuint64_t)o.rows;      // any legal value for an extent-1 dimension
  cuuint64_t strides[3] = {row_bytes, dj > 1 ? (cuuint64_t)o.stride_inner * 2 : dflt,
                           di > 1 ? (cuuint64_t)o.stride_outer * 2 : dflt};
  cuuint32_t box[4] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                  reinterpret_cast<void*>(o.ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { g_last_cuda_error = (int)r; return CACTI_B200_ERR_LAUNCH; }
  return CACTI_B200_OK;
}

// Repacked operands are padded to a multiple of 64 columns (one 128-byte swizzle span) with zeros, so that no
// TMA box of theirs is partly out of range: measured on B200, boxes that needed out-of-range fill made the
// head_dim-100 block matmuls 1.45x slower than the same kernel on head_dim 128.
static long long packed_cols(long long cols) { return (cols + 63) / 64 * 64; }
static size_t packed_bytes(long long rows, long long cols, long long nblk) {
  const long long cp = packed_cols(cols);
  return ((size_t)nblk * rows * cp * 2 + 255) / 256 * 256;
}

// Copy an operand that TMA cannot address into `dst` (packed_bytes), rows padded with zeros to packed_cols, and describe the
// copy in its place.
static int repack_operand(Operand& o, int nbi, int nbo, uint64_t dst, cudaStream_t st) {
  const long long nblk = (long long)((o.has_j ? nbi : 1)) * (o.has_i ? nbo : 1);
  const long long cp = packed_cols(o.cols);
  const int eff_nbi = o.has_j ? nbi : 1;
  const long long so_ = o.has_i ? o.stride_outer : 0, si_ = o.has_j ? o.stride_inner : 0;
  // widest unit (in elements) that divides every offset involved
  const unsigned long long all = (unsigned long long)(o.ptr / 2) | (unsigned long long)o.ld | (unsigned long long)so_ |
                                 (unsigned long long)si_ | (unsigned long long)o.cols;
  const int ue = (all & 3) == 0 ? 4 : (all & 1) == 0 ? 2 : 1;       // elements per unit
  const long long total_units = nblk * o.rows * (cp / ue);
  long long grid = (total_units + 255) / 256;
  if (grid > (long long)kNumSMs * 32) grid = (long long)kNumSMs * 32;
#define CB_PACK(U_)                                                                                              \
  pack_blocks_kernel<U_><<<(unsigned)grid, 256, 0, st>>>(reinterpret_cast<U_*>(dst),                             \
      reinterpret_cast<const U_*>(o.ptr), (unsigned)o.rows, (unsigned)(o.cols / ue), (unsigned)(cp / ue),        \
      o.ld / ue, (unsigned)eff_nbi, so_ / ue, si_ / ue, total_units)
  if (ue == 4) CB_PACK(uint2); else if (ue == 2) CB_PACK(uint32_t); else CB_PACK(uint16_t);
#undef CB_PACK
  const int rc = check_launch();
  if (rc) return rc;
  o.ptr = dst; o.ld = cp; o.map_cols = cp;
  o.stride_inner = o.rows * cp;
  o.stride_outer = o.rows * cp * eff_nbi;
  return CACTI_B200_OK;
}

}  // namespace cb
