// G1 / G2: dense and block (strided-batched) matmul on the 5th-generation tensor cores.
//
// Replaces MatrixMulF16F32GpuThunkImpl (cublasGemmEx, src/thunk/op.rs:4413-4716) and
// BlockMatrixMulF16F32GpuThunkImpl (cublasGemmBatchedEx over host-built pointer arrays,
// src/thunk/op.rs:5025-5471): C = f16(alpha * op(A) op(B) + beta * C), 16-bit operands, fp32
// accumulation, no split-K and no atomics (cacti_gpu_cu_ffi/src/lib.rs:749,766-767), row-major with
// leading dimensions, all four transpose combinations (src/thunk/op.rs:4336-4365, :4883-4911).
// The block form addresses block (i, j) by two affine strides per operand, which is what the
// reference computes on the host for its pointer arrays (src/thunk/op.rs:5174-5189); a stride of 0
// broadcasts the block.
//
// Kernel: one persistent CTA per SM, 192 threads.
//   warp 0      : TMA producer.  Operand tiles are fetched with cp.async.bulk.tensor (4-D tensor maps:
//                 inner, outer, block j, block i) into a ring of 128-byte-swizzled shared-memory stages;
//                 out-of-range rows/columns/K are zero-filled by the TMA unit.
//   warp 1      : allocates TMEM and issues tcgen05.mma (UMMA 128 x BN x 16, kind::f16) from one thread;
//                 tcgen05.commit releases shared-memory stages and publishes finished accumulators.
//   warps 2..5  : epilogue.  tcgen05.ld brings the fp32 accumulator out of TMEM, alpha/beta are applied,
//                 the result is rounded once to the 16-bit type and stored.
// Two accumulators (2 x BN of the 512 TMEM columns) let the epilogue of one tile overlap the main
// loop of the next.  Operands may be K-major or MN-major in memory; the transpose flags only change
// the tensor-map box and the "major" bits of the descriptors, never the data.  No load uses cluster
// multicast.  Every wait is bounded; on a timeout the CTA records kDevErrGemmTimeout, drains, frees
// its TMEM and returns.
//
// Operands that TMA cannot address (base or a stride not a multiple of 16 bytes, e.g. head_dim 100
// slices at 200-byte offsets) are first repacked into the caller's workspace with the inner
// dimension zero-padded to a multiple of 64 elements; the reference pads the same operands to 16 bytes
// with a separate thunk before calling cuBLAS (src/op.rs:1454-1482).  Outputs need no alignment.
#include "gemm_common.cuh"

namespace cb {

// ---- k-split ("stream-K") schedule ------------------------------------------------------------------------------
// A persistent grid of W workers over T tiles runs ceil(T / W) waves; when T is not a multiple of W the last wave is
// partly idle (104 tiles on 74 SM pairs: 2 waves for 1.4 waves of work).  Here the first sk_tiles tiles are treated
// as one run of sk_tiles * nkb k-blocks that is cut into W equal consecutive ranges; worker w computes range w and
// then whole tiles sk_tiles + w, sk_tiles + w + W, ...  A range starts inside at most one tile.  That first piece is
// a *contribution*: its f32 accumulator goes to the worker's slot of `sk_part` and a flag is raised.  The worker
// whose range holds a tile's first k-block *owns* the tile: it computes its piece last, then adds the
// contributions in increasing k order and runs the normal epilogue.  Every output element is therefore summed in
// an order fixed by (shape, W): results do not change from run to run.  Contributions are the first thing a worker
// computes and owned pieces the last thing of its range, so an owner finds them ready unless the contributing CTA
// has not been scheduled yet; the wait for it is bounded (kDevErrGemmSplitTimeout).  Waits only ever point from
// worker w to workers > w, so no cycle exists.
constexpr int kSkSlots = 128;                       // launches in flight at once share flags only 128 launches apart
constexpr int kSkMaxWorkers = kNumSMs / 2;
__device__ unsigned g_sk_flags[kSkSlots][kSkMaxWorkers][2][4];    // zero at load; every flag is cleared by its reader

struct WorkItem { long long tile; int kb0, kb1, kind; };
struct WorkIter {
  long long pos, end, dp_next, dp_step, total;
  int nkb;
  __device__ __forceinline__ static long long range_begin(const GemmParams& p, long long w, long long nworkers) {
    return p.sk_units * w / nworkers;
  }
  __device__ __forceinline__ void init(const GemmParams& p, long long w, long long nworkers, long long total_tiles, int nkb_) {
    nkb = nkb_; total = total_tiles; dp_step = nworkers;
    pos = range_begin(p, w, nworkers); end = range_begin(p, w + 1, nworkers);
    dp_next = p.sk_tiles + w;
  }
  __device__ __forceinline__ bool next(WorkItem& it) {
    if (pos < end) {
      const long long t = pos / nkb, tile_end = (t + 1) * nkb;
      const long long e = end < tile_end ? end : tile_end;
      it.tile = t; it.kb0 = (int)(pos - t * nkb); it.kb1 = (int)(e - t * nkb);
      it.kind = it.kb0 ? kItemContrib : (it.kb1 == nkb ? kItemFull : kItemOwner);
      pos = e;
      return true;
    }
    if (dp_next < total) {
      it.tile = dp_next; it.kb0 = 0; it.kb1 = nkb; it.kind = kItemFull;
      dp_next += dp_step;
      return true;
    }
    return false;
  }
};

// ---- dynamic tile schedule ---------------------------------------------------------------------------------------
// A persistent grid that walks tiles with a fixed stride (worker w takes tiles w, w + W, ...) assumes all W workers
// run at once.  When another kernel holds some SMs (the gradient all-reduce beside the backward pass) the CTAs that
// find no SM start only when others have finished, and then still compute their whole share: the matmul takes two
// rounds instead of one and a fraction.  Here a worker's first tile is its own index and every further tile comes
// from a global counter, so the tiles go to whichever workers are running; a worker that starts late finds the
// counter exhausted and leaves.  Every tile is still computed whole by one worker in the same k order, so the
// results are bit-identical to the fixed-stride walk.
// The producer thread draws the tile indices and hands them to the other roles of its CTA (and, in the two-SM
// kernel, of the peer CTA) through a ring of kSchedDepth entries in shared memory guarded by mbarriers; -1 ends the
// walk.  The counter of a launch is g_tile_next[slot]; the last worker to finish (g_tile_done[slot]) puts both back
// to zero for the next launch that uses the slot.
__device__ unsigned g_tile_next[kSkSlots];
__device__ unsigned g_tile_done[kSkSlots];

// Next tile for the scheduling thread: workers' first tiles are their own indices, the rest come from the counter.
__device__ __forceinline__ long long sched_draw(int slot, long long nworkers, long long total) {
  const long long t = nworkers + (long long)atomicAdd(&g_tile_next[slot], 1u);
  return t < total ? t : -1;
}
// Called once per worker by its scheduling thread when it is done drawing.
__device__ __forceinline__ void sched_retire(int slot, long long nworkers) {
  __threadfence();
  if (atomicAdd(&g_tile_done[slot], 1u) == (unsigned)(nworkers - 1)) {
    __threadfence();
    g_tile_next[slot] = 0;
    g_tile_done[slot] = 0;
  }
}

template <typename T, int BN, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kGemmThreads, 1)
gemm_tc_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
               const __grid_constant__ CUtensorMap tmC, T* __restrict__ C, const GemmParams p) {
  constexpr int STAGES = BN >= 192 ? 4 : 6;
  constexpr uint32_t A_BYTES = kBM * kBK * 2, B_BYTES = BN * kBK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + (size_t)STAGES * STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  SchedSmem* sched = reinterpret_cast<SchedSmem*>(tmem_slot + 4);
  uint64_t* cbar = reinterpret_cast<uint64_t*>(sched + 1);        // one per epilogue warp: old C boxes have arrived
  // epilogue staging: per epilogue warp two [32 rows][64 cols] buffers in the 128-byte-swizzled layout of a
  // TMA box (4 KB each), 1024-byte aligned
  unsigned char* cstage = tiles + (size_t)STAGES * STAGE_BYTES + 1024;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(tfull + a, 1); mbar_init(tempty + a, 4); }
    // schedule ring: read by the MMA thread and by the four epilogue warps
    for (int i = 0; i < kSchedDepth; ++i) { mbar_init(sched->full + i, 1); mbar_init(sched->empty + i, 5); mbar_init(sched->empty_peer + i, 5); }
    for (int w = 0; w < 4; ++w) mbar_init(cbar + w, 1);
    mbar_fence_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int nkb = (p.K + kBK - 1) / kBK;
  const long long tiles_per_block = (long long)p.tiles_m * p.tiles_n;
  const long long total = tiles_per_block * p.nb_inner * p.nb_outer;

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer (and, with the dynamic schedule, the thread that draws the tiles) ----------------
    int s = 0; unsigned ph = 0;
    auto produce = [&](long long tile) -> bool {
      int blk, tm, tn;
      decode_tile(tile, tiles_per_block, p, blk, tm, tn);
      const int bi = blk / p.nb_inner, bj = blk - bi * p.nb_inner;
      const int aj = p.a_j ? bj : 0, ai = p.a_i ? bi : 0, bjj = p.b_j ? bj : 0, bii = p.b_i ? bi : 0;
      if (tile_skipped(p, tm * kBM, kBM, tn * BN)) return true;
      int kb0, kb1;
      k_block_range(p, tm * kBM, kBM, nkb, kb0, kb1);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(empty + s, ph ^ 1, kDevErrGemmTimeout)) return false;
        unsigned char* sa = tiles + (size_t)s * STAGE_BYTES;
        unsigned char* sb = sa + A_BYTES;
        mbar_expect_tx(full + s, STAGE_BYTES);
        if (!A_MN) tma_load_4d(sa, &tmA, full + s, kb * kBK, tm * kBM, aj, ai);
        else {
#pragma unroll
          for (int h = 0; h < kBM / 64; ++h) tma_load_4d(sa + h * 8192, &tmA, full + s, tm * kBM + h * 64, kb * kBK, aj, ai);
        }
        if (!B_MN) tma_load_4d(sb, &tmB, full + s, kb * kBK, tn * BN, bjj, bii);
        else {
#pragma unroll
          for (int h = 0; h < BN / 64; ++h) tma_load_4d(sb + h * 8192, &tmB, full + s, tn * BN + h * 64, kb * kBK, bjj, bii);
        }
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
      return true;
    };
    if (p.dyn) {
      unsigned sn = 0;
      long long tile = blockIdx.x;                       // the grid never exceeds the tile count
      for (;;) {
        if (!sched_publish<false>(sched, sn, (int)tile)) break;
        if (tile < 0) break;
        const long long nxt = sched_draw(p.sk_slot, gridDim.x, total);     // in flight while this tile's loads are issued
        if (!produce(tile)) break;
        tile = nxt;
      }
    } else {
      for (long long tile = blockIdx.x; tile < total; tile += gridDim.x)
        if (!produce(tile)) break;
    }
  } else if (warp == 1 && lane == 0) {
    // ---------------- MMA issuer ----------------
    int s = 0; unsigned ph = 0;
    long long local = 0;
    auto mma_tile = [&](long long tile) -> bool {
      int kb0 = 0, kb1 = nkb;
      int blk, tm, tn;
      decode_tile(tile, tiles_per_block, p, blk, tm, tn);
      if (p.tri) {
        if (tile_skipped(p, tm * kBM, kBM, tn * BN)) return true;
        k_block_range(p, tm * kBM, kBM, nkb, kb0, kb1);
      }
      // the last column tile multiplies only the columns that exist (rounded up to the MMA's granularity of 16)
      const int nvalid = p.N - tn * BN;
      const uint32_t idesc = nvalid >= BN ? p.idesc : idesc_with_n(p.idesc, (nvalid + 15) & ~15);
      const int acc = (int)(local & 1);
      if (!mbar_wait_bounded(tempty + acc, (unsigned)((local >> 1) & 1) ^ 1, kDevErrGemmTimeout)) return false;
      tc_fence_after();
      const uint32_t tacc = tmem_base + (uint32_t)acc * BN;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(full + s, ph, kDevErrGemmTimeout)) return false;
        tc_fence_after();
        const uint32_t sa = smem_u32(tiles + (size_t)s * STAGE_BYTES), sb = sa + A_BYTES;
#pragma unroll
        for (int k4 = 0; k4 < kBK / 16; ++k4) {
          const uint64_t da = A_MN ? make_desc(sa + k4 * 2048, 512, 64) : make_desc(sa + k4 * 32, 1, 64);
          const uint64_t db = B_MN ? make_desc(sb + k4 * 2048, 512, 64) : make_desc(sb + k4 * 32, 1, 64);
          tc_mma_f16(tacc, da, db, idesc, (kb > kb0 || k4) ? 1u : 0u);
        }
        tc_commit(empty + s);                 // stage free once these MMAs have read it
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
      tc_commit(tfull + acc);                 // accumulator complete
      ++local;
      return true;
    };
    if (p.dyn) {
      unsigned sn = 0;
      for (;;) {
        const int tile = sched_take<false>(sched, sn, true, 0);
        if (tile < 0 || !mma_tile(tile)) break;
      }
    } else {
      for (long long tile = blockIdx.x; tile < total; tile += gridDim.x)
        if (!mma_tile(tile)) break;
    }
  } else if (warp >= 2) {
    // ---------------- epilogue ----------------
    const int q = warp & 3;                   // TMEM lane quarter this warp may read
    long long local = 0;
    unsigned cpar = 0;                        // phase of this warp's old-C barrier
    auto epi_tile = [&](long long tile) -> bool {
      int blk, tm, tn;
      decode_tile(tile, tiles_per_block, p, blk, tm, tn);
      if (tile_skipped(p, tm * kBM, kBM, tn * BN)) return true;
      const int bi = blk / p.nb_inner, bj = blk - bi * p.nb_inner;
      const int acc = (int)(local & 1);
      // all 32 lanes leave together: a wait that ran out on some lanes only must not split the warp before the
      // warp-wide tcgen05.ld of the epilogue
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(tfull + acc, (unsigned)((local >> 1) & 1), kDevErrGemmTimeout))) return false;
      tc_fence_after();
      epilogue_tile<T, BN>(p, tmC, C, tmem_base, acc, tm * kBM + q * 32, tn, bj, bi, q, lane,
                           cstage + (size_t)(warp - 2) * 8192, smem_u32(tempty + acc), cbar + (warp - 2), cpar);
      ++local;
      return true;
    };
    if (p.dyn) {
      unsigned sn = 0;
      for (;;) {
        const int tile = sched_take_warp<false>(sched, sn, lane, 0);
        if (tile < 0 || !epi_tile(tile)) break;
      }
    } else {
      for (long long tile = blockIdx.x; tile < total; tile += gridDim.x)
        if (!epi_tile(tile)) break;
    }
  }
  if (p.dyn && warp == 0 && lane == 0) sched_retire(p.sk_slot, gridDim.x);     // on every path, or the counter stays dirty
  if (warp >= 2 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  }
}

// ---- two-SM variant (cta_group::2) -------------------------------------------------------------------------
// A cluster of two CTAs on one SM pair computes a 256 x 256 output tile.  Each CTA stages its own 128 rows of A
// and one half (128 rows) of the B tile; the leader CTA (cluster rank 0) issues tcgen05.mma.cta_group::2 with
// M = 256, which reads A from both CTAs, both halves of B, and accumulates rows 0..127 into the leader's TMEM and
// rows 128..255 into the peer's.  Per flop each SM reads a third less shared memory and L2 than the
// one-SM 128 x 256 tile.  Signalling:
//   full[s]   (leader only) : 1 arrival (the leader's expect_tx for both CTAs' bytes); both CTAs' TMA loads
//                             complete their bytes on it (the load's cta_group::2 form allows a peer barrier)
//   empty[s]  (both CTAs)   : the leader's tcgen05.commit, multicast to both CTAs
//   tfull[a]  (both CTAs)   : same, when an accumulator is complete
//   tempty[a] (leader only) : 8 arrivals, one per epilogue warp of either CTA
// No load uses cluster multicast.  Every wait is bounded; all threads of both CTAs meet on the cluster barrier
// before TMEM is freed, and the producers wait for the last stage releases, so neither CTA exits while the other
// can still signal into its shared memory.
constexpr int kPairBM = 256, kPairBN = 256, kPairStages = 6;
constexpr size_t kPairSmem = (size_t)kPairStages * (kBM * kBK * 2 + (kPairBN / 2) * kBK * 2) + 1024 + 1024 + 4 * 8192;

template <typename T, bool A_MN, bool B_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1)
gemm_tc_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmC, T* __restrict__ C, const GemmParams p) {
  constexpr int BN = kPairBN, HB = BN / 2, STAGES = kPairStages;
  constexpr uint32_t A_BYTES = kBM * kBK * 2, B_BYTES = HB * kBK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + (size_t)STAGES * STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  SchedSmem* sched = reinterpret_cast<SchedSmem*>(tmem_slot + 4);
  uint64_t* cbar = reinterpret_cast<uint64_t*>(sched + 1);        // one per epilogue warp: old C boxes have arrived
  unsigned char* cstage = tiles + (size_t)STAGES * STAGE_BYTES + 1024;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const long long pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(tfull + a, 1); mbar_init(tempty + a, 8); }
    // schedule ring: in the leader read by the MMA thread and four epilogue warps (empty), in the peer by the producer
    // thread and four epilogue warps, which report to the leader's empty_peer
    for (int i = 0; i < kSchedDepth; ++i) { mbar_init(sched->full + i, 1); mbar_init(sched->empty + i, 5); mbar_init(sched->empty_peer + i, 5); }
    for (int w = 0; w < 4; ++w) mbar_init(cbar + w, 1);
    mbar_fence_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                         // the peer's barriers are initialised before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int nkb = (p.K + kBK - 1) / kBK;
  const long long tiles_per_block = (long long)p.tiles_m * p.tiles_n;
  const long long total = tiles_per_block * p.nb_inner * p.nb_outer;

  // the leader's barriers on which the peer CTA's consumers report their reads of the schedule ring
  const uint32_t leader_empty_peer0 = map_to_rank(smem_u32(sched->empty_peer), 0);

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer (both CTAs); the leader's also draws the tiles of the dynamic schedule ----------------
    int s = 0; unsigned ph = 0;
    const int row_off = (int)rank * kBM;
    auto produce = [&](const WorkItem& wi) -> bool {
      int blk, tm, tn;
      decode_tile(wi.tile, tiles_per_block, p, blk, tm, tn);
      const int bi = blk / p.nb_inner, bj = blk - bi * p.nb_inner;
      const int aj = p.a_j ? bj : 0, ai = p.a_i ? bi : 0, bjj = p.b_j ? bj : 0, bii = p.b_i ? bi : 0;
      // a last column tile with at most 128 columns runs as an N = 128 MMA: each CTA then supplies 64 rows of B
      // (the first 64 of the box it loads), so the CTAs' boxes start 64 rows apart instead of 128
      const int hb = (p.N - tn * BN <= HB) ? HB / 2 : HB;
      const int m0 = tm * kPairBM + row_off, n0 = tn * BN + (int)rank * hb;
      if (tile_skipped(p, tm * kPairBM, kPairBM, tn * BN)) return true;
      int kb0 = wi.kb0, kb1 = wi.kb1;
      if (p.tri) k_block_range(p, tm * kPairBM, kPairBM, nkb, kb0, kb1);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(empty + s, ph ^ 1, kDevErrGemmTimeout)) return false;
        unsigned char* sa = tiles + (size_t)s * STAGE_BYTES;
        unsigned char* sb = sa + A_BYTES;
        const uint32_t fb = map_to_rank(smem_u32(full + s), 0);
        if (rank == 0) mbar_expect_tx(full + s, 2 * STAGE_BYTES);
        if (!A_MN) tma_load_4d_pair(sa, &tmA, fb, kb * kBK, m0, aj, ai);
        else {
#pragma unroll
          for (int h = 0; h < kBM / 64; ++h) tma_load_4d_pair(sa + h * 8192, &tmA, fb, m0 + h * 64, kb * kBK, aj, ai);
        }
        if (!B_MN) tma_load_4d_pair(sb, &tmB, fb, kb * kBK, n0, bjj, bii);
        else {
#pragma unroll
          for (int h = 0; h < HB / 64; ++h) tma_load_4d_pair(sb + h * 8192, &tmB, fb, n0 + h * 64, kb * kBK, bjj, bii);
        }
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
      return true;
    };
    bool ok = true;
    WorkItem wi;
    if (p.dyn) {
      unsigned sn = 0;
      wi.kb0 = 0; wi.kb1 = nkb; wi.kind = kItemFull;
      if (rank == 0) {
        long long tile = pair;                             // the grid never has more pairs than tiles
        for (;;) {
          if (!sched_publish<true>(sched, sn, (int)tile)) { ok = false; break; }
          if (tile < 0) break;
          const long long nxt = sched_draw(p.sk_slot, npairs, total);    // in flight while this tile's loads are issued
          wi.tile = tile;
          if (!produce(wi)) { ok = false; break; }
          tile = nxt;
        }
      } else {
        for (;;) {
          const int tile = sched_take<true>(sched, sn, true, leader_empty_peer0);
          if (tile < 0) { ok = tile == -1; break; }
          wi.tile = tile;
          if (!produce(wi)) { ok = false; break; }
        }
      }
    } else {
      WorkIter it;
      it.init(p, pair, npairs, total, nkb);
      while (ok && it.next(wi)) ok = produce(wi);
    }
    // the leader's last commits still arrive on this CTA's empty barriers: wait for them before leaving
    for (int i = 0; ok && i < STAGES; ++i) {
      ok = mbar_wait_bounded(empty + s, ph ^ 1, kDevErrGemmTimeout);
      if (++s == STAGES) { s = 0; ph ^= 1; }
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ---------------- MMA issuer (leader CTA) ----------------
    int s = 0; unsigned ph = 0;
    long long local = 0;
    auto mma_item = [&](const WorkItem& wi) -> bool {
      int kb0 = wi.kb0, kb1 = wi.kb1;
      int blk, tm, tn;
      decode_tile(wi.tile, tiles_per_block, p, blk, tm, tn);
      if (p.tri) {
        if (tile_skipped(p, tm * kPairBM, kPairBM, tn * BN)) return true;
        k_block_range(p, tm * kPairBM, kPairBM, nkb, kb0, kb1);
      }
      const uint32_t idesc = (p.N - tn * BN <= HB) ? idesc_with_n(p.idesc, HB) : p.idesc;      // see the producer
      const int acc = (int)(local & 1);
      if (!mbar_wait_bounded(tempty + acc, (unsigned)((local >> 1) & 1) ^ 1, kDevErrGemmTimeout)) return false;
      tc_fence_after();
      const uint32_t tacc = tmem_base + (uint32_t)acc * BN;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(full + s, ph, kDevErrGemmTimeout)) return false;
        tc_fence_after();
        const uint32_t sa = smem_u32(tiles + (size_t)s * STAGE_BYTES), sb = sa + A_BYTES;
#pragma unroll
        for (int k4 = 0; k4 < kBK / 16; ++k4) {
          const uint64_t da = A_MN ? make_desc(sa + k4 * 2048, 512, 64) : make_desc(sa + k4 * 32, 1, 64);
          const uint64_t db = B_MN ? make_desc(sb + k4 * 2048, 512, 64) : make_desc(sb + k4 * 32, 1, 64);
          tc_mma_f16_pair(tacc, da, db, idesc, (kb > kb0 || k4) ? 1u : 0u);
        }
        tc_commit_pair(empty + s);
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
      tc_commit_pair(tfull + acc);
      ++local;
      return true;
    };
    WorkItem wi;
    if (p.dyn) {
      unsigned sn = 0;
      wi.kb0 = 0; wi.kb1 = nkb; wi.kind = kItemFull;
      for (;;) {
        const int tile = sched_take<false>(sched, sn, true, 0);
        if (tile < 0) break;
        wi.tile = tile;
        if (!mma_item(wi)) break;
      }
    } else {
      WorkIter it;
      it.init(p, pair, npairs, total, nkb);
      while (it.next(wi))
        if (!mma_item(wi)) break;
    }
  } else if (warp >= 2) {
    // ---------------- epilogue (both CTAs, each on its own 128 rows) ----------------
    const int q = warp & 3;
    long long local = 0;
    unsigned cpar = 0;                        // phase of this warp's old-C barrier
    auto epi_item = [&](const WorkItem& wi) -> bool {
      int blk, tm, tn;
      decode_tile(wi.tile, tiles_per_block, p, blk, tm, tn);
      if (tile_skipped(p, tm * kPairBM, kPairBM, tn * BN)) return true;
      const int bi = blk / p.nb_inner, bj = blk - bi * p.nb_inner;
      const int acc = (int)(local & 1);
      SkEpi sk{};
      sk.kind = wi.kind;
      if (wi.kind == kItemContrib) {
        sk.my_part = p.sk_part + ((size_t)pair * 2 + rank) * kSkPartFloats;
        sk.my_flags = &g_sk_flags[p.sk_slot][pair][rank][0];
      } else if (wi.kind == kItemOwner) {
        // the rest of this tile lies in the ranges of the next workers
        const long long tile_end = (wi.tile + 1) * nkb;
        int n = 0;
        for (long long w2 = pair + 1; w2 < npairs && WorkIter::range_begin(p, w2, npairs) < tile_end; ++w2) ++n;
        sk.ncontrib = n;
        sk.part0 = p.sk_part + ((size_t)(pair + 1) * 2 + rank) * kSkPartFloats;
        sk.flags0 = &g_sk_flags[p.sk_slot][pair + 1][rank][0];
      }
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(tfull + acc, (unsigned)((local >> 1) & 1), kDevErrGemmTimeout))) return false;
      tc_fence_after();
      epilogue_tile<T, BN>(p, tmC, C, tmem_base, acc, tm * kPairBM + (int)rank * kBM + q * 32, tn, bj, bi, q, lane,
                           cstage + (size_t)(warp - 2) * 8192, map_to_rank(smem_u32(tempty + acc), 0), cbar + (warp - 2), cpar, sk);
      ++local;
      return true;
    };
    WorkItem wi;
    if (p.dyn) {
      unsigned sn = 0;
      wi.kb0 = 0; wi.kb1 = nkb; wi.kind = kItemFull;
      for (;;) {
        const int tile = rank == 0 ? sched_take_warp<false>(sched, sn, lane, 0) : sched_take_warp<true>(sched, sn, lane, leader_empty_peer0);
        if (tile < 0) break;
        wi.tile = tile;
        if (!epi_item(wi)) break;
      }
    } else {
      WorkIter it;
      it.init(p, pair, npairs, total, nkb);
      while (it.next(wi))
        if (!epi_item(wi)) break;
    }
  }
  if (p.dyn && warp == 0 && lane == 0 && rank == 0) sched_retire(p.sk_slot, npairs);   // on every path, or the counter stays dirty
  if (warp >= 2 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                         // both CTAs have finished reading TMEM and signalling each other
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  }
}

int g_gemm_bn = 0;   // 0: choose by N; 128 or 256 forces the tile width (measurement knob)
int g_gemm_group_m = 0;
int g_gemm_sms = 0;   // 0: all 148
int g_gemm_pair = 1;  // 1: 256-wide tiles may run as two-SM (cta_group::2) 256 x 256 tiles; 0: one-SM tiles only
// 1: the two-SM kernel may share tiles out in k-blocks when a workspace is given (see WorkIter).  Off unless asked
// for: timed alone at one sequence per GPU (M = 2048) the schedule brought the forward and input-gradient matmuls to
// the per-flop rate they have at M = 16384 (2048 x 3200 x 8640: 124 -> 107 us), but a whole training step ran 5 %
// slower with it (50.8 -> 53.6 ms at M = 2048): these matmuls are power-limited, the SMs a partly filled last wave
// leaves idle let the others clock higher, and the partial sums displace 19 MB of the L2 per matmul.
int g_gemm_split = 0;
int g_gemm_dynamic = 1;  // 1: tiles beyond a worker's first are drawn from a global counter (see "dynamic tile schedule")

// Workers and k-split tiles for `tiles` two-SM tiles of `nkb` k-blocks on at most `max_workers` SM pairs.  Splitting
// pays when the last wave of whole tiles would leave more than about 5 % of the grid idle.
struct SplitPlan { long long workers, sk_tiles; };
// `tiles_n`, `group_m`, `N`, `K`: to bound the operand bytes the split tiles touch.  Whole tiles that run at the same
// time walk k together, so each operand panel is fetched from HBM once and shared through L2; workers of the k-split
// region sit at different k, and the region's operands must stay in L2 (126 MB) as a whole or every panel is fetched
// again per tile (measured: the 2048 x 3200 x 32000 input-gradient matmul of the output head, 336 MB of operands,
// ran 14 % slower split than whole; the 90 MB of the 8640-deep projections 8 to 15 % faster).
static SplitPlan plan_split(long long tiles, int nkb, long long max_workers, long long tiles_n, long long group_m, long long M,
                            long long N, long long K) {
  SplitPlan s{tiles < max_workers ? tiles : max_workers, 0};
  if (max_workers < 2 || tiles * 2 < max_workers) return s;          // a handful of tiles: not worth the partial traffic
  const long long rem = tiles % max_workers;
  if (rem == 0) return s;
  const long long waves = (tiles + max_workers - 1) / max_workers;
  if ((double)(max_workers - rem) / (double)(waves * max_workers) <= 0.05) return s;
  const long long sk_tiles = tiles < max_workers ? tiles : max_workers + rem;
  if (sk_tiles * nkb / max_workers < 4) return s;                    // pieces shorter than the operand ring
  const long long per_group = (group_m > 0 ? group_m : 1) * tiles_n;
  long long rows = (sk_tiles + per_group - 1) / per_group * group_m * 256;
  if (rows > M) rows = M;
  if ((rows + N) * K * 2 > 100ll * 1024 * 1024) return s;
  s.workers = max_workers; s.sk_tiles = sk_tiles;
  return s;
}
static long long pair_group_m(long long tiles_m) {
  const long long g = g_gemm_group_m > 0 ? g_gemm_group_m : 8;
  return g > tiles_m ? tiles_m : g;
}
static size_t split_bytes() { return (size_t)kSkMaxWorkers * 2 * kSkPartFloats * sizeof(float); }

template <typename T>
static int gemm_run(uint64_t c, Operand A, Operand B, bool a_mn, bool b_mn, long long M, long long N, long long K,
                    long long ldc, long long cso, long long csi, int nbi, int nbo, float alpha, float beta,
                    int tri, long long diag, int opflags, uint64_t ws, size_t ws_bytes, cudaStream_t st) {
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  size_t ws_off = 0;
  // repack what TMA cannot address
  for (Operand* o : {&A, &B}) {
    if (tma_ok(*o, nbi, nbo)) {
      // rows stored zero-padded to a multiple of 64 elements: let the tensor map cover the padding, so that no box
      // is partly out of range (the slow path of the TMA unit) and nothing has to be repacked
      if (opflags & (o == &A ? CACTI_B200_OPERAND_A_PADDED : CACTI_B200_OPERAND_B_PADDED)) {
        if (o->ld < packed_cols(o->cols)) return CACTI_B200_ERR_INVALID_VALUE;
        o->map_cols = packed_cols(o->cols);
      }
      continue;
    }
    const long long nblk = (long long)((o->has_j ? nbi : 1)) * (o->has_i ? nbo : 1);
    const size_t need = packed_bytes(o->rows, o->cols, nblk);
    if (!ws || (ws & 255) || ws_off + need > ws_bytes) return CACTI_B200_ERR_WORKSPACE;
    const int rc = repack_operand(*o, nbi, nbo, ws + ws_off, st);
    if (rc) return rc;
    ws_off += need;
  }
  // Tile shape: the persistent grid runs ceil(tiles / CTAs) waves; pick the shape with the least wave-time.
  // Per-flop cost relative to the one-SM 256-wide tile with K-major operands, from sustained interleaved runs of
  // the projection shapes: 1.08 for 192-wide and 1.3 for 128-wide tiles; one-SM tiles with an MN-major operand
  // 1.25 (their shared-memory reads conflict more); the two-SM 256 x 256 tile 0.93 with either operand layout (the
  // 3200 x 3200 x 16384 weight-gradient matmul: 1041 TFLOP/s in 3 waves of 256 x 256 against 963 in 3 waves of 128 x 192).
  int BN = g_gemm_bn;
  bool pair = false;
  const int sms = g_gemm_sms > 0 && g_gemm_sms < kNumSMs ? g_gemm_sms : kNumSMs;
  const long long pair_workers = sms / 2;
  const int nkb_host = (int)((K + kBK - 1) / kBK);
  // the k-split schedule needs room for the partial accumulators behind whatever was repacked; dense matmuls only
  // (block matmuls bring hundreds of tiles, and their hinted forms promise bits equal to the unhinted ones)
  const size_t split_off = (ws_off + 255) / 256 * 256;
  const bool split_ok = g_gemm_split && tri == 0 && nbi == 1 && nbo == 1 && ws && !(ws & 255) &&
                        split_off + split_bytes() <= ws_bytes;
  if (!BN) {
    if (N <= 128) BN = 128;
    else {
      const bool mn = a_mn || b_mn;
      double best = 1e300;
      for (int bn : {256, 192, 128}) {
        const long long tiles = ((M + kBM - 1) / kBM) * ((N + bn - 1) / bn) * nbi * nbo;
        const double cost = (double)((tiles + kNumSMs - 1) / kNumSMs) * bn * (bn == 128 ? 1.3 : bn == 192 ? 1.08 : 1.0) *
                            (mn ? 1.25 : 1.0);
        if (cost < best * 0.999) { best = cost; BN = bn; }
      }
      if (g_gemm_pair && M > kBM) {
        const long long tiles2 = ((M + kPairBM - 1) / kPairBM) * ((N + kPairBN - 1) / kPairBN) * nbi * nbo;
        double cost = (double)((tiles2 + kNumSMs / 2 - 1) / (kNumSMs / 2)) * kPairBN * 0.93;
        // with the k-split schedule the two-SM grid has no idle last wave (3 % for the partial sums)
        const long long tm2 = (M + kPairBM - 1) / kPairBM, tn2 = (N + kPairBN - 1) / kPairBN;
        if (split_ok && plan_split(tiles2, nkb_host, pair_workers, tn2, pair_group_m(tm2), M, N, K).sk_tiles)
          cost = (double)tiles2 / (double)pair_workers * kPairBN * 0.93 * 1.03;
        if (cost < best) { best = cost; BN = kPairBN; pair = true; }
      }
    }
  } else {
    pair = g_gemm_pair != 0 && BN == kPairBN && M > kBM;
  }
  const int tile_m = pair ? kPairBM : kBM;
  CUtensorMap tmA, tmB;
  // K-major operand: stored [mn][k] -> box {64 k, tile mn}; MN-major: stored [k][mn] -> box {64 mn, 64 k}
  int rc = encode_operand(&tmA, A, nbi, nbo, 64, a_mn ? 64 : kBM, bf16);
  if (rc) return rc;
  rc = encode_operand(&tmB, B, nbi, nbo, 64, b_mn ? 64 : (pair ? BN / 2 : BN), bf16);
  if (rc) return rc;
  GemmParams p;
  p.M = (int)M; p.N = (int)N; p.K = (int)K;
  p.nb_inner = nbi; p.nb_outer = nbo;
  p.tiles_m = (int)((M + tile_m - 1) / tile_m); p.tiles_n = (int)((N + BN - 1) / BN);
  p.a_j = A.has_j && nbi > 1; p.a_i = A.has_i && nbo > 1; p.b_j = B.has_j && nbi > 1; p.b_i = B.has_i && nbo > 1;
  p.ldc = ldc; p.c_stride_inner = csi; p.c_stride_outer = cso;
  p.alpha = alpha; p.beta = beta;
  p.tri = tri; p.diag = (int)diag;
  p.idesc = (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) |
            ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(tile_m >> 4) << 24);
  const uint64_t all = c | (uint64_t)(ldc * 2) | (uint64_t)(nbi > 1 ? csi * 2 : 0) | (uint64_t)(nbo > 1 ? cso * 2 : 0);
  p.c_align = (all & 15) == 0 ? 16 : (all & 7) == 0 ? 8 : (all & 3) == 0 ? 4 : 2;
  // TMA store (and, with beta != 0, TMA load) of C needs a 16-byte aligned base and strides
  CUtensorMap tmC = tmA;
  p.c_tma = 0;
  {
    Operand Co{c, M, N, ldc, csi, cso, nbi > 1, nbo > 1};
    if (tma_ok(Co, nbi, nbo) && (nbi == 1 || csi != 0) && (nbo == 1 || cso != 0)) {
      rc = encode_operand(&tmC, Co, nbi, nbo, 64, 32, bf16);
      if (rc) return rc;
      p.c_tma = 1;
    }
  }
  // about 16 m-tiles of A (2048 rows) stay hot in L2 while the B panels stream
  p.group_m = pair ? (int)pair_group_m(p.tiles_m) : (g_gemm_group_m > 0 ? g_gemm_group_m : 16);
  if (p.group_m > p.tiles_m) p.group_m = p.tiles_m;
  const long long total = (long long)p.tiles_m * p.tiles_n * nbi * nbo;
  // g_gemm_sms < 148 leaves SMs free for a concurrent kernel (the gradient all-reduce): a persistent grid that
  // cannot be fully resident would otherwise run its last CTAs as a second wave
  const int grid = (int)(total < sms ? total : sms);
  p.sk_tiles = 0; p.sk_units = 0; p.sk_part = nullptr; p.sk_slot = 0;
  static std::atomic<unsigned> launch_seq{0};       // flag / counter slot of a launch: consecutive launches use different ones
  p.dyn = (g_gemm_dynamic && total < 0x7fffffffLL) ? 1 : 0;
  if (p.dyn) p.sk_slot = (int)(launch_seq.fetch_add(1) % kSkSlots);
  const int stages = BN >= 192 ? 4 : 6;
  const size_t smem = (size_t)stages * (kBM * kBK * 2 + BN * kBK * 2) + 1024 /*align*/ + 1024 /*barriers*/ + 4 * 8192;
  T* C = reinterpret_cast<T*>(c);
  if (pair) {
    long long pairs = total < sms / 2 ? total : sms / 2;
    if (split_ok) {
      const SplitPlan sp = plan_split(total, nkb_host, pair_workers, p.tiles_n, p.group_m, M, N, K);
      if (sp.sk_tiles) {                                // the k-split walk is static: it replaces the dynamic one
        pairs = sp.workers;
        p.sk_tiles = sp.sk_tiles; p.sk_units = sp.sk_tiles * nkb_host;
        p.sk_part = reinterpret_cast<float*>(ws + split_off);
        if (!p.dyn) p.sk_slot = (int)(launch_seq.fetch_add(1) % kSkSlots);
        p.dyn = 0;
      }
    }
#define CB_GEMM2(AM_, BM_)                                                                             \
  do {                                                                                                 \
    auto kern = gemm_tc_pair_kernel<T, AM_, BM_>;                                                      \
    static bool attr_set[kMaxDevices] = {};                                                                      \
    ensure_dynamic_smem(kern, kPairSmem, attr_set); \
    kern<<<(unsigned)(2 * pairs), kGemmThreads, kPairSmem, st>>>(tmA, tmB, tmC, C, p);                 \
  } while (0)
    if (!a_mn && !b_mn) CB_GEMM2(false, false); else if (!a_mn && b_mn) CB_GEMM2(false, true);
    else if (a_mn && !b_mn) CB_GEMM2(true, false); else CB_GEMM2(true, true);
#undef CB_GEMM2
    return check_launch();
  }
#define CB_GEMM(BN_, AM_, BM_)                                                                         \
  do {                                                                                                 \
    auto kern = gemm_tc_kernel<T, BN_, AM_, BM_>;                                                      \
    static bool attr_set[kMaxDevices] = {};                                                                      \
    ensure_dynamic_smem(kern, smem, attr_set); \
    kern<<<grid, kGemmThreads, smem, st>>>(tmA, tmB, tmC, C, p);                                            \
  } while (0)
  if (BN == 256) {
    if (!a_mn && !b_mn) CB_GEMM(256, false, false); else if (!a_mn && b_mn) CB_GEMM(256, false, true);
    else if (a_mn && !b_mn) CB_GEMM(256, true, false); else CB_GEMM(256, true, true);
  } else if (BN == 192) {
    if (!a_mn && !b_mn) CB_GEMM(192, false, false); else if (!a_mn && b_mn) CB_GEMM(192, false, true);
    else if (a_mn && !b_mn) CB_GEMM(192, true, false); else CB_GEMM(192, true, true);
  } else {
    if (!a_mn && !b_mn) CB_GEMM(128, false, false); else if (!a_mn && b_mn) CB_GEMM(128, false, true);
    else if (a_mn && !b_mn) CB_GEMM(128, true, false); else CB_GEMM(128, true, true);
  }
#undef CB_GEMM
  return check_launch();
}

static int gemm_entry(uint64_t c, uint64_t a, uint64_t b, long long m, long long n, long long k, long long lda,
                      long long ldb, long long ldc, int ta, int tb, const float* alpha, const float* beta, int nbo, int nbi,
                      long long sao, long long sai, long long sbo, long long sbi, long long sco, long long sci, int tri,
                      long long diag, int opflags, int dtype, uint64_t ws, size_t ws_bytes, void* stream) {
  if (m < 0 || n < 0 || k < 0 || nbo < 0 || nbi < 0 || !alpha || !beta) return CACTI_B200_ERR_INVALID_VALUE;
  if (m > 0x7fffffffLL || n > 0x7fffffffLL || k > 0x7fffffffLL) return CACTI_B200_ERR_SHAPE;
  if ((ta & ~1) || (tb & ~1)) return CACTI_B200_ERR_INVALID_VALUE;
  if (tri < CACTI_B200_TRI_NONE || tri > CACTI_B200_TRI_A_UPPER || diag > 0x3fffffffLL || diag < -0x3fffffffLL)
    return CACTI_B200_ERR_INVALID_VALUE;
  if (dtype != CACTI_B200_R_16F && dtype != CACTI_B200_R_16BF) return CACTI_B200_ERR_DTYPE;
  if (m == 0 || n == 0 || nbo == 0 || nbi == 0) return CACTI_B200_OK;
  if (!c || (k > 0 && (!a || !b))) return CACTI_B200_ERR_INVALID_VALUE;
  // stored shapes: A is [m,k] (ta = 0) or [k,m]; B is [k,n] (tb = 0) or [n,k]
  const long long a_rows = ta ? k : m, a_cols = ta ? m : k, b_rows = tb ? n : k, b_cols = tb ? k : n;
  if (lda < a_cols || ldb < b_cols || ldc < n) return CACTI_B200_ERR_INVALID_VALUE;
  if (k == 0) return CACTI_B200_ERR_SHAPE;      // the reference never stages an empty contraction
  Operand A{a, a_rows, a_cols, lda, sai, sao, sai != 0, sao != 0};
  Operand B{b, b_rows, b_cols, ldb, sbi, sbo, sbi != 0, sbo != 0};
  if (nbi == 1) { A.has_j = B.has_j = 0; }
  if (nbo == 1) { A.has_i = B.has_i = 0; }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // A as [m][k] is K-major; as [k][m] it is MN-major.  B as [n][k] (tb = 1) is K-major; as [k][n] MN-major.
  const bool a_mn = ta != 0, b_mn = tb == 0;
  if (dtype == CACTI_B200_R_16F)
    return gemm_run<__half>(c, A, B, a_mn, b_mn, m, n, k, ldc, sco, sci, nbi, nbo, *alpha, *beta, tri, diag, opflags, ws, ws_bytes, st);
  return gemm_run<__nv_bfloat16>(c, A, B, a_mn, b_mn, m, n, k, ldc, sco, sci, nbi, nbo, *alpha, *beta, tri, diag, opflags, ws, ws_bytes, st);
}

}  // namespace cb

extern "C" {

size_t cacti_b200_gemm_workspace_bytes(int64_t m, int64_t n, int64_t k, int64_t batch_outer, int64_t batch_inner) {
  if (m < 0 || n < 0 || k < 0 || batch_outer < 0 || batch_inner < 0) return 0;
  const long long nb = (batch_outer ? batch_outer : 1) * (batch_inner ? batch_inner : 1);
  // worst case: both operands repacked, either orientation
  auto worst = [&](long long r, long long c) {
    const size_t x = cb::packed_bytes(r, c, nb), y = cb::packed_bytes(c, r, nb);
    return x > y ? x : y;
  };
  return worst(m, k) + worst(k, n) + 512 + cb::split_bytes() + 256;
}

int cacti_b200_gemm(cacti_b200_dptr c, cacti_b200_dptr a, cacti_b200_dptr b, int64_t m, int64_t n, int64_t k, int64_t lda,
                    int64_t ldb, int64_t ldc, int trans_a, int trans_b, const float* alpha, const float* beta, int dtype,
                    cacti_b200_dptr workspace, size_t workspace_bytes, cacti_b200_stream stream) {
  return cb::gemm_entry(c, a, b, m, n, k, lda, ldb, ldc, trans_a, trans_b, alpha, beta, 1, 1, 0, 0, 0, 0, 0, 0,
                        CACTI_B200_TRI_NONE, 0, 0, dtype, workspace, workspace_bytes, stream);
}

int cacti_b200_gemm_strided_batched(cacti_b200_dptr c, cacti_b200_dptr a, cacti_b200_dptr b, int64_t m, int64_t n,
                                    int64_t k, int64_t lda, int64_t ldb, int64_t ldc, int trans_a, int trans_b,
                                    const float* alpha, const float* beta, int64_t batch_outer, int64_t batch_inner,
                                    int64_t stride_a_outer, int64_t stride_a_inner, int64_t stride_b_outer,
                                    int64_t stride_b_inner, int64_t stride_c_outer, int64_t stride_c_inner, int dtype,
                                    cacti_b200_dptr workspace, size_t workspace_bytes, cacti_b200_stream stream) {
  if (batch_outer > 0x7fffffffLL || batch_inner > 0x7fffffffLL) return CACTI_B200_ERR_SHAPE;
  return cb::gemm_entry(c, a, b, m, n, k, lda, ldb, ldc, trans_a, trans_b, alpha, beta, (int)batch_outer, (int)batch_inner,
                        stride_a_outer, stride_a_inner, stride_b_outer, stride_b_inner, stride_c_outer, stride_c_inner,
                        CACTI_B200_TRI_NONE, 0, 0, dtype, workspace, workspace_bytes, stream);
}

int cacti_b200_gemm_strided_batched_tri(cacti_b200_dptr c, cacti_b200_dptr a, cacti_b200_dptr b, int64_t m, int64_t n,
                                        int64_t k, int64_t lda, int64_t ldb, int64_t ldc, int trans_a, int trans_b,
                                        const float* alpha, const float* beta, int64_t batch_outer, int64_t batch_inner,
                                        int64_t stride_a_outer, int64_t stride_a_inner, int64_t stride_b_outer,
                                        int64_t stride_b_inner, int64_t stride_c_outer, int64_t stride_c_inner, int tri_mode,
                                        int64_t diag, int operand_flags, int dtype, cacti_b200_dptr workspace,
                                        size_t workspace_bytes,
                                        cacti_b200_stream stream) {
  if (batch_outer > 0x7fffffffLL || batch_inner > 0x7fffffffLL) return CACTI_B200_ERR_SHAPE;
  return cb::gemm_entry(c, a, b, m, n, k, lda, ldb, ldc, trans_a, trans_b, alpha, beta, (int)batch_outer, (int)batch_inner,
                        stride_a_outer, stride_a_inner, stride_b_outer, stride_b_inner, stride_c_outer, stride_c_inner,
                        tri_mode, diag, operand_flags, dtype, workspace, workspace_bytes, stream);
}
}
