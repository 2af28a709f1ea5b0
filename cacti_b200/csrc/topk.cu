// The largest K logits of each row, sorted, and the row's log of the sum of its exponentials: what a teacher's forward pass
// hands to the distillation loss instead of its whole logits tensor.
//
// No counterpart in the reference (its arg-max, src/librarium/llama.rs:546, is the case K = 1).  Order: larger values first,
// equal values (+0 equals -0) by ascending index, NaN above +inf.
//
// One CTA a row, the row read twice (the second time from L2):
//   pass 1: 512 groups of positions (by thread and lane of a pair) each keep a running maximum, and every warp sums exponentials.
//           The K-th largest of the 512 maxima is a lower bound t of the K-th largest logit (K positions at or above it are known);
//           one warp finds it, or a value just below it, by bisection on counts.
//   pass 2: vectors with a position at or above t are put aside, then these positions, hardly more than K for ordinary rows, are
//           collected and ranked by counting.
// The exponentials are taken against 1; a row whose sum then leaves 2^-60 .. 2^60 (all logits beyond about 41 temperatures from 0) is swept
// once more for its sum: 8192 x 32000 f16 182 us around 0, 252 us around -60.
// Fewer than K groups that hold anything (16-bit rows of fewer than 16 K words read by 1024 threads): the bound is -inf, and the exact
// search below runs on ordinary rows too: 4 x 3000 with K = 256 61 us, with K = 64 12 us.
// More than kTopkCap of them: with many equal to t (few distinct values, masks) only those above t are collected, and the first
// positions equal to t fill the rest in index order.  More than kTopkCap above t (values arranged against the kernel's order): the
// exact K-th largest is found by bisection over the whole row, and at most K - 1 lie above that.  Nothing depends on the order in
// which positions are collected.
//
// Bound: the logits read once, 8192 x 32000 f16: 0.52 GB, 81 us at the measured copy rate.  Measured 171 us (3.1 TB/s, 0.47; DRAM reads
// 1.00 of the row bytes, so the second pass does come from L2), 1001 x 50001 f32 62 us, one row of 32000 9 us.  Issue slots are 57 percent
// busy and the exponentials' unit 41 percent; the rest is the serial part of a row (search of the bound, hits, ranking: about 3 us)
// that six CTAs on an SM do not hide completely.  A search by eight warps instead of one took 239 us, a bulk prefetch of the next row into
// L2 211 us (against 184 us at that step).
#include "row_vec.cuh"

namespace cb {

constexpr int kTopkMaxK = 256;
constexpr int64_t kTopkMaxVocab = 1 << 18;
constexpr int kTopkCap = 1024;
constexpr int kTopkGroups = 512;

__device__ __forceinline__ unsigned order_key(float v) {
  if (v != v) return 0xffffffffu;
  const unsigned b = __float_as_uint(v == 0.f ? 0.f : v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_value(unsigned key) {                    // of a key that is no NaN's
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// f(vector, index) for every whole vector of the row, UN at a time, all their loads first; f1(j) for the elements of the vectors at
// its edges that belong to it, one a thread.
template <typename T, int THREADS, int UN, typename F, typename F1>
__device__ __forceinline__ void topk_sweep(const RowVecs<T>& rv, int V, int t, F&& f, F1&& f1) {
  constexpr int VEC = Elem<T>::VEC;
  const int ilo = rv.head ? 1 : 0, ihi = rv.nvec * VEC - rv.head > V ? rv.nvec - 1 : rv.nvec;
  const uint4* p = reinterpret_cast<const uint4*>(rv.base);
  int i = ilo + t;
#pragma unroll 1
  for (; i + (UN - 1) * THREADS < ihi; i += UN * THREADS) {
    uint4 v[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) v[u] = __ldg(p + i + u * THREADS);
#pragma unroll
    for (int u = 0; u < UN; ++u) f(v[u], i + u * THREADS);
  }
#pragma unroll 1
  for (; i < ihi; i += THREADS) f(__ldg(p + i), i);
  if (t < 2 * VEC) {
    // vector 0, and the last one where it is another
    const bool tail = t >= VEC;
    const int v = tail ? rv.nvec - 1 : 0, j = v * VEC - rv.head + (tail ? t - VEC : t);
    if ((v < ilo || v >= ihi) && !(tail && v == 0) && j >= 0 && j < V) f1(j);
  }
}

// The largest value of T below t; NaN below -inf, with which every value compares as not less or equal.
template <typename T> __device__ __forceinline__ float topk_below(float t) {
  if (t == 0.f) t = 0.f;                                       // of -0 and +0 alike: the smallest negative number
  if (t == -INFINITY) return __int_as_float(0x7fc00000);
  if constexpr (sizeof(T) == 2) {
    const T v = Elem<T>::from_f32(t);
    unsigned short b = *reinterpret_cast<const unsigned short*>(&v);
    b = b == 0 ? 0x8001 : (b & 0x8000u) ? b + 1 : b - 1;
    return Elem<T>::to_f32(*reinterpret_cast<const T*>(&b));
  } else {
    const unsigned b = __float_as_uint(t);
    return __uint_as_float(b == 0 ? 0x80000001u : (b & 0x80000000u) ? b + 1 : b - 1);
  }
}

// Any element of the vector above t, or NaN?
template <typename T> __device__ __forceinline__ bool topk_any(const uint4& v, float t) {
  if constexpr (sizeof(T) == 2) {
    using P2 = typename Pair16<T>::type;
    const P2* q = reinterpret_cast<const P2*>(&v);
    const P2 t2{Elem<T>::from_f32(t), Elem<T>::from_f32(t)};                    // exact: t is a logit
    return (__hgtu2_mask(q[0], t2) | __hgtu2_mask(q[1], t2) | __hgtu2_mask(q[2], t2) | __hgtu2_mask(q[3], t2)) != 0u;
  } else {
    float x[4];
    unpack<float>(v, x);
    return !(x[0] <= t) || !(x[1] <= t) || !(x[2] <= t) || !(x[3] <= t);
  }
}
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1536 / THREADS)
logits_topk_kernel(T* __restrict__ values, int* __restrict__ indices, float* __restrict__ lse, const T* __restrict__ L,
                   int rows, int V, int K, double inv_temp) {
  constexpr int VEC = Elem<T>::VEC, NW = THREADS / 32;
  __shared__ float s_max[kTopkGroups];
  __shared__ uint4 s_hit[kTopkCap];                            // vectors that hold a candidate ...
  __shared__ int s_hit_at[kTopkCap];                           // ... and their indices
  // candidates: key, then the complement of the index (18 bits; larger is earlier), then 1 for -0
  __shared__ alignas(16) unsigned long long s_cand[kTopkCap + 8];
  __shared__ float s_red[33];
  __shared__ float s_z[NW];                                    // a warp's sum of exponentials
  __shared__ int s_n, s_hits, s_warp[NW];
  __shared__ float s_t;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const float c = (float)(inv_temp * 1.4426950408889634);
  for (int row = blockIdx.x; row < rows; row += gridDim.x) {
    // exponentials are 2^(x c + off), off a whole number: 0, and where the sum leaves its range it is formed once more with the off
    // that suits the row's maximum.  (The off of the row before would spare rows of large logits that second sum, but a row's last bits
    // would then depend on its neighbours.)
    float off = 0.f;
    const T* x = L + (int64_t)row * V;
    const RowVecs<T> rv(x, V);
    // ---- pass 1 ----
    const float2 c2 = make_float2(c, c);
    float2 off2 = make_float2(off, off);
    float2 zq[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    float2 mx = make_float2(-INFINITY, -INFINITY);
    using P2 = typename Pair16<T>::type;
    P2 mp = Pair16<T>::neg_inf();
    auto take1 = [&](int j) {
      const float a = Elem<T>::to_f32(x[j]);
      mx.x = fmaxf(mx.x, a);
      if (lse) zq[0].x += exp2f_approx(fmaf(a, c, off));
    };
    auto take = [&](const uint4& v, int) {
      if constexpr (sizeof(T) == 2) {
        const P2* q = reinterpret_cast<const P2*>(&v);
        mp = __hmax2(mp, __hmax2(__hmax2(q[0], q[1]), __hmax2(q[2], q[3])));
      } else {
        float a[4];
        unpack<float>(v, a);
        mx.x = fmaxf(mx.x, fmaxf(a[0], a[2]));
        mx.y = fmaxf(mx.y, fmaxf(a[1], a[3]));
      }
      if (lse) {
        float a[VEC];
        unpack<T>(v, a);
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) {
          float2 y = fma2(make_float2(a[2 * e], a[2 * e + 1]), c2, off2);
          y.x = exp2f_approx(y.x);
          y.y = exp2f_approx(y.y);
          zq[e & 1] = add2(zq[e & 1], y);
        }
      }
    };
    float z = 0.f;
    for (int attempt = 0;; ++attempt) {
      topk_sweep<T, THREADS, 4>(rv, V, t, take, take1);
      if constexpr (sizeof(T) == 2) mx = make_float2(fmaxf(mx.x, Elem<T>::to_f32(mp.x)), fmaxf(mx.y, Elem<T>::to_f32(mp.y)));
      if constexpr (THREADS == 256) { s_max[t] = mx.x; s_max[256 + t] = mx.y; }
      else {
        float m = fmaxf(mx.x, mx.y);
        if constexpr (THREADS == 1024) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        if (THREADS == 512 || (t & 1) == 0) s_max[THREADS == 512 ? t : t >> 1] = m;
      }
      if (lse) {
        const float2 zz = add2(zq[0], zq[1]);
        const float zw = warp_reduce<SumOp>(zz.x + zz.y);
        if (lane == 0) s_z[warp] = zw;
      }
      if (t == 0) { s_n = 0; s_hits = 0; }
      __syncthreads();
      if (!lse) break;
      z = 0.f;
      for (int u = 0; u < NW; ++u) z += s_z[u];
      if (attempt || (z > 8.6736174e-19f && z < 1.1529215e18f)) break;            // 2^-60, 2^60
      float m = -INFINITY;
      for (int u = t; u < kTopkGroups; u += THREADS) m = fmaxf(m, s_max[u]);
      m = block_reduce<MaxOp>(m, s_red);
      if (!(fabsf(m * c) < 4194304.f)) break;                    // infinite, or near the type's largest magnitudes: below
      off = -rintf(m * c);
      off2 = make_float2(off, off);
      zq[0] = zq[1] = make_float2(0.f, 0.f);
      __syncthreads();
    }
    if (warp == 0) {
      // ---- a lower bound of the K-th largest: three thresholds a step, their counts in one word ----
      constexpr int PER = kTopkGroups / 32;
      unsigned key[PER];
      unsigned kmin = 0xffffffffu, kmax = 0u;
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        key[u] = order_key(s_max[u * 32 + lane]);
        kmin = key[u] < kmin ? key[u] : kmin;
        kmax = key[u] > kmax ? key[u] : kmax;
      }
      unsigned lo = __reduce_min_sync(0xffffffffu, kmin), hi = __reduce_max_sync(0xffffffffu, kmax);
      // K of the maxima are always at or above `lo` (K <= 512, and empty groups count as -inf), fewer above `hi`
      while (lo < hi) {
        const unsigned d = hi - lo;
        const unsigned m1 = lo + d / 4 + 1 <= hi ? lo + d / 4 + 1 : hi, m2 = lo + d / 2 + 1 <= hi ? lo + d / 2 + 1 : hi;
        const unsigned m3 = lo + d / 2 + d / 4 + 1 <= hi ? lo + d / 2 + d / 4 + 1 : hi;
        unsigned n = 0;
#pragma unroll
        for (int u = 0; u < PER; ++u) n += (key[u] >= m1 ? 1u : 0u) + (key[u] >= m2 ? 1u << 10 : 0u) + (key[u] >= m3 ? 1u << 20 : 0u);
        n = __reduce_add_sync(0xffffffffu, n);                  // at most 512 each: no carries
        const int n1 = (int)(n & 1023u), n2 = (int)((n >> 10) & 1023u), n3 = (int)(n >> 20);
        int at;
        if (n3 >= K) { lo = m3; at = n3; }
        else if (n2 >= K) { lo = m2; hi = m3 - 1; at = n2; }
        else if (n1 >= K) { lo = m1; hi = m2 - 1; at = n1; }
        else { hi = m1 - 1; continue; }
        if (at <= K + K / 8) break;
      }
      // a logit's own value, so that it converts to T exactly: the smallest of the maxima at or above the bound
      unsigned up = 0xffffffffu;
#pragma unroll
      for (int u = 0; u < PER; ++u) up = key[u] >= lo && key[u] < up ? key[u] : up;
      up = __reduce_min_sync(0xffffffffu, up);
      if (lane == 0) s_t = order_value(up);
    }
    __syncthreads();
    if (lse) {
      float sub = 0.f;
      double ln_off = (double)off * 0.6931471805599453;
      if (!(z > 8.6736174e-19f && z < 1.1529215e18f)) {         // still: against the true maximum, differences first
        float m = -INFINITY;
        for (int u = t; u < kTopkGroups; u += THREADS) m = fmaxf(m, s_max[u]);
        m = block_reduce<MaxOp>(m, s_red);
        sub = isinf(m) ? 0.f : m;                               // no inf - inf: the sum is then 0 or inf
        ln_off = 0.;
        z = 0.f;
        topk_sweep<T, THREADS, 1>(rv, V, t, [&](const uint4& v, int) {
          float a[VEC];
          unpack<T>(v, a);
#pragma unroll
          for (int e = 0; e < VEC; ++e) z += exp2f_approx((a[e] - sub) * c);
        }, [&](int j) { z += exp2f_approx((Elem<T>::to_f32(x[j]) - sub) * c); });
        z = block_reduce<SumOp>(z, s_red);
      }
      if (t == THREADS - 32) lse[row] = (float)(log((double)z) - ln_off + inv_temp * (double)sub);
    }
    // ---- pass 2 ----
    float bound = s_t, above = topk_below<T>(bound);           // collected: what is not less than or equal to `above`
    int n = 0;
    for (int attempt = 0; attempt < 3; ++attempt) {
      auto push = [&](float a, int j) {
        if (!(a <= above)) {
          const int slot = atomicAdd(&s_n, 1);
          if (slot < kTopkCap)
            s_cand[slot] = ((unsigned long long)order_key(a) << 32) | ((0x3ffffu - (unsigned)j) << 1) | (a == 0.f && signbit(a) ? 1u : 0u);
        }
      };
      topk_sweep<T, THREADS, 4>(rv, V, t, [&](const uint4& v, int at) {
        if (topk_any<T>(v, above)) {
          const int slot = atomicAdd(&s_hits, 1);
          if (slot < kTopkCap) { s_hit[slot] = v; s_hit_at[slot] = at; }
        }
      }, [&](int j) { push(Elem<T>::to_f32(x[j]), j); });
      __syncthreads();
      const int hits = s_hits;
      for (int q = t; q < (hits < kTopkCap ? hits : 0) * VEC; q += THREADS)
        push(Elem<T>::to_f32(reinterpret_cast<const T*>(s_hit)[q]), s_hit_at[q / VEC] * VEC - rv.head + q % VEC);
      __syncthreads();
      n = hits > kTopkCap ? hits : s_n;
      if (n <= kTopkCap) break;
      __syncthreads();                                          // everyone has read the counts
      if (t == 0) { s_n = 0; s_hits = 0; }
      __syncthreads();
      above = bound;
      if (attempt == 0) continue;                               // the same bound, without its equals
      // the exact K-th largest: at most K - 1 positions are above it
      unsigned lo = order_key(bound), hi = 0xffffffffu;
      while (lo < hi) {
        const unsigned mid = lo + (hi - lo) / 2 + 1;
        float cnt = 0.f;                                        // counts below 2^24 are exact in f32
        topk_sweep<T, THREADS, 1>(rv, V, t, [&](const uint4& v, int) {
          float a[VEC];
          unpack<T>(v, a);
#pragma unroll
          for (int e = 0; e < VEC; ++e) cnt += order_key(a[e]) >= mid ? 1.f : 0.f;
        }, [&](int j) { cnt += order_key(Elem<T>::to_f32(x[j])) >= mid ? 1.f : 0.f; });
        if (block_reduce<SumOp>(cnt, s_red) >= (float)K) lo = mid;
        else hi = mid - 1;
      }
      // K NaNs or more: the bound is NaN, nothing is above it and its positions are the ties
      bound = lo == 0xffffffffu ? __int_as_float(0x7fc00000) : order_value(lo);
      above = bound;
      if (bound != bound) { n = 0; break; }
    }
    // ---- the candidates in order ----
    auto put = [&](unsigned long long cand, int rank) {
      const unsigned key = (unsigned)(cand >> 32);
      const float v = key == 0xffffffffu ? __int_as_float(0x7fc00000) : (cand & 1ull) ? -0.f : order_value(key);
      values[(int64_t)row * K + rank] = Elem<T>::from_f32(v);
      indices[(int64_t)row * K + rank] = (int)(0x3ffffu - (((unsigned)cand >> 1) & 0x3ffffu));
    };
    if (n <= 160) {
      // few: a candidate's rank is the number of larger ones, its comparisons shared by `parts` neighbouring lanes (n^2 of them:
      // above about 160 sorting is cheaper)
      const int parts = n * 4 <= THREADS ? 4 : n * 2 <= THREADS ? 2 : 1;
      for (int q0 = 0; q0 < n * parts; q0 += THREADS) {         // whole warps take part in the shuffles
        const int q = (q0 + t) / parts, part = t & (parts - 1);
        const unsigned long long own = q < n ? s_cand[q] : ~0ull;
        int rank = 0;
        for (int u = part * 2; u < n; u += 2 * parts) {
          const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(s_cand + u);
          rank += (o.x > own ? 1 : 0) + (u + 1 < n && o.y > own ? 1 : 0);
        }
        if (parts > 1) rank += __shfl_xor_sync(0xffffffffu, rank, 1);
        if (parts > 2) rank += __shfl_xor_sync(0xffffffffu, rank, 2);
        if (q < n && part == 0 && rank < K) put(own, rank);
      }
    } else {
      // a bitonic sort, largest first; 0 is below every candidate
      const int size = n <= 256 ? 256 : n <= 512 ? 512 : 1024;
      for (int q = n + t; q < size; q += THREADS) s_cand[q] = 0ull;
      __syncthreads();
      for (int len = 2; len <= size; len *= 2) {
        for (int gap = len / 2; gap > 0; gap /= 2) {
          for (int q = t; q < size / 2; q += THREADS) {
            const int i = 2 * q - (q & (gap - 1)), j = i + gap;
            const unsigned long long a = s_cand[i], b = s_cand[j];
            if ((a < b) == ((i & len) == 0)) { s_cand[i] = b; s_cand[j] = a; }
          }
          __syncthreads();
        }
      }
      for (int q = t; q < (n < K ? n : K); q += THREADS) put(s_cand[q], q);
    }
    // ---- the first positions equal to the bound, in index order ----
    for (int j0 = 0, have = n; have < K && j0 < V; j0 += THREADS) {
      const int j = j0 + t;
      const float a = j < V ? Elem<T>::to_f32(x[j]) : 0.f;
      const bool tie = j < V && (a == bound || (bound != bound && a != a));
      const unsigned b = __ballot_sync(0xffffffffu, tie);
      if (lane == 0) s_warp[warp] = __popc(b);
      __syncthreads();
      int at = have + __popc(b & ((1u << lane) - 1u)), total = 0;
#pragma unroll
      for (int u = 0; u < NW; ++u) { if (u < warp) at += s_warp[u]; total += s_warp[u]; }
      if (tie && at < K) { values[(int64_t)row * K + at] = x[j]; indices[(int64_t)row * K + at] = j; }
      have += total;
      __syncthreads();
    }
    __syncthreads();
  }
}

template <typename T>
static int launch_topk(uint64_t values, uint64_t indices, uint64_t lse, uint64_t logits, int64_t rows, int64_t vocab, int64_t k,
                       double inv_temp, cudaStream_t st) {
  T* v = reinterpret_cast<T*>(values);
  int* ix = reinterpret_cast<int*>(indices);
  float* ls = reinterpret_cast<float*>(lse);
  const T* l = reinterpret_cast<const T*>(logits);
  // The rows at work have to stay in the 126 MB of L2 between their two passes, and a CTA's serial steps have to be covered by
  // others on its SM: six CTAs an SM for short rows, three for longer ones, one for the longest; one also for few rows, where 1024
  // threads bring a row's bytes sooner.
  const int64_t bytes = vocab * (int64_t)sizeof(T);
  const int64_t per_sm = rows <= kNumSMs || bytes > 200 * 1024 ? 1 : bytes > 80 * 1024 ? 3 : 6;
  const int64_t cap = (int64_t)kNumSMs * per_sm;
  const unsigned grid = (unsigned)(rows < cap ? rows : cap);
  if (per_sm == 1) logits_topk_kernel<T, 1024><<<grid, 1024, 0, st>>>(v, ix, ls, l, (int)rows, (int)vocab, (int)k, inv_temp);
  else if (per_sm == 3) logits_topk_kernel<T, 512><<<grid, 512, 0, st>>>(v, ix, ls, l, (int)rows, (int)vocab, (int)k, inv_temp);
  else logits_topk_kernel<T, 256><<<grid, 256, 0, st>>>(v, ix, ls, l, (int)rows, (int)vocab, (int)k, inv_temp);
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
  if (vocab > kTopkMaxVocab || k > kTopkMaxK || k < 1 || k > vocab || rows > 0x3fffffffLL) return CACTI_B200_ERR_SHAPE;
  if (rows == 0) return CACTI_B200_OK;
  const int es = dtype == CACTI_B200_R_32F ? 4 : 2;
  if (!values || !indices || !logits || values % es || logits % es || (indices & 3) || (lse & 3)) return CACTI_B200_ERR_INVALID_VALUE;
  const Span in{logits, (uint64_t)rows * vocab * es};
  for (const Span& out : {Span{values, (uint64_t)rows * k * es}, Span{indices, (uint64_t)rows * k * 4}, Span{lse, (uint64_t)rows * 4}})
    if (overlap(out, in)) return CACTI_B200_ERR_INVALID_VALUE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dispatch_dtype(dtype, [&](auto tag) -> int {
    return launch_topk<decltype(tag)>(values, indices, lse, logits, rows, vocab, k, 1.0 / (double)temperature, st);
  });
}
}
