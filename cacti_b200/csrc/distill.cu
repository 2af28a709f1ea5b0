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
//
// Bound: logits read and gradient written once, 8192 x 32000 f16: 1.05 GB, 162 us at the measured copy rate.  Measured 218 us with a list
// of 64 (4.8 TB/s, 0.74 of that rate); 2048 x 131072 bf16 325 us with its clusters (3.3 TB/s, 0.51); a reading of each logit in three
// sweeps, as softmax_nll does it, and lists handled by the same warps took 2.32 ms.  What is left is not bandwidth: a row's phases
// follow one another (listed logits out of the row, exponentials and sum, gradient, listed positions, copy out), and with one
// row in work a CTA and two waiting the instruction issue is a third busy.  Shared memory holds no fourth row of 64 KB.
// Other forms, 8192 x 32000 f16 with a list of 64: forward only 146 us; Accumulate mode 568 us (the old values are loaded where they are
// needed, nothing ahead).  Where gradient and logits start at different places in a 16-byte vector, a list warp copies the row out by
// elements: 443 us, 6.6 ms in Accumulate mode.  f32 rows above about 135000 words have one slot and form their exponentials twice:
// 1024 x 151936 697 us (0.28 of the copy rate), 1024 x 131072 265 us (0.63).
#include "row_vec.cuh"
#include <type_traits>

namespace cb {

constexpr int kDistillMaxK = 256;
constexpr int64_t kDistillMaxVocab = 1 << 18;

int g_distill_part = 4096;     // 16-byte vectors of a row that one CTA takes at most (launch_distill)

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

__device__ __forceinline__ float teacher_value(const DistillParams& p, int64_t i) {
  if (p.t_dtype == CACTI_B200_R_32F) return reinterpret_cast<const float*>(p.t_values)[i];
  if (p.t_dtype == CACTI_B200_R_16F) return __half2float(reinterpret_cast<const __half*>(p.t_values)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.t_values)[i]);
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

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Roles of a CTA (a cluster of C CTAs shares a row, each a run of its vectors):
//   list warps, one per ring slot: fetch the slot's row (bulk copy), turn the teacher's list into probabilities, take the listed
//     student logits out of the staged row (they become -inf there), and, when the row's gradient lies in the slot, put the listed
//     positions' gradient in, send it off (bulk copy) and write the loss;
//   MW main warps: maximum and exponentials of the unlisted positions, one combination of (maximum, sum) over the CTA and the
//     cluster, then gradient = exponential times a factor, written over the staged row.
// NV > 0: a CTA's part of a row is at most MW * 32 * NV vectors: the exponentials stay in registers, one a position.  NV = 0: they are
// formed again for the gradient.
constexpr int kDistillMaxC = 8;
constexpr int kDistillSeen = 512;                              // words of a list's index filter
// What exponentials are taken against: e(x) = 2^((x - sub) c + off).  Ordinarily sub = 0 and off = -(a large logit times c,
// rounded to a whole number): one multiply-add an exponential, and two references differ by an exact power of two.  Where that
// product is no longer a small whole number (rows near the type's largest magnitudes) sub is the row's maximum and off = 0.
struct DistillRef { float sub, off; };
struct DistillRow {              // from the list warp to the main warps
  DistillRef ref;                // from the listed logits and a sample of the others; off = NaN: none to be had
  int skip;                      // weight 0
  double z_top;                  // sum of the listed exponentials (of this CTA's vectors)
  double g_mass, g_r;            // w c P and w c r
  double px, pown;               // sum of p log2 e(x) and of p over this CTA's listed positions
};
// A sum of exponentials under its reference.  Listed and unlisted positions keep references of their own until the end: where
// the list holds nearly everything, the rest is still known.  f64 from a warp's sum on, and the listed exponentials are f64 (good to
// 3e-10 for the c they are given; c itself is f32, the same for listed and unlisted positions: the temperature is off by up to 2^-24
// relative).  Near the teacher both the loss and the gradient are small differences, in which the errors of single exponentials average
// out or are multiplied by a difference, but an error of the whole sum is not.
struct alignas(16) DistillSum { DistillRef ref; double z; };
struct DistillFin { DistillRef ref; double z_all, z_rest, shift_rest, px; };             // back to the list warp
struct alignas(16) DistillRec { DistillSum rest, top; double px, pown; };  // a CTA's part of a row, to the cluster

template <int MW, int R> struct alignas(16) DistillSmem {
  uint64_t full[R], marked[R], stored[R];
  uint64_t rec_bar[2];
  DistillRec rec[2][kDistillMaxC];
  double red[2][MW];
  DistillRow row[R];
  DistillFin fin[R];
  alignas(16) unsigned seen[R][kDistillSeen];
};
// behind it: a list a slot, then the ring
struct DistillList {             // KP = k rounded up to 32 entries of each
  double* p;                     // scaled teacher logit, later the probability
  float* x;                      // listed student logit, where it is in this CTA's part
  int* idx;                      // -1: no entry
};
constexpr unsigned kDistillListBytes = 16;                     // per entry

__device__ __forceinline__ uint32_t distill_ctarank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t distill_nctas() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void distill_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool distill_wait_cluster(uint64_t* bar, unsigned parity) {
  for (unsigned it = 0; it < kMbarPolls; ++it) {
    unsigned ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(g_mbar_suspend_ns) : "memory");
    if (ok) return true;
  }
  atomicMax(&g_dev_error, kDevErrStageTimeout);
  return false;
}

__device__ __forceinline__ float distill_arg(float x, const DistillRef& r, float c) { return fmaf(x - r.sub, c, r.off); }
__device__ __forceinline__ float distill_exp(float x, const DistillRef& r, float c) { return exp2f_approx(distill_arg(x, r, c)); }
// The reference for a largest logit m.
__device__ __forceinline__ DistillRef distill_ref(float m, float c) {
  const float a = m * c;
  return fabsf(a) < 4194304.f ? DistillRef{0.f, -rintf(a)} : DistillRef{m, 0.f};
}
// log2 of e under a over e under b; positive where b's logits are the larger ones
__device__ __forceinline__ double distill_shift64(const DistillRef& a, const DistillRef& b, float c) {
  return ((double)b.sub - (double)a.sub) * (double)c + ((double)a.off - (double)b.off);
}
// 2^s, exact for whole numbers
__device__ __forceinline__ double distill_pow2(double s) {
  return s == rint(s) && fabs(s) < 1000. ? __hiloint2double(((int)s + 1023) << 20, 0) : exp2(s);
}
// a + b under the larger reference
__device__ __forceinline__ DistillSum distill_add(const DistillSum& a, const DistillSum& b, float c) {
  if (a.z == 0.) return b;
  if (b.z == 0.) return a;
  const double s = distill_shift64(a.ref, b.ref, c);
  if (s > 0.) return DistillSum{b.ref, a.z * distill_pow2(-s) + b.z};
  return DistillSum{a.ref, b.z * distill_pow2(s) + a.z};
}

// CTA-wide sum or maximum over the main warps, on barrier 1; `any` ORs a flag on the way.  A sum is f32 inside a warp and f64 from there on:
// the roundings of the warps' sums average out (below 2^-25 of the sum), those of a last f32 addition would not.
template <int MW> __device__ __forceinline__ bool distill_meet(bool any) {
  unsigned r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %2, 0;\n\tbar.red.or.pred p, 1, %1, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r) : "n"(MW * 32), "r"((unsigned)any) : "memory");
  return r != 0;
}
template <int MW> __device__ __forceinline__ double distill_sum(float z, double (&red)[MW], int warp, int lane, bool& any) {
  z = warp_reduce<SumOp>(z);
  if (lane == 0) red[warp] = (double)z;
  any = distill_meet<MW>(any);
  double s[2] = {red[0], red[1]};
#pragma unroll
  for (int i = 2; i < MW; ++i) s[i & 1] += red[i];
  return s[0] + s[1];
}
template <int MW> __device__ __forceinline__ float distill_max(float m, double (&red)[MW], int warp, int lane, bool& any) {
  m = warp_reduce<MaxOp>(m);
  if (lane == 0) red[warp] = (double)m;
  any = distill_meet<MW>(any);
#pragma unroll
  for (int i = 0; i < MW; ++i) m = fmaxf(m, (float)red[i]);
  return m;
}
// a / b to about 1e-11: the hardware's reciprocal estimate (20 bits) and one Newton step.  NaN where b is 0 or infinite.
__device__ __forceinline__ double quotient(double a, double b) {
  double r;
  asm("rcp.approx.ftz.f64 %0, %1;" : "=d"(r) : "d"(b));
  return a * fma(r, fma(-b, r, 1.), r);
}

template <typename T> __device__ __forceinline__ void distill_put(T* o, float v, int beta) {
  *o = beta ? Elem<T>::from_f32(Elem<T>::to_f32(*o) + round_to<T>(v)) : Elem<T>::from_f32(v);
}

// What a list warp knows of a row.
struct DistillHead { float w; double psum, ent, r; bool bad; };

// exp(d) to 3e-10 relative: 2^n times the Taylor series of exp(f ln2), |f| <= 1/2, to the eighth power (the next term is
// (ln2 / 2)^9 / 9! = 2e-10, and the series is at least 0.7).  A third of the latency of the library's, which a single warp does not hide.  The f32 functions
// would do for ordinary rows; where the student gives a listed word a logit of -65504, the loss shows their 1e-7.
__device__ __forceinline__ double exp_list(double d) {
  const double y = d * 1.4426950408889634;
  if (!(y > -1000.)) return y != y ? y : 0.;
  if (y > 1000.) return INFINITY;
  const double n = rint(y), x = (y - n) * 0.6931471805599453;
  double s = 1. / 40320.;
  s = fma(s, x, 1. / 5040.);
  s = fma(s, x, 1. / 720.);
  s = fma(s, x, 1. / 120.);
  s = fma(s, x, 1. / 24.);
  s = fma(s, x, 1. / 6.);
  s = fma(s, x, 0.5);
  s = fma(s, x, 1.);
  s = fma(s, x, 1.);
  return s * __hiloint2double(((int)n + 1023) << 20, 0);
}

// ln z to 3e-10 absolute: the f32 logarithm and one Newton step on exp_list, whose error passes on.
__device__ __forceinline__ double log_list(double z) {
  const float y = logf((float)z);
  if (!(fabsf(y) < 80.f)) return log(z);                        // 0, infinities, NaN, the ends of f32's range
  const double d = fma(z, exp_list(-(double)y), -1.);
  return (double)y + d - 0.5 * d * d;
}

// What is fetched of a row's list ahead of its preparation: the weight, the teacher's lse and the first two entries of each lane.
struct DistillAhead { float w, lse; int id[2]; float z[2]; };
__device__ __forceinline__ void distill_fetch(const DistillParams& p, int64_t row, int lane, DistillAhead& f) {
  f.w = p.w_rows ? p.w_rows[row] : p.w_scalar;
  f.lse = p.t_lse ? p.t_lse[row] : 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int k = i * 32 + lane;
    f.id[i] = -1; f.z[i] = 0.f;
    if (k < p.k) { f.id[i] = teacher_index(p, row * p.k + k); f.z[i] = teacher_value(p, row * p.k + k); }
  }
}

// Prepare the list of `row`: indices and validity, probabilities, their sums.
__device__ __forceinline__ void distill_prepare(const DistillParams& p, int64_t row, const DistillAhead& f, const DistillList& li,
                                                unsigned* seen, int KP, int lane, DistillHead& h) {
  h.w = f.w;
  h.psum = h.ent = h.r = 0.;
  h.bad = false;
  if (h.w == 0.f) return;
#pragma unroll
  for (int i = 0; i < kDistillSeen / 128; ++i) reinterpret_cast<uint4*>(seen)[i * 32 + lane] = make_uint4(0, 0, 0, 0);
  __syncwarp();
  // An index listed twice: of two equal ones at least one finds its bit in the filter set; only groups of 32 slots with such a
  // one are compared with the whole list.
  bool bad = false;
  unsigned suspects = 0;                                        // bit i: group i
#pragma unroll 1
  for (int i = 0; i * 32 < KP; ++i) {
    const int k = i * 32 + lane;
    int id = -1;
    float z = 0.f;
    if (i < 2) { id = i ? f.id[1] : f.id[0]; z = i ? f.z[1] : f.z[0]; }
    else if (k < p.k) { id = teacher_index(p, row * p.k + k); z = teacher_value(p, row * p.k + k); }
    bad |= id == -2;
    bool suspect = false;
    if (id >= 0) {
      const unsigned hash = ((unsigned)id * 2654435761u) >> 18;                 // 14 bits
      const unsigned bit = 1u << (hash & 31);
      suspect = (atomicOr(seen + (hash >> 5), bit) & bit) != 0;
    }
    if (__any_sync(0xffffffffu, suspect)) suspects |= 1u << i;
    li.idx[k] = id < 0 ? -1 : id;
    li.p[k] = id < 0 ? -INFINITY : p.inv_temp * (double)z;
  }
  __syncwarp();
  if (suspects) {
    bool twice = false;
#pragma unroll 1
    for (int i = 0; i * 32 < KP; ++i) {
      if (!((suspects >> i) & 1u)) continue;
      const int own = li.idx[i * 32 + lane];
      int hits = 0;
#pragma unroll 2
      for (int j = 0; j < KP; j += 4) {
        const int4 o = *reinterpret_cast<const int4*>(li.idx + j);
        hits += (o.x == own) + (o.y == own) + (o.z == own) + (o.w == own);
      }
      twice |= own >= 0 && hits > 1;
    }
    if (__any_sync(0xffffffffu, twice)) {                       // every slot but the first of its index goes
      bad = true;
#pragma unroll 1
      for (int k = lane; k < KP; k += 32) {
        bool earlier = false;
        for (int j = 0; j < k; ++j) earlier |= li.idx[j] == li.idx[k];
        li.x[k] = earlier ? 1.f : 0.f;
      }
      __syncwarp();
      for (int k = lane; k < KP; k += 32) if (li.x[k] != 0.f) { li.idx[k] = -1; li.p[k] = -INFINITY; }
      __syncwarp();
    }
  }
  h.bad = __any_sync(0xffffffffu, bad);
  double lse_t = (double)f.lse;
  int cnt = 0;
  if (p.t_lse) {
#pragma unroll 1
    for (int k = lane; k < KP; k += 32) cnt += li.idx[k] >= 0;
    cnt = __reduce_add_sync(0xffffffffu, cnt);
  } else {
    double zm = -INFINITY;
#pragma unroll 1
    for (int k = lane; k < KP; k += 32) { const double z = li.p[k]; zm = z > zm || z != z ? z : zm; }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { const double v = __shfl_xor_sync(0xffffffffu, zm, o); zm = v > zm || v != v ? v : zm; }
    double e = 0.;
#pragma unroll 1
    for (int k = lane; k < KP; k += 32) if (li.p[k] != -INFINITY) e += exp_list(li.p[k] - zm);
    lse_t = zm + log_list(warp_sum_f64(e));
  }
#pragma unroll 1
  for (int k = lane; k < KP; k += 32) {
    const double z = li.p[k];
    double pk = 0.;
    if (z != -INFINITY) {
      pk = exp_list(z - lse_t);
      h.psum += pk;
      if (pk != 0.) h.ent += pk * (z - lse_t);
    }
    li.p[k] = pk;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    h.psum += __shfl_xor_sync(0xffffffffu, h.psum, o);
    h.ent += __shfl_xor_sync(0xffffffffu, h.ent, o);
  }
  if (p.t_lse && cnt && cnt < p.vocab) h.r = fmax(0., 1. - h.psum);
}

// CTAs an SM is to hold: by registers (NV * 8 exponentials and about 30 more a thread), each scheduler's 16384 shared by its warps
constexpr int distill_residency(int MW, int R, int NV) { return NV == 0 || MW * NV > 64 ? 1 : MW * NV > 32 ? 2 : 3; }

enum { kDistillFwd = 0, kDistillBwd = 1, kDistillAcc = 2 };

template <typename T, int MW, int R, int NVH, int MODE>
__global__ void __launch_bounds__((MW + R) * 32, distill_residency(MW, R, NVH))
distill_kernel(T* __restrict__ dL, const T* __restrict__ L, const __grid_constant__ DistillParams p, unsigned slot_bytes) {
  constexpr int VEC = Elem<T>::VEC, MT = MW * 32;
  constexpr bool BWD = MODE != kDistillFwd;
  constexpr int beta = MODE == kDistillAcc;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  using Smem = DistillSmem<MW, R>;
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int KP = (p.k + 31) / 32 * 32;
  unsigned char* lists = smem_raw + sizeof(Smem);
  unsigned char* ring = smem_raw + (sizeof(Smem) + (size_t)R * KP * kDistillListBytes + 127) / 128 * 128;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, V = p.vocab;
  const int C = (int)distill_nctas(), rank = (int)distill_ctarank();
  const int rows = (int)p.rows, row0 = (int)blockIdx.x / C, stride = (int)gridDim.x / C;
  const float c = (float)(p.inv_temp * 1.4426950408889634);
  if (threadIdx.x == 0) {
    for (int s = 0; s < R; ++s) { mbar_init(sm.full + s, 1); mbar_init(sm.marked + s, 1); mbar_init(sm.stored + s, MW); }
    for (int i = 0; i < 2; ++i) mbar_init(sm.rec_bar + i, 1);
    mbar_fence_init();
  }
  __syncthreads();
  if (C > 1) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");

  if (warp >= MW) {
    // ---------------- list warp of slot s ----------------
    const int s = warp - MW;
    T* sx = reinterpret_cast<T*>(ring + (size_t)s * slot_bytes);
    const uint64_t t_begin = reinterpret_cast<uint64_t>(L), t_end = t_begin + (uint64_t)p.rows * V * sizeof(T);
    unsigned char* at0 = lists + (size_t)s * KP * kDistillListBytes;
    const DistillList li{reinterpret_cast<double*>(at0), reinterpret_cast<float*>(at0 + 8 * KP), reinterpret_cast<int*>(at0 + 12 * KP)};
    // fetch a row's vectors of this CTA; whole vectors inside the tensor only
    auto issue = [&](int row) {
      if (lane == 0) {
        const RowVecs<T> rv(L + (int64_t)row * V, V);
        const int v0 = rv.nvec * rank / C, v1 = rv.nvec * (rank + 1) / C;
        const unsigned char *a = rv.base + (size_t)v0 * 16, *b = rv.base + (size_t)v1 * 16;
        unsigned skip = 0;
        if (reinterpret_cast<uint64_t>(a) < t_begin) { a += 16; skip = 16; }
        if (reinterpret_cast<uint64_t>(b) > t_end) b -= 16;
        const unsigned bytes = b > a ? (unsigned)(b - a) : 0u;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // marks in the slot before the copy over them
        mbar_expect_tx(sm.full + s, bytes);
        if (bytes) bulk_g2s(reinterpret_cast<unsigned char*>(sx) + skip, a, bytes, sm.full + s);
      }
    };
    unsigned ph = 0, full_ph = 0;                               // rows of weight 0 do not pass through `full`
    DistillHead h;
    DistillAhead ahead;
    int row = row0 + s * stride;
    if (row < rows) {
      distill_fetch(p, row, lane, ahead);
      if (ahead.w != 0.f) issue(row);
      distill_prepare(p, row, ahead, li, sm.seen[s], KP, lane, h);
    }
    // vectors of gradient and logits coincide: whole vectors leave by bulk copy, otherwise the slot is copied out by element
    const bool same = ((reinterpret_cast<uint64_t>(dL) ^ reinterpret_cast<uint64_t>(L)) & 15) == 0;
    for (; row < rows; row += R * stride) {
      const bool skip = h.w == 0.f;
      const RowVecs<T> rv(L + (int64_t)row * V, V);
      const int v0 = rv.nvec * rank / C, n = rv.nvec * (rank + 1) / C - v0;
      const int j0 = v0 * VEC - rv.head, j1 = j0 + n * VEC;                  // row elements of this CTA: [j0, j1)
      const int ilo = j0 < 0 ? 1 : 0, ihi = j1 > V ? n - 1 : n;              // vectors [ilo, ihi) lie wholly inside the row
      DistillRef ref{0.f, 0.f};                                 // of the listed exponentials
      if (!skip) {
        // ---- the listed logits out of the staged row ----
        if (!mbar_wait_bounded_warp(sm.full + s, full_ph, kDevErrStageTimeout)) break;
        full_ph ^= 1u;
        if (lane < VEC) {
          // foreign elements, and edge vectors that were not copied because they reach outside the tensor
          for (int side = 0; side < 2; ++side) {
            const int i = side ? n - 1 : 0;
            if (i < 0 || (side && i == 0) || (i >= ilo && i < ihi)) continue;
            const uint64_t a = reinterpret_cast<uint64_t>(rv.base) + (uint64_t)(v0 + i) * 16;
            const int j = j0 + i * VEC + lane;
            if (j < 0 || j >= V) sx[i * VEC + lane] = Elem<T>::from_f32(-INFINITY);
            else if (a < t_begin || a + 16 > t_end) sx[i * VEC + lane] = L[(int64_t)row * V + j];
          }
        }
        __syncwarp();
        // a large logit of this part: the listed ones, and one vector a lane of the rest
        float mt = -INFINITY;
        for (int k = lane; k < KP; k += 32) {
          const int id = li.idx[k];
          float x = -INFINITY;
          if (id >= 0 && id >= j0 && id < j1) { x = Elem<T>::to_f32(sx[id - j0]); sx[id - j0] = Elem<T>::from_f32(-INFINITY); }
          li.x[k] = x;
          mt = fmaxf(mt, x);
        }
        if (n > 0) {
          float x[VEC];
          unpack<T>(reinterpret_cast<const uint4*>(sx)[lane * n / 32], x);
#pragma unroll
          for (int e = 0; e < VEC; ++e) mt = fmaxf(mt, x[e]);
        }
        mt = warp_reduce<MaxOp>(mt);
        ref = isinf(mt) ? DistillRef{0.f, 0.f} : distill_ref(mt, c);
        double zt = 0., px = 0., pown = 0.;
        for (int k = lane; k < KP; k += 32) {
          const float x = li.x[k];
          const int id = li.idx[k];
          const double arg = ((double)x - (double)ref.sub) * (double)c + (double)ref.off, ek = exp_list(arg * 0.6931471805599453);
          zt += ek;
          li.x[k] = (float)ek;                                  // from here on the exponential
          const double pk = id >= j0 && id < j1 && id >= 0 ? li.p[k] : 0.;
          if (pk != 0.) { pown += pk; px += pk * arg; }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          zt += __shfl_xor_sync(0xffffffffu, zt, o);
          px += __shfl_xor_sync(0xffffffffu, px, o);
          pown += __shfl_xor_sync(0xffffffffu, pown, o);
        }
        if (lane == 0) {
          const double wc = (double)h.w * p.inv_temp;
          // without a usable sample the main warps look for the maximum themselves
          sm.row[s] = DistillRow{DistillRef{ref.sub, isinf(mt) ? __int_as_float(0x7fc00000) : ref.off}, 0, zt, wc * (h.psum + h.r), wc * h.r, px, pown};
        }
      } else if (lane == 0) {
        sm.row[s] = DistillRow{DistillRef{0.f, 0.f}, 1, 0., 0., 0., 0., 0.};
      }
      __syncwarp();
      if (lane == 0) distill_arrive(sm.marked + s);
      const int next = row + R * stride;
      if (next < rows) distill_fetch(p, next, lane, ahead);      // used once this row is out of the slot
      // ---- the row's gradient is in the slot: listed positions, off with it, loss ----
      if (!mbar_wait_bounded_warp(sm.stored + s, ph, kDevErrStageTimeout)) break;
      ph ^= 1u;
      if (skip) {
        if (lane == 0 && rank == 0 && p.loss_rows) p.loss_rows[row] = 0.f;
        if (next < rows) {
          if (ahead.w != 0.f) issue(next);
          distill_prepare(p, next, ahead, li, sm.seen[s], KP, lane, h);
        }
        continue;
      }
      const DistillFin f = sm.fin[s];
      const double mass = h.psum + h.r;
      if (BWD) {
        T* dpart = dL + (int64_t)row * V + j0;
        const double wc = (double)h.w * p.inv_temp;
        const double ga = quotient(wc * mass, f.z_all) * (f.ref.off == ref.off && f.ref.sub == ref.sub ? 1. : distill_pow2(distill_shift64(f.ref, ref, c)));
        for (int k = lane; k < KP; k += 32) {
          const int at = li.idx[k] - j0;
          if (li.idx[k] >= 0 && at >= 0 && at < j1 - j0) {
            // (in Accumulate mode the old value is there already, unless it is added when the element is copied out)
            const int i = at / VEC;
            distill_put<T>(sx + at, mass != 0. ? (float)(ga * (double)li.x[k] - wc * li.p[k]) : 0.f, beta && same && i >= ilo && i < ihi);
          }
        }
        __syncwarp();
        if (same) {
          if (lane < VEC) {
            for (int side = 0; side < 2; ++side) {
              const int i = side ? n - 1 : 0;
              if (i < 0 || (side && i == 0) || (i >= ilo && i < ihi)) continue;
              const int e = i * VEC + lane;
              if (j0 + e >= 0 && j0 + e < V) distill_put<T>(dpart + e, Elem<T>::to_f32(sx[e]), beta);
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0 && ihi > ilo) {
            bulk_s2g(dpart + ilo * VEC, sx + ilo * VEC, (unsigned)(ihi - ilo) * 16u);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {
          const int e0 = j0 < 0 ? -j0 : 0, e1 = j1 > V ? V - j0 : j1 - j0;
          for (int e = e0 + lane; e < e1; e += 32) distill_put<T>(dpart + e, Elem<T>::to_f32(sx[e]), beta);
          __syncwarp();
        }
      }
      if (row % C == rank && p.loss_rows) {                     // the CTAs of a cluster take turns
        // the three logarithms side by side
        const double lg = log_list(lane == 0 ? f.z_all : lane == 1 ? h.r : f.z_rest);
        const double la = __shfl_sync(0xffffffffu, lg, 0), lr = __shfl_sync(0xffffffffu, lg, 1), lz = __shfl_sync(0xffffffffu, lg, 2);
        if (lane == 0) {
          double loss = mass != 0. ? h.ent - 0.6931471805599453 * f.px + h.psum * la : 0.;
          if (h.r > 0.) loss += h.r * (lr - lz - 0.6931471805599453 * f.shift_rest + la);
          p.loss_rows[row] = h.bad ? __int_as_float(0x7fc00000) : (float)loss;
        }
      }
      if (lane == 0 && rank == 0 && h.bad && p.status) atomicMax(p.status, (unsigned)CACTI_B200_ERR_INDEX_RANGE);
      // the slot may be filled again once the copy out has read it
      if (BWD && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      __syncwarp();
      if (next < rows) {
        if (ahead.w != 0.f) issue(next);
        distill_prepare(p, next, ahead, li, sm.seen[s], KP, lane, h);       // while the row is on its way
      }
    }
    if (BWD && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  } else {
    // ---------------- main warps ----------------
    const int t = threadIdx.x;
    int s = 0;
    unsigned ph = 0, par = 0, rpar = 0, rph[2] = {0, 0};
    // A wait that ran out: the warp goes on with what is there up to the CTA's next barrier, in this row or behind the last one, where
    // all leave together.  (Held over several rows, the flag costs registers: 8192 x 32000 f16 took 240 us instead of 218.)
    bool gave_up = false, agreed = false;
    for (int row = row0; row < rows; row += stride) {
      gave_up = !mbar_wait_bounded_warp(sm.marked + s, ph, kDevErrStageTimeout);
      const struct { DistillRef ref; int skip; } info{sm.row[s].ref, sm.row[s].skip};
      const RowVecs<T> rv(L + (int64_t)row * V, V);
      const int v0 = rv.nvec * rank / C, n = rv.nvec * (rank + 1) / C - v0;
      const int j0 = v0 * VEC - rv.head;                        // row element of this part's first vector
      // vectors [ilo, ihi) of this part lie wholly inside the row
      const int ilo = j0 < 0 ? 1 : 0, ihi = j0 + n * VEC > V ? n - 1 : n;
      T* dpart = BWD ? dL + (int64_t)row * V + j0 : nullptr;
      const bool same = BWD && ((reinterpret_cast<uint64_t>(dL) ^ reinterpret_cast<uint64_t>(L)) & 15) == 0;
      if (info.skip) {
        if (BWD && !beta) {
          const T zero = Elem<T>::from_f32(0.f);
          for (int i = t; i < n; i += MT) {
            if (same && i >= ilo && i < ihi) st_stream(dpart + i * VEC, make_uint4(0, 0, 0, 0));
            else for (int e = 0; e < VEC; ++e) if (j0 + i * VEC + e >= 0 && j0 + i * VEC + e < V) dpart[i * VEC + e] = zero;
          }
        }
        if (lane == 0) distill_arrive(sm.stored + s);
        if (++s == R) { s = 0; ph ^= 1u; }
        if (gave_up) break;
        continue;
      }
      uint4* srow = reinterpret_cast<uint4*>(ring + (size_t)s * slot_bytes);
      constexpr bool HOLD = NVH > 0;
      constexpr int NV = HOLD ? NVH : 1;
      float2 a[NV][VEC / 2];
      DistillSum rest{info.ref, 0.};
      const bool sampled = info.ref.off == info.ref.off;
      bool held = HOLD && sampled && info.ref.sub == 0.f;
      if (held) {
        // ordinary rows: every logit read and exponentiated once
        float2 zq[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        const float2 c2 = make_float2(c, c), off2 = make_float2(info.ref.off, info.ref.off);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          if (t + k * MT < n) {
            float x[VEC];
            unpack<T>(srow[t + k * MT], x);
#pragma unroll
            for (int e = 0; e < VEC / 2; ++e) {
              a[k][e] = fma2(make_float2(x[2 * e], x[2 * e + 1]), c2, off2);
              a[k][e].x = exp2f_approx(a[k][e].x);
              a[k][e].y = exp2f_approx(a[k][e].y);
              zq[e & 1] = add2(zq[e & 1], a[k][e]);
            }
          }
        }
        zq[0] = add2(zq[0], zq[1]);
        rest.z = distill_sum<MW>(zq[0].x + zq[0].y, sm.red[par], warp, lane, gave_up);
        par ^= 1u;
        if (gave_up) { agreed = true; break; }
        // a logit far above the reference, all of them far below, an infinity, NaN: the CTA starts over with the true maximum
        held = rest.z > 8.6736174e-19 && rest.z < 1.1529215e18;             // 2^-60, 2^60
      }
      if (!held) {
        float m = -INFINITY, z = 0.f;
        for (int i = t; i < n; i += MT) {
          float x[VEC];
          unpack<T>(srow[i], x);
#pragma unroll
          for (int e = 0; e < VEC; ++e) m = fmaxf(m, x[e]);
        }
        m = distill_max<MW>(m, sm.red[par], warp, lane, gave_up);
        par ^= 1u;
        if (gave_up) { agreed = true; break; }
        rest.ref = m == -INFINITY ? DistillRef{0.f, 0.f} : distill_ref(m, c);
        for (int i = t; i < n; i += MT) {
          float x[VEC];
          unpack<T>(srow[i], x);
#pragma unroll
          for (int e = 0; e < VEC; ++e) z += distill_exp(x[e], rest.ref, c);
        }
        rest.z = distill_sum<MW>(z, sm.red[par], warp, lane, gave_up);
        par ^= 1u;
        if (gave_up) { agreed = true; break; }
      }
      const DistillRef own = rest.ref;
      const bool empty = rest.z == 0.;                          // nothing but -inf in this part: its reference means nothing
      DistillSum top{sampled ? info.ref : DistillRef{0.f, 0.f}, sm.row[s].z_top};
      if (C > 1) {
        // every CTA hands its part to all of the cluster; the parts are combined in rank order everywhere
        if (warp == 0) {
          if (lane == 0) mbar_expect_tx(sm.rec_bar + rpar, (unsigned)(C * sizeof(DistillRec)));
          if (lane < C) {
            uint32_t dst, bar;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(smem_u32(&sm.rec[rpar][rank])), "r"(lane));
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(smem_u32(&sm.rec_bar[rpar])), "r"(lane));
            auto send = [&](uint32_t at, double lo, double hi) {
              asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f64 [%0], {%1, %2}, [%3];"
                           ::"r"(dst + at), "d"(lo), "d"(hi), "r"(bar) : "memory");
            };
            auto refs = [](const DistillRef& r) { return __hiloint2double(__float_as_int(r.off), __float_as_int(r.sub)); };
            send(0u, refs(rest.ref), rest.z);
            send(16u, refs(top.ref), top.z);
            send(32u, sm.row[s].px, sm.row[s].pown);
          }
        }
        gave_up = !__all_sync(0xffffffffu, distill_wait_cluster(sm.rec_bar + rpar, rph[rpar]));
        rph[rpar] ^= 1u;
        const DistillSum nothing{DistillRef{0.f, 0.f}, 0.};
        const DistillSum ro = lane < C ? sm.rec[rpar][lane].rest : nothing, to = lane < C ? sm.rec[rpar][lane].top : nothing;
        if (__all_sync(0xffffffffu, ro.ref.sub == 0.f && to.ref.sub == 0.f)) {
          // the largest reference has the smallest offset; sums over the lanes in a fixed order
          float ra = ro.z != 0. ? ro.ref.off : INFINITY, ta = to.z != 0. ? to.ref.off : INFINITY;
#pragma unroll
          for (int o = kDistillMaxC / 2; o > 0; o >>= 1) {
            ra = fminf(ra, __shfl_xor_sync(0xffffffffu, ra, o));
            ta = fminf(ta, __shfl_xor_sync(0xffffffffu, ta, o));
          }
          double rz = ro.z != 0. ? ro.z * distill_pow2((double)(ra - ro.ref.off)) : 0., tz = to.z != 0. ? to.z * distill_pow2((double)(ta - to.ref.off)) : 0.;
#pragma unroll
          for (int o = kDistillMaxC / 2; o > 0; o >>= 1) {
            rz += __shfl_xor_sync(0xffffffffu, rz, o);
            tz += __shfl_xor_sync(0xffffffffu, tz, o);
          }
          // (the lanes beyond the cluster's CTAs have followed lanes of their own)
          rest = DistillSum{DistillRef{0.f, __shfl_sync(0xffffffffu, isinf(ra) ? 0.f : ra, 0)}, __shfl_sync(0xffffffffu, rz, 0)};
          top = DistillSum{DistillRef{0.f, __shfl_sync(0xffffffffu, isinf(ta) ? 0.f : ta, 0)}, __shfl_sync(0xffffffffu, tz, 0)};
        } else {
          rest = sm.rec[rpar][0].rest;
          top = sm.rec[rpar][0].top;
          for (int q = 1; q < C; ++q) {
            rest = distill_add(rest, sm.rec[rpar][q].rest, c);
            top = distill_add(top, sm.rec[rpar][q].top, c);
          }
        }
      }
      const bool one = C == 1 && held;                          // one reference for everything
      const DistillSum all = one ? DistillSum{own, rest.z + top.z} : distill_add(rest, top, c);
      if (t == 0) {
        // sum p log2 e(x) under the row's reference
        double px = 0.;
        if (one) px = sm.row[s].px;
        else if (C == 1) px = sm.row[s].pown != 0. ? sm.row[s].px + sm.row[s].pown * distill_shift64(all.ref, top.ref, c) : 0.;
        else
          for (int q = 0; q < C; ++q) {
            const DistillRec& o = sm.rec[rpar][q];
            if (o.pown != 0.) px += o.px + o.pown * distill_shift64(all.ref, o.top.ref, c);
          }
        sm.fin[s] = DistillFin{all.ref, all.z, rest.z, one || rest.z == 0. ? 0. : distill_shift64(all.ref, rest.ref, c), px};
      }
      if (C > 1) rpar ^= 1u;
      if (BWD) {
        // (P / E - r / E_rest) e, e formed against this CTA's reference
        const double num = lane == 0 ? sm.row[s].g_mass : sm.row[s].g_r, den = lane == 0 ? all.z : rest.z;
        double ga = num != 0. && (lane == 0 || den > 0.) ? quotient(num, den) : 0., gr = __shfl_sync(0xffffffffu, ga, 1);      // one division
        ga = __shfl_sync(0xffffffffu, ga, 0);
        if (!one && !empty) {
          if (ga != 0.) ga *= distill_pow2(distill_shift64(all.ref, own, c));
          if (gr != 0.) gr *= distill_pow2(distill_shift64(rest.ref, own, c));
        }
        const float g = (float)(ga - gr);
        if (held) {
          const float2 g2 = make_float2(g, g);
#pragma unroll
          for (int k = 0; k < NV; ++k) {
            const int i = t + k * MT;
            if (i < n) {
              float d[VEC];
#pragma unroll
              for (int e = 0; e < VEC / 2; ++e) {
                const float2 v = mul2(a[k][e], g2);
                d[2 * e] = v.x; d[2 * e + 1] = v.y;
              }
              if (beta && same && i >= ilo && i < ihi) srow[i] = pack_accumulate<T>(d, ld_stream(dpart + i * VEC));
              else srow[i] = pack<T>(d);
            }
          }
        } else {
          // a factor of 0 (no probability on the list and none beside it): 0 also where the logits are no numbers
          for (int i = t; i < n; i += MT) {
            float x[VEC];
            unpack<T>(srow[i], x);
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] = g != 0.f ? distill_exp(x[e], empty ? all.ref : own, c) * g : 0.f;
            if (beta && same && i >= ilo && i < ihi) srow[i] = pack_accumulate<T>(x, ld_stream(dpart + i * VEC));
            else srow[i] = pack<T>(x);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // written here, read by the copy out
      }
      __syncwarp();
      if (lane == 0) distill_arrive(sm.stored + s);
      if (++s == R) { s = 0; ph ^= 1u; }
      if (gave_up) break;
    }
    if (!agreed) (void)distill_meet<MW>(gave_up);
  }
  __syncwarp();
  // no CTA leaves while another may still write into its records
  if (C > 1) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
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

template <typename T, int MW, int R, int NVH>
static int launch_distill_as(uint64_t dl, uint64_t l, const DistillParams& p, int C, unsigned slot_bytes, cudaStream_t st) {
  const size_t lists = (size_t)R * ((p.k + 31) / 32 * 32) * kDistillListBytes;
  const size_t smem = (sizeof(DistillSmem<MW, R>) + lists + 127) / 128 * 128 + (size_t)R * slot_bytes;
  auto kern = !dl ? distill_kernel<T, MW, R, NVH, kDistillFwd>
                  : p.beta ? distill_kernel<T, MW, R, NVH, kDistillAcc> : distill_kernel<T, MW, R, NVH, kDistillBwd>;
  const int per_sm = resident_ctas(kern, (MW + R) * 32, smem);
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3((MW + R) * 32); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)C; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  // rows are dealt to clusters in turn: exactly as many clusters as run at once (a GPC's SMs are no multiple of C)
  int64_t clusters = (int64_t)kNumSMs * per_sm;
  if (C > 1) {
    struct Key { const void* k; int dev, C; size_t smem; int n; };
    static thread_local Key cache[64];
    static thread_local int used = 0;
    const void* kp = reinterpret_cast<const void*>(kern);
    const int dev = device_ordinal();
    int n = 0;
    for (int i = 0; i < used && !n; ++i)
      if (cache[i].k == kp && cache[i].dev == dev && cache[i].C == C && cache[i].smem == smem) n = cache[i].n;
    if (!n) {
      cfg.gridDim = dim3((unsigned)C);
      if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) { (void)cudaGetLastError(); n = kNumSMs / C / 2; }
      if (used < 64) cache[used++] = Key{kp, dev, C, smem, n};
    }
    clusters = n;
  }
  if (clusters > p.rows) clusters = p.rows;
  cfg.gridDim = dim3((unsigned)(clusters * C));
  cudaLaunchKernelEx(&cfg, kern, reinterpret_cast<T*>(dl), reinterpret_cast<const T*>(l), p, slot_bytes);
  return check_launch();
}

template <typename T>
static int launch_distill(uint64_t dl, uint64_t l, const DistillParams& p, cudaStream_t st) {
  constexpr int VEC = Elem<T>::VEC;
  // vectors of a row; of the worst-aligned one where rows start at different places
  const int nvec = p.vocab % VEC == 0 && (l & 15) == 0 ? p.vocab / VEC : (p.vocab + 2 * VEC - 2) / VEC;
  int C = 1;
  while (C < kDistillMaxC && (nvec + C - 1) / C > g_distill_part) C *= 2;
  const int per = (nvec + C - 1) / C;
  const unsigned slot = ((unsigned)(per + 1) * 16 + 127) / 128 * 128;
  // Warps and vectors a thread, by a row's (or part's) length: few warps that hold much, as long as two or three CTAs share an SM or
  // one has the registers to itself.  Measured, us, k 64: 8192 x 32000 f16 with 12 x 11: 204, 16 x 8 (spills): 221, 9 x 15: 226,
  // 8 x 16: 266, 24 x 6: 288; 8192 x 16000 with 8 x 8 on two CTAs: 133, 6 x 11: 179; 16384 x 8000 with 4 x 8 on three CTAs: 149,
  // 8 x 4: 177.
  if (per <= 4 * 32 * 8) return launch_distill_as<T, 4, 2, 8>(dl, l, p, C, slot, st);
  if (per <= 8 * 32 * 8) return launch_distill_as<T, 8, 2, 8>(dl, l, p, C, slot, st);
  if (per <= 12 * 32 * 11) return launch_distill_as<T, 12, 3, 11>(dl, l, p, C, slot, st);
  return launch_distill_as<T, 16, 1, 0>(dl, l, p, C, slot, st);
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
  if (rows > 0x3fffffffLL) return CACTI_B200_ERR_SHAPE;           // row indices of the kernel and a grid's stride fit 32 bits
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
  const uint64_t bytes = (uint64_t)rows * vocab * es;
  if (overlap({dlogits, bytes}, {logits, bytes})) return CACTI_B200_ERR_INVALID_VALUE;
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
