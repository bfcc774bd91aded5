// logprob.cu -- log probability of a given token in each row of logits, with
// the row's entropy and its k most likely tokens, and the gradient.
//
// Mathematics, with z = x / temperature and y = (x - max x) log2(e) / temperature:
//   S = sum 2^y,  W = sum 2^y y,   log p_j = ln2 (y_j - log2 S),
//   H = -sum p ln p = ln2 (log2 S - W / S)
//   dL/dx_j = (1/temperature) (dlogp (1{j = id} - p_j) - dH p_j (ln p_j + H)).
// The forward reads a row once, with the running maximum and sums of an
// online softmax in every thread; the backward reads it a second time, since
// p is cheaper to form again than to store.
//
// Top k without a second pass: every thread knows the largest value it has
// seen.  The k-th largest of those is a bound that at least k elements reach,
// so only the threads whose maximum reaches it (k of them, more with ties)
// look through their elements again, from L2, and hand those that reach the
// bound to the CTA.  Candidates are ordered as 64-bit keys, value first (NaN
// last) and then the lower index, so the result does not depend on any order of
// arrival.
//
// Bound: HBM for many rows (forward: one read of the logits; backward: one
// read and one write).  4096 x 151936 bf16 with entropy: forward 209 us (5.96
// TB/s), backward 363 us (6.87 TB/s, the logits' last rows still in L2);
// 2048 rows with top 1: 118 us (5.28 TB/s; ncu, each).  Few rows are split over the CTAs
// of a cluster, which join their partial sums and candidates through
// distributed shared memory (32 rows with top 5: 13.7 us); small vocabularies
// take a warp a row.
#include <cooperative_groups.h>

#include <cfloat>

#include "mma16.cuh"
#include "op_util.cuh"

namespace cg = cooperative_groups;

namespace gdn2 {
namespace {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpUnroll = 4;       // vectors of a thread in flight
constexpr int kMaxTop = 128;
constexpr int kRoundKeys = kLpWarps * 32 * 8;   // most candidates of one round
constexpr int kSpare = 512;                     // candidates kept between rounds
constexpr int kCandidates = kRoundKeys + kSpare;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLow = -1e4f;      // 2^kLow = 0: stands for y = -inf where 0 * y is formed

struct LogprobArgs {
  int64_t rows, ld, ignore;
  int V, k;
  float c;  // log2(e) / temperature
  float inv_temperature;
  const void* x;
  const int64_t* ids;
  float *logp, *entropy, *top_logp;
  int64_t* top_ids;
  float4* stats;  // max, 1 / S, log2 S, entropy
  const float *dlogp, *dentropy;
  void* dx;
};

// max and sums of a set of logits; m is finite.
struct Soft {
  float m, s, w;
};

__device__ __forceinline__ Soft rescale(Soft a, float m, float c) {
  if (m > a.m) {
    const float y = (a.m - m) * c, f = fast_exp2(y);
    a.w = f * fmaf(a.s, fmaxf(y, kLow), a.w);
    a.s *= f;
    a.m = m;
  }
  return a;
}

__device__ __forceinline__ Soft merge(Soft a, Soft b, float c) {
  const float m = fmaxf(a.m, b.m);
  a = rescale(a, m, c);
  b = rescale(b, m, c);
  return Soft{m, a.s + b.s, a.w + b.w};
}

// Largest of the packed elements; a NaN does not count.
template <typename T, int N> __device__ __forceinline__ float raw_max(const Raw<T, N>& r) {
  if constexpr (sizeof(T) == 4) {
    float m = __uint_as_float(r.u[0]);
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, __uint_as_float(r.u[i]));
    return m;
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    __nv_bfloat162 m = *reinterpret_cast<const __nv_bfloat162*>(&r.u[0]);
#pragma unroll
    for (int i = 1; i < N / 2; ++i)
      m = __hmax2(m, *reinterpret_cast<const __nv_bfloat162*>(&r.u[i]));
    const float2 f = __bfloat1622float2(m);
    return fmaxf(f.x, f.y);
  } else {
    __half2 m = *reinterpret_cast<const __half2*>(&r.u[0]);
#pragma unroll
    for (int i = 1; i < N / 2; ++i) m = __hmax2(m, *reinterpret_cast<const __half2*>(&r.u[i]));
    const float2 f = __half22float2(m);
    return fmaxf(f.x, f.y);
  }
}

template <typename T, int N> __device__ __forceinline__ float2 raw_pair(const Raw<T, N>& r, int i) {
  if constexpr (sizeof(T) == 4)
    return make_float2(__uint_as_float(r.u[2 * i]), __uint_as_float(r.u[2 * i + 1]));
  else
    return unpack2<T>(r.u[i]);
}

// Order-preserving map of a float to 32 bits; -0 counts as 0, NaN as least.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  if (o == 0u) return __uint_as_float(0x7fffffffu);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ uint64_t key_of(float x, int idx) {
  return ((uint64_t)order_of(x) << 32) | (uint32_t)~(uint32_t)idx;
}

// A row as aligned 16-byte vectors: vector j holds the elements j*VE - off
// .. j*VE - off + VE - 1 of which those in [0, V) exist.
template <typename T> struct RowView {
  static constexpr int VE = 16 / (int)sizeof(T);
  const T* base;  // element -off
  int off, V, nvec;
  __device__ __forceinline__ RowView(const T* row, int v) : V(v) {
    off = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    base = row - off;
    nvec = (int)(((int64_t)V + off + VE - 1) / VE);
  }
  __device__ __forceinline__ bool whole(int j) const {
    return (j > 0 || off == 0) && (int64_t)(j + 1) * VE - off <= V;
  }
  // absent elements, and all of a vector that is not below `hi`, read as -inf
  __device__ __forceinline__ Raw<T, VE> load(int j, int hi) const {
    if (j < hi) return load(j);
    float f[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) f[e] = -INFINITY;
    return raw_from<T, VE>(f);
  }
  __device__ __forceinline__ Raw<T, VE> load(int j) const {
    if (whole(j)) return load_raw<T, VE>(base + (int64_t)j * VE);
    float f[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const int64_t i = (int64_t)j * VE + e - off;
      f[e] = i >= 0 && i < V ? to_f<T>(base[(int64_t)j * VE + e]) : -INFINITY;
    }
    return raw_from<T, VE>(f);
  }
};

struct LogprobShared {
  float warp_max[kLpWarps];
  float2 warp_sum[kLpWarps];
  Soft total;
  uint32_t most[kLpThreads];
  int who[kLpThreads];
  uint64_t cand[kCandidates];
  uint64_t best[kMaxTop];
  uint64_t least;
  uint32_t bound;
  int n_who, n_cand, n_best;
};

// The k largest of s.cand[0 .. n) into s.best, in order.
__device__ __forceinline__ void select_best(LogprobShared& s, int n, int k) {
  for (int i = threadIdx.x; i < n; i += kLpThreads) {
    const uint64_t key = s.cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += s.cand[j] > key;
    if (rank < k) s.best[rank] = key;
  }
  if (threadIdx.x == 0) s.n_best = n < k ? n : k;
}

// Hands the elements of vector j that reach `least` to the CTA.
template <typename T>
__device__ __forceinline__ void collect(LogprobShared& s, const RowView<T>& row, int j,
                                        uint64_t least) {
  constexpr int VE = RowView<T>::VE;
  const Raw<T, VE> r = row.load(j);
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    const int64_t i = (int64_t)j * VE + e - row.off;
    if (i < 0 || i >= row.V) continue;
    const uint64_t key = key_of(raw_get(r, e), (int)i);
    if (key < least) continue;
    const int at = atomicAdd(&s.n_cand, 1);
    if (at < kCandidates) s.cand[at] = key;
  }
}

// The same for 32 vectors of the thread s.who[u / segs], one for each lane.
template <typename T>
__device__ __forceinline__ void collect_unit(LogprobShared& s, const RowView<T>& row, int lo, int hi,
                                             int u, int segs, uint64_t least) {
  const int step = (u % segs) * 32 + (threadIdx.x & 31);
  const int64_t j = (int64_t)lo + s.who[u / segs] + (int64_t)step * kLpThreads;
  if (j < hi) collect(s, row, (int)j, least);
}

// The k-th largest of the threads' values into s.bound (0 if fewer have one).
// Up to 32 are found among the k largest of each warp, which a bitonic sort
// puts in order; more by counting among all threads'.
__device__ __forceinline__ void find_bound(LogprobShared& s, uint32_t mine, int k) {
  const int tid = threadIdx.x, lane = tid & 31;
  int n = kLpThreads;
  if (k <= 32) {
    uint32_t x = mine;
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
      for (int o = size / 2; o > 0; o /= 2) {
        const uint32_t y = __shfl_xor_sync(0xffffffffu, x, o);
        const bool falling = (lane & size) == 0, low = (lane & o) == 0;
        x = low == falling ? max(x, y) : min(x, y);
      }
    n = kLpWarps * k;
    if (lane < k) s.most[(tid >> 5) * k + lane] = x;
  } else {
    s.most[tid] = mine;
  }
  __syncthreads();
  if (tid < n) {
    const uint32_t x = s.most[tid];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) {
      const uint32_t y = s.most[j];
      rank += y > x || (y == x && j < tid);
    }
    if (rank == k - 1) s.bound = x;
  }
  __syncthreads();
}

// The CTA's k largest elements of vectors [lo, hi), given every thread's largest.
template <typename T>
__device__ void cta_top(LogprobShared& s, const RowView<T>& row, int lo, int hi, float most,
                        int k) {
  const int tid = threadIdx.x, warp = tid >> 5;
  const bool any = lo + tid < hi;
  const uint32_t mine = any ? order_of(most) : 0u;
  if (tid == 0) { s.n_who = 0; s.n_cand = 0; }
  find_bound(s, mine, k);
  // -inf is also what a thread reports that has read NaN alone, so it bounds
  // nothing: below it come the NaN, which fill up the places that are left
  const uint32_t bound = s.bound == order_of(-INFINITY) ? 0u : s.bound;
  const int steps = (hi - lo + kLpThreads - 1) / kLpThreads, segs = (steps + 31) / 32;
  const bool reach = any && mine >= bound;
  if (steps <= 4) {  // few vectors: a thread looks through its own
    if (reach)
      for (int j = lo + tid; j < hi; j += kLpThreads) collect(s, row, j, (uint64_t)bound << 32);
    __syncthreads();
    if (s.n_cand <= kCandidates) {
      select_best(s, s.n_cand, k);
      __syncthreads();
      return;
    }
  }
  if (reach) s.who[atomicAdd(&s.n_who, 1)] = tid;
  __syncthreads();
  const int units = s.n_who * segs;
  if (steps > 4) {
    for (int u = warp; u < units; u += kLpWarps)
      collect_unit(s, row, lo, hi, u, segs, (uint64_t)bound << 32);
    __syncthreads();
  }
  const int n = s.n_cand;
  if (n <= kCandidates) {
    select_best(s, n, k);
    __syncthreads();
    return;
  }
  // More elements reach the bound than the list holds (many equal values, or
  // the largest all with few threads): again in rounds that fit, raising the
  // bound to the k-th best so far after each.
  __syncthreads();
  if (tid == 0) { s.n_cand = 0; s.least = (uint64_t)bound << 32; }
  __syncthreads();
  for (int u0 = 0; u0 < units; u0 += kLpWarps) {
    if (u0 + warp < units) collect_unit(s, row, lo, hi, u0 + warp, segs, s.least);
    __syncthreads();
    const int have = s.n_cand;
    const bool last = u0 + kLpWarps >= units;
    __syncthreads();  // everyone has read the count before the next round adds to it
    if (have > kSpare || last) {
      select_best(s, have, k);
      __syncthreads();
      const int kept = s.n_best;
      for (int i = tid; i < kept; i += kLpThreads) s.cand[i] = s.best[i];
      if (tid == 0) {
        s.n_cand = kept;
        if (kept == k) s.least = s.best[k - 1];
      }
      __syncthreads();
    }
  }
}

// Running maximum and sums of a thread's elements, four vectors at a time.
template <typename T, bool ENT> struct Running {
  static constexpr int VE = RowView<T>::VE;
  float m = -FLT_MAX, most = -INFINITY;  // finite; the largest element itself
  float2 s = make_float2(0.f, 0.f), w = make_float2(0.f, 0.f);

  template <int N> __device__ __forceinline__ void add(const Raw<T, VE> (&v)[N], float c) {
    float top = raw_max(v[0]);
#pragma unroll
    for (int u = 1; u < N; ++u) top = fmaxf(top, raw_max(v[u]));
    most = fmaxf(most, top);
    if (top > m) lift(top, c);
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int i = 0; i < VE / 2; ++i) {
        const float2 y = mul2(add2(raw_pair(v[u], i), f2(-m)), f2(c));
        const float2 e = exp2_2(y);
        s = add2(s, e);
        if constexpr (ENT) w = fma2(e, make_float2(fmaxf(y.x, kLow), fmaxf(y.y, kLow)), w);
      }
  }
  // the sums with respect to a larger maximum
  __device__ __forceinline__ void lift(float top, float c) {
    const float y = (m - top) * c, f = fast_exp2(y), g = fmaxf(y, kLow);
    if constexpr (ENT) w = mul2(f2(f), fma2(s, f2(g), w));
    s = mul2(s, f2(f));
    m = top;
  }
};

__device__ __forceinline__ float warp_most(float x) {  // NaN does not count
  const uint32_t o = __reduce_max_sync(0xffffffffu, order_of(x));
  return value_of(o);
}

// A row's results from its sums: log probability of x (NaN for a token outside
// the vocabulary), entropy, and what the backward needs.
struct RowEnd {
  float lg, ent;
  bool none;  // every logit is -inf
  __device__ __forceinline__ RowEnd(const Soft& t) {
    none = t.s == 0.f;
    lg = log2f(t.s);
    ent = none ? 0.f : kLn2 * (lg - t.w / t.s);
  }
  __device__ __forceinline__ float logp(const Soft& t, float x, float c) const {
    return none ? -INFINITY : kLn2 * ((x - t.m) * c - lg);
  }
  __device__ __forceinline__ void write(const LogprobArgs& a, const Soft& t, int64_t r, int64_t id,
                                        float x) const {
    a.logp[r] = id >= 0 && id < a.V ? logp(t, x, a.c) : __uint_as_float(0x7fffffffu);
    if (a.entropy) a.entropy[r] = ent;
    if (a.stats) a.stats[r] = make_float4(t.m, none ? 0.f : 1.f / t.s, none ? 0.f : lg, ent);
  }
};

__device__ __forceinline__ void write_ignored(const LogprobArgs& a, int64_t r, int thread, int threads) {
  if (thread == 0) {
    a.logp[r] = 0.f;
    if (a.entropy) a.entropy[r] = 0.f;
  }
  for (int i = thread; i < a.k; i += threads) {
    a.top_logp[r * a.k + i] = -INFINITY;
    a.top_ids[r * a.k + i] = -1;
  }
}

template <typename T, bool ENT, bool TOP>
__global__ void __launch_bounds__(kLpThreads, 5) k_logprob_fwd(const LogprobArgs a, const int parts) {
  constexpr int VE = RowView<T>::VE;
  __shared__ LogprobShared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x / (unsigned)parts;
  const int part = (int)(blockIdx.x - r * parts);
  const int64_t id = a.ids[r];
  if (id == a.ignore) {  // the same for the whole cluster
    if (part == 0) write_ignored(a, r, tid, kLpThreads);
    return;
  }
  const T* xr = (const T*)a.x + r * a.ld;
  const RowView<T> row(xr, a.V);
  const int per = (row.nvec + parts - 1) / parts;
  const int lo = min(part * per, row.nvec), hi = min(lo + per, row.nvec);
  const float c = a.c;
  float given = 0.f;  // the token's logit, on its way early
  if (tid == 0 && part == 0 && id >= 0 && id < a.V) given = to_f<T>(xr[id]);

  Running<T, ENT> run;
  Raw<T, VE> v[kLpUnroll];
  int j = lo + tid;
  for (; j + (kLpUnroll - 1) * kLpThreads < hi; j += kLpUnroll * kLpThreads) {
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) v[u] = row.load(j + u * kLpThreads);
    run.add(v, c);
  }
  if (j < hi) {
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) v[u] = row.load(j + u * kLpThreads, hi);
    run.add(v, c);
  }

  // the CTA's maximum, then its sums with respect to it
  {
    const float m = warp_most(run.m);
    if (lane == 0) s.warp_max[warp] = m;
  }
  if constexpr (TOP) cta_top(s, row, lo, hi, run.most, a.k);
  else __syncthreads();
  float m = s.warp_max[0];
#pragma unroll
  for (int i = 1; i < kLpWarps; ++i) m = fmaxf(m, s.warp_max[i]);
  run.lift(m, c);
  const float ps = warp_sum(run.s.x + run.s.y), pw = ENT ? warp_sum(run.w.x + run.w.y) : 0.f;
  if (lane == 0) s.warp_sum[warp] = make_float2(ps, pw);
  __syncthreads();
  Soft t{m, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kLpWarps; ++i) {
    t.s += s.warp_sum[i].x;
    t.w += s.warp_sum[i].y;
  }

  if (parts > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    if (tid == 0) s.total = t;
    cluster.sync();
    if (part == 0) {
      for (int q = 1; q < parts; ++q) t = merge(t, *cluster.map_shared_rank(&s.total, q), c);
      if constexpr (TOP) {
        int n = 0;
        for (int q = 0; q < parts; ++q) {
          const LogprobShared* o = cluster.map_shared_rank(&s, q);
          const int have = o->n_best;
          for (int i = tid; i < have; i += kLpThreads) s.cand[n + i] = o->best[i];
          n += have;
        }
        __syncthreads();
        select_best(s, n, a.k);
        __syncthreads();
      }
    }
    cluster.sync();  // no CTA leaves while another reads its shared memory
    if (part != 0) return;
  }

  if (TOP || tid == 0) {
    const RowEnd end(t);
    if (tid == 0) end.write(a, t, r, id, given);
    if constexpr (TOP)
      for (int i = tid; i < a.k; i += kLpThreads) {
        const uint64_t key = s.best[i];
        a.top_logp[r * a.k + i] = end.logp(t, value_of((uint32_t)(key >> 32)), c);
        a.top_ids[r * a.k + i] = (int64_t)(uint32_t)~(uint32_t)key;
      }
  }
}

// Rows of up to 32 * kLpUnroll vectors: a warp each, the row in registers
// (8192 x 500 bf16 with top 1: 25 us a call, 51 us with a CTA each).  The
// top k come out one by one: the lanes' best by two reductions (value, then the
// lower index), and the lane that held it looks for its next.
template <typename T, bool ENT, bool TOP>
__global__ void __launch_bounds__(kLpThreads) k_logprob_small(const LogprobArgs a) {
  constexpr int VE = RowView<T>::VE;
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * kLpWarps + (threadIdx.x >> 5);
  if (r >= a.rows) return;
  const int64_t id = a.ids[r];
  if (id == a.ignore) return write_ignored(a, r, lane, 32);
  const T* xr = (const T*)a.x + r * a.ld;
  const RowView<T> row(xr, a.V);
  float given = 0.f;
  if (lane == 0 && id >= 0 && id < a.V) given = to_f<T>(xr[id]);
  Raw<T, VE> v[kLpUnroll];
#pragma unroll
  for (int u = 0; u < kLpUnroll; ++u) v[u] = row.load(lane + 32 * u, row.nvec);
  Running<T, ENT> run;
  run.add(v, a.c);
  run.lift(warp_most(run.m), a.c);
  const Soft t{run.m, warp_sum(run.s.x + run.s.y), ENT ? warp_sum(run.w.x + run.w.y) : 0.f};
  const RowEnd end(t);
  if (lane == 0) end.write(a, t, r, id, given);
  if constexpr (TOP) {
    uint64_t last = ~0ull, best = 0;  // this lane's largest key below `last`
    bool look = true;
    for (int n = 0; n < a.k; ++n) {
      if (look) {
        best = 0;
#pragma unroll
        for (int u = 0; u < kLpUnroll; ++u)
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const int64_t i = (int64_t)(lane + 32 * u) * VE + e - row.off;
            const uint64_t key = key_of(raw_get(v[u], e), (int)i);
            if (i >= 0 && i < row.V && key < last && key > best) best = key;
          }
      }
      const uint32_t hi = (uint32_t)(best >> 32), top = __reduce_max_sync(0xffffffffu, hi);
      const uint32_t lo = __reduce_max_sync(0xffffffffu, best && hi == top ? (uint32_t)best : 0u);
      look = best && hi == top && (uint32_t)best == lo;
      if (look) last = best;
      if (lane == 0) {
        a.top_logp[r * a.k + n] = end.logp(t, value_of(top), a.c);
        a.top_ids[r * a.k + n] = (int64_t)(uint32_t)~lo;
      }
    }
  }
}

// dL/dx = 2^y (A + B y) + 1{j = id} dlogp / temperature, with
//   A = (1/S)(1/temperature) (-dlogp - dH (H - ln S)),  B = -(1/S)(1/temperature) ln2 dH.
template <typename T, bool ENT>
__global__ void __launch_bounds__(kLpThreads) k_logprob_bwd(const LogprobArgs a, const int blocks) {
  constexpr int VE = RowView<T>::VE;
  const int64_t r = blockIdx.x / (unsigned)blocks;
  const int block = (int)(blockIdx.x - r * blocks);
  const T* xr = (const T*)a.x + r * a.ld;
  T* dr = (T*)a.dx + r * a.V;
  const RowView<T> row(xr, a.V);
  const bool same = ((reinterpret_cast<uintptr_t>(xr) ^ reinterpret_cast<uintptr_t>(dr)) & 15) == 0;
  const int64_t id = a.ids[r];
  const float4 st = a.stats[r];
  const float dl = a.dlogp ? a.dlogp[r] : 0.f, de = ENT && a.dentropy ? a.dentropy[r] : 0.f;
  const bool skip = id == a.ignore || st.y == 0.f;
  const bool known = id >= 0 && id < a.V;
  const float scale = st.y * a.inv_temperature;
  // a token outside the vocabulary has no log probability to move
  const float A = scale * (-(known ? dl : 0.f) - de * (st.w - kLn2 * st.z)), B = -scale * kLn2 * de;
  const float hot = dl * a.inv_temperature;
  const int j0 = block * (kLpThreads * kLpUnroll) + threadIdx.x;
  Raw<T, VE> v[kLpUnroll];
  if (!skip) {
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u)
      if (j0 + u * kLpThreads < row.nvec) v[u] = row.load(j0 + u * kLpThreads);
  }
#pragma unroll
  for (int u = 0; u < kLpUnroll; ++u) {
    const int j = j0 + u * kLpThreads;
    if (j >= row.nvec) break;
    float d[VE];
    const int64_t first = (int64_t)j * VE - row.off;
    if (skip) {
#pragma unroll
      for (int e = 0; e < VE; ++e) d[e] = 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < VE / 2; ++i) {
        const float2 y = mul2(add2(raw_pair(v[u], i), f2(-st.x)), f2(a.c));
        float2 k = f2(A);
        if constexpr (ENT)
          k = fma2(f2(B), make_float2(fmaxf(y.x, kLow), fmaxf(y.y, kLow)), k);
        const float2 g = mul2(exp2_2(y), k);
        d[2 * i] = g.x;
        d[2 * i + 1] = g.y;
      }
      const int64_t at = id - first;
      if (at >= 0 && at < VE) {
#pragma unroll
        for (int e = 0; e < VE; ++e)
          if (e == at) d[e] += hot;
      }
    }
    if (same && row.whole(j)) {
      store_raw<T, VE>(dr + first, raw_from<T, VE>(d));
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (first + e >= 0 && first + e < a.V) dr[first + e] = from_f<T>(d[e]);
    }
  }
}

// ---------------------------------------------------------------------------
// entry points
// ---------------------------------------------------------------------------
int check_logprob(const gdn2_logprob_problem* p, const char* fn) {
  if (!p) return fail(GDN2_ERR_INVALID, "%s: null problem", fn);
  if (p->rows < 0 || p->vocab <= 0)
    return fail(GDN2_ERR_INVALID, "%s: needs rows >= 0 and vocab > 0 (got %lld, %d)", fn,
                (long long)p->rows, p->vocab);
  if (!dtype_valid(p->dtype)) return fail(GDN2_ERR_INVALID, "%s: unknown dtype %d", fn, p->dtype);
  if (p->ld < p->vocab)
    return fail(GDN2_ERR_INVALID, "%s: the row stride must be at least vocab", fn);
  // log2(e) / temperature overflows below 4.3e-39
  if (!(p->temperature > 0.f) || p->temperature > FLT_MAX || kLog2e / p->temperature > FLT_MAX)
    return fail(GDN2_ERR_INVALID, "%s: temperature must be positive and finite, and so its inverse",
                fn);
  if (p->top_k < 0 || p->top_k > p->vocab)
    return fail(GDN2_ERR_INVALID, "%s: top_k must be in 0 .. vocab (got %d)", fn, p->top_k);
  if (p->top_k > kMaxTop)
    return fail(GDN2_ERR_UNSUPPORTED, "%s: top_k up to %d is supported (got %d)", fn, kMaxTop,
                p->top_k);
  const int64_t blocks = (int64_t)p->vocab / 256 / 4 + 2;  // of a row, at most
  if (p->rows > 2147483647LL / blocks)
    return fail(GDN2_ERR_UNSUPPORTED, "%s: too many rows", fn);
  return GDN2_OK;
}

LogprobArgs logprob_args(const gdn2_logprob_problem* p) {
  LogprobArgs a{};
  a.rows = p->rows;
  a.ld = p->ld;
  a.ignore = p->ignore_index;
  a.V = p->vocab;
  a.k = p->top_k;
  a.inv_temperature = 1.f / p->temperature;
  a.c = kLog2e / p->temperature;
  return a;
}

// CTAs of a row: one when the rows alone fill the GPU, else as many (2, 4, 8)
// as keep the grid within two CTAs per SM and 16 KB for each (bf16, between
// events: 2048 rows of 151936 with top 1 one 115 us, two 132 us; 32 rows with top
// 5 one 21.2 us, two 15.1, eight 13.0 us).
cudaError_t row_parts(int64_t rows, int64_t row_bytes, int* parts) {
  int sms = 0;
  const cudaError_t e = num_sms(&sms);
  *parts = 1;
  while (*parts < 8 && rows * *parts * 2 <= 2 * sms && row_bytes / (*parts * 2) >= 16384)
    *parts *= 2;
  return e;
}

template <typename T, bool ENT, bool TOP>
cudaError_t launch_logprob(const LogprobArgs& a, int parts, cudaStream_t st) {
  // with one vector to spare for a row that starts inside one
  if (a.V <= (32 * kLpUnroll - 1) * RowView<T>::VE) {
    k_logprob_small<T, ENT, TOP>
        <<<(unsigned)((a.rows + kLpWarps - 1) / kLpWarps), kLpThreads, 0, st>>>(a);
    return cudaGetLastError();
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.rows * parts));
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)parts;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, k_logprob_fwd<T, ENT, TOP>, a, parts);
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

int gdn2_logprob_fwd(const gdn2_logprob_problem* p, const void* logits, const int64_t* token_ids,
                     float* logprobs, float* entropy, float* top_logprobs, int64_t* top_ids,
                     float* stats, void* stream) {
  const char* fn = "gdn2_logprob_fwd";
  int rc = check_logprob(p, fn);
  if (rc) return rc;
  if (p->rows == 0) return GDN2_OK;
  if (!logits || !token_ids || !logprobs || (p->top_k > 0 && (!top_logprobs || !top_ids)))
    return fail(GDN2_ERR_INVALID, "%s: null pointer", fn);
  if (stats && !aligned_to(stats, 16))
    return fail(GDN2_ERR_INVALID, "%s: stats must start on a 16-byte boundary", fn);
  LogprobArgs a = logprob_args(p);
  a.x = logits; a.ids = token_ids; a.logp = logprobs; a.entropy = entropy;
  a.top_logp = top_logprobs; a.top_ids = top_ids; a.stats = reinterpret_cast<float4*>(stats);
  int parts = 1;
  cudaError_t e = row_parts(p->rows, (int64_t)p->vocab * dtype_size(p->dtype), &parts);
  if (e != cudaSuccess) return cuda_status(e, fn);
  const cudaStream_t st = (cudaStream_t)stream;
  e = with_dtype(p->dtype, [&](auto t) {
    using T = decltype(t);
    if (p->top_k > 0)
      return entropy ? launch_logprob<T, true, true>(a, parts, st)
                     : launch_logprob<T, false, true>(a, parts, st);
    return entropy ? launch_logprob<T, true, false>(a, parts, st)
                   : launch_logprob<T, false, false>(a, parts, st);
  });
  return cuda_status(e, fn);
}

int gdn2_logprob_bwd(const gdn2_logprob_problem* p, const void* logits, const int64_t* token_ids,
                     const float* stats, const float* dlogprobs, const float* dentropy,
                     void* dlogits, void* stream) {
  const char* fn = "gdn2_logprob_bwd";
  int rc = check_logprob(p, fn);
  if (rc) return rc;
  if (p->rows == 0) return GDN2_OK;
  if (!logits || !token_ids || !stats || !dlogits)
    return fail(GDN2_ERR_INVALID, "%s: null pointer", fn);
  if (!aligned_to(stats, 16))
    return fail(GDN2_ERR_INVALID, "%s: stats must start on a 16-byte boundary", fn);
  LogprobArgs a = logprob_args(p);
  a.x = logits; a.ids = token_ids; a.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
  a.dlogp = dlogprobs; a.dentropy = dentropy; a.dx = dlogits;
  const cudaStream_t st = (cudaStream_t)stream;
  return cuda_status(with_dtype(p->dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int per = RowView<T>::VE * kLpThreads * kLpUnroll;
    // one vector more than the row fills where it starts inside one
    const int blocks = (int)(((int64_t)a.V + RowView<T>::VE - 1 + per - 1) / per);
    const unsigned grid = (unsigned)(a.rows * blocks);
    if (dentropy) k_logprob_bwd<T, true><<<grid, kLpThreads, 0, st>>>(a, blocks);
    else k_logprob_bwd<T, false><<<grid, kLpThreads, 0, st>>>(a, blocks);
    return cudaGetLastError();
  }), fn);
}

}  // extern "C"
