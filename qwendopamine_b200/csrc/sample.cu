// sample.cu -- one token for each row of logits from one given random number.
//
// Mathematics, with m = max x and w_i = exp((x_i - m) / temperature) = 2^-y_i:
//   kept by min-p:  w_i >= min_p;   by top-k: the k largest of those;
//   by top-p: of what is left, in falling order, up to the first running sum
//   that reaches top_p of the sum;  equal logits rank by rising index
//   token = the lowest index whose running sum of kept weights, in the order of
//   the vocabulary, exceeds uniform * (their sum).
//
// A token far down the vocabulary may hold a millionth of the sum, so whether
// the running sum has passed the target is decided by digits that fp32 does not
// have: weights and sums are fp64 (2^-y from a table of 16 roots and the Taylor
// polynomial of 2^f, |f| <= 1/32, to f^5: 2e-13 relative).  Sums are formed in a
// fixed order or as whole numbers: equal inputs give equal tokens.
//
// Top-k, top-p and min-p need no sort of the row.  The k-th largest of the threads'
// largest values bounds the k largest from below (min-p bounds what it keeps
// itself), so that a second sweep, which skips most vectors by their largest value,
// hands a short list to the cluster's first CTA; it sorts the list, applies the
// rules and takes the token.  Top-p alone, and what the list does not hold, go by a
// histogram over bins of equal width in x: counts, and the values' mean place in the
// bin.  A bin's weight is close to its count times the weight at that place, which
// gives the bin that has top-p's bound; the next sweep forms the exact sum above it
// and lists the bin, and if the bound is not in it the next bin is taken.  Where the
// bin and all above it are few, the list decides as before.
// A bin with more values than the list holds (equal logits, or logits within a
// hundredth) is cut by the digits of the values' ordered bits, 11 at a time, with
// weights as whole numbers of 2^-44 (larger units for vocabularies beyond 2^18), and
// among equal values the lower indices are counted out.
//
// Bound: by temperature alone the row is read once, with 44 instructions for a value,
// 12 of them fp64 (256 x 151936 bf16: 88 us a call, of which the fp64 pipe is busy for
// 42 % and the issue of instructions for 59 %; 40 of 148 SMs have one row, the others
// two); with a short list the row is read once from memory and once from L2 (64 x
// 151936 with top-k 50 31 us, 256 rows 51 us); with top-p 0.6 alone 98 and 272 us.
// Few rows are split over the CTAs of a cluster, which exchange through distributed
// shared memory: what is counted is added to the first CTA's histogram by remote
// atomics, which nobody waits for.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "mma16.cuh"
#include "op_util.cuh"

namespace cg = cooperative_groups;

namespace gdn2 {
namespace {

constexpr int kSmThreads = 512;
constexpr int kSmWarps = kSmThreads / 32;
constexpr int kBins = 2048;
constexpr int kBinsPer = kBins / kSmThreads;   // bins of a thread
constexpr int kList = 2048;                    // longest list that is sorted
constexpr int kShort = kSmThreads;             // of a list that is sorted by counting
constexpr int kPlaces = 4096;                  // of a bin; 2^20 values' sum fits 32 bits
constexpr float kBinsPerUnit = 46.f;           // bins of a logit: 44 units below the maximum

struct SampleArgs {
  int64_t rows, ld;
  int V;
  double weight_unit;  // 2^(52 - s), with weights counted in 2^-s
  const void* x;
  const float *uniform, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  double temperature1, top_p1, min_p1;  // for all rows, where there is no pointer
  int64_t top_k1;
  int64_t* ids;
};

// What the cluster agrees on; the leader's copy counts.
struct Decision {
  uint64_t bound;    // keys of at least this are kept
  int bin;           // of the histogram that holds the bound, -1 where none does
  uint32_t above, in;          // values above the bin and in it
  uint64_t mass_above, mass;   // weights above the bin, and in all
  int64_t at;        // index found
};

struct SampleShared {
  double root[16];               // 2^(i/16)
  double warp_sum[kSmWarps];
  double total;                  // of this CTA
  uint32_t warp_max[kSmWarps], warp_bad[kSmWarps];
  uint32_t most, bad;            // of this CTA: the maximum's key, whether there is a NaN
  uint32_t warp_count[kSmWarps];
  uint64_t warp_mass[kSmWarps];
  Decision d;
  int n_list, first, reached;
  uint32_t count[kBins];
  union {
    uint64_t mass[kBins];
    uint32_t place[kBins];       // sums of the places in a bin, in parts of kPlaces
  };
  uint64_t list[kList];
};

// 2^-y for y >= +0 as fp64; 0 beyond 1022, for infinity and NaN
__device__ __forceinline__ double pow2_neg(const double* root, double y) {
  constexpr double magic = 6755399441055744.;  // 1.5 * 2^52: rounds to whole numbers
  constexpr double c1 = 0.69314718055994531, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4,
                   c5 = c4 * c1 / 5;
  const double t = fma(y, -16., magic);
  const int k = __double2loint(t);
  const double f = fma(t - magic, -.0625, -y);
  double p = fma(fma(fma(fma(fma(c5, f, c4), f, c3), f, c2), f, c1), f, 1.);
  p *= root[k & 15];
  const double w = __hiloint2double(__double2hiint(p) + ((k >> 4) << 20), __double2loint(p));
  // numbers that are not negative order as their bits do
  return (uint32_t)__double2hiint(y) <= 0x408ff000u ? w : 0.;
}

__device__ __forceinline__ uint32_t abs_bits(uint32_t w, float) { return w & 0x7fffffffu; }
__device__ __forceinline__ uint32_t abs_bits(uint32_t w, __nv_bfloat16) { return w & 0x7fff7fffu; }
__device__ __forceinline__ uint32_t abs_bits(uint32_t w, __half) { return w & 0x7fff7fffu; }

// Largest magnitude's bits, NaN above infinity (two 16-bit halves, or one word).
template <typename T, int N>
__device__ __forceinline__ uint32_t largest_bits(const Raw<T, N>& r, uint32_t most) {
#pragma unroll
  for (int i = 0; i < Raw<T, N>::kWords; ++i) {
    const uint32_t b = abs_bits(r.u[i], T{});
    if constexpr (sizeof(T) == 4) most = max(most, b);
    else most = __vmaxu2(most, b);
  }
  return most;
}
template <typename T> __device__ __forceinline__ bool bits_are_nan(uint32_t m) {
  if constexpr (sizeof(T) == 4) return m > 0x7f800000u;
  else {
    constexpr uint32_t inf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    return (m & 0xffffu) > inf || (m >> 16) > inf;
  }
}

// A CTA's part of a row, in the order of the row: parts, then warps.
template <typename T> struct RowShare {
  RowView<T> row;
  int plo, phi, wper, part, parts;
  static constexpr int VE = RowView<T>::VE;
  __device__ __forceinline__ RowShare(const T* p, int V, int part_, int parts_)
      : row(p, V), part(part_), parts(parts_) {
    const int per = (row.nvec + parts - 1) / parts;
    plo = min(part * per, row.nvec);
    phi = min(plo + per, row.nvec);
    wper = (phi - plo + kSmWarps - 1) / kSmWarps;
  }
  __device__ __forceinline__ int lo(int warp) const { return min(plo + warp * wper, phi); }
  // which warp of all parts has vector j
  __device__ __forceinline__ int warp_of(int j) const {
    const int per = (row.nvec + parts - 1) / parts, p = j / per;
    const int n = min(per, row.nvec - p * per), w = (n + kSmWarps - 1) / kSmWarps;
    return p * kSmWarps + (j - p * per) / w;
  }
  __device__ __forceinline__ int64_t index(int j, int e) const { return (int64_t)j * VE + e - row.off; }
  // f(vector, its place) for the lane's vectors of [lo, hi), U of them in flight
  template <int U, typename F> __device__ __forceinline__ void sweep(int lo, int hi, F&& f) const {
    int j = lo + (int)(threadIdx.x & 31);
    if constexpr (U > 1) {
      for (; j + (U - 1) * 32 < hi; j += U * 32) {
        Raw<T, VE> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = row.load(j + u * 32);
#pragma unroll
        for (int u = 0; u < U; ++u) f(v[u], j + u * 32);
      }
    }
#pragma unroll 1
    for (; j < hi; j += 32) f(row.load(j), j);
  }
  template <int U, typename F> __device__ __forceinline__ void sweep(F&& f) const {
    const int warp = threadIdx.x >> 5;
    sweep<U>(lo(warp), lo(warp + 1), f);
  }
};

__device__ __forceinline__ double warp_total(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// The parameters of one row, and which values they keep.
struct RowRule {
  float m;
  double c, most_y;  // weights 2^-y, y = (m - x) c; kept up to y = most_y
  uint64_t bound;    // and from this key
  float tau;         // the bound's value
  bool all_y, all_keys;
  const double* root;
  // falling values have rising bins; the same function wherever a bin is asked for
  __device__ __forceinline__ int bin(float x) const {
    return min((int)(__fmul_rn(__fsub_rn(m, x), kBinsPerUnit)), kBins - 1);
  }
  // the least value in bins up to b: bins fall as the ordered bits rise.  By all lanes
  // of a warp, a 32nd of the range at a time.
  __device__ __forceinline__ float least(int b) const {
    if (b < 0) return INFINITY;
    uint32_t lo = order_of(-FLT_MAX), hi = order_of(m);  // hi's bin is 0
    while (lo < hi) {
      const uint32_t step = (hi - lo) / 32 + 1, lane = threadIdx.x & 31;
      const uint32_t mine = hi - lo > lane * step ? lo + lane * step : hi;
      const unsigned in = __ballot_sync(0xffffffffu, bin(value_of(mine)) <= b);
      const int first = __ffs(in) - 1;  // none: beyond the last lane's
      const uint32_t from = lo;
      lo = first == 0 ? from : min(from + (first < 0 ? 31u : first - 1u) * step, hi) + 1u;
      if (first >= 0) hi = min(from + first * step, hi);
    }
    return value_of(hi);
  }
  __device__ __forceinline__ double weight(float x) const { return pow2_neg(root, ((double)m - x) * c); }
  __device__ __forceinline__ bool keeps(float x, int64_t i) const {
    if (x == -INFINITY) return false;
    if (!all_keys && !(x > tau) && (x < tau || key_of(x, (int)i) < bound)) return false;
    return all_y || ((double)m - x) * c <= most_y;
  }
};

// The first of kSmWarps sums with which the running sum, from `before` on, exceeds
// goal; -1 and `some` the last that is not zero where rounding leaves none.
__device__ __forceinline__ int which_warp(const double* sums, double goal, double& before, int& some) {
  double run = before;
  int who = -1;
  some = 0;
  for (int i = 0; i < kSmWarps; ++i) {
    const double t = sums[i];
    if (t > 0.) {
      some = i;
      if (who < 0 && run + t > goal) {
        who = i;
        before = run;
      }
    }
    run += t;
  }
  return who;
}

// The index at which the running sum of f(x, index) >= 0 over the row, in fp64,
// exceeds target(sum); where rounding leaves none, the last with f > 0.  The
// result is in the leader's d.at.  The warps' sums are given in s.warp_sum if
// `have`.  Called by all threads of the cluster.
template <typename T, typename F, typename G>
__device__ __forceinline__ void locate(cg::cluster_group& cluster, SampleShared& s, const RowShare<T>& sh,
                                       bool have, F&& f, G&& target) {
  constexpr int VE = RowView<T>::VE;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto sum_of = [&](int lo, int hi) {
    double mine = 0.;
    sh.template sweep<1>(lo, hi, [&](const Raw<T, VE>& v, int j) {
#pragma unroll
      for (int e = 0; e < VE; ++e) mine += f(raw_get(v, e), sh.index(j, e));
    });
    return warp_total(mine);
  };
  if (!have) {
    const double mine = sum_of(sh.lo(warp), sh.lo(warp + 1));
    if (lane == 0) s.warp_sum[warp] = mine;
  }
  __syncthreads();
  if (tid == 0) {
    double t = 0.;
    for (int i = 0; i < kSmWarps; ++i) t += s.warp_sum[i];
    s.total = t;
    s.d.at = -1;
  }
  cluster.sync();
  double before = 0., sum = 0.;
  int owner = -1, last = 0;  // the part with the target, the last that has a weight
  for (int q = 0; q < sh.parts; ++q) sum += *cluster.map_shared_rank(&s.total, q);
  const double goal = target(sum);
  double run = 0.;
  for (int q = 0; q < sh.parts; ++q) {
    const double t = *cluster.map_shared_rank(&s.total, q);
    if (t > 0.) last = q;
    if (owner < 0 && run + t > goal && t > 0.) { owner = q; before = run; }
    run += t;
  }
  bool none = owner < 0;
  if (none) owner = last;
  if (owner == sh.part) {
    // the warp whose vectors have the target, then a sixteenth of them, by the same
    // sums in the same order
    int some;
    int who = which_warp(s.warp_sum, none ? INFINITY : goal, before, some);
    if (who < 0) {
      who = some;
      none = true;
    }
    int lo = sh.lo(who), hi = sh.lo(who + 1);
    const int per = (hi - lo + kSmWarps - 1) / kSmWarps;
    const double mine = sum_of(min(lo + warp * per, hi), min(lo + (warp + 1) * per, hi));
    __syncthreads();  // the first sums have been read
    if (lane == 0) s.warp_sum[warp] = mine;
    __syncthreads();
    who = which_warp(s.warp_sum, none ? INFINITY : goal, before, some);
    if (who < 0) {
      who = some;
      none = true;
    }
    hi = min(lo + (who + 1) * per, hi);
    lo = min(lo + who * per, hi);
    if (warp == who) {
      int64_t found = -1, tail = -1;  // tail: the last index with a weight
      double at = before;
      for (int j0 = lo; j0 < hi && found < 0; j0 += 32) {
        const int j = j0 + lane;
        Raw<T, VE> v;
        double own = 0.;
        int64_t mytail = -1;
        if (j < hi) {
          v = sh.row.load(j);
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const double w = f(raw_get(v, e), sh.index(j, e));
            if (w > 0.) mytail = sh.index(j, e);
            own += w;
          }
        }
        double incl = own;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const double y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, !none && own > 0. && at + incl > goal);
        if (hit) {
          const int l = __ffs(hit) - 1;
          int64_t mineat = -1;
          if (lane == l) {
            double r = at + (incl - own);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              const double w = f(raw_get(v, e), sh.index(j, e));
              r += w;
              if (mineat < 0 && w > 0. && r > goal) mineat = sh.index(j, e);
            }
            if (mineat < 0) mineat = mytail;
          }
          found = __shfl_sync(0xffffffffu, mineat, l);
        }
        const unsigned has = __ballot_sync(0xffffffffu, mytail >= 0);
        if (has) tail = __shfl_sync(0xffffffffu, mytail, 31 - __clz(has));
        at += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) cluster.map_shared_rank(&s.d, 0)->at = found >= 0 ? found : tail;
    }
  }
  cluster.sync();
}

// Adds the parts' histograms into the leader's and finds the first bin at which
// the running count reaches k (MASS false) or the running weight share * (all).
template <bool MASS>
__device__ __forceinline__ void find_bin(cg::cluster_group& cluster, SampleShared& s, int part, int parts,
                                         uint32_t k, double share, uint32_t above0, uint64_t mass0,
                                         uint64_t mass_all) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cluster.sync();  // histograms complete
  if (part == 0) {
    uint32_t c[kBinsPer], cs = 0u;
    uint64_t w[kBinsPer], ws = 0u;
#pragma unroll
    for (int i = 0; i < kBinsPer; ++i) {
      const int b = tid * kBinsPer + i;
      c[i] = s.count[b];
      w[i] = s.mass[b];
    }
    for (int q = 1; q < parts; ++q) {
      const SampleShared* o = cluster.map_shared_rank(&s, q);
#pragma unroll
      for (int i = 0; i < kBinsPer; ++i) {
        c[i] += o->count[tid * kBinsPer + i];
        w[i] += o->mass[tid * kBinsPer + i];
      }
    }
#pragma unroll
    for (int i = 0; i < kBinsPer; ++i) {
      cs += c[i];
      ws += w[i];
    }
    uint32_t ci = cs;
    uint64_t wi = ws;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const uint32_t a = __shfl_up_sync(0xffffffffu, ci, o);
      const uint64_t b = __shfl_up_sync(0xffffffffu, wi, o);
      if (lane >= o) { ci += a; wi += b; }
    }
    if (lane == 31) { s.warp_count[warp] = ci; s.warp_mass[warp] = wi; }
    if (tid == 0) s.d.bin = -1;
    __syncthreads();
    uint32_t cb = above0, call = above0;
    uint64_t wb = mass0, wall = mass0;
    for (int i = 0; i < kSmWarps; ++i) {
      if (i < warp) { cb += s.warp_count[i]; wb += s.warp_mass[i]; }
      call += s.warp_count[i];
      wall += s.warp_mass[i];
    }
    cb += ci - cs;
    wb += wi - ws;
    // whole numbers up to 2^62 as fp64: the bound moves by 2^-53 of itself at most
    const uint64_t all = mass_all ? mass_all : wall;
    const double goal = share * (double)all;
#pragma unroll
    for (int i = 0; i < kBinsPer; ++i) {
      const bool here = MASS ? (double)wb < goal && (double)(wb + w[i]) >= goal
                             : cb < k && cb + c[i] >= k;
      if (here) {  // one bin of all
        s.d.bin = tid * kBinsPer + i;
        s.d.above = cb;
        s.d.mass_above = wb;
        s.d.in = c[i];
      }
      cb += c[i];
      wb += w[i];
    }
    if (tid == 0) s.d.mass = all;
  }
  cluster.sync();
}

// Sorts s.list[0 .. n) in falling order: up to kShort values, one for each thread,
// by counting the larger ones (100 values: 0.6 us), more by a bitonic sort (2048
// values: 20 us; with the exchanges inside a warp by shuffles 25 us).
__device__ __forceinline__ void sort_list(SampleShared& s, int n) {
  const int tid = threadIdx.x;
  if (n <= kShort) {
    __syncthreads();
    const uint64_t key = tid < n ? s.list[tid] : 0u;
    int rank = 0;
    if ((tid & ~31) < n) {
#pragma unroll 8
      for (int j = 0; j < n; ++j) rank += s.list[j] > key;
    }
    __syncthreads();
    if (tid < n) s.list[rank] = key;
    __syncthreads();
    return;
  }
  int size = 2;
  while (size < n) size *= 2;
  for (int i = tid + n; i < size; i += kSmThreads) s.list[i] = 0u;
  for (int k = 2; k <= size; k *= 2)
    for (int o = k / 2; o > 0; o /= 2) {
      __syncthreads();
      for (int i = tid; i < size / 2; i += kSmThreads) {
        const int a = 2 * i - (i & (o - 1)), b = a + o;
        const uint64_t x = s.list[a], y = s.list[b];
        if ((x < y) == ((a & k) == 0)) { s.list[a] = y; s.list[b] = x; }
      }
    }
  __syncthreads();
}

// A weight as a whole number of 2^-s (unit = 2^(52 - s)).
__device__ __forceinline__ uint64_t whole_weight(double w, double unit) {
  return (uint64_t)__double_as_longlong(w + unit) & 0xfffffffffffffull;
}

// Of the first n of the sorted list, how many are kept while the weights before
// them, on top of `above`, are below share * all (all = 0: the list's own weight);
// at least one.  Called by all threads of the leader.
__device__ __forceinline__ int count_by_mass(SampleShared& s, int n, uint64_t above, double share,
                                             uint64_t all, const RowRule& rule, double unit) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int per = kList / kSmThreads;
  uint64_t w[per], ws = 0u;
#pragma unroll
  for (int i = 0; i < per; ++i) {
    const int at = tid * per + i;
    w[i] = at < n ? whole_weight(rule.weight(value_of((uint32_t)(s.list[at] >> 32))), unit) : 0u;
    ws += w[i];
  }
  uint64_t before = ws;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const uint64_t b = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += b;
  }
  if (lane == 31) s.warp_mass[warp] = before;
  __syncthreads();
  before += above - ws;
  uint64_t own = above;
  for (int i = 0; i < kSmWarps; ++i) {
    if (i < warp) before += s.warp_mass[i];
    own += s.warp_mass[i];
  }
  const double goal = share * (double)(all ? all : own);
  if (tid == 0) s.reached = (double)own >= goal;
  int kept = 0;
#pragma unroll
  for (int i = 0; i < per; ++i) {
    kept += tid * per + i < n && (tid * per + i == 0 || (double)before < goal);
    before += w[i];
  }
  kept = __reduce_add_sync(0xffffffffu, kept);
  if (lane == 0) s.warp_count[warp] = (uint32_t)kept;
  __syncthreads();
  kept = 0;
  for (int i = 0; i < kSmWarps; ++i) kept += (int)s.warp_count[i];
  return kept;
}

// Narrows rule.bound to the k largest kept values (MASS false), or to those whose
// weight before them is below share * (all).
template <typename T, bool MASS>
__device__ __forceinline__ void narrow(cg::cluster_group& cluster, SampleShared& s, const RowShare<T>& sh,
                                       const SampleArgs& a, RowRule& rule, int64_t k, double share) {
  constexpr int VE = RowView<T>::VE;
  const int tid = threadIdx.x;
  SampleShared* lead = cluster.map_shared_rank(&s, 0);
  int bin = -1, shift = 32;   // the bin that was cut, the bits of `prefix` are those above shift
  uint32_t prefix = 0u, above = 0u;
  uint64_t mass_above = 0u, mass_all = 0u;
  for (int round = 0;; ++round) {
    // round 0: bins of equal width; then digits of the ordered bits, in the bin
    const int width = round == 3 ? 10 : 11;
    if (round > 0) shift -= width;
    for (int i = tid; i < kBins; i += kSmThreads) { s.count[i] = 0u; s.mass[i] = 0u; }
    if (tid == 0) s.n_list = 0;
    __syncthreads();
    sh.template sweep<1>([&](const Raw<T, VE>& v, int j) {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float x = raw_get(v, e);
        if (!rule.keeps(x, sh.index(j, e))) continue;
        int b = rule.bin(x);
        if (round > 0) {
          if (b != bin) continue;
          const uint32_t o = order_of(x);
          if (round > 1 && (o >> (shift + width)) != prefix) continue;
          b = (1 << width) - 1 - (int)((o >> shift) & ((1u << width) - 1u));
        }
        atomicAdd(&s.count[b], 1u);
        if constexpr (MASS)
          atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[b]),
                    (unsigned long long)whole_weight(rule.weight(x), a.weight_unit));
      }
    });
    __syncthreads();
    find_bin<MASS>(cluster, s, sh.part, sh.parts, (uint32_t)min(k, (int64_t)0x7fffffff), share, above,
                   mass_above, mass_all);
    const int b = lead->d.bin;
    if (b < 0) {  // fewer values than k: all are kept
      cluster.sync();
      return;
    }
    above = lead->d.above;
    mass_above = lead->d.mass_above;
    mass_all = lead->d.mass;
    const uint32_t in = lead->d.in;
    if (in <= kList) {
      sh.template sweep<1>([&](const Raw<T, VE>& v, int j) {
        const float most = raw_max(v);
        if (most == -INFINITY || (round == 0 ? rule.bin(most) > b : rule.bin(most) > bin)) return;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float x = raw_get(v, e);
          if (!rule.keeps(x, sh.index(j, e))) continue;
          const int c = rule.bin(x);
          if (round == 0) {
            if (c != b) continue;
          } else {
            if (c != bin) continue;
            const uint32_t o = order_of(x);
            if (round > 1 && (o >> (shift + width)) != prefix) continue;
            if ((1 << width) - 1 - (int)((o >> shift) & ((1u << width) - 1u)) != b) continue;
          }
          const int at = atomicAdd(&lead->n_list, 1);  // as many as were counted
          if (at < kList) lead->list[at] = key_of(x, (int)sh.index(j, e));
        }
      });
      cluster.sync();
      if (sh.part == 0) {
        const int n = min(s.n_list, kList);
        sort_list(s, n);
        int kept;
        if constexpr (MASS) kept = count_by_mass(s, n, mass_above, share, mass_all, rule, a.weight_unit);
        else kept = (int)min(k - above, (int64_t)n);
        if (tid == 0) s.d.bound = s.list[kept - 1];
      }
      cluster.sync();
      rule.bound = lead->d.bound;
      rule.tau = value_of((uint32_t)(rule.bound >> 32));
      rule.all_keys = false;
      cluster.sync();
      return;
    }
    if (round == 0) {
      bin = b;
    } else {
      prefix = (round == 1 ? 0u : prefix << width) | (uint32_t)((1 << width) - 1 - b);
    }
    cluster.sync();  // the decision has been read
    if (round == 3) {
      // `in` values are equal: the first of them by index are kept
      const float x0 = value_of(prefix);
      int64_t need;
      if constexpr (MASS) {
        const double w = (double)whole_weight(rule.weight(x0), a.weight_unit);
        const double left = share * (double)mass_all - (double)mass_above;
        need = w > 0. ? (int64_t)fmin(ceil(left / w), (double)in) : (int64_t)in;
      } else {
        need = k - above;
      }
      if (need < 1) need = 1;
      locate<T>(cluster, s, sh, false,
                [&](float x, int64_t i) { return x == x0 && rule.keeps(x, i) ? 1. : 0.; },
                [&](double) { return (double)need - .5; });
      rule.bound = key_of(x0, (int)lead->d.at);
      rule.tau = x0;
      rule.all_keys = false;
      cluster.sync();
      return;
    }
  }
}

// The token among the first `kept` of the sorted list (the leader's threads): into
// s.d.at.
__device__ __forceinline__ void pick_from_list(SampleShared& s, int kept, const RowRule& rule, double u) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __syncthreads();
  for (int i = tid; i < kept; i += kSmThreads) {  // by rising index, values behind it
    const uint64_t key = s.list[i];
    s.list[i] = key << 32 | key >> 32;
  }
  __syncthreads();
  sort_list(s, kept);
  constexpr int per = kList / kSmThreads;
  double w[per], ws = 0.;
#pragma unroll
  for (int i = 0; i < per; ++i) {
    const int at = tid * per + i;
    w[i] = at < kept ? rule.weight(value_of((uint32_t)s.list[at])) : 0.;
    ws += w[i];
  }
  double run = ws;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const double y = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += y;
  }
  if (lane == 31) s.warp_sum[warp] = run;
  if (tid == 0) s.first = kept - 1;
  __syncthreads();
  run -= ws;
  double sum = 0.;
  for (int i = 0; i < kSmWarps; ++i) {
    if (i < warp) run += s.warp_sum[i];
    sum += s.warp_sum[i];
  }
  const double goal = u * sum;
#pragma unroll
  for (int i = 0; i < per; ++i) {
    run += w[i];
    if (w[i] > 0. && run > goal) {
      atomicMin(&s.first, tid * per + i);
      break;
    }
  }
  __syncthreads();
  if (tid == 0) s.d.at = (int64_t)(uint32_t)~(uint32_t)(s.list[s.first] >> 32);
}

// Hands the values in [least, below) that the rule keeps to the leader's list.
template <typename T>
__device__ __forceinline__ void list_values(SampleShared* lead, const RowShare<T>& sh, const RowRule& rule,
                                            float least, float below) {
  constexpr int VE = RowView<T>::VE;
  sh.template sweep<4>([&](const Raw<T, VE>& v, int j) {
    if (!(raw_max(v) >= least)) return;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float x = raw_get(v, e);
      if (!(x >= least) || x >= below || !rule.keeps(x, sh.index(j, e))) continue;
      const int at = atomicAdd(&lead->n_list, 1);
      if (at < kList) lead->list[at] = key_of(x, (int)sh.index(j, e));
    }
  });
}

// The first of the leader's bins at which the running count reaches k, or (MASS)
// the running weight, each bin's taken at its mean place, reaches goal; the last bin
// with a value where rounding leaves none.  Into s.d.bin (-1: fewer than k), with the
// counts above and in it and its neighbours'.  The leader's threads.
template <bool MASS>
__device__ __forceinline__ void scan_bins(SampleShared& s, uint32_t k, double goal, int places,
                                          const RowRule& rule) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t c[kBinsPer], cs = 0u;
  double w[kBinsPer], ws = 0.;
#pragma unroll
  for (int i = 0; i < kBinsPer; ++i) {
    const int b = tid * kBinsPer + i;
    c[i] = s.count[b];
    cs += c[i];
    const double place = MASS && c[i] ? b + (double)s.place[b] / (places * (double)c[i]) : 0.;
    w[i] = MASS && c[i] ? c[i] * pow2_neg(rule.root, place * (1. / kBinsPerUnit) * rule.c) : 0.;
    ws += w[i];
  }
  uint32_t ci = cs;
  double wi = ws;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, ci, o);
    const double b = __shfl_up_sync(0xffffffffu, wi, o);
    if (lane >= o) { ci += a; wi += b; }
  }
  if (lane == 31) { s.warp_count[warp] = ci; s.warp_sum[warp] = wi; }
  if (tid == 0) { s.d.bin = -1; s.first = -1; }
  __syncthreads();
  uint32_t cb = ci - cs;
  double wb = wi - ws;
  for (int i = 0; i < warp; ++i) { cb += s.warp_count[i]; wb += s.warp_sum[i]; }
  int last = -1;
#pragma unroll
  for (int i = 0; i < kBinsPer; ++i) {
    const int b = tid * kBinsPer + i;
    if (c[i]) last = b;
    const bool here = MASS ? c[i] && wb < goal && wb + w[i] >= goal : cb < k && cb + c[i] >= k;
    if (here) s.d.bin = b;  // rounding may leave two neighbours: either will do
    cb += c[i];
    wb += w[i];
  }
  if constexpr (MASS) {
    if (last >= 0) atomicMax(&s.first, last);
    __syncthreads();
    if (tid == 0 && s.d.bin < 0) s.d.bin = s.first;
  }
  __syncthreads();
}

// Values in bins up to b (the leader's threads, all get it).
__device__ __forceinline__ uint32_t count_to(SampleShared& s, int b) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t c = 0u;
#pragma unroll
  for (int i = 0; i < kBinsPer; ++i)
    if (tid * kBinsPer + i <= b) c += s.count[tid * kBinsPer + i];
  c = __reduce_add_sync(0xffffffffu, c);
  __syncthreads();
  if (lane == 0) s.warp_count[warp] = c;
  __syncthreads();
  c = 0u;
  for (int i = 0; i < kSmWarps; ++i) c += s.warp_count[i];
  return c;
}

// What a list of at most kList values can decide: the values in bins up to that of
// the k-th largest of the threads' largest values (k < 0: all that the rule keeps)
// are sorted, top-k and top-p applied, and the token taken.  Returns whether the
// list held the set.  `mine` is the thread's largest value.
template <typename T>
__device__ __forceinline__ bool take_from_list(cg::cluster_group& cluster, SampleShared& s,
                                               const RowShare<T>& sh, const SampleArgs& a, const RowRule& rule,
                                               float mine, int k, int64_t top_k, double top_p, double u) {
  const int tid = threadIdx.x;
  SampleShared* lead = cluster.map_shared_rank(&s, 0);
  float least = -FLT_MAX;
  if (sh.part == 0) {
    for (int i = tid; i < kBins; i += kSmThreads) s.count[i] = 0u;
    if (tid == 0) s.n_list = 0;
  }
  cluster.sync();
  if (k >= 0) {
    if (mine != -INFINITY) atomicAdd(&lead->count[rule.bin(mine)], 1u);
    cluster.sync();
    if (sh.part == 0) scan_bins<false>(s, (uint32_t)k, 0., 1, rule);
    cluster.sync();
    const int most = lead->d.bin;
    cluster.sync();
    if (most < 0) return false;  // fewer threads than k have a value
    least = rule.least(most);
  }
  list_values(lead, sh, rule, least, INFINITY);
  cluster.sync();
  if (sh.part == 0) {
    const int n = s.n_list;
    int kept = 0;
    if (n <= kList) {
      sort_list(s, n);
      kept = top_k > 1 ? (int)min(top_k, (int64_t)n) : n;
      if (top_p < 1.) kept = count_by_mass(s, kept, 0u, top_p, 0u, rule, a.weight_unit);
      pick_from_list(s, kept, rule, u);
    }
    if (tid == 0) s.d.bin = kept;
  }
  cluster.sync();
  const bool done = lead->d.bin > 0;
  cluster.sync();
  return done;
}

enum { kNarrowed, kTaken, kCrowded };

// The bound of top-k (MASS false: the k largest of what the rule keeps), or of top-p
// with `goal` of the weights' sum, by a histogram.  kTaken: a list held all that is
// kept, and the token is taken (with then_share < 1 after top-p of the k largest);
// kNarrowed: the rule has the bound; kCrowded: a bin has more values than the list.
// `rest` (MASS): the sum's part beyond goal.  The values whose weights are below
// rest / vocab weigh less than it together, so they are not among those kept and
// are not counted.  With kNarrowed by MASS, s.warp_sum has the sums of what is kept.
template <typename T, bool MASS>
__device__ __forceinline__ int by_window(cg::cluster_group& cluster, SampleShared& s, const RowShare<T>& sh,
                                         const SampleArgs& a, RowRule& rule, int64_t k, double goal, double rest,
                                         double then_share, double u) {
  constexpr int VE = RowView<T>::VE;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // a little below the bound, for fp32's sake
  float low = -INFINITY;
  if (MASS && rest > 0.) {
    const double y = log2(a.V / rest) / rule.c;
    low = (float)(rule.m - y) - (float)(fabs((double)rule.m) + fabs(y)) * 1e-6f;
  }
  SampleShared* lead = cluster.map_shared_rank(&s, 0);
  for (int i = tid; i < kBins; i += kSmThreads) {
    s.count[i] = 0u;
    s.place[i] = 0u;
  }
  cluster.sync();
  const int places = a.V <= 1 << 20 ? kPlaces : 1;  // beyond, the bin's start: more bins are tried
  uint32_t far = 0u;  // in the last bin, where masks by low values all are
  sh.template sweep<2>([&](const Raw<T, VE>& v, int j) {
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float x = raw_get(v, e);
      if (!(x >= low) || !rule.keeps(x, sh.index(j, e))) continue;
      const float at = __fmul_rn(__fsub_rn(rule.m, x), kBinsPerUnit);
      const int b = min((int)at, kBins - 1);  // as rule.bin
      if (b == kBins - 1) {
        ++far;
        continue;
      }
      atomicAdd(&s.count[b], 1u);
      if constexpr (MASS) atomicAdd(&s.place[b], (uint32_t)((at - b) * places));
    }
  });
  far = __reduce_add_sync(0xffffffffu, far);
  if (lane == 0 && far) atomicAdd(&s.count[kBins - 1], far);
  __syncthreads();
  if (sh.part != 0)
    for (int i = tid; i < kBins; i += kSmThreads)
      if (s.count[i]) {
        atomicAdd(&lead->count[i], s.count[i]);
        if constexpr (MASS) atomicAdd(&lead->place[i], s.place[i]);
      }
  cluster.sync();
  if (sh.part == 0) scan_bins<MASS>(s, (uint32_t)min(k, (int64_t)0x7fffffff), goal, places, rule);
  cluster.sync();
  int at = lead->d.bin;
  if (at < 0) {
    cluster.sync();
    return kNarrowed;  // fewer values than k: all are kept
  }
  cluster.sync();  // the bin has been read
  for (int way = 0;;) {
    // the window: the bin, with all above it where they are few
    if (sh.part == 0) {
      const uint32_t to1 = count_to(s, at);
      uint32_t to0 = to1 <= kShort || at == 0 ? 0u : count_to(s, at - 1);
      if (tid == 0) {
        s.d.bin = to1 - to0 > kList ? -1 : to0 ? at : 0;
        s.d.in = (uint32_t)at;
        s.d.above = to0;
        s.n_list = 0;
      }
      const uint32_t all = MASS ? count_to(s, kBins - 1) : 0u;
      if (tid == 0) s.d.mass = to1 == all;  // nothing is below the window
    }
    cluster.sync();
    const int b0 = lead->d.bin, b1 = (int)lead->d.in;
    if (b0 < 0) {
      cluster.sync();
      return kCrowded;
    }
    const float least = rule.least(b1), below = rule.least(b0 - 1);
    double sum = 0.;
    if (MASS && b0 > 0) {  // with the exact sum above the window
      sh.template sweep<2>([&](const Raw<T, VE>& v, int j) {
        if (!(raw_max(v) >= least)) return;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float x = raw_get(v, e);
          if (!(x >= least) || !rule.keeps(x, sh.index(j, e))) continue;
          if (x >= below) {
            sum += rule.weight(x);
          } else {
            const int to = atomicAdd(&lead->n_list, 1);
            if (to < kList) lead->list[to] = key_of(x, (int)sh.index(j, e));
          }
        }
      });
      sum = warp_total(sum);
    } else {
      list_values(lead, sh, rule, least, below);
    }
    __syncthreads();
    if (lane == 0) s.warp_sum[warp] = sum;
    __syncthreads();
    if (tid == 0) {
      double t = 0.;
      for (int i = 0; i < kSmWarps; ++i) t += s.warp_sum[i];
      s.total = t;
    }
    cluster.sync();
    if (sh.part == 0) {
      const int n = min(s.n_list, kList);
      double above = 0.;
      for (int q = 0; q < sh.parts; ++q) above += *cluster.map_shared_rank(&s.total, q);
      sort_list(s, n);
      int kept = MASS ? 0 : (int)min(k - (int64_t)s.d.above, (int64_t)n), miss = 0;
      if constexpr (MASS) {
        const double unit = 4503599627370496. / a.weight_unit;  // whole weights of the goal's part in the list
        if (above < goal) {
          const double rest = (goal - above) * unit;
          kept = count_by_mass(s, n, 0u, 1., (uint64_t)__double2ll_ru(rest), rule, a.weight_unit);
          if (!s.reached && !s.d.mass) miss = 1;        // the bound is below the window
        } else {
          miss = -1;                                    // or above it
        }
      } else if (b0 == 0 && then_share < 1.) {
        kept = count_by_mass(s, kept, 0u, then_share, 0u, rule, a.weight_unit);
      }
      if (miss == 0 && kept < 1) miss = -1;
      // values that were not counted, in the bin that their bound cuts
      if (s.n_list > kList) miss = 2;
      if (miss == 0) {
        const uint64_t bound = s.list[kept - 1];
        if (b0 == 0) {
          pick_from_list(s, kept, rule, u);
        } else if (MASS) {
          // what the window keeps, in whole numbers, for the warps that have it
          for (int i = tid; i < kSmWarps * sh.parts; i += kSmThreads) s.mass[i] = 0u;
          __syncthreads();
          for (int i = tid; i < kept; i += kSmThreads) {
            const uint64_t key = s.list[i];
            const int64_t idx = (int64_t)(uint32_t)~(uint32_t)key;
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[sh.warp_of((int)((idx + sh.row.off) / VE))]),
                      (unsigned long long)whole_weight(rule.weight(value_of((uint32_t)(key >> 32))), a.weight_unit));
          }
        }
        if (tid == 0) s.d.bound = bound;
      }
      __syncthreads();
      // a window that missed: the next bin that has values, below it or above
      if (tid == 0) {
        s.d.bin = miss;
        s.first = miss > 0 ? kBins - 1 : 0;
      }
      __syncthreads();
      if (MASS && (miss == 1 || miss == -1))
#pragma unroll
        for (int i = 0; i < kBinsPer; ++i) {
          const int b = tid * kBinsPer + i;
          if (!s.count[b]) continue;
          if (miss > 0 && b > b1) atomicMin(&s.first, b);
          if (miss < 0 && b < b0) atomicMax(&s.first, b);
        }
    }
    cluster.sync();
    const int miss = lead->d.bin, next = lead->first;
    if (miss == 0) rule.bound = lead->d.bound;  // a window that missed has none: the rule's own stays
    if (MASS && miss == 0 && b0 > 0 && tid < kSmWarps)
      s.warp_sum[tid] += (double)lead->mass[sh.part * kSmWarps + tid] * (a.weight_unit / 4503599627370496.);
    cluster.sync();
    if (miss == 0) {
      rule.tau = value_of((uint32_t)(rule.bound >> 32));
      rule.all_keys = false;
      return b0 == 0 ? kTaken : kNarrowed;
    }
    // the sums' roundings at a bin's edge may send it back and forth: once is enough
    if (!MASS || miss == 2 || (way && way != miss)) return kCrowded;
    way = miss;
    at = next;
  }
}

template <typename T>
__global__ void __launch_bounds__(kSmThreads, 2) k_sample(const SampleArgs a, const int parts) {
  constexpr int VE = RowView<T>::VE;
  __shared__ SampleShared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x / (unsigned)parts;
  const int part = (int)(blockIdx.x - r * parts);
  const RowShare<T> sh((const T*)a.x + r * a.ld, a.V, part, parts);
  const double temperature = a.temperature ? (double)a.temperature[r] : a.temperature1;
  const double top_p = a.top_p ? (double)a.top_p[r] : a.top_p1;
  const double min_p = a.min_p ? (double)a.min_p[r] : a.min_p1;
  const int64_t top_k = a.top_k ? (int64_t)a.top_k[r] : a.top_k1;
  const float uniform = a.uniform[r];
  const bool greedy = temperature <= 0. || top_k == 1 || top_p <= 0.;
  const bool by_k = !greedy && top_k > 1 && top_k < a.V, by_p = !greedy && top_p < 1.;
  const bool by_min = !greedy && min_p > 0.;
  if (tid < 16) s.root[tid] = exp2(tid / 16.);
  __syncthreads();

  // The row's maximum; where nothing is cut off, the weights' sums with it, each
  // lane's in units of its own running maximum.
  // (a factor of at most 1e300 keeps the maximum's weight at 2^0)
  RowRule rule{0.f, fmin(1.4426950408889634 / temperature, 1e300), 0., 0u, -INFINITY, true, true, s.root};
  const bool at_once = !greedy && !by_k && !by_min;  // the sums with the maximum: temperature, top-p
  float mine = -INFINITY;
  double sum = 0.;
  uint32_t bits = 0u;
  if (at_once) {
    sh.template sweep<2>([&](const Raw<T, VE>& v, int) {
      bits = largest_bits(v, bits);
      const float top = raw_max(v);
      if (top > mine) {
        if (sum > 0.) sum *= pow2_neg(s.root, ((double)top - mine) * rule.c);
        mine = top + 0.f;  // not -0, from which +0 would be a negative zero away
      }
      if (mine == -INFINITY) return;
      const double m = mine;
#pragma unroll
      for (int e = 0; e < VE; ++e) sum += pow2_neg(s.root, (m - (double)raw_get(v, e)) * rule.c);
    });
  } else {
    sh.template sweep<4>([&](const Raw<T, VE>& v, int) {
      bits = largest_bits(v, bits);
      mine = fmaxf(mine, raw_max(v));
    });
  }
  // absent elements read as -inf, whose bits are those of infinity
  const bool nan = bits_are_nan<T>(bits);
  {
    const uint32_t o = __reduce_max_sync(0xffffffffu, order_of(mine));
    const unsigned bad = __ballot_sync(0xffffffffu, nan);
    if (lane == 0) { s.warp_max[warp] = o; s.warp_bad[warp] = bad; }
  }
  __syncthreads();
  if (tid == 0) {
    uint32_t o = 0u, bad = 0u;
    for (int i = 0; i < kSmWarps; ++i) { o = max(o, s.warp_max[i]); bad |= s.warp_bad[i]; }
    s.most = o;
    s.bad = bad;
  }
  cluster.sync();
  uint32_t most = 0u, bad = 0u;
  for (int q = 0; q < parts; ++q) {
    most = max(most, *cluster.map_shared_rank(&s.most, q));
    bad |= *cluster.map_shared_rank(&s.bad, q);
  }
  cluster.sync();
  rule.m = value_of(most);
  // no distribution: NaN, +inf, nothing but -inf, or options that are NaN
  if (bad || rule.m == INFINITY || rule.m == -INFINITY || temperature != temperature || top_p != top_p ||
      min_p != min_p || uniform != uniform) {
    if (part == 0 && tid == 0) a.ids[r] = -1;
    return;
  }

  if (greedy) {  // the first index of the maximum
    locate<T>(cluster, s, sh, false, [&](float x, int64_t) { return x == rule.m ? 1. : 0.; },
              [](double) { return 0.; });
  } else {
    if (by_min) {
      rule.all_y = false;
      rule.most_y = min_p < 1. ? -log2(min_p) : 0.;
    }
    const double u = fmin(fmax((double)uniform, 0.), 1.);
    if (at_once) {
      const double f = mine == -INFINITY ? 0. : pow2_neg(s.root, ((double)rule.m - mine) * rule.c);
      sum = warp_total(sum * f);
      if (lane == 0) s.warp_sum[warp] = sum;
    }
    bool done = false, summed = at_once;  // whether s.warp_sum has the sums of what is kept
    if (by_k || by_min) {
      // more than a few hundred would make a list that is slow to sort
      const int k = a.V <= kShort || !by_k ? -1 : (int)top_k;
      if (k <= kShort * 3 / 4)
        done = take_from_list<T>(cluster, s, sh, a, rule, mine, k, by_k ? top_k : 0, by_p ? top_p : 1., u);
    }
    if (!done && by_k) {
      const int how = by_window<T, false>(cluster, s, sh, a, rule, top_k, 0., 0., by_p ? top_p : 1., u);
      if (how == kCrowded) narrow<T, false>(cluster, s, sh, a, rule, top_k, 0.);
      done = how == kTaken;
    }
    if (!done && by_p) {
      // the weights' sum: formed with the maximum, or of what the rule keeps
      if (!at_once) {
        double own = 0.;
        sh.template sweep<1>([&](const Raw<T, VE>& v, int j) {
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float x = raw_get(v, e);
            if (rule.keeps(x, sh.index(j, e))) own += rule.weight(x);
          }
        });
        own = warp_total(own);
        if (lane == 0) s.warp_sum[warp] = own;
      }
      __syncthreads();
      if (tid == 0) {
        double t = 0.;
        for (int i = 0; i < kSmWarps; ++i) t += s.warp_sum[i];
        s.total = t;
      }
      cluster.sync();
      double total = 0.;
      for (int q = 0; q < parts; ++q) total += *cluster.map_shared_rank(&s.total, q);
      cluster.sync();
      const int how = by_window<T, true>(cluster, s, sh, a, rule, 0, top_p * total, (1. - top_p) * total, 1., u);
      if (how == kCrowded) narrow<T, true>(cluster, s, sh, a, rule, 0, top_p);
      done = how == kTaken;
      summed = how == kNarrowed;
    }
    if (!done)
      locate<T>(cluster, s, sh, summed,
                [&](float x, int64_t i) { return rule.keeps(x, i) ? rule.weight(x) : 0.; },
                [&](double w) { return u * w; });
  }
  if (part == 0 && tid == 0) a.ids[r] = s.d.at;
}

// ---------------------------------------------------------------------------
// entry point
// ---------------------------------------------------------------------------
template <typename T> cudaError_t launch_sample(const SampleArgs& a, int parts, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.rows * parts));
  cfg.blockDim = dim3(kSmThreads);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)parts;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_sample<T>, a, parts);
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

int gdn2_sample(const gdn2_sample_problem* p, const void* logits, const float* uniform,
                const float* temperature, const int32_t* top_k, const float* top_p,
                const float* min_p, int64_t* token_ids, void* stream) {
  const char* fn = "gdn2_sample";
  if (!p) return fail(GDN2_ERR_INVALID, "%s: null problem", fn);
  if (p->rows < 0 || p->vocab <= 0)
    return fail(GDN2_ERR_INVALID, "%s: needs rows >= 0 and vocab > 0 (got %lld, %d)", fn,
                (long long)p->rows, p->vocab);
  if (!dtype_valid(p->dtype)) return fail(GDN2_ERR_INVALID, "%s: unknown dtype %d", fn, p->dtype);
  if (p->ld < p->vocab)
    return fail(GDN2_ERR_INVALID, "%s: the row stride must be at least vocab", fn);
  if (!(temperature || (p->temperature >= 0. && std::isfinite(p->temperature))) ||
      !(top_k || p->top_k >= 0) || !(top_p || (p->top_p >= 0. && p->top_p <= 1.)) ||
      !(min_p || (p->min_p >= 0. && p->min_p <= 1.)))
    return fail(GDN2_ERR_INVALID,
                "%s: needs a finite temperature >= 0, top_k >= 0, top_p and min_p in [0, 1]", fn);
  // CTAs of a row: one where the rows fill the GPU, else as many (2, 4, 8) as keep
  // the grid within two CTAs per SM and 16 KB for each
  int sms = 0, parts = 1;
  if (p->rows > 2147483647LL / 8) return fail(GDN2_ERR_UNSUPPORTED, "%s: too many rows", fn);
  if (p->rows == 0) return GDN2_OK;
  if (!logits || !uniform || !token_ids) return fail(GDN2_ERR_INVALID, "%s: null pointer", fn);
  if (!aligned_to(logits, dtype_size(p->dtype)) || !aligned_to(token_ids, 8) ||
      !all_aligned(4, uniform, temperature, top_k, top_p, min_p))
    return fail(GDN2_ERR_INVALID, "%s: a pointer is not aligned to its elements", fn);
  const cudaError_t e = num_sms(&sms);
  if (e != cudaSuccess) return cuda_status(e, fn);
  const int64_t row_bytes = (int64_t)p->vocab * (int64_t)dtype_size(p->dtype);
  while (parts < 8 && p->rows * parts * 2 <= 2 * sms && row_bytes / (parts * 2) >= 16384) parts *= 2;
  SampleArgs a{};
  a.rows = p->rows;
  a.ld = p->ld;
  a.V = p->vocab;
  // sums of vocab weights of at most 2^s stay below 2^63
  int bits = 1;
  while (bits < 31 && (1LL << bits) <= p->vocab) ++bits;
  a.weight_unit = std::ldexp(1., 52 - std::min(44, 62 - bits));
  a.x = logits; a.uniform = uniform; a.temperature = temperature; a.top_k = top_k;
  a.top_p = top_p; a.min_p = min_p;
  a.temperature1 = p->temperature; a.top_k1 = p->top_k; a.top_p1 = p->top_p; a.min_p1 = p->min_p;
  a.ids = token_ids;
  const cudaStream_t st = (cudaStream_t)stream;
  return cuda_status(with_dtype(p->dtype, [&](auto t) {
    return launch_sample<decltype(t)>(a, parts, st);
  }), fn);
}

}  // extern "C"
