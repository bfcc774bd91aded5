// scan.cu -- gated linear recurrence over token rows, per channel,
//
//   h_t = exp(g_t) h_{t-1} + w_t v_t,    y_t = round(h_t)
//
// (GDN-2's decay and write gate without keys), its backward pass and its
// single-token form on a state pool.
//
// Mathematics.  A run of rows acts on the state entering it as h -> A h + H
// with A the product of its decays; runs compose as
// (A1, H1) then (A2, H2) = (A1 A2, A2 H1 + H2).  All B*T rows are one long
// scan: the first row of a sequence replaces the state by h0 (or 0), so a run
// that holds one ignores what enters it, marked by A = -1 (a product of
// exponentials is never negative) and selected, never multiplied, so that an
// infinity or NaN of one sequence does not reach the next.  The backward is
// the same scan in reverse on c_t = a_t dh_t:
//   dh_t = dy_t + c_{t+1},   c_t = a_t dh_t   (c after a last row: dht or 0)
//   dv = w dh,  dw = v dh,  dg_t = a_t h_{t-1} dh_t,  dh0 = c at a first row
// with h recomputed in fp32 from states that the forward keeps every 64 rows:
// reading v again costs what reading a stored y would.
//
// Bound: HBM (a handful of flops per element).  Each tensor is read and
// written once.  A cluster of CTAs walks a chain: kSlab channels of a stretch
// of rows that starts with a sequence, one tile of rows per CTA and turn.  A
// thread holds its rows of the tile in registers across the exchange of runs
// -- shuffles between a warp's two slots of rows, shared memory between warps,
// distributed shared memory between the cluster's CTAs -- and walks them a
// second time with the right entering state.  The next turn's rows come in by
// cp.async meanwhile.  The state passes from turn to turn inside the cluster:
// no CTA waits for another cluster, and the order of all products is fixed.
//
// Chains: whole sequences are dealt to stretches while there are enough of
// them to fill the GPU; clusters of 2 to 16 CTAs make up for too few.
#include <cooperative_groups.h>

#include "mma16.cuh"
#include "op_util.cuh"

namespace cg = cooperative_groups;

namespace gdn2 {
namespace {

constexpr int kSlab = 64;         // channels of a tile
constexpr int kLanes = 16;        // threads across a tile's channels
constexpr int kCpt = 4;           // channels of a thread
constexpr int kSlots = 16;        // threads down a tile's rows
constexpr int kScanThreads = kLanes * kSlots;
constexpr int kWarps = kScanThreads / 32;
constexpr int kKeep = 64;         // rows between the states kept for the backward
constexpr int kMaxCluster = 16;
constexpr int kCtas = 2;          // CTAs that share an SM

// Rows of a thread: as many as its registers hold (16-bit tensors, forward).
template <typename T, bool BWD> constexpr int rows_of() { return sizeof(T) == 2 && !BWD ? 8 : 4; }

struct ScanArgs {
  int64_t rows, T;     // T: rows of a sequence, fixed length
  int64_t stretch;     // rows of a chain (the last may have fewer)
  int64_t keeps;       // states kept of a chain
  int D, n_seqs, nslab, cluster;
  const int32_t* cu;
  const void *v, *g, *w, *dy;
  int64_t ldv, ldg, ldw, lddy;
  const float *h0, *dht;
  void *y, *dv, *dg, *dw;
  float *ht, *dh0, *saved;
};

// A run of rows: A in x (-1: it holds a reset), H in y.
__device__ __forceinline__ float2 compose(float2 p, float2 q) {
  if (q.x < 0.f) return q;
  return make_float2(p.x < 0.f ? -1.f : p.x * q.x, fmaf(q.x, p.y, q.y));
}

// State after a run that is entered with h.
__device__ __forceinline__ float leave(float2 p, float h) {
  return p.x < 0.f ? p.y : fmaf(p.x, h, p.y);
}

template <int TILE> struct ScanShared {
  float2 part[kWarps][kSlab];   // runs of the warps' slot pairs, then the runs before them
  float carry[kSlab];           // state entering the tile
  // of this turn and, while it is finished, the next:
  int seq[2][TILE];                      // the row's sequence
  uint32_t first[2][TILE / 32], last[2][TILE / 32];  // whether it is its first / last row
  float2 runs[2][kMaxCluster][kSlab];    // of the cluster's tiles, by turn
};

// A warp holds two slots of rows.  Puts their joint run into part[warp] and
// returns the run of the warp's rows before this thread's.
template <bool UP>
__device__ __forceinline__ void join_pair(float2 (*part)[kSlab], const float2 (&A2)[2],
                                          const float2 (&H2)[2], float2 (&before)[kCpt]) {
  const float A[kCpt] = {A2[0].x, A2[0].y, A2[1].x, A2[1].y};
  const float H[kCpt] = {H2[0].x, H2[0].y, H2[1].x, H2[1].y};
  const int lane = threadIdx.x & 31, lc = (lane % kLanes) * kCpt;
  const bool leads = (lane < kLanes) != UP;
#pragma unroll
  for (int j = 0; j < kCpt; ++j) {
    const float2 mine = make_float2(A[j], H[j]);
    const float2 other = make_float2(__shfl_xor_sync(0xffffffffu, A[j], kLanes),
                                     __shfl_xor_sync(0xffffffffu, H[j], kLanes));
    before[j] = leads ? make_float2(1.f, 0.f) : other;
    if (leads) part[threadIdx.x >> 5][lc + j] = compose(mine, other);
  }
}

// Turns part[] into the runs before each warp; returns the tile's run.
template <bool UP> __device__ __forceinline__ float2 fold_warps(float2 (*part)[kSlab], int ch) {
  float2 p[kWarps], run = make_float2(1.f, 0.f);
#pragma unroll
  for (int k = 0; k < kWarps; ++k) p[k] = part[UP ? kWarps - 1 - k : k][ch];
#pragma unroll
  for (int k = 0; k < kWarps; ++k) {
    part[UP ? kWarps - 1 - k : k][ch] = run;
    run = compose(run, p[k]);
  }
  return run;
}

// Sets s.carry, the state that enters this CTA's tile, from s.part of
// join_pair, and moves `state` (threads 0 .. 63, one per channel) from the
// state that enters the turn's first tile to the one that leaves its last.
// Called by all threads after a barrier; ends with one.  The runs of turn i+2
// overwrite those of turn i: every CTA has folded those before it arrived at
// the cluster barrier of turn i+1.
template <bool UP, int TILE>
__device__ __forceinline__ void exchange(const ScanArgs& a, ScanShared<TILE>& s, int rank, int turn,
                                         float& state) {
  const int ch = threadIdx.x;
  if (a.cluster == 1) {
    if (ch < kSlab) {
      const float2 run = fold_warps<UP>(s.part, ch);
      s.carry[ch] = state;
      state = leave(run, state);
    }
  } else {
    cg::cluster_group cluster = cg::this_cluster();
    if (ch < kSlab) {
      const float2 run = fold_warps<UP>(s.part, ch);
      float2* const slot = &s.runs[turn][rank][ch];
      for (int k = 0; k < a.cluster; ++k) *cluster.map_shared_rank(slot, k) = run;
    }
    cluster.sync();
    if (ch < kSlab) {
      float carry = state;
#pragma unroll 4
      for (int k = 0; k < a.cluster; ++k) {
        if (k == rank) carry = state;
        state = leave(s.runs[turn][k][ch], state);
      }
      s.carry[ch] = carry;
    }
  }
  __syncthreads();
}

// Follows a row (one for each of the first TILE threads) from turn to turn:
// its sequence, and where in it the row is.
struct RowWalk {
  int64_t at, len;  // place in the sequence, and the sequence's rows
  int n;

  __device__ __forceinline__ void find(const ScanArgs& a, int64_t r) {
    if (!a.cu) {
      n = (int)(r / a.T);
      at = r - (int64_t)n * a.T;
      len = a.T;
      return;
    }
    int lo = 0, hi = a.n_seqs;  // the last n with cu[n] <= r owns the row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(a.cu + mid) <= r) lo = mid; else hi = mid;
    }
    n = lo;
    at = r - __ldg(a.cu + lo);
    len = (int64_t)__ldg(a.cu + lo + 1) - __ldg(a.cu + lo);
  }
  // `r` is the row now, `by` (either sign) rows from the last one
  __device__ __forceinline__ void move(const ScanArgs& a, int64_t r, int64_t by) {
    at += by;
    if (at >= 0 && at < len) return;
    if (a.cu || a.T < 4096) return find(a, r);  // a turn is at most 2048 rows
    const int s = at < 0 ? -1 : 1;  // into the neighbour
    at -= s * a.T;
    n += s;
  }
};

// Marks the rows of the tile that starts at row `tile` for a turn; rows outside
// the chain have none.
template <int TILE>
__device__ __forceinline__ void mark_rows(const ScanArgs& a, ScanShared<TILE>& s, RowWalk& w,
                                          int which, int64_t tile, int64_t by, int64_t lo,
                                          int64_t hi) {
  if (threadIdx.x >= TILE) return;
  const int64_t r = tile + threadIdx.x;
  const bool in = r >= lo && r < hi;
  if (in) {
    if (by == 0) w.find(a, r);
    else w.move(a, r, by);
  }
  const uint32_t f = __ballot_sync(0xffffffffu, in && w.at == 0);
  const uint32_t l = __ballot_sync(0xffffffffu, in && w.at == w.len - 1);
  s.seq[which][threadIdx.x] = w.n;
  if ((threadIdx.x & 31) == 0) {
    s.first[which][threadIdx.x >> 5] = f;
    s.last[which][threadIdx.x >> 5] = l;
  }
}

// Sequences without rows: their state passes through (`from` NULL: zero).
__device__ __forceinline__ void pass_empty(const ScanArgs& a, int slab, const float* from,
                                           float* to) {
  if (!to || (!a.cu && a.T > 0)) return;
  const int c = slab * kSlab + (threadIdx.x & (kSlab - 1));
  if (c >= a.D) return;
  for (int n = threadIdx.x / kSlab; n < a.n_seqs; n += kScanThreads / kSlab)
    if (!a.cu || __ldg(a.cu + n) == __ldg(a.cu + n + 1))
      to[(int64_t)n * a.D + c] = from ? from[(int64_t)n * a.D + c] : 0.f;
}

// A thread's own rows of a tile in shared memory, filled asynchronously by
// the thread itself (no barrier) and read by it alone: group i of tensor k at
// k's section, row i, thread.
template <typename T, int R> struct Stage {
  static constexpr int kGroupBytes = kCpt * (int)sizeof(T);
  static constexpr int kBytes = R * kScanThreads * kGroupBytes;
  __device__ static __forceinline__ char* at(char* base, int i) {
    return base + (i * kScanThreads + threadIdx.x) * kGroupBytes;
  }
  __device__ static __forceinline__ void copy(char* base, int i, const T* src, int have) {
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(at(base, i));
    if constexpr (kGroupBytes == 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(have) : "memory");
    else
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(have) : "memory");
  }
  // rows r0 .. r0 + R - 1 of which those in [lo, hi) exist (`whole`: all, and
  // all channels); what does not exist reads as zero
  template <bool VEC>
  __device__ static __forceinline__ void fill(char* base, const void* x, int64_t ld, int64_t r0,
                                              int64_t lo, int64_t hi, int c, int nc, bool whole) {
    const T* p = (const T*)x + r0 * ld + c;
    if (VEC && whole) {
#pragma unroll
      for (int i = 0; i < R; ++i, p += ld) copy(base, i, p, kGroupBytes);
      return;
    }
#pragma unroll 1
    for (int i = 0; i < R; ++i, p += ld) {
      const int n = r0 + i >= lo && r0 + i < hi ? nc : 0;
      if constexpr (VEC)
        copy(base, i, n > 0 ? p : (const T*)x, n > 0 ? kGroupBytes : 0);
      else
        *reinterpret_cast<Raw<T, kCpt>*>(at(base, i)) = load_group<T, kCpt, false>(p, n);
    }
  }
  __device__ static __forceinline__ Raw<T, kCpt> get(char* base, int i) {
    Raw<T, kCpt> r;
    if constexpr (kGroupBytes == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(at(base, i));
      r.u[0] = v.x; r.u[1] = v.y; r.u[2] = v.z; r.u[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(at(base, i));
      r.u[0] = v.x; r.u[1] = v.y;
    }
    return r;
  }
};

__device__ __forceinline__ void stage_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Sections of a stage: g, v, w, dy.
template <typename T, typename G, bool GATE, bool BWD, int R> struct StageLayout {
  static constexpr int g = 0, v = Stage<G, R>::kBytes, w = v + Stage<T, R>::kBytes;
  static constexpr int dy = w + (GATE ? Stage<T, R>::kBytes : 0);
  static constexpr int bytes = dy + (BWD ? Stage<T, R>::kBytes : 0);
};

// A CTA's chain and place in it.
struct Place {
  int64_t lo, hi;   // rows of the chain
  int64_t chain;    // which stretch
  int rank, slab, turns;
};
template <int TILE> __device__ __forceinline__ Place place_of(const ScanArgs& a) {
  Place p;
  const unsigned id = blockIdx.x / (unsigned)a.cluster;
  p.rank = (int)(blockIdx.x - id * a.cluster);
  p.chain = id / (unsigned)a.nslab;
  p.slab = (int)(id - p.chain * a.nslab);
  p.lo = p.chain * a.stretch;
  p.hi = min(p.lo + a.stretch, a.rows);
  const int64_t step = (int64_t)a.cluster * TILE;
  p.turns = (int)((p.hi - p.lo + step - 1) / step);
  return p;
}

// Groups of four channels as two packed pairs.
template <typename T> __device__ __forceinline__ float2 pair_of(const Raw<T, kCpt>& r, int k) {
  if constexpr (sizeof(T) == 4)
    return make_float2(__uint_as_float(r.u[2 * k]), __uint_as_float(r.u[2 * k + 1]));
  else
    return unpack2<T>(r.u[k]);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_pairs(T* p, const float2 (&x)[2], int n) {
  const float f[kCpt] = {x[0].x, x[0].y, x[1].x, x[1].y};
  store_group<T, kCpt, VEC>(p, f, n);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// exp of log-decays: 2^(g log2 e), the hardware's base-2 exponential.  Its
// error and that of the product are about 2^-23 for decays near one, where
// errors add up over the steps; results below 2^-126 are zero.
__device__ __forceinline__ float2 decay_of(float2 g) { return exp2_2(mul2(g, both(kLog2e))); }

// Four channels of the states [n_seqs][D] (NULL: zero).
__device__ __forceinline__ void state_at(const float* x, int64_t seq, int D, int c, int nc,
                                         float2 (&h)[2]) {
  float f[kCpt];
#pragma unroll
  for (int j = 0; j < kCpt; ++j) f[j] = x && j < nc ? __ldg(x + seq * D + c + j) : 0.f;
  h[0] = make_float2(f[0], f[1]);
  h[1] = make_float2(f[2], f[3]);
}
__device__ __forceinline__ void put_state(float* x, int64_t seq, int D, int c, int nc,
                                          const float2 (&h)[2]) {
  const float f[kCpt] = {h[0].x, h[0].y, h[1].x, h[1].y};
#pragma unroll
  for (int j = 0; j < kCpt; ++j)
    if (j < nc) x[seq * D + c + j] = f[j];
}

// What enters a thread's rows: through the runs of the pair's rows and of the
// warps before them from the state entering the tile.
__device__ __forceinline__ void entering(const float2 (&pair)[kCpt], const float2* warps,
                                         const float* tile, float2 (&h)[2]) {
  float f[kCpt];
#pragma unroll
  for (int j = 0; j < kCpt; ++j) f[j] = leave(pair[j], leave(warps[j], tile[j]));
  h[0] = make_float2(f[0], f[1]);
  h[1] = make_float2(f[2], f[3]);
}

template <typename T, typename G, bool GATE, bool VEC>
__global__ void __launch_bounds__(kScanThreads, kCtas) k_scan_fwd(const ScanArgs a) {
  constexpr int R = rows_of<T, false>(), TILE = R * kSlots;
  using L = StageLayout<T, G, GATE, false, R>;
  extern __shared__ __align__(16) char st[];
  __shared__ ScanShared<TILE> s;
  const Place p = place_of<TILE>(a);
  const int slot = threadIdx.x / kLanes, warp = threadIdx.x >> 5;
  const int lc = (threadIdx.x % kLanes) * kCpt, c = p.slab * kSlab + lc, nc = a.D - c;
  const int64_t step = (int64_t)a.cluster * TILE;
  int64_t tile = p.lo + (int64_t)p.rank * TILE;  // first row of this turn's tile
  auto fill = [&](int64_t row) {
    const int64_t r0 = row + slot * R;
    const bool whole = r0 + R <= p.hi && nc >= kCpt;
    Stage<G, R>::template fill<VEC>(st + L::g, a.g, a.ldg, r0, p.lo, p.hi, c, nc, whole);
    Stage<T, R>::template fill<VEC>(st + L::v, a.v, a.ldv, r0, p.lo, p.hi, c, nc, whole);
    if constexpr (GATE)
      Stage<T, R>::template fill<VEC>(st + L::w, a.w, a.ldw, r0, p.lo, p.hi, c, nc, whole);
  };
  if (p.chain == 0 && p.rank == 0) pass_empty(a, p.slab, a.h0, a.ht);
  if (p.turns > 0) fill(tile);
  if (a.cluster > 1) cg::this_cluster().sync();  // all CTAs run before one writes to another
  float state = 0.f;
  RowWalk walk{};
  mark_rows(a, s, walk, 0, tile, 0, p.lo, p.hi);

  for (int turn = 0; turn < p.turns; ++turn, tile += step) {
    const int b = turn & 1;
    stage_wait();
    float2 d[R][2];
    // the inputs w v, packed as v where there is no gate
    typename std::conditional<GATE, Raw<float, kCpt>, Raw<T, kCpt>>::type x[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const Raw<G, kCpt> g = Stage<G, R>::get(st + L::g, i);
      const Raw<T, kCpt> v = Stage<T, R>::get(st + L::v, i);
      if constexpr (GATE) {
        const Raw<T, kCpt> w = Stage<T, R>::get(st + L::w, i);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 y = mul2(pair_of<T>(v, k), pair_of<T>(w, k));
          x[i].u[2 * k] = __float_as_uint(y.x);
          x[i].u[2 * k + 1] = __float_as_uint(y.y);
        }
      } else {
        x[i] = v;
      }
      d[i][0] = decay_of(pair_of<G>(g, 0));
      d[i][1] = decay_of(pair_of<G>(g, 1));
    }
    using X = typename std::conditional<GATE, float, T>::type;
    if (turn + 1 < p.turns) fill(tile + step);
    __syncthreads();
    const uint32_t first = (s.first[b][slot * R / 32] >> (slot * R % 32)) & ((1u << R) - 1);
    const uint32_t last = (s.last[b][slot * R / 32] >> (slot * R % 32)) & ((1u << R) - 1);
    const int* const seq = s.seq[b] + slot * R;

    float2 lead[kCpt];
    {
      float2 A[2] = {both(1.f), both(1.f)}, H[2] = {both(0.f), both(0.f)};
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (first >> i & 1) state_at(a.h0, seq[i], a.D, c, nc, H);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          H[k] = fma2(d[i][k], H[k], pair_of<X>(x[i], k));
          A[k] = mul2(A[k], d[i][k]);
        }
      }
      if (first) A[0] = A[1] = both(-1.f);
      join_pair<false>(s.part, A, H, lead);
    }
    __syncthreads();
    if (turn + 1 < p.turns) mark_rows(a, s, walk, b ^ 1, tile + step, step, p.lo, p.hi);
    exchange<false>(a, s, p.rank, b, state);

    float2 h[2];
    entering(lead, s.part[warp] + lc, s.carry + lc, h);
    const int64_t r0 = tile + slot * R;
    if (a.saved && (slot * R) % kKeep == 0 && r0 < p.hi)
      put_state(a.saved, p.chain * a.keeps + (r0 - p.lo) / kKeep, a.D, c, nc, h);
    const int here = (int)min((int64_t)R, p.hi - r0);  // rows that exist
    T* y = (T*)a.y + r0 * a.D + c;
#pragma unroll
    for (int i = 0; i < R; ++i, y += a.D) {
      if (first >> i & 1) state_at(a.h0, seq[i], a.D, c, nc, h);
#pragma unroll
      for (int k = 0; k < 2; ++k) h[k] = fma2(d[i][k], h[k], pair_of<X>(x[i], k));
      store_pairs<T, VEC>(y, h, i < here ? nc : 0);
      if ((last >> i & 1) && a.ht) put_state(a.ht, seq[i], a.D, c, nc, h);
    }
  }
}

template <typename T, typename G, bool GATE, bool VEC>
__global__ void __launch_bounds__(kScanThreads, kCtas) k_scan_bwd(const ScanArgs a) {
  constexpr int R = rows_of<T, true>(), TILE = R * kSlots;
  static_assert(TILE == kKeep, "a kept state enters every tile of the backward");
  using L = StageLayout<T, G, GATE, true, R>;
  extern __shared__ __align__(16) char st[];
  __shared__ ScanShared<TILE> s;
  __shared__ float2 ahead[kWarps][kSlab];  // s.part of the recomputed states
  __shared__ float enter[kSlab];           // the state entering the tile
  const Place p = place_of<TILE>(a);
  const int slot = threadIdx.x / kLanes, warp = threadIdx.x >> 5;
  const int lc = (threadIdx.x % kLanes) * kCpt, c = p.slab * kSlab + lc, nc = a.D - c;
  const int64_t step = (int64_t)a.cluster * TILE;
  // from the chain's last tile down; before the first there is nothing
  int64_t tile = p.lo + ((p.hi - p.lo + TILE - 1) / TILE - 1 - p.rank) * TILE;
  auto fill = [&](int64_t row) {
    const int64_t r0 = row + slot * R;
    const bool whole = r0 >= p.lo && r0 + R <= p.hi && nc >= kCpt;
    Stage<G, R>::template fill<VEC>(st + L::g, a.g, a.ldg, r0, p.lo, p.hi, c, nc, whole);
    Stage<T, R>::template fill<VEC>(st + L::v, a.v, a.ldv, r0, p.lo, p.hi, c, nc, whole);
    Stage<T, R>::template fill<VEC>(st + L::dy, a.dy, a.lddy, r0, p.lo, p.hi, c, nc, whole);
    if constexpr (GATE)
      Stage<T, R>::template fill<VEC>(st + L::w, a.w, a.ldw, r0, p.lo, p.hi, c, nc, whole);
  };
  if (p.chain == 0 && p.rank == 0) pass_empty(a, p.slab, a.dht, a.dh0);
  if (p.turns > 0) fill(tile);
  if (a.cluster > 1) cg::this_cluster().sync();  // all CTAs run before one writes to another
  float state = 0.f;
  RowWalk walk{};
  bool walking = tile + threadIdx.x < p.hi && tile >= p.lo;  // this thread's row was found
  mark_rows(a, s, walk, 0, tile, 0, p.lo, p.hi);

  for (int turn = 0; turn < p.turns; ++turn, tile -= step) {
    const int b = turn & 1;
    const bool some = tile >= p.lo;
    float kept = 0.f;
    if (threadIdx.x / kSlab == 1) {
      const int ch = p.slab * kSlab + threadIdx.x - kSlab;
      if (some && ch < a.D)
        kept = __ldg(a.saved + (p.chain * a.keeps + (tile - p.lo) / kKeep) * a.D + ch);
    }
    stage_wait();
    float2 d[R][2];
    Raw<T, kCpt> v[R], w[GATE ? R : 1], dy[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const Raw<G, kCpt> g = Stage<G, R>::get(st + L::g, i);
      v[i] = Stage<T, R>::get(st + L::v, i);
      dy[i] = Stage<T, R>::get(st + L::dy, i);
      if constexpr (GATE) w[i] = Stage<T, R>::get(st + L::w, i);
      d[i][0] = decay_of(pair_of<G>(g, 0));
      d[i][1] = decay_of(pair_of<G>(g, 1));
    }
    auto input = [&](int i, int k) {
      const float2 x = pair_of<T>(v[i], k);
      if constexpr (GATE) return mul2(x, pair_of<T>(w[i], k));
      return x;
    };
    if (turn + 1 < p.turns) fill(tile - step);
    __syncthreads();
    const uint32_t first = (s.first[b][slot * R / 32] >> (slot * R % 32)) & ((1u << R) - 1);
    const uint32_t last = (s.last[b][slot * R / 32] >> (slot * R % 32)) & ((1u << R) - 1);
    const int* const seq = s.seq[b] + slot * R;

    float2 lead[kCpt], trail[kCpt];  // runs of the pair's rows before / after these
    {
      float2 A[2] = {both(1.f), both(1.f)}, H[2] = {both(0.f), both(0.f)};
      float2 C[2] = {both(0.f), both(0.f)};
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (first >> i & 1) state_at(a.h0, seq[i], a.D, c, nc, H);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          H[k] = fma2(d[i][k], H[k], input(i, k));
          A[k] = mul2(A[k], d[i][k]);
        }
      }
#pragma unroll
      for (int i = R - 1; i >= 0; --i) {
        if (last >> i & 1) state_at(a.dht, seq[i], a.D, c, nc, C);
#pragma unroll
        for (int k = 0; k < 2; ++k) C[k] = mul2(d[i][k], add2(pair_of<T>(dy[i], k), C[k]));
      }
      const float2 Z[2] = {last ? both(-1.f) : A[0], last ? both(-1.f) : A[1]};
      if (first) A[0] = A[1] = both(-1.f);
      join_pair<false>(ahead, A, H, lead);
      join_pair<true>(s.part, Z, C, trail);
    }
    __syncthreads();
    if (threadIdx.x / kSlab == 1) {
      enter[threadIdx.x - kSlab] = kept;
      fold_warps<false>(ahead, threadIdx.x - kSlab);
    }
    if (turn + 1 < p.turns) {
      mark_rows(a, s, walk, b ^ 1, tile - step, walking ? -step : 0, p.lo, p.hi);
      walking = walking || tile - step + (int64_t)threadIdx.x < p.hi;
    }
    exchange<true>(a, s, p.rank, b, state);

    float2 before[R][2];  // a_t h_{t-1}
    {
      float2 h[2];
      entering(lead, ahead[warp] + lc, enter + lc, h);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (first >> i & 1) state_at(a.h0, seq[i], a.D, c, nc, h);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          before[i][k] = mul2(d[i][k], h[k]);
          h[k] = add2(before[i][k], input(i, k));
        }
      }
    }
    float2 cc[2];
    entering(trail, s.part[warp] + lc, s.carry + lc, cc);
    const int64_t r0 = tile + slot * R, at = r0 * a.D + c;
    const int here = some ? (int)min((int64_t)R, p.hi - r0) : 0;  // rows that exist
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      const int n = i < here ? nc : 0;
      const int64_t o = at + (int64_t)i * a.D;
      if (last >> i & 1) state_at(a.dht, seq[i], a.D, c, nc, cc);
      float2 dh[2], z[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        dh[k] = add2(pair_of<T>(dy[i], k), cc[k]);
        cc[k] = mul2(d[i][k], dh[k]);
        z[k] = mul2(before[i][k], dh[k]);
      }
      store_pairs<G, VEC>((G*)a.dg + o, z, n);
      if constexpr (GATE) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          z[k] = mul2(pair_of<T>(v[i], k), dh[k]);
          dh[k] = mul2(dh[k], pair_of<T>(w[i], k));
        }
        store_pairs<T, VEC>((T*)a.dw + o, z, n);
      }
      store_pairs<T, VEC>((T*)a.dv + o, dh, n);
      if ((first >> i & 1) && a.dh0) put_state(a.dh0, seq[i], a.D, c, nc, cc);
    }
  }
}

// One token for each of n sequences: the state pool's slot is read, updated
// and written back in place.  A slot index outside the pool marks padding:
// its state stays and its y is zero.
struct StepArgs {
  int n, D, pool;
  const void *v, *g, *w;
  int64_t ldv, ldg, ldw, lds;
  float* state;
  const int32_t* slots;
  void* y;
};

template <typename T, typename G, bool GATE, bool VEC>
__global__ void __launch_bounds__(256) k_scan_step(const StepArgs a) {
  const int groups = (a.D + kCpt - 1) / kCpt;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = id / groups;
  if (row >= a.n) return;
  const int c = (int)(id - row * groups) * kCpt, nc = a.D - c;
  const int slot = a.slots ? __ldg(a.slots + row) : (int)row;
  float h[kCpt] = {0.f, 0.f, 0.f, 0.f};
  if (slot >= 0 && slot < a.pool) {
    const auto g = load_group<G, kCpt, VEC>((const G*)a.g + row * a.ldg + c, nc);
    const auto v = load_group<T, kCpt, VEC>((const T*)a.v + row * a.ldv + c, nc);
    float* st = a.state + (int64_t)slot * a.lds + c;
#pragma unroll
    for (int j = 0; j < kCpt; ++j) h[j] = j < nc ? st[j] : 0.f;
    if constexpr (GATE) {
      const auto w = load_group<T, kCpt, VEC>((const T*)a.w + row * a.ldw + c, nc);
#pragma unroll
      for (int j = 0; j < kCpt; ++j)
        h[j] = fmaf(expf(raw_get(g, j)), h[j], raw_get(v, j) * raw_get(w, j));
    } else {
#pragma unroll
      for (int j = 0; j < kCpt; ++j) h[j] = fmaf(expf(raw_get(g, j)), h[j], raw_get(v, j));
    }
    store_group<float, kCpt, VEC>(st, h, nc);
  }
  store_group<T, kCpt, VEC>((T*)a.y + row * a.D + c, h, nc);
}

// ---------------------------------------------------------------------------
// entry points
// ---------------------------------------------------------------------------
int check_scan(const gdn2_scan_problem* p, const char* fn) {
  if (!p) return fail(GDN2_ERR_INVALID, "%s: null problem", fn);
  if (p->B < 0 || p->T < 0 || p->D <= 0 || p->n_seqs < 0)
    return fail(GDN2_ERR_INVALID, "%s: needs B, T, n_seqs >= 0 and D > 0 (got %d, %lld, %d, %d)",
                fn, p->B, (long long)p->T, p->n_seqs, p->D);
  if (!dtype_valid(p->dtype) || !dtype_valid(p->g_dtype))
    return fail(GDN2_ERR_INVALID, "%s: unknown dtype %d / %d", fn, p->dtype, p->g_dtype);
  if (p->g_dtype != p->dtype && p->g_dtype != GDN2_DTYPE_F32)
    return fail(GDN2_ERR_UNSUPPORTED, "%s: g must be fp32 or have v's dtype", fn);
  if (p->cu_seqlens ? p->B != 1 || p->T > 2147483647LL : p->n_seqs != p->B)
    return fail(GDN2_ERR_INVALID,
                "%s: packed sequences need B = 1 (T < 2^31), others n_seqs = B", fn);
  if (p->ld_v < p->D || p->ld_g < p->D || p->ld_w < 0 || p->ld_dy < 0)
    return fail(GDN2_ERR_INVALID, "%s: row strides must be at least D", fn);
  const int64_t rows = (int64_t)p->B * p->T;
  const int64_t nslab = (p->D + kSlab - 1) / kSlab;
  if ((p->T > 0 && rows / p->T != p->B) ||
      (rows / kKeep + p->B + kMaxCluster) > 2147483647LL / nslab)
    return fail(GDN2_ERR_UNSUPPORTED, "%s: too many rows x channels", fn);
  return GDN2_OK;
}

// How the rows are dealt out: `stretches` chains (each of whole sequences) and
// `cluster` CTAs for a chain.
struct ScanPlan {
  int64_t stretches;
  int64_t rows;     // of a stretch
  int cluster;
};

// The largest number of CTAs that any SM slot works through, in tiles, is what
// a plan costs; of equal ones the smaller cluster is taken (its exchange is
// cheaper).  A GPC places clusters of 8 and 16 on all but a few of its SMs.
ScanPlan scan_plan(const gdn2_scan_problem* p, int sms, int tile) {
  const int64_t rows = (int64_t)p->B * p->T, nslab = (p->D + kSlab - 1) / kSlab;
  ScanPlan best{1, rows, 1};
  int64_t least = -1;
  for (int c = 1; c <= kMaxCluster; c *= 2) {
    const int64_t slots = (int64_t)sms * kCtas * (c >= 8 ? 86 : 100) / 100 / c;  // clusters at once
    int64_t s = p->cu_seqlens ? 1 : slots / nslab;
    if (s > p->B) s = p->B;
    if (s < 1) s = 1;
    const int64_t each = p->B > 0 ? (p->B + s - 1) / s : 0;  // sequences of a stretch
    s = each > 0 ? (p->B + each - 1) / each : 1;
    const int64_t r = p->cu_seqlens ? rows : each * p->T;
    const int64_t waves = (s * nslab + slots - 1) / slots;
    const int64_t cost = waves * ((r + (int64_t)c * tile - 1) / ((int64_t)c * tile));
    if (least < 0 || cost < least) {
      least = cost;
      best = ScanPlan{s, r, c};
    }
  }
  return best;
}

int64_t scan_keeps(const ScanPlan& l) { return (l.rows + kKeep - 1) / kKeep; }

// The stretches are those of the backward's tiles in both directions, so that
// the kept states are found again; the cluster follows the kernel's own tile.
ScanArgs scan_args(const gdn2_scan_problem* p, int sms, int tile, int64_t* ctas) {
  ScanArgs a{};
  a.rows = (int64_t)p->B * p->T;
  a.T = p->T;
  a.D = p->D;
  a.n_seqs = p->n_seqs;
  a.nslab = (p->D + kSlab - 1) / kSlab;
  a.cu = p->cu_seqlens;
  a.ldv = p->ld_v;
  a.ldg = p->ld_g;
  a.ldw = p->ld_w;
  a.lddy = p->ld_dy;
  const ScanPlan l = scan_plan(p, sms, kKeep);
  a.stretch = l.rows;
  a.keeps = scan_keeps(l);
  a.cluster = l.cluster;
  while (a.cluster > 1 && (int64_t)(a.cluster / 2) * tile >= l.rows) a.cluster /= 2;
  *ctas = l.stretches * a.nslab * a.cluster;
  return a;
}

template <typename K>
cudaError_t launch_scan(K kernel, const ScanArgs& a, int64_t ctas, int smem, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess && a.cluster > 8)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kScanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)a.cluster;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = a.cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

// Whether every group of kCpt channels of a row can be moved as one vector.
bool group_ok(const void* p, int64_t ld, size_t es) {
  return aligned_to(p, kCpt * es) && ld % kCpt == 0;
}

// f(T, G, gate) over the element types and the presence of w.
template <typename F> cudaError_t scan_dispatch(const gdn2_scan_problem* p, bool gate, F&& f) {
  return with_dtype(p->dtype, [&](auto t) {
    using T = decltype(t);
    auto pick = [&](auto g) {
      return gate ? f(t, g, std::true_type{}) : f(t, g, std::false_type{});
    };
    return p->g_dtype == p->dtype ? pick(T{}) : pick(float{});
  });
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

size_t gdn2_scan_saved_bytes(const gdn2_scan_problem* p) {
  if (check_scan(p, "gdn2_scan_saved_bytes") != GDN2_OK) return 0;
  // whatever the stretches are: a state for every 64 rows and one for the rest
  // of each stretch, of which there are at most B
  const size_t rows = (size_t)p->B * p->T;
  return (rows / kKeep + p->B) * p->D * sizeof(float);
}

int gdn2_scan_fwd(const gdn2_scan_problem* p, const void* v, const void* g, const void* w,
                  const float* h0, void* y, float* ht, float* saved, void* stream) {
  const char* fn = "gdn2_scan_fwd";
  int rc = check_scan(p, fn);
  if (rc) return rc;
  const int64_t rows = (int64_t)p->B * p->T;
  if (rows > 0 && (!v || !g || !y)) return fail(GDN2_ERR_INVALID, "%s: null pointer", fn);
  if (w && p->ld_w < p->D) return fail(GDN2_ERR_INVALID, "%s: ld_w must be at least D", fn);
  if (p->n_seqs == 0 || (rows == 0 && !ht)) return GDN2_OK;
  const cudaStream_t st = (cudaStream_t)stream;
  int sms = 0;
  const cudaError_t e = num_sms(&sms);
  if (e != cudaSuccess) return cuda_status(e, fn);
  int64_t ctas = 0;
  ScanArgs a = scan_args(p, sms, kSlots * (p->dtype == GDN2_DTYPE_F32 ? rows_of<float, false>()
                                                                      : rows_of<__half, false>()),
                         &ctas);
  a.v = v; a.g = g; a.w = w; a.h0 = h0; a.y = y; a.ht = ht; a.saved = saved;
  const size_t es = dtype_size(p->dtype);
  const bool vec = a.D % kCpt == 0 && group_ok(v, a.ldv, es) && group_ok(y, a.D, es) &&
                   group_ok(g, a.ldg, dtype_size(p->g_dtype)) && (!w || group_ok(w, a.ldw, es));
  return cuda_status(scan_dispatch(p, w != nullptr, [&](auto t, auto gt, auto gate) {
    using T = decltype(t);
    using G = decltype(gt);
    constexpr bool W = decltype(gate)::value;
    constexpr int smem = StageLayout<T, G, W, false, rows_of<T, false>()>::bytes;
    return vec ? launch_scan(k_scan_fwd<T, G, W, true>, a, ctas, smem, st)
               : launch_scan(k_scan_fwd<T, G, W, false>, a, ctas, smem, st);
  }), fn);
}

int gdn2_scan_bwd(const gdn2_scan_problem* p, const void* v, const void* g, const void* w,
                  const float* h0, const float* saved, const void* dy, const float* dht,
                  void* dv, void* dg, void* dw, float* dh0, void* stream) {
  const char* fn = "gdn2_scan_bwd";
  int rc = check_scan(p, fn);
  if (rc) return rc;
  const int64_t rows = (int64_t)p->B * p->T;
  if (rows > 0 && (!v || !g || !saved || !dy || !dv || !dg || (w && !dw)))
    return fail(GDN2_ERR_INVALID, "%s: null pointer", fn);
  if (p->ld_dy < p->D || (w && p->ld_w < p->D))
    return fail(GDN2_ERR_INVALID, "%s: row strides must be at least D", fn);
  if (p->n_seqs == 0 || (rows == 0 && !dh0)) return GDN2_OK;
  const cudaStream_t st = (cudaStream_t)stream;
  int sms = 0;
  const cudaError_t e = num_sms(&sms);
  if (e != cudaSuccess) return cuda_status(e, fn);
  int64_t ctas = 0;
  ScanArgs a = scan_args(p, sms, kKeep, &ctas);
  a.v = v; a.g = g; a.w = w; a.h0 = h0; a.saved = const_cast<float*>(saved);
  a.dy = dy; a.dht = dht; a.dv = dv; a.dg = dg; a.dw = dw; a.dh0 = dh0;
  const size_t es = dtype_size(p->dtype), eg = dtype_size(p->g_dtype);
  const bool vec = a.D % kCpt == 0 && group_ok(v, a.ldv, es) && group_ok(dy, a.lddy, es) &&
                   group_ok(g, a.ldg, eg) && group_ok(dv, a.D, es) && group_ok(dg, a.D, eg) &&
                   (!w || (group_ok(w, a.ldw, es) && group_ok(dw, a.D, es)));
  return cuda_status(scan_dispatch(p, w != nullptr, [&](auto t, auto gt, auto gate) {
    using T = decltype(t);
    using G = decltype(gt);
    constexpr bool W = decltype(gate)::value;
    constexpr int smem = StageLayout<T, G, W, true, rows_of<T, true>()>::bytes;
    return vec ? launch_scan(k_scan_bwd<T, G, W, true>, a, ctas, smem, st)
               : launch_scan(k_scan_bwd<T, G, W, false>, a, ctas, smem, st);
  }), fn);
}

int gdn2_scan_step(const gdn2_scan_problem* p, const void* v, const void* g, const void* w,
                   float* state, int64_t state_stride, int32_t pool, const int32_t* state_indices,
                   void* y, void* stream) {
  const char* fn = "gdn2_scan_step";
  int rc = check_scan(p, fn);
  if (rc) return rc;
  if (p->T != 1 || p->cu_seqlens)
    return fail(GDN2_ERR_INVALID, "%s: one token per sequence (T = 1, no cu_seqlens)", fn);
  if (p->B == 0) return GDN2_OK;
  if (!v || !g || !state || !y) return fail(GDN2_ERR_INVALID, "%s: null pointer", fn);
  if (state_stride < p->D || pool <= 0 || (!state_indices && pool < p->B) ||
      (w && p->ld_w < p->D))
    return fail(GDN2_ERR_INVALID,
                "%s: needs state rows of at least D values and a row per sequence", fn);
  StepArgs a{};
  a.n = p->B; a.D = p->D; a.pool = pool;
  a.v = v; a.g = g; a.w = w; a.state = state; a.slots = state_indices; a.y = y;
  a.ldv = p->ld_v; a.ldg = p->ld_g; a.ldw = p->ld_w; a.lds = state_stride;
  const size_t es = dtype_size(p->dtype);
  const bool vec = a.D % kCpt == 0 && group_ok(v, a.ldv, es) && group_ok(y, a.D, es) &&
                   group_ok(g, a.ldg, dtype_size(p->g_dtype)) && group_ok(state, a.lds, 4) &&
                   (!w || group_ok(w, a.ldw, es));
  const int64_t blocks = ((int64_t)a.n * ((a.D + kCpt - 1) / kCpt) + 255) / 256;
  if (blocks > 2147483647LL) return fail(GDN2_ERR_UNSUPPORTED, "%s: too many channels", fn);
  const unsigned grid = (unsigned)blocks;
  const cudaStream_t st = (cudaStream_t)stream;
  return cuda_status(scan_dispatch(p, w != nullptr, [&](auto t, auto gt, auto gate) {
    using T = decltype(t);
    using G = decltype(gt);
    constexpr bool W = decltype(gate)::value;
    if (vec) k_scan_step<T, G, W, true><<<grid, 256, 0, st>>>(a);
    else k_scan_step<T, G, W, false><<<grid, 256, 0, st>>>(a);
    return cudaGetLastError();
  }), fn);
}

}  // extern "C"
