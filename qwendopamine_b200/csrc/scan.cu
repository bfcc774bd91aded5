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
// written once: a CTA takes kSlab channels x a tile of rows, its threads hold
// their rows in registers across the exchange of (A, H) between the CTA's row
// slots and between CTAs (below), and walk them a second time with the right
// entering state.
//
// Between CTAs.  Tiles are taken in row order from a counter, so every tile
// before a running one is done or running.  A tile publishes its (A, H); it
// reads those of the tiles before it in its group of kGroup tiles, and the
// state leaving the previous group, which that group's last tile publishes.
// The order of the products is fixed by the positions alone: results do not
// depend on timing.  A published pair is one 64-bit word that is all ones
// before (no decay product is that NaN), so it needs no flag and no fence, and
// a tile has all it reads in flight at once, eight words to a thread.  Waits
// are bounded; one that runs out sets bit 4 of the fault word and turns the
// tile's carry into NaN.
#include "op_util.cuh"

namespace gdn2 {
namespace {

constexpr int kSlab = 64;         // channels of a tile
constexpr int kLanes = 16;        // threads across a tile's channels
constexpr int kCpt = 4;           // channels of a thread
constexpr int kSlots = 16;        // threads down a tile's rows
constexpr int kScanThreads = kLanes * kSlots;
constexpr int kWarps = kScanThreads / 32;
constexpr int kFwdRows = 8;       // rows of a thread, forward
constexpr int kBwdRows = 4;       // and backward (twice the tensors in registers)
constexpr int kSaveRows = kSlots * kBwdRows;  // rows between states kept for the backward
constexpr int kGroup = 32;        // tiles between published states
constexpr unsigned kScanFault = 16u;
constexpr uint64_t kScanWaitNs = 1000000000ull;

struct ScanArgs {
  int64_t rows, T;     // T: rows of a sequence, fixed length
  int D, n_seqs, nslab, chained;
  int64_t ntiles;
  const int32_t* cu;
  const void *v, *g, *w, *dy;
  int64_t ldv, ldg, ldw, lddy;
  const float *h0, *dht;
  void *y, *dv, *dg, *dw;
  float *ht, *dh0, *saved;
  unsigned *ticket, *fault;
  uint64_t *runs, *states;
};

struct ScanWorkspace {
  size_t runs, states, total;
};

ScanWorkspace scan_workspace(int64_t rows, int D, int tile) {
  ScanWorkspace w;
  const size_t nslab = (size_t)(D + kSlab - 1) / kSlab;
  const size_t nt = (size_t)((rows + tile - 1) / tile), ng = (nt + kGroup - 1) / kGroup;
  size_t off = 256;  // the tile counter
  w.runs = off; off += nt * nslab * kSlab * sizeof(uint64_t);
  w.states = off; off += ng * nslab * kSlab * sizeof(uint64_t);
  w.total = off;
  return w;
}

// A run of rows: A in x (-1: it holds a reset), H in y.
__device__ __forceinline__ float2 compose(float2 p, float2 q) {
  if (q.x < 0.f) return q;
  return make_float2(p.x < 0.f ? -1.f : p.x * q.x, fmaf(q.x, p.y, q.y));
}

// State after a run that is entered with h.
__device__ __forceinline__ float leave(float2 p, float h) {
  return p.x < 0.f ? p.y : fmaf(p.x, h, p.y);
}

__device__ __forceinline__ uint64_t load_word(const uint64_t* p) {
  uint64_t v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ bool is_there(uint64_t v) { return (uint32_t)v != 0xffffffffu; }
__device__ __forceinline__ float2 run_of(uint64_t v) {
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}
__device__ __forceinline__ void publish(uint64_t* p, float2 r) {
  const uint32_t x = r.x != r.x ? 0x7fffffffu : __float_as_uint(r.x);
  const uint64_t v = ((uint64_t)__float_as_uint(r.y) << 32) | x;
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

// Polls until the word is there; false if the time ran out.
__device__ __forceinline__ bool wait_word(const uint64_t* p, uint64_t& v) {
  if (is_there(v)) return true;
  const uint64_t t0 = now_ns();
  for (int round = 0; round < (1 << 24); ++round) {
    v = load_word(p);
    if (is_there(v)) return true;
    if (now_ns() - t0 > kScanWaitNs) return false;
  }
  return false;
}

struct ScanShared {
  float2 part[kWarps][kSlab];   // runs of the warps' slot pairs, then the runs before them
  float2 past[4][kSlab];        // runs of eight tiles of the group each
  float carry[kSlab];           // state entering the tile
  unsigned item;
};

// A warp holds two slots of rows.  Puts their joint run into part[warp] and
// returns the run of the warp's rows before this thread's.
template <bool UP>
__device__ __forceinline__ void join_pair(float2 (*part)[kSlab], const float (&A)[kCpt],
                                          const float (&H)[kCpt], float2 (&before)[kCpt]) {
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

// Sets s.carry, the state that enters the tile, given s.part of join_pair;
// `pos` is the tile's place in processing order.  Called by all threads after
// a barrier; ends with one.
template <bool UP>
__device__ __forceinline__ void exchange(const ScanArgs& a, ScanShared& s, int64_t pos, int slab) {
  const int ch = threadIdx.x % kSlab, q = threadIdx.x / kSlab;
  const int64_t group = pos / kGroup, first = group * kGroup;
  const int n = (int)(pos - first);
  const int64_t stride = (int64_t)a.nslab * kSlab, at = (int64_t)slab * kSlab + ch;
  float2 run;
  uint64_t state = 0;
  bool ok = true;
  if (q == 0) {
    run = fold_warps<UP>(s.part, ch);
    if (a.chained) {
      // the last tile's run is only needed in the group's state
      if (n < kGroup - 1) publish(a.runs + pos * stride + at, run);
      if (group > 0) state = load_word(a.states + (group - 1) * stride + at);
    }
  }
  if (a.chained) {
    const uint64_t* p = a.runs + (first + q * (kGroup / 4)) * stride + at;
    uint64_t v[kGroup / 4];
#pragma unroll
    for (int k = 0; k < kGroup / 4; ++k)
      if (q * (kGroup / 4) + k < n) v[k] = load_word(p + k * stride);
    float2 acc = make_float2(1.f, 0.f);
#pragma unroll
    for (int k = 0; k < kGroup / 4; ++k)
      if (q * (kGroup / 4) + k < n) {
        ok = wait_word(p + k * stride, v[k]) && ok;
        acc = compose(acc, run_of(v[k]));
      }
    s.past[q][ch] = acc;
    ok = __syncthreads_and(ok);
  }
  if (q == 0) {
    float carry = 0.f;
    if (a.chained) {
      float2 acc = s.past[0][ch];
#pragma unroll
      for (int k = 1; k < 4; ++k) acc = compose(acc, s.past[k][ch]);
      carry = acc.y;
      if (group > 0 && !(acc.x < 0.f)) {
        ok = wait_word(a.states + (group - 1) * stride + at, state) && ok;
        carry = leave(acc, run_of(state).y);
      }
      if (!ok) {
        carry = __int_as_float(0x7fffffff);
        atomicOr(a.fault, kScanFault);
      }
      if (n == kGroup - 1)
        publish(a.states + group * stride + at, make_float2(0.f, leave(run, carry)));
    }
    s.carry[ch] = carry;
  }
  __syncthreads();
}

// The sequence that owns row r, and whether r is its first / last row.
struct RowMark {
  int first, last;  // sequence index, or -1
};
__device__ __forceinline__ RowMark mark_row(const ScanArgs& a, int64_t r) {
  RowMark m{-1, -1};
  if (r >= a.rows) return m;
  if (!a.cu) {
    const int64_t n = r / a.T, t = r - n * a.T;
    if (t == 0) m.first = (int)n;
    if (t == a.T - 1) m.last = (int)n;
    return m;
  }
  int lo = 0, hi = a.n_seqs;  // the last n with cu[n] <= r owns the row
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(a.cu + mid) <= r) lo = mid; else hi = mid;
  }
  if (__ldg(a.cu + lo) == r) m.first = lo;
  if (__ldg(a.cu + lo + 1) == r + 1) m.last = lo;
  return m;
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

__device__ __forceinline__ unsigned take_item(const ScanArgs& a, ScanShared& s) {
  if (!a.chained) return blockIdx.x;
  if (threadIdx.x == 0) s.item = atomicAdd(a.ticket, 1u) + 1u;  // starts at all ones
  __syncthreads();
  return s.item;
}

template <typename T, typename G, bool GATE, bool VEC>
__global__ void __launch_bounds__(kScanThreads, 2) k_scan_fwd(const ScanArgs a) {
  constexpr int R = kFwdRows;
  __shared__ ScanShared s;
  __shared__ int first_s[kSlots * R], last_s[kSlots * R];
  const unsigned item = take_item(a, s);
  const int64_t pos = item / (unsigned)a.nslab;
  const int slab = (int)(item - pos * a.nslab);
  const int slot = threadIdx.x / kLanes, lc = (threadIdx.x % kLanes) * kCpt;
  const int c = slab * kSlab + lc, nc = a.D - c;
  const int64_t r0 = pos * (kSlots * R) + slot * R;

  Raw<T, kCpt> v[R], w[GATE ? R : 1];
  float d[R][kCpt];  // log-decays, then decays
  {
    Raw<G, kCpt> g[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t r = r0 + i;
      const int n = r < a.rows ? nc : 0;
      g[i] = load_group<G, kCpt, VEC>((const G*)a.g + r * a.ldg + c, n);
      v[i] = load_group<T, kCpt, VEC>((const T*)a.v + r * a.ldv + c, n);
      if constexpr (GATE) w[i] = load_group<T, kCpt, VEC>((const T*)a.w + r * a.ldw + c, n);
    }
    if (threadIdx.x < kSlots * R) {
      const RowMark m = mark_row(a, pos * (kSlots * R) + threadIdx.x);
      first_s[threadIdx.x] = m.first;
      last_s[threadIdx.x] = m.last;
    }
    if (pos == 0) pass_empty(a, slab, a.h0, a.ht);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < kCpt; ++j) d[i][j] = expf(raw_get(g[i], j));
  }
  __syncthreads();

  auto input = [&](int i, int j) {
    const float x = raw_get(v[i], j);
    if constexpr (GATE) return x * raw_get(w[i], j);
    return x;
  };
  auto start = [&](int seq, int j) {
    return a.h0 && j < nc ? __ldg(a.h0 + (int64_t)seq * a.D + c + j) : 0.f;
  };

  float A[kCpt], H[kCpt];
  bool seen = false;
#pragma unroll
  for (int j = 0; j < kCpt; ++j) { A[j] = 1.f; H[j] = 0.f; }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int seq = first_s[slot * R + i];
    if (seq >= 0) {
      seen = true;
#pragma unroll
      for (int j = 0; j < kCpt; ++j) H[j] = start(seq, j);
    }
#pragma unroll
    for (int j = 0; j < kCpt; ++j) {
      H[j] = fmaf(d[i][j], H[j], input(i, j));
      A[j] *= d[i][j];
    }
  }
#pragma unroll
  for (int j = 0; j < kCpt; ++j)
    if (seen) A[j] = -1.f;
  float2 lead[kCpt];
  join_pair<false>(s.part, A, H, lead);
  __syncthreads();
  exchange<false>(a, s, pos, slab);

  float h[kCpt];
#pragma unroll
  for (int j = 0; j < kCpt; ++j)
    h[j] = leave(lead[j], leave(s.part[threadIdx.x >> 5][lc + j], s.carry[lc + j]));
  if (a.saved && (slot * R) % kSaveRows == 0 && r0 < a.rows) {
    float* keep = a.saved + r0 / kSaveRows * a.D + c;
#pragma unroll
    for (int j = 0; j < kCpt; ++j)
      if (j < nc) keep[j] = h[j];
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t r = r0 + i;
    const int seq = first_s[slot * R + i], end = last_s[slot * R + i];
    if (seq >= 0) {
#pragma unroll
      for (int j = 0; j < kCpt; ++j) h[j] = start(seq, j);
    }
#pragma unroll
    for (int j = 0; j < kCpt; ++j) h[j] = fmaf(d[i][j], h[j], input(i, j));
    store_group<T, kCpt, VEC>((T*)a.y + r * a.D + c, h, r < a.rows ? nc : 0);
    if (end >= 0 && a.ht) {
#pragma unroll
      for (int j = 0; j < kCpt; ++j)
        if (j < nc) a.ht[(int64_t)end * a.D + c + j] = h[j];
    }
  }
}

template <typename T, typename G, bool GATE, bool VEC>
__global__ void __launch_bounds__(kScanThreads, 2) k_scan_bwd(const ScanArgs a) {
  constexpr int R = kBwdRows;
  __shared__ ScanShared s;
  __shared__ float2 ahead[kWarps][kSlab];  // the same for the recomputed states
  __shared__ float enter[kSlab];
  __shared__ int first_s[kSlots * R], last_s[kSlots * R];
  const unsigned item = take_item(a, s);
  const int64_t pos = item / (unsigned)a.nslab;
  const int slab = (int)(item - pos * a.nslab);
  const int64_t tile = a.ntiles - 1 - pos;
  const int slot = threadIdx.x / kLanes, lc = (threadIdx.x % kLanes) * kCpt;
  const int c = slab * kSlab + lc, nc = a.D - c;
  const int64_t r0 = tile * (kSlots * R) + slot * R;

  Raw<T, kCpt> v[R], w[GATE ? R : 1], dy[R];
  float d[R][kCpt];
  {
    Raw<G, kCpt> g[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t r = r0 + i;
      const int n = r < a.rows ? nc : 0;
      g[i] = load_group<G, kCpt, VEC>((const G*)a.g + r * a.ldg + c, n);
      dy[i] = load_group<T, kCpt, VEC>((const T*)a.dy + r * a.lddy + c, n);
      v[i] = load_group<T, kCpt, VEC>((const T*)a.v + r * a.ldv + c, n);
      if constexpr (GATE) w[i] = load_group<T, kCpt, VEC>((const T*)a.w + r * a.ldw + c, n);
    }
    if (threadIdx.x < kSlots * R) {
      const RowMark m = mark_row(a, tile * (kSlots * R) + threadIdx.x);
      first_s[threadIdx.x] = m.first;
      last_s[threadIdx.x] = m.last;
    }
    if (pos == 0) pass_empty(a, slab, a.dht, a.dh0);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < kCpt; ++j) d[i][j] = expf(raw_get(g[i], j));
  }
  __syncthreads();

  auto input = [&](int i, int j) {
    const float x = raw_get(v[i], j);
    if constexpr (GATE) return x * raw_get(w[i], j);
    return x;
  };
  auto start = [&](int seq, int j) {
    return a.h0 && j < nc ? __ldg(a.h0 + (int64_t)seq * a.D + c + j) : 0.f;
  };
  auto finish = [&](int seq, int j) {
    return a.dht && j < nc ? __ldg(a.dht + (int64_t)seq * a.D + c + j) : 0.f;
  };

  float2 lead[kCpt], trail[kCpt];  // runs of the pair's rows before / after these
  {
    float A[kCpt], H[kCpt], C[kCpt];
    bool began = false, ended = false;
#pragma unroll
    for (int j = 0; j < kCpt; ++j) { A[j] = 1.f; H[j] = 0.f; C[j] = 0.f; }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int seq = first_s[slot * R + i];
      if (seq >= 0) {
        began = true;
#pragma unroll
        for (int j = 0; j < kCpt; ++j) H[j] = start(seq, j);
      }
#pragma unroll
      for (int j = 0; j < kCpt; ++j) {
        H[j] = fmaf(d[i][j], H[j], input(i, j));
        A[j] *= d[i][j];
      }
    }
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      const int seq = last_s[slot * R + i];
      if (seq >= 0) {
        ended = true;
#pragma unroll
        for (int j = 0; j < kCpt; ++j) C[j] = finish(seq, j);
      }
#pragma unroll
      for (int j = 0; j < kCpt; ++j) C[j] = d[i][j] * (raw_get(dy[i], j) + C[j]);
    }
    float A2[kCpt];
#pragma unroll
    for (int j = 0; j < kCpt; ++j) {
      A2[j] = ended ? -1.f : A[j];
      if (began) A[j] = -1.f;
    }
    join_pair<false>(ahead, A, H, lead);
    join_pair<true>(s.part, A2, C, trail);
  }
  __syncthreads();
  if (threadIdx.x / kSlab == 1) {
    const int ch = threadIdx.x - kSlab;
    const bool have = slab * kSlab + ch < a.D && tile * (kSlots * R) < a.rows;
    enter[ch] = have ? a.saved[tile * a.D + slab * kSlab + ch] : 0.f;
    fold_warps<false>(ahead, ch);
  }
  exchange<true>(a, s, pos, slab);

  float before[R][kCpt];  // a_t h_{t-1}
  {
    float h[kCpt];
#pragma unroll
    for (int j = 0; j < kCpt; ++j)
      h[j] = leave(lead[j], leave(ahead[threadIdx.x >> 5][lc + j], enter[lc + j]));
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int seq = first_s[slot * R + i];
      if (seq >= 0) {
#pragma unroll
        for (int j = 0; j < kCpt; ++j) h[j] = start(seq, j);
      }
#pragma unroll
      for (int j = 0; j < kCpt; ++j) {
        before[i][j] = d[i][j] * h[j];
        h[j] = before[i][j] + input(i, j);
      }
    }
  }
  float cc[kCpt];
#pragma unroll
  for (int j = 0; j < kCpt; ++j)
    cc[j] = leave(trail[j], leave(s.part[threadIdx.x >> 5][lc + j], s.carry[lc + j]));
#pragma unroll
  for (int i = R - 1; i >= 0; --i) {
    const int64_t r = r0 + i;
    const int n = r < a.rows ? nc : 0;
    const int seq = first_s[slot * R + i], end = last_s[slot * R + i];
    if (end >= 0) {
#pragma unroll
      for (int j = 0; j < kCpt; ++j) cc[j] = finish(end, j);
    }
    float dh[kCpt], o[kCpt];
#pragma unroll
    for (int j = 0; j < kCpt; ++j) {
      dh[j] = raw_get(dy[i], j) + cc[j];
      cc[j] = d[i][j] * dh[j];
      o[j] = before[i][j] * dh[j];
    }
    store_group<G, kCpt, VEC>((G*)a.dg + r * a.D + c, o, n);
    if constexpr (GATE) {
#pragma unroll
      for (int j = 0; j < kCpt; ++j) o[j] = raw_get(v[i], j) * dh[j];
      store_group<T, kCpt, VEC>((T*)a.dw + r * a.D + c, o, n);
#pragma unroll
      for (int j = 0; j < kCpt; ++j) dh[j] *= raw_get(w[i], j);
    }
    store_group<T, kCpt, VEC>((T*)a.dv + r * a.D + c, dh, n);
    if (seq >= 0 && a.dh0) {
#pragma unroll
      for (int j = 0; j < kCpt; ++j)
        if (j < nc) a.dh0[(int64_t)seq * a.D + c + j] = cc[j];
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
      (rows / kSaveRows + 1) > 2147483647LL / nslab)
    return fail(GDN2_ERR_UNSUPPORTED, "%s: too many rows x channels", fn);
  return GDN2_OK;
}

ScanArgs scan_args(const gdn2_scan_problem* p, int tile) {
  ScanArgs a{};
  a.rows = (int64_t)p->B * p->T;
  a.T = p->T;
  a.D = p->D;
  a.n_seqs = p->n_seqs;
  a.nslab = (p->D + kSlab - 1) / kSlab;
  a.cu = p->cu_seqlens;
  a.ntiles = (a.rows + tile - 1) / tile;
  if (a.ntiles == 0) a.ntiles = 1;  // sequences without rows still have end states
  a.chained = a.ntiles > 1;
  a.ldv = p->ld_v;
  a.ldg = p->ld_g;
  a.ldw = p->ld_w;
  a.lddy = p->ld_dy;
  return a;
}

int scan_chain(ScanArgs& a, int tile, void* ws, size_t bytes, cudaStream_t st, const char* fn) {
  if (!a.chained) return GDN2_OK;
  const ScanWorkspace L = scan_workspace(a.rows, a.D, tile);
  if (!ws || bytes < L.total)
    return fail(GDN2_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", fn, ws ? bytes : (size_t)0,
                L.total);
  if (!aligned_to(ws, 16))
    return fail(GDN2_ERR_INVALID, "%s: workspace must start on a 16-byte boundary", fn);
  char* b = static_cast<char*>(ws);
  a.ticket = reinterpret_cast<unsigned*>(b);
  a.runs = reinterpret_cast<uint64_t*>(b + L.runs);
  a.states = reinterpret_cast<uint64_t*>(b + L.states);
  cudaError_t e = fault_word(&a.fault);
  if (e == cudaSuccess) e = cudaMemsetAsync(ws, 0xff, L.total, st);
  return cuda_status(e, fn);
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
  const int64_t rows = (int64_t)p->B * p->T;
  return (size_t)((rows + kSaveRows - 1) / kSaveRows) * p->D * sizeof(float);
}

size_t gdn2_scan_workspace_bytes(const gdn2_scan_problem* p) {
  if (check_scan(p, "gdn2_scan_workspace_bytes") != GDN2_OK) return 0;
  return scan_workspace((int64_t)p->B * p->T, p->D, kSlots * kBwdRows).total;
}

int gdn2_scan_fwd(const gdn2_scan_problem* p, const void* v, const void* g, const void* w,
                  const float* h0, void* y, float* ht, float* saved, void* workspace,
                  size_t workspace_bytes, void* stream) {
  const char* fn = "gdn2_scan_fwd";
  int rc = check_scan(p, fn);
  if (rc) return rc;
  ScanArgs a = scan_args(p, kSlots * kFwdRows);
  if (a.rows > 0 && (!v || !g || !y)) return fail(GDN2_ERR_INVALID, "%s: null pointer", fn);
  if (w && p->ld_w < p->D) return fail(GDN2_ERR_INVALID, "%s: ld_w must be at least D", fn);
  if (a.n_seqs == 0 || (a.rows == 0 && !ht)) return GDN2_OK;
  const cudaStream_t st = (cudaStream_t)stream;
  if ((rc = scan_chain(a, kSlots * kFwdRows, workspace, workspace_bytes, st, fn))) return rc;
  a.v = v; a.g = g; a.w = w; a.h0 = h0; a.y = y; a.ht = ht; a.saved = saved;
  const size_t es = dtype_size(p->dtype);
  const bool vec = a.D % kCpt == 0 && group_ok(v, a.ldv, es) && group_ok(y, a.D, es) &&
                   group_ok(g, a.ldg, dtype_size(p->g_dtype)) && (!w || group_ok(w, a.ldw, es));
  const unsigned grid = (unsigned)(a.ntiles * a.nslab);
  return cuda_status(scan_dispatch(p, w != nullptr, [&](auto t, auto gt, auto gate) {
    using T = decltype(t);
    using G = decltype(gt);
    constexpr bool W = decltype(gate)::value;
    if (vec) k_scan_fwd<T, G, W, true><<<grid, kScanThreads, 0, st>>>(a);
    else k_scan_fwd<T, G, W, false><<<grid, kScanThreads, 0, st>>>(a);
    return cudaGetLastError();
  }), fn);
}

int gdn2_scan_bwd(const gdn2_scan_problem* p, const void* v, const void* g, const void* w,
                  const float* h0, const float* saved, const void* dy, const float* dht,
                  void* dv, void* dg, void* dw, float* dh0, void* workspace,
                  size_t workspace_bytes, void* stream) {
  const char* fn = "gdn2_scan_bwd";
  int rc = check_scan(p, fn);
  if (rc) return rc;
  ScanArgs a = scan_args(p, kSlots * kBwdRows);
  if (a.rows > 0 && (!v || !g || !saved || !dy || !dv || !dg || (w && !dw)))
    return fail(GDN2_ERR_INVALID, "%s: null pointer", fn);
  if (p->ld_dy < p->D || (w && p->ld_w < p->D))
    return fail(GDN2_ERR_INVALID, "%s: row strides must be at least D", fn);
  if (a.n_seqs == 0 || (a.rows == 0 && !dh0)) return GDN2_OK;
  const cudaStream_t st = (cudaStream_t)stream;
  if ((rc = scan_chain(a, kSlots * kBwdRows, workspace, workspace_bytes, st, fn))) return rc;
  a.v = v; a.g = g; a.w = w; a.h0 = h0; a.saved = const_cast<float*>(saved);
  a.dy = dy; a.dht = dht; a.dv = dv; a.dg = dg; a.dw = dw; a.dh0 = dh0;
  const size_t es = dtype_size(p->dtype), eg = dtype_size(p->g_dtype);
  const bool vec = a.D % kCpt == 0 && group_ok(v, a.ldv, es) && group_ok(dy, a.lddy, es) &&
                   group_ok(g, a.ldg, eg) && group_ok(dv, a.D, es) && group_ok(dg, a.D, eg) &&
                   (!w || (group_ok(w, a.ldw, es) && group_ok(dw, a.D, es)));
  const unsigned grid = (unsigned)(a.ntiles * a.nslab);
  return cuda_status(scan_dispatch(p, w != nullptr, [&](auto t, auto gt, auto gate) {
    using T = decltype(t);
    using G = decltype(gt);
    constexpr bool W = decltype(gate)::value;
    if (vec) k_scan_bwd<T, G, W, true><<<grid, kScanThreads, 0, st>>>(a);
    else k_scan_bwd<T, G, W, false><<<grid, kScanThreads, 0, st>>>(a);
    return cudaGetLastError();
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
