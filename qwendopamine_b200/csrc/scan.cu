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
// written once.  A cluster of CTAs walks a chain: W channels of a stretch of
// rows that starts with a sequence, one tile of rows per CTA and turn.  A
// thread holds its rows of the tile in registers across the exchange of runs
// (shared memory in a CTA, distributed shared memory in a cluster) and walks
// them a second time from the state that enters them.  The next turn's rows come in by
// cp.async meanwhile.  The state passes from turn to turn inside the cluster:
// no CTA waits for another cluster, and the order of all products is fixed.
// Two to four CTAs share an SM and cover one another's barriers, while a thread
// still has enough rows to spread the cost of the exchange over.  A tile
// without a sequence's edge takes a path without the checks for one.
//
// Chains: whole sequences are dealt to stretches while there are enough of
// them to fill the GPU; clusters of 2 to 16 CTAs and half-width slabs make up
// for too few.
#include <cooperative_groups.h>

#include "op_util.cuh"
#include "tc.cuh"

namespace cg = cooperative_groups;

namespace gdn2 {
namespace {

constexpr int kCpt = 4;           // channels of a thread
constexpr int kKeep = 64;         // rows between the states kept for the backward
constexpr int kMaxStride = 1 << 22;  // a tile's offsets are held in 32 bits
constexpr int kMaxCluster = 16;
constexpr unsigned kScanFault = 16u;  // of the device's fault word

// A tile of W channels: `lanes` threads across and `slots` threads down, R rows
// and kCpt channels each.
template <int W, int R> struct Shape {
  static constexpr int threads = 1024 / R;
  static constexpr int lanes = W / kCpt, slots = threads / lanes, tile = slots * R;
  static_assert(tile % kKeep == 0, "a kept state enters every tile");
};

// Rows of a thread, and CTAs that share an SM (what their registers allow).
// Forward: four CTAs of 128 threads with eight rows each (B = 8, T = 4096,
// D = 2048, bf16 with a gate: 123 us between events, 84 % of the measured copy
// bandwidth; two of 256 with four rows 119 us, but 254 against 213 us on one
// sequence of 131,072 x 1024 and 98 against 78 us on 512 of 64 x 1024).
// Backward, with twice the tensors in registers: two CTAs of 256 threads with
// four rows (211 us, 89 %; three of 128 with eight rows 242 us).
template <bool BWD> constexpr int rows_of() { return BWD ? 4 : 8; }
template <typename T, bool BWD> constexpr int ctas_of() {
  return BWD ? 2 : (sizeof(T) == 2 ? 4 : 3);
}

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
  unsigned* fault;
  uint64_t wait_ns;  // limit of a wait for the cluster's runs
  int expect;        // bytes of them that come in a turn
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

// Runs of a tile's rows on their way, in groups of `own` slots: with own = 1 the
// slots themselves, else a warp's, which it folds itself before and after the
// tile's barriers, so that fewer are left between them.  That pays forward
// (131,072 x 128: 137 -> 133 us, 60,000 x 1001: 305 -> 293 us), not with the
// backward's two folds (B = 8, T = 4096, D = 2048: 211 -> 219 us).  Read and written four channels at a time.
template <int W, int R> struct alignas(16) Runs {
  using S = Shape<W, R>;
  static constexpr int own = R == rows_of<false>() ? 32 / S::lanes : 1, groups = S::slots / own;
  float A[groups][W], H[groups][W];
  float enter[groups][W];  // the states entering the groups
  // a warp's slots (own > 1); in sH later the states entering them
  float sA[own > 1 ? S::slots : 1][W], sH[own > 1 ? S::slots : 1][W];
};

// Whole lines, so that the stages behind it start on one (16 bytes more of it alone
// cost B = 8, T = 4096, D = 2048 forward 123 -> 127 us).
template <int W, int R> struct alignas(128) ScanShared {
  static constexpr int tile = Shape<W, R>::tile;
  Runs<W, R> runs;
  uint64_t bar[2];  // the cluster's runs have come, by turn's parity
  int lost;         // a wait for them has run out
  // of a turn with sequence edges in its tile
  int seq[tile];                               // the row's sequence
  uint32_t first[tile / 32], last[tile / 32];  // whether it is its first / last row
};

__device__ __forceinline__ float4 quad(const float2 (&x)[2]) {
  return make_float4(x[0].x, x[0].y, x[1].x, x[1].y);
}
__device__ __forceinline__ void unquad(float2 (&x)[2], const float4 f) {
  x[0] = make_float2(f.x, f.y);
  x[1] = make_float2(f.z, f.w);
}

// The fold of a tile's runs, in the order of the scan.
template <int W, int R, bool UP> struct Fold {
  using S = Runs<W, R>;
  // a thread's run, and its group's
  __device__ static __forceinline__ void put(S& s, int slot, int lc, const float4& A, const float4& H) {
    float (&a)[W] = S::own > 1 ? s.sA[slot] : s.A[slot];
    float (&h)[W] = S::own > 1 ? s.sH[slot] : s.H[slot];
    *reinterpret_cast<float4*>(a + lc) = A;
    *reinterpret_cast<float4*>(h + lc) = H;
    if constexpr (S::own > 1) {
      __syncwarp();
      const int w = threadIdx.x >> 5;
#pragma unroll
      for (int ch = threadIdx.x & 31; ch < W; ch += 32) {
        float2 all = make_float2(1.f, 0.f);
#pragma unroll
        for (int i = 0; i < S::own; ++i) {
          const int k = w * S::own + (UP ? S::own - 1 - i : i);
          all = compose(all, make_float2(s.sA[k][ch], s.sH[k][ch]));
        }
        s.A[w][ch] = all.x;
        s.H[w][ch] = all.y;
      }
    }
  }
  // one channel of the groups' runs: the tile's
  __device__ static __forceinline__ float2 run(const S& s, int ch) {
    float2 all = make_float2(1.f, 0.f);
#pragma unroll
    for (int i = 0; i < S::groups; ++i) {
      const int k = UP ? S::groups - 1 - i : i;
      all = compose(all, make_float2(s.A[k][ch], s.H[k][ch]));
    }
    return all;
  }
  // one channel of the states entering the groups; returns the one that leaves
  __device__ static __forceinline__ float enter(S& s, int ch, float state) {
#pragma unroll
    for (int i = 0; i < S::groups; ++i) {
      const int k = UP ? S::groups - 1 - i : i;
      s.enter[k][ch] = state;
      state = leave(make_float2(s.A[k][ch], s.H[k][ch]), state);
    }
    return state;
  }
  // the state entering a thread's rows
  __device__ static __forceinline__ float4 get(S& s, int slot, int lc) {
    if constexpr (S::own == 1) {
      return *reinterpret_cast<const float4*>(&s.enter[slot][lc]);
    } else {
      const int w = threadIdx.x >> 5;
#pragma unroll
      for (int ch = threadIdx.x & 31; ch < W; ch += 32) {
        float state = s.enter[w][ch];
#pragma unroll
        for (int i = 0; i < S::own; ++i) {
          const int k = w * S::own + (UP ? S::own - 1 - i : i);
          const float2 r = make_float2(s.sA[k][ch], s.sH[k][ch]);
          s.sH[k][ch] = state;
          state = leave(r, state);
        }
      }
      __syncwarp();
      return *reinterpret_cast<const float4*>(&s.sH[slot][lc]);
    }
  }
};

// A 64-bit store into another CTA's shared memory that counts on a barrier there.
__device__ __forceinline__ void store_async(uint32_t to, uint32_t bar, float2 x) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(to),
               "l"(*reinterpret_cast<const uint64_t*>(&x)), "r"(bar)
               : "memory");
}
__device__ __forceinline__ uint32_t address_at(uint32_t a, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}

// Before the first turn: the cluster's barriers, known to all its CTAs.
template <int W, int R>
__device__ __forceinline__ void open_exchange(const ScanArgs& a, ScanShared<W, R>& s) {
  if (a.cluster == 1) return;
  if (threadIdx.x == 0) {
    tc::mbar_init(&s.bar[0], 1);
    tc::mbar_init(&s.bar[1], 1);
    tc::fence_mbar_init();
    s.lost = 0;
  }
  cg::this_cluster().sync();
}

// After the last turn.  A CTA that has received all runs of its last turn could
// leave, since nothing more is sent to it; after a wait that ran out that is not
// known, so all stay until all have sent what they send.
__device__ __forceinline__ void close_exchange(const ScanArgs& a) {
  if (a.cluster > 1) cg::this_cluster().sync();
}

// Finds the states that enter the groups of this CTA's tile and moves `state`
// (threads 0 .. W-1, one per channel) from the state that enters the turn's
// first tile to the one that leaves its last.  Called by all threads after a
// barrier; ends with one.
//
// In a cluster every CTA sends its tile's run to all, into `runs` by turn's
// parity, and waits for as many; a cluster-wide barrier would also wait for
// the last turn's stores to reach memory.  A thread sends the run of turn i+1
// after it has read those of turn i, and receives all of turn i+1 before it
// sends turn i+2: the same places are free by then.
//
// A wait that runs out sets a fault bit and `lost`.  The CTA then gives up: what
// lies in `runs` is of no turn, and its barrier, whose phase is still open, cannot
// be used again.  It sends nothing more, so the others' waits run out as well.
template <int W, int R, bool UP>
__device__ __forceinline__ void exchange(const ScanArgs& a, ScanShared<W, R>& s, float2* runs, int rank,
                                         int turn, float& state) {
  const int ch = threadIdx.x, b = turn & 1;
  if (ch < W) {
    if (a.cluster == 1) {
      state = Fold<W, R, UP>::enter(s.runs, ch, state);
    } else {
      runs += b * a.cluster * W;
      const float2 all = Fold<W, R, UP>::run(s.runs, ch);
      if (ch == 0) tc::mbar_expect_tx(&s.bar[b], a.expect);
      const uint32_t to = smem_u32(runs + rank * W + ch), bar = smem_u32(&s.bar[b]);
      for (int k = 0; k < a.cluster; ++k) store_async(address_at(to, k), address_at(bar, k), all);
      if (!tc::mbar_wait(&s.bar[b], (turn >> 1) & 1, a.wait_ns)) {
        atomicOr(a.fault, kScanFault);
        s.lost = 1;
      }
      float carry = state;
#pragma unroll 4
      for (int k = 0; k < a.cluster; ++k) {
        if (k == rank) carry = state;
        state = leave(runs[k * W + ch], state);
      }
      Fold<W, R, UP>::enter(s.runs, ch, carry);
    }
  }
  __syncthreads();
}

// The sequence that owns row r, and r's place in it.
struct RowPlace {
  int64_t at, len;
  int n;
  __device__ __forceinline__ void find(const ScanArgs& a, int64_t r) {
    if (!a.cu) {
      n = (int)(r / a.T);
      at = r - (int64_t)n * a.T;
      len = a.T;
      return;
    }
    int lo = 0, hi = a.n_seqs;  // the last n with cu[n] <= r
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(a.cu + mid) <= r) lo = mid; else hi = mid;
    }
    n = lo;
    at = r - __ldg(a.cu + lo);
    len = (int64_t)__ldg(a.cu + lo + 1) - __ldg(a.cu + lo);
  }
  // Moves to row r, `by` rows on (the same for the CTA); true if the tile of
  // rows from there holds a sequence's first or last row or leaves [lo, hi).
  __device__ __forceinline__ bool edges(const ScanArgs& a, int64_t r, int64_t by, int tile,
                                        int64_t lo, int64_t hi) {
    if (r < lo || r + tile > hi) {
      len = 0;  // to be found again
      return true;
    }
    at += by;
    if (at < 0 || at >= len) find(a, r);
    return at <= 0 || at + tile >= len;
  }
};

// Marks the rows of the tile that starts at row `tile`; rows outside [lo, hi)
// have no marks.
template <int W, int R>
__device__ __forceinline__ void mark_rows(const ScanArgs& a, ScanShared<W, R>& s, int64_t tile,
                                          int64_t lo, int64_t hi) {
  if (threadIdx.x >= Shape<W, R>::tile) return;
  const int64_t r = tile + threadIdx.x;
  const bool in = r >= lo && r < hi;
  RowPlace p{-1, 0, 0};
  if (in) p.find(a, r);
  const uint32_t f = __ballot_sync(0xffffffffu, in && p.at == 0);
  const uint32_t l = __ballot_sync(0xffffffffu, in && p.at == p.len - 1);
  s.seq[threadIdx.x] = p.n;
  if ((threadIdx.x & 31) == 0) {
    s.first[threadIdx.x >> 5] = f;
    s.last[threadIdx.x >> 5] = l;
  }
}

// Sequences without rows: their state passes through (`from` NULL: zero).
template <int W, int THREADS>
__device__ __forceinline__ void pass_empty(const ScanArgs& a, int slab, const float* from,
                                           float* to) {
  if (!to || (!a.cu && a.T > 0)) return;
  const int c = slab * W + (int)threadIdx.x % W;
  if (c >= a.D) return;
  for (int n = threadIdx.x / W; n < a.n_seqs; n += THREADS / W)
    if (!a.cu || __ldg(a.cu + n) == __ldg(a.cu + n + 1))
      to[(int64_t)n * a.D + c] = from ? from[(int64_t)n * a.D + c] : 0.f;
}

// A thread's own rows of a tile in shared memory, filled asynchronously by
// the thread itself (no barrier) and read by it alone: group i of a tensor at
// its section, row i, thread.  AL elements (4, 2 or 1) of the tensor are
// aligned together.  Single 16-bit elements are too small to be copied
// asynchronously: such a group comes in as the three words that hold it and is
// shifted into place when it is read.
template <typename T, int R, int AL> struct Stage {
  static constexpr bool kWords = AL * sizeof(T) < 4;
  static constexpr int kGroupBytes = kWords ? 16 : kCpt * (int)sizeof(T);
  static constexpr int kBytes = 1024 * kGroupBytes;
  static constexpr int kPiece = kWords ? 4 : AL * (int)sizeof(T);  // bytes of a copy

  __device__ static __forceinline__ char* at(char* base, int i) {
    return base + (i * (1024 / R) + threadIdx.x) * kGroupBytes;
  }
  // a piece at byte `e` of a row's group; zeros where there is nothing
  __device__ static __forceinline__ void copy(char* base, int i, int e, const void* src, bool there) {
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(at(base, i)) + e;
    const int n = there ? kPiece : 0;
    if constexpr (kPiece == 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else
      asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(n), "n"(kPiece) : "memory");
  }
  // The thread's rows of the tile at row `tile` (the same for the CTA), of
  // which those in [lo, hi) exist, `nc` channels wide; what does not exist
  // reads as zero, but a thread without channels reads nothing.
  template <int W>
  __device__ static __forceinline__ void fill(char* base, const void* x, int64_t ld, int64_t tile,
                                              int64_t lo, int64_t hi, int64_t rows, int slab, int nc) {
    if (nc <= 0) return;
    const int r0 = (int)threadIdx.x / Shape<W, R>::lanes * R;
    const int lc = (int)threadIdx.x % Shape<W, R>::lanes * kCpt;
    const bool inside = tile >= lo && tile + Shape<W, R>::tile <= hi;
    const char* p = (const char*)x + (tile * ld + slab * W) * (int64_t)sizeof(T);
    if constexpr (kWords) {
      // the three words may reach into the neighbouring rows, but not out of the
      // tensor: its first and last elements come one by one
      const T* q = (const T*)p + r0 * ld + lc;
#pragma unroll
      for (int i = 0; i < R; ++i, q += ld) {
        const int64_t r = tile + r0 + i;
        const uintptr_t a = reinterpret_cast<uintptr_t>(q) & ~(uintptr_t)3;
        const bool row = inside || (r >= lo && r < hi);
        const int odd = (int)(reinterpret_cast<uintptr_t>(q) >> 1) & 1;
        if (row && r * ld + slab * W + lc > 0 && (rows - 1 - r) * ld + nc >= 6) {
#pragma unroll
          for (int e = 0; e < 12; e += 4) copy(base, i, e, (const void*)(a + e), e < 8 || odd);
        } else {
#pragma unroll
          for (int e = 0; e < kCpt; ++e)
            *reinterpret_cast<T*>(at(base, i) + (e + odd) * 2) = row && e < nc ? q[e] : from_f<T>(0.f);
        }
      }
    } else if (inside && nc >= kCpt) {
      const uint32_t off = (uint32_t)(r0 * (int)ld + lc) * (uint32_t)sizeof(T);
#pragma unroll
      for (int i = 0; i < R; ++i, p += ld * (int64_t)sizeof(T))
#pragma unroll
        for (int e = 0; e < kGroupBytes; e += kPiece) copy(base, i, e, p + off + e, true);
    } else {
      const T* q = (const T*)p + r0 * ld + lc;
#pragma unroll 1
      for (int i = 0; i < R; ++i, q += ld) {
        const int64_t r = tile + r0 + i;
        const int n = r >= lo && r < hi ? nc : 0;
#pragma unroll
        for (int e = 0; e < kCpt; e += AL)
          copy(base, i, e * (int)sizeof(T), n > e ? (const void*)(q + e) : x, n > e);
      }
    }
  }
  // `odd`: whether the row starts in the middle of a word
  __device__ static __forceinline__ Raw<T, kCpt> get(char* base, int i, bool odd) {
    Raw<T, kCpt> r;
    if constexpr (kWords) {
      const uint4 v = *reinterpret_cast<const uint4*>(at(base, i));
      r.u[0] = odd ? __funnelshift_r(v.x, v.y, 16) : v.x;
      r.u[1] = odd ? __funnelshift_r(v.y, v.z, 16) : v.y;
    } else if constexpr (kGroupBytes == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(at(base, i));
      r.u[0] = v.x; r.u[1] = v.y; r.u[2] = v.z; r.u[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(at(base, i));
      r.u[0] = v.x; r.u[1] = v.y;
    }
    return r;
  }
  // whether row r starts in the middle of a word (16-bit elements)
  __device__ static __forceinline__ bool odd_row(const void* x, int64_t ld, int64_t r) {
    if constexpr (!kWords) return false;
    return ((reinterpret_cast<uintptr_t>(x) >> 1) + (uintptr_t)(r * ld)) & 1;
  }
};

__device__ __forceinline__ void stage_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Sections of a stage: g, v, w, dy.
template <typename T, typename G, bool GATE, bool BWD, int AL> struct StageLayout {
  static constexpr int sg = Stage<G, 8, AL>::kBytes, st = Stage<T, 8, AL>::kBytes;
  static constexpr int g = 0, v = sg, w = v + st;
  static constexpr int dy = w + (GATE ? st : 0);
  static constexpr int bytes = dy + (BWD ? st : 0);
};

// A CTA's chain and place in it.
struct Place {
  int64_t lo, hi;   // rows of the chain
  int64_t chain;    // which stretch
  int rank, slab, turns;
};
template <int W, int R> __device__ __forceinline__ Place place_of(const ScanArgs& a) {
  Place p;
  const unsigned id = blockIdx.x / (unsigned)a.cluster;
  p.rank = (int)(blockIdx.x - id * a.cluster);
  p.chain = id / (unsigned)a.nslab;
  p.slab = (int)(id - p.chain * a.nslab);
  p.lo = p.chain * a.stretch;
  p.hi = min(p.lo + a.stretch, a.rows);
  const int64_t step = (int64_t)a.cluster * Shape<W, R>::tile;
  p.turns = (int)((p.hi - p.lo + step - 1) / step);
  return p;
}

// each(r, c) for the rows of the CTA's tiles from the one at row `tile` on, and
// their channels (after it has given up).
template <int W, int R, typename F>
__device__ __forceinline__ void for_rest(const ScanArgs& a, const Place& p, int64_t tile, int64_t step,
                                         int turns, F&& each) {
  const int c = p.slab * W + (int)threadIdx.x % W;
  if (c >= a.D) return;
  for (; turns > 0; --turns, tile += step) {
    const int64_t end = min(tile + Shape<W, R>::tile, p.hi);
    for (int64_t r = tile + threadIdx.x / W; r < end; r += Shape<W, R>::threads / W)
      if (r >= p.lo) each(r, c);
  }
}

// Groups of four channels as two packed pairs.
template <typename T> __device__ __forceinline__ float2 pair_of(const Raw<T, kCpt>& r, int k) {
  if constexpr (sizeof(T) == 4)
    return make_float2(__uint_as_float(r.u[2 * k]), __uint_as_float(r.u[2 * k + 1]));
  else
    return unpack2<T>(r.u[k]);
}

// Where a thread's rows of a contiguous output go: the tile's first element
// (the same for the CTA) and the thread's place from there.
template <typename T, int W, int R> struct Target {
  char* base;
  uint32_t off;
  int row_bytes;
  __device__ __forceinline__ Target(void* x, int64_t tile, int slab, int D) {
    base = (char*)x + (tile * D + slab * W) * (int64_t)sizeof(T);
    const int r0 = (int)threadIdx.x / Shape<W, R>::lanes * R;
    const int lc = (int)threadIdx.x % Shape<W, R>::lanes * kCpt;
    off = (uint32_t)(r0 * D + lc) * (uint32_t)sizeof(T);
    row_bytes = D * (int)sizeof(T);
  }
  template <int AL> __device__ __forceinline__ void put(int i, const float2 (&x)[2], int n) const {
    T* const p = (T*)(base + (int64_t)i * row_bytes + off);
    if constexpr (AL == 2) {
      const float f[2][2] = {{x[0].x, x[0].y}, {x[1].x, x[1].y}};
      if (n > 0) store_raw<T, 2>(p, raw_from<T, 2>(f[0]));
      if (n > 2) store_raw<T, 2>(p + 2, raw_from<T, 2>(f[1]));
    } else {
      const float f[kCpt] = {x[0].x, x[0].y, x[1].x, x[1].y};
      store_group<T, kCpt, AL == 4>(p, f, n);
    }
  }
};
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

template <typename T, typename G, bool GATE, int W, int R, int AL>
__global__ void __launch_bounds__(1024 / R, ctas_of<T, false>()) k_scan_fwd(const ScanArgs a) {
  constexpr int TILE = Shape<W, R>::tile;
  using L = StageLayout<T, G, GATE, false, AL>;
  extern __shared__ __align__(16) char st[];
  __shared__ ScanShared<W, R> s;
  const Place p = place_of<W, R>(a);
  float2* const runs = reinterpret_cast<float2*>(st + L::bytes);
  const int slot = threadIdx.x / Shape<W, R>::lanes, r0 = slot * R;
  const int lc = (threadIdx.x % Shape<W, R>::lanes) * kCpt, c = p.slab * W + lc, nc = a.D - c;
  const int64_t step = (int64_t)a.cluster * TILE;
  int64_t tile = p.lo + (int64_t)p.rank * TILE;  // first row of this turn's tile
  auto fill = [&](int64_t row) {
    Stage<G, R, AL>::template fill<W>(st + L::g, a.g, a.ldg, row, p.lo, p.hi, a.rows, p.slab, nc);
    Stage<T, R, AL>::template fill<W>(st + L::v, a.v, a.ldv, row, p.lo, p.hi, a.rows, p.slab, nc);
    if constexpr (GATE)
      Stage<T, R, AL>::template fill<W>(st + L::w, a.w, a.ldw, row, p.lo, p.hi, a.rows, p.slab, nc);
  };
  if (p.chain == 0 && p.rank == 0) pass_empty<W, Shape<W, R>::threads>(a, p.slab, a.h0, a.ht);
  if (p.turns > 0) fill(tile);
  open_exchange(a, s);
  float state = 0.f;
  RowPlace place{0, 0, 0};

  int turn = 0;
  for (; turn < p.turns; ++turn, tile += step) {
    const bool edges = place.edges(a, tile, step, TILE, p.lo, p.hi);
    if (edges) mark_rows(a, s, tile, p.lo, p.hi);
    stage_wait();
    auto odd = [&](const void* x, int64_t ld, int i) {
      return Stage<T, R, AL>::odd_row(x, ld, tile + r0 + i);
    };
    float2 d[R][2];
    // the inputs w v, packed as v where there is no gate
    using X = typename std::conditional<GATE, float, T>::type;
    Raw<X, kCpt> x[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const Raw<G, kCpt> g = Stage<G, R, AL>::get(st + L::g, i, odd(a.g, a.ldg, i));
      const Raw<T, kCpt> v = Stage<T, R, AL>::get(st + L::v, i, odd(a.v, a.ldv, i));
      if constexpr (GATE) {
        const Raw<T, kCpt> w = Stage<T, R, AL>::get(st + L::w, i, odd(a.w, a.ldw, i));
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
    if (turn + 1 < p.turns) fill(tile + step);
    uint32_t first = 0, last = 0;
    if (edges) {
      __syncthreads();
      first = (s.first[r0 / 32] >> (r0 % 32)) & ((1u << R) - 1);
      last = (s.last[r0 / 32] >> (r0 % 32)) & ((1u << R) - 1);
    }

    float2 A[2] = {both(1.f), both(1.f)}, h[2] = {both(0.f), both(0.f)};
    auto walk = [&](auto edge, auto&& each) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if constexpr (decltype(edge)::value)
          if (first >> i & 1) state_at(a.h0, s.seq[r0 + i], a.D, c, nc, h);
#pragma unroll
        for (int k = 0; k < 2; ++k) h[k] = fma2(d[i][k], h[k], pair_of<X>(x[i], k));
        each(i);
      }
    };
    auto product = [&](int i) {
#pragma unroll
      for (int k = 0; k < 2; ++k) A[k] = mul2(A[k], d[i][k]);
    };
    if (edges) {
      walk(std::true_type{}, product);
      if (first) A[0] = A[1] = both(-1.f);
    } else {
      walk(std::false_type{}, product);
    }
    Fold<W, R, false>::put(s.runs, slot, lc, quad(A), quad(h));
    __syncthreads();
    exchange<W, R, false>(a, s, runs, p.rank, turn, state);
    if (a.cluster > 1 && s.lost) break;

    unquad(h, Fold<W, R, false>::get(s.runs, slot, lc));
    const int64_t left = p.hi - tile - r0;  // rows that exist from here
    if (a.saved && r0 % kKeep == 0 && left > 0)
      put_state(a.saved, p.chain * a.keeps + (tile + r0 - p.lo) / kKeep, a.D, c, nc, h);
    const Target<T, W, R> y(a.y, tile, p.slab, a.D);
    if (edges) {
      walk(std::true_type{}, [&](int i) {
        y.template put<AL>(i, h, i < left ? nc : 0);
        if ((last >> i & 1) && a.ht) put_state(a.ht, s.seq[r0 + i], a.D, c, nc, h);
      });
      __syncthreads();  // the marks have been read
    } else {
      walk(std::false_type{}, [&](int i) { y.template put<AL>(i, h, nc); });
    }
  }
  if (turn < p.turns) {
    const float nan = __int_as_float(0x7fffffff);
    stage_wait();  // the next turn's rows
    for_rest<W, R>(a, p, tile, step, p.turns - turn, [&](int64_t r, int c) {
      ((T*)a.y)[r * a.D + c] = from_f<T>(nan);
      if (a.saved && (r - p.lo) % kKeep == 0)
        a.saved[(p.chain * a.keeps + (r - p.lo) / kKeep) * a.D + c] = nan;
      place.find(a, r);
      if (a.ht && place.at == place.len - 1) a.ht[(int64_t)place.n * a.D + c] = nan;
    });
  }
  close_exchange(a);
}

template <typename T, typename G, bool GATE, int W, int R, int AL>
__global__ void __launch_bounds__(1024 / R, ctas_of<T, true>()) k_scan_bwd(const ScanArgs a) {
  constexpr int TILE = Shape<W, R>::tile;
  using L = StageLayout<T, G, GATE, true, AL>;
  extern __shared__ __align__(16) char st[];
  __shared__ ScanShared<W, R> s;
  __shared__ Runs<W, R> ahead;  // of the recomputed states
  const Place p = place_of<W, R>(a);
  float2* const runs = reinterpret_cast<float2*>(st + L::bytes);
  const int slot = threadIdx.x / Shape<W, R>::lanes, r0 = slot * R;
  const int lc = (threadIdx.x % Shape<W, R>::lanes) * kCpt, c = p.slab * W + lc, nc = a.D - c;
  const int64_t step = (int64_t)a.cluster * TILE;
  // from the chain's last tile down; before the first there is nothing
  int64_t tile = p.lo + ((p.hi - p.lo + TILE - 1) / TILE - 1 - p.rank) * TILE;
  auto fill = [&](int64_t row) {
    Stage<G, R, AL>::template fill<W>(st + L::g, a.g, a.ldg, row, p.lo, p.hi, a.rows, p.slab, nc);
    Stage<T, R, AL>::template fill<W>(st + L::v, a.v, a.ldv, row, p.lo, p.hi, a.rows, p.slab, nc);
    Stage<T, R, AL>::template fill<W>(st + L::dy, a.dy, a.lddy, row, p.lo, p.hi, a.rows, p.slab, nc);
    if constexpr (GATE)
      Stage<T, R, AL>::template fill<W>(st + L::w, a.w, a.ldw, row, p.lo, p.hi, a.rows, p.slab, nc);
  };
  if (p.chain == 0 && p.rank == 0) pass_empty<W, Shape<W, R>::threads>(a, p.slab, a.dht, a.dh0);
  if (p.turns > 0) fill(tile);
  open_exchange(a, s);
  float state = 0.f;
  RowPlace place{0, 0, 0};

  int turn = 0;
  for (; turn < p.turns; ++turn, tile -= step) {
    const bool some = tile >= p.lo;
    const bool edges = place.edges(a, tile, -step, TILE, p.lo, p.hi);
    float kept = 0.f;  // the state entering the tile
    if (threadIdx.x / W == 1) {
      const int ch = p.slab * W + threadIdx.x - W;
      if (some && ch < a.D)
        kept = __ldg(a.saved + (p.chain * a.keeps + (tile - p.lo) / kKeep) * a.D + ch);
    }
    if (edges) mark_rows(a, s, tile, p.lo, p.hi);
    stage_wait();
    auto odd = [&](const void* x, int64_t ld, int i) {
      return Stage<T, R, AL>::odd_row(x, ld, tile + r0 + i);
    };
    float2 d[R][2];
    Raw<T, kCpt> v[R], w[GATE ? R : 1], dy[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const Raw<G, kCpt> g = Stage<G, R, AL>::get(st + L::g, i, odd(a.g, a.ldg, i));
      v[i] = Stage<T, R, AL>::get(st + L::v, i, odd(a.v, a.ldv, i));
      dy[i] = Stage<T, R, AL>::get(st + L::dy, i, odd(a.dy, a.lddy, i));
      if constexpr (GATE) w[i] = Stage<T, R, AL>::get(st + L::w, i, odd(a.w, a.ldw, i));
      d[i][0] = decay_of(pair_of<G>(g, 0));
      d[i][1] = decay_of(pair_of<G>(g, 1));
    }
    auto input = [&](int i, int k) {
      const float2 x = pair_of<T>(v[i], k);
      if constexpr (GATE) return mul2(x, pair_of<T>(w[i], k));
      return x;
    };
    if (turn + 1 < p.turns) fill(tile - step);
    uint32_t first = 0, last = 0;
    if (edges) {
      __syncthreads();
      first = (s.first[r0 / 32] >> (r0 % 32)) & ((1u << R) - 1);
      last = (s.last[r0 / 32] >> (r0 % 32)) & ((1u << R) - 1);
    }

    auto runs_of_rows = [&](auto edge) {
      constexpr bool EDGE = decltype(edge)::value;
      float2 A[2] = {both(1.f), both(1.f)}, H[2] = {both(0.f), both(0.f)};
      float2 C[2] = {both(0.f), both(0.f)};
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (EDGE && (first >> i & 1)) state_at(a.h0, s.seq[r0 + i], a.D, c, nc, H);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          H[k] = fma2(d[i][k], H[k], input(i, k));
          A[k] = mul2(A[k], d[i][k]);
        }
      }
#pragma unroll
      for (int i = R - 1; i >= 0; --i) {
        if (EDGE && (last >> i & 1)) state_at(a.dht, s.seq[r0 + i], a.D, c, nc, C);
#pragma unroll
        for (int k = 0; k < 2; ++k) C[k] = mul2(d[i][k], add2(pair_of<T>(dy[i], k), C[k]));
      }
      const float4 reset = make_float4(-1.f, -1.f, -1.f, -1.f);
      Fold<W, R, false>::put(ahead, slot, lc, EDGE && first ? reset : quad(A), quad(H));
      Fold<W, R, true>::put(s.runs, slot, lc, EDGE && last ? reset : quad(A), quad(C));
    };
    if (edges) runs_of_rows(std::true_type{});
    else runs_of_rows(std::false_type{});
    __syncthreads();
    if (threadIdx.x / W == 1)
      Fold<W, R, false>::enter(ahead, threadIdx.x - W, kept);
    exchange<W, R, true>(a, s, runs, p.rank, turn, state);
    if (a.cluster > 1 && s.lost) break;

    const int64_t left = some ? p.hi - tile - r0 : 0;  // rows that exist from here
    const Target<G, W, R> dg(a.dg, tile, p.slab, a.D);
    const Target<T, W, R> dv(a.dv, tile, p.slab, a.D), dw(a.dw, tile, p.slab, a.D);
    auto gradients = [&](auto edge) {
      constexpr bool EDGE = decltype(edge)::value;
      float2 before[R][2];  // a_t h_{t-1}
      float2 h[2], cc[2];
      unquad(h, Fold<W, R, false>::get(ahead, slot, lc));
      unquad(cc, Fold<W, R, true>::get(s.runs, slot, lc));
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (EDGE && (first >> i & 1)) state_at(a.h0, s.seq[r0 + i], a.D, c, nc, h);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          before[i][k] = mul2(d[i][k], h[k]);
          h[k] = add2(before[i][k], input(i, k));
        }
      }
#pragma unroll
      for (int i = R - 1; i >= 0; --i) {
        const int n = !EDGE || i < left ? nc : 0;
        if (EDGE && (last >> i & 1)) state_at(a.dht, s.seq[r0 + i], a.D, c, nc, cc);
        float2 dh[2], z[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          dh[k] = add2(pair_of<T>(dy[i], k), cc[k]);
          cc[k] = mul2(d[i][k], dh[k]);
          z[k] = mul2(before[i][k], dh[k]);
        }
        dg.template put<AL>(i, z, n);
        if constexpr (GATE) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            z[k] = mul2(pair_of<T>(v[i], k), dh[k]);
            dh[k] = mul2(dh[k], pair_of<T>(w[i], k));
          }
          dw.template put<AL>(i, z, n);
        }
        dv.template put<AL>(i, dh, n);
        if (EDGE && (first >> i & 1) && a.dh0) put_state(a.dh0, s.seq[r0 + i], a.D, c, nc, cc);
      }
    };
    if (edges) {
      gradients(std::true_type{});
      __syncthreads();  // the marks have been read
    } else {
      gradients(std::false_type{});
    }
  }
  if (turn < p.turns) {
    const float nan = __int_as_float(0x7fffffff);
    stage_wait();  // the next turn's rows
    for_rest<W, R>(a, p, tile, -step, p.turns - turn, [&](int64_t r, int c) {
      ((T*)a.dv)[r * a.D + c] = from_f<T>(nan);
      ((G*)a.dg)[r * a.D + c] = from_f<G>(nan);
      if constexpr (GATE) ((T*)a.dw)[r * a.D + c] = from_f<T>(nan);
      place.find(a, r);
      if (a.dh0 && place.at == 0) a.dh0[(int64_t)place.n * a.D + c] = nan;
    });
  }
  close_exchange(a);
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
  if (p->cu_seqlens && p->n_seqs == 0 && p->T > 0)
    return fail(GDN2_ERR_INVALID, "%s: cu_seqlens without a sequence cannot end at T = %lld", fn,
                (long long)p->T);
  if (p->ld_v < p->D || p->ld_g < p->D || p->ld_w < 0 || p->ld_dy < 0)
    return fail(GDN2_ERR_INVALID, "%s: row strides must be at least D", fn);
  if (p->ld_v > kMaxStride || p->ld_g > kMaxStride || p->ld_w > kMaxStride || p->ld_dy > kMaxStride)
    return fail(GDN2_ERR_UNSUPPORTED, "%s: D and row strides up to %d are supported", fn, kMaxStride);
  const int64_t rows = (int64_t)p->B * p->T;
  const int64_t nslab = (p->D + 31) / 32;
  if ((p->T > 0 && rows / p->T != p->B) ||
      (rows / kKeep + p->B + kMaxCluster) > 2147483647LL / nslab)
    return fail(GDN2_ERR_UNSUPPORTED, "%s: too many rows x channels", fn);
  return GDN2_OK;
}

// How the rows are dealt out.
struct ScanPlan {
  int64_t stretches;  // chains of a slab, each of whole sequences
  int64_t rows;       // of a stretch
  int64_t sequences;  // and its sequences
  int slab, cluster;
};

// Stretches: as many as leave two or three CTAs for every SM.  They are the
// same forward and backward, so that the kept states are found again.
ScanPlan scan_stretches(const gdn2_scan_problem* p, int sms) {
  ScanPlan l{1, (int64_t)p->B * p->T, p->n_seqs, 64, 1};
  if (p->cu_seqlens || p->B == 0) return l;
  int64_t s = (int64_t)sms * 3 / ((p->D + 63) / 64);
  if (s > p->B) s = p->B;
  if (s < 1) s = 1;
  const int64_t each = (p->B + s - 1) / s;  // sequences of a stretch
  l.stretches = (p->B + each - 1) / each;
  l.rows = each * p->T;
  l.sequences = each;
  return l;
}

// Slab and cluster: what takes the least time by a model of a turn, fitted to
// runs of both directions over slabs and clusters (seven shapes from 9001 x 1000
// to 131,072 x 1024).  A turn takes its latency, which grows with the cluster
// and with a sequence's edge in it, or what its SM needs for all its CTAs.  Scans
// of a few hundred channels and packed training were not among the shapes.
// GPCs have 16 to 20 SMs, so large clusters leave some of them out.
void scan_fit(const gdn2_scan_problem* p, int sms, int ctas, bool bwd, ScanPlan& l) {
  static constexpr struct { int size; double reach; } kClusters[] = {
      {1, 1.}, {2, 1.}, {4, .94}, {6, .9}, {8, .865}, {10, .83}, {12, .8}, {14, .77}, {16, .75}};
  double least = -1.;
  for (const auto& c : kClusters)
    for (int w = 64; w >= 32; w /= 2) {
      const int64_t slots = (int64_t)(sms * ctas * c.reach);
      const int64_t need = l.stretches * ((p->D + w - 1) / w) * c.size;
      const int64_t rows = (int64_t)c.size * (1024 * kCpt / w);
      const double on_sm = (double)(need < slots ? need : slots) / sms;
      // microseconds
      const int64_t turns = (l.rows + rows - 1) / rows;
      const double edge = turns > l.sequences ? (double)l.sequences / turns : 1.;
      const double latency =
          1.2 * edge + (c.size > 1 ? (bwd ? 2.8 : 1.7) + .03 * c.size : (bwd ? 2.2 : 1.2));
      const double work = on_sm * (bwd ? 1.93 : w == 64 ? 1.1 : 1.22);
      const double turn = .25 + (latency > work ? latency : work);
      // what a second wave holds starts as the first ends
      const double waves = .5 * ((double)((need + slots - 1) / slots) +
                                 (need > slots ? (double)need / slots : 1.));
      const double cost = waves * (double)(turns + 2) * turn;
      if (least < 0. || cost < least) {
        least = cost;
        l.slab = w;
        l.cluster = c.size;
      }
    }
}

ScanArgs scan_args(const gdn2_scan_problem* p, const ScanPlan& l) {
  ScanArgs a{};
  a.rows = (int64_t)p->B * p->T;
  a.T = p->T;
  a.D = p->D;
  a.n_seqs = p->n_seqs;
  a.cu = p->cu_seqlens;
  a.ldv = p->ld_v;
  a.ldg = p->ld_g;
  a.ldw = p->ld_w;
  a.lddy = p->ld_dy;
  a.stretch = l.rows;
  a.keeps = (l.rows + kKeep - 1) / kKeep;
  a.nslab = (p->D + l.slab - 1) / l.slab;
  a.cluster = l.cluster;
  return a;
}

template <typename K>
cudaError_t launch_scan(K kernel, const ScanArgs& a, const ScanPlan& l, int threads, int stage,
                        cudaStream_t st) {
  const int run = 2 * l.slab * (int)sizeof(float2);  // of a CTA of the cluster, both parities
  const int smem = stage + (l.cluster > 1 ? l.cluster * run : 0);
  // The limit belongs to the kernel, and other host threads launch it with other
  // clusters: always what the largest needs.
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       stage + kMaxCluster * run);
  if (e == cudaSuccess && l.cluster > 8)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(l.stretches * a.nslab * l.cluster));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)l.cluster;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = l.cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

// Whether every `n` channels of a row can be moved together.
bool group_ok(const void* p, int64_t ld, size_t es, int n = kCpt) {
  return aligned_to(p, n * es) && ld % n == 0;
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

// How long a wait for the cluster's runs may take, and whether it waits for more
// than comes (a test).
struct Wait {
  uint64_t ns = tc::kWaitLimitNs;
  bool in_vain = false;
};

int scan_fwd(const char* fn, const gdn2_scan_problem* p, const void* v, const void* g,
             const void* w, const float* h0, void* y, float* ht, float* saved, void* stream,
             const Wait& wait) {
  int rc = check_scan(p, fn);
  if (rc) return rc;
  const int64_t rows = (int64_t)p->B * p->T;
  if (rows > 0 && (!v || !g || !y)) return fail(GDN2_ERR_INVALID, "%s: null pointer", fn);
  if (w && p->ld_w < p->D) return fail(GDN2_ERR_INVALID, "%s: ld_w must be at least D", fn);
  if (p->n_seqs == 0 || (rows == 0 && !ht)) return GDN2_OK;
  const cudaStream_t st = (cudaStream_t)stream;
  int sms = 0;
  cudaError_t e = num_sms(&sms);
  if (e != cudaSuccess) return cuda_status(e, fn);
  ScanPlan l = scan_stretches(p, sms);
  ScanArgs a = scan_args(p, l);
  if ((e = fault_word(&a.fault)) != cudaSuccess) return cuda_status(e, fn);
  a.v = v; a.g = g; a.w = w; a.h0 = h0; a.y = y; a.ht = ht; a.saved = saved;
  const size_t es = dtype_size(p->dtype);
  int al = kCpt;  // channels aligned together
  for (; al > 1; al /= 2)
    if (a.D % al == 0 && group_ok(v, a.ldv, es, al) && group_ok(y, a.D, es, al) &&
        group_ok(g, a.ldg, dtype_size(p->g_dtype), al) && (!w || group_ok(w, a.ldw, es, al)))
      break;
  return cuda_status(scan_dispatch(p, w != nullptr, [&](auto t, auto gt, auto gate) {
    using T = decltype(t);
    using G = decltype(gt);
    constexpr bool GATE = decltype(gate)::value;
    scan_fit(p, sms, ctas_of<T, false>(), false, l);
    ScanArgs b = a;
    b.nslab = (a.D + l.slab - 1) / l.slab;
    b.cluster = l.cluster;
    if (wait.in_vain && l.cluster == 1) return cudaErrorNotSupported;
    b.wait_ns = wait.ns;
    b.expect = (l.cluster * l.slab + wait.in_vain) * (int)sizeof(float2);
    auto go = [&](auto w) {
      constexpr int W = decltype(w)::value;
      constexpr int R = rows_of<false>();
      auto run = [&](auto k, auto aligned) {
        constexpr int stage = StageLayout<T, G, GATE, false, decltype(aligned)::value>::bytes;
        return launch_scan(k, b, l, 1024 / R, stage, st);
      };
      if (al == 4) return run(k_scan_fwd<T, G, GATE, W, R, 4>, std::integral_constant<int, 4>{});
      if constexpr (sizeof(T) == 2)  // two fp32 channels gain nothing over one
        if (al == 2) return run(k_scan_fwd<T, G, GATE, W, R, 2>, std::integral_constant<int, 2>{});
      return run(k_scan_fwd<T, G, GATE, W, R, 1>, std::integral_constant<int, 1>{});
    };
    return l.slab == 64 ? go(std::integral_constant<int, 64>{})
                        : go(std::integral_constant<int, 32>{});
  }), fn);
}

int scan_bwd(const char* fn, const gdn2_scan_problem* p, const void* v, const void* g,
             const void* w, const float* h0, const float* saved, const void* dy, const float* dht,
             void* dv, void* dg, void* dw, float* dh0, void* stream, const Wait& wait) {
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
  cudaError_t e = num_sms(&sms);
  if (e != cudaSuccess) return cuda_status(e, fn);
  ScanPlan l = scan_stretches(p, sms);
  ScanArgs a = scan_args(p, l);
  if ((e = fault_word(&a.fault)) != cudaSuccess) return cuda_status(e, fn);
  a.v = v; a.g = g; a.w = w; a.h0 = h0; a.saved = const_cast<float*>(saved);
  a.dy = dy; a.dht = dht; a.dv = dv; a.dg = dg; a.dw = dw; a.dh0 = dh0;
  const size_t es = dtype_size(p->dtype), eg = dtype_size(p->g_dtype);
  int al = kCpt;  // channels aligned together
  for (; al > 1; al /= 2)
    if (a.D % al == 0 && group_ok(v, a.ldv, es, al) && group_ok(dy, a.lddy, es, al) &&
        group_ok(g, a.ldg, eg, al) && group_ok(dv, a.D, es, al) && group_ok(dg, a.D, eg, al) &&
        (!w || (group_ok(w, a.ldw, es, al) && group_ok(dw, a.D, es, al))))
      break;
  return cuda_status(scan_dispatch(p, w != nullptr, [&](auto t, auto gt, auto gate) {
    using T = decltype(t);
    using G = decltype(gt);
    constexpr bool GATE = decltype(gate)::value;
    scan_fit(p, sms, ctas_of<T, true>(), true, l);
    ScanArgs b = a;
    b.nslab = (a.D + l.slab - 1) / l.slab;
    b.cluster = l.cluster;
    if (wait.in_vain && l.cluster == 1) return cudaErrorNotSupported;
    b.wait_ns = wait.ns;
    b.expect = (l.cluster * l.slab + wait.in_vain) * (int)sizeof(float2);
    auto go = [&](auto w) {
      constexpr int W = decltype(w)::value;
      constexpr int R = rows_of<true>();
      auto run = [&](auto k, auto aligned) {
        constexpr int stage = StageLayout<T, G, GATE, true, decltype(aligned)::value>::bytes;
        return launch_scan(k, b, l, 1024 / R, stage, st);
      };
      if (al == 4) return run(k_scan_bwd<T, G, GATE, W, R, 4>, std::integral_constant<int, 4>{});
      if constexpr (sizeof(T) == 2)  // two fp32 channels gain nothing over one
        if (al == 2) return run(k_scan_bwd<T, G, GATE, W, R, 2>, std::integral_constant<int, 2>{});
      return run(k_scan_bwd<T, G, GATE, W, R, 1>, std::integral_constant<int, 1>{});
    };
    return l.slab == 64 ? go(std::integral_constant<int, 64>{})
                        : go(std::integral_constant<int, 32>{});
  }), fn);
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
  return scan_fwd("gdn2_scan_fwd", p, v, g, w, h0, y, ht, saved, stream, Wait{});
}

int gdn2_scan_bwd(const gdn2_scan_problem* p, const void* v, const void* g, const void* w,
                  const float* h0, const float* saved, const void* dy, const float* dht,
                  void* dv, void* dg, void* dw, float* dh0, void* stream) {
  return scan_bwd("gdn2_scan_bwd", p, v, g, w, h0, saved, dy, dht, dv, dg, dw, dh0, stream, Wait{});
}

int gdn2_test_scan_wait_timeout(const gdn2_scan_problem* p, const void* v, const void* g, void* y,
                                float* saved, const void* dy, void* dv, void* dg,
                                uint64_t wait_ns, void* stream) {
  const char* fn = "gdn2_test_scan_wait_timeout";
  if (wait_ns == 0 || wait_ns > tc::kWaitLimitNs)
    return fail(GDN2_ERR_INVALID, "%s: wait_ns must be in 1 .. 1e9 (got %llu)", fn,
                (unsigned long long)wait_ns);
  const Wait wait{wait_ns, true};
  if (dy)
    return scan_bwd(fn, p, v, g, nullptr, nullptr, saved, dy, nullptr, dv, dg, nullptr, nullptr,
                    stream, wait);
  return scan_fwd(fn, p, v, g, nullptr, nullptr, y, nullptr, saved, stream, wait);
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
