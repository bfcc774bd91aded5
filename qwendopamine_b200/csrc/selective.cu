// selective.cu -- selective state space scan: N states for each channel, decays
// and inputs that depend on the token; its gradient, and one token on a pool of
// states.
//
// Mathematics, for channel d, state n, with dt after its bias and softplus and
// B, C shared by the channels of a group:
//   a_t = exp(dt_t A),  h_t = a_t h_{t-1} + dt_t x_t B_t,  y_t = (sum_n C_t h_t + D x_t) silu(z_t)
// Backward, with o_t = dy_t silu(z_t) and e_t = dL/dh_t:
//   e_t = o_t C_t + a_{t+1} e_{t+1},  dC_t = sum_d o_t h_t,  dB_t = sum_d dt_t x_t e_t
//   dx_t = dt_t sum_n B_t e_t + D o_t,  ddt_t = sum_n A a_t h_{t-1} e_t + x_t sum_n B_t e_t
//   dA = sum_t dt_t a_t h_{t-1} e_t,  dD = sum_t o_t x_t,  dz_t = dy_t (sum_n C_t h_t + D x_t) silu'(z_t)
//
// A channel's states stay in registers from row to row, four to a lane forward and
// two of each of two channels backward.  Rows come in 16 at a time by asynchronous
// copies, one block ahead; what a row needs of a channel (dt, dt x, o) is formed once
// for all lanes, in shared memory, and there the lanes leave their shares of sums over
// a channel's states.  The sums over channels, dB and dC, are products on the tensor
// core (operands of two TF32 values, fp32 sums): a lane has its operands' values as
// they are.
//
// The time axis is cut where channels and sequences alone leave SMs idle: each
// chunk's end state is formed from a zero start, a second launch carries them from
// chunk to chunk (a chunk's decay is exp(A sum dt)), and the third starts every
// chunk from its state.  The backward does the same with e.  The forward keeps the
// state in front of every 16 rows; the backward forms the 16 rows' states again and
// holds four rows' at a time.  The CTAs' shares of dB and dC are summed by a launch of
// their own: every sum has a fixed order, equal inputs give equal bits.
//
// Bound: shared memory's bandwidth and the exponentials forward (8 x 4096 tokens x
// 2048 channels x 16 states in bf16: 699 us, of which one exponential a state and
// row takes 239); backward (2.5 ms, 3.8 times the forward's instructions) the issue of
// instructions, 57 % busy, and waits for shared memory and the tensor core with 14
// warps an SM.  Rows read as they were needed and sums exchanged between lanes took
// 1523 us and 4.6 ms.
#include "mma16.cuh"
#include "op_util.cuh"

#include <algorithm>
#include <cfloat>

namespace gdn2 {
namespace {

constexpr int kSelThreads = 128;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSub = 16;   // rows of a block: one kept state for each
constexpr int kHeld = 4;   // rows whose states the backward holds at a time
constexpr int kHalf = 8;   // rows whose sums it hands on at a time
constexpr int kMostChunks = 640;  // of the time axis
constexpr float kSelLn2 = 0.6931471805599453f;
constexpr float kLog2eRest = 1.92596299e-8f;  // log2(e) - kLog2e

struct SelSource {  // a token tensor's rows
  const void* p;
  int64_t ld;
};

struct SelArgs {
  int B, D, G, N, NP, n_seqs;   // NP: N rounded up to 4
  int64_t T;
  const int32_t* cu;
  SelSource tok[4];   // x, dy (backward only), z, dt where it has their type
  SelSource dt32;     // dt where it is fp32
  SelSource vec[2];   // B, C
  const void *x, *dt, *z, *Bv, *Cv;  // of one token
  int64_t ldx, lddt, ldz, ldb, ldc, lddy;
  const float *A, *Dk, *bias, *h0;
  bool dt_f32, softplus;
  void* y;
  float* ht;
  float* saved;       // [B][subs][D][NP]: the states in front of every 16 rows
  int64_t chunk, subs;
  int chunks, tiles_per_group, tiles;
  float* carry;       // [B][chunks][D][NP]
  float* decay;       // [B][chunks][D]: sums of dt
  // backward
  const float* dht;
  void *dx, *ddt, *dz;
  float* dh0;
  float* part_bc;     // [tiles][B T][2][N]
  float* part_a;      // [B][chunks][D][NP]
  float* part_d;      // [2][B][chunks][D]: dD, ddt_bias
};

// ---------------------------------------------------------------------------
// elementary functions of a token's values
// ---------------------------------------------------------------------------
__device__ __forceinline__ float rcp_fast(float x) {  // relative error 2^-23
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float2 rcp2(float2 x) { return make_float2(rcp_fast(x.x), rcp_fast(x.y)); }

// ln(1 + e^v) = max(v, 0) + ln(1 + t), t = e^-|v|, without loss for very negative
// v: with s = t / (2 + t) <= 1/3, ln(1 + t) = 2 artanh s = 2 (s + s^3/3 + s^5/5 ...),
// whose terms from s^17 on are below 1e-9 of it.  t = 2^e (1 + r ln 2), where r is what
// the exponent e = -|v| log2(e) loses to its rounding (up to |v| 2^-24) and log2(e) to
// its own.  Within 3 * 2^-22 for v from -87 on; below, t is flushed to zero.
__device__ __forceinline__ float2 softplus2(float2 v) {
  // beyond 128 t is zero; the difference of two infinities would be NaN
  const float2 w = make_float2(fminf(fabsf(v.x), 128.f), fminf(fabsf(v.y), 128.f));
  const float2 e = mul2(w, f2(-kLog2e));
  const float2 r = fma2(w, f2(-kLog2eRest), fma2(w, f2(-kLog2e), neg2(e)));
  const float2 t0 = exp2_2(e), t = fma2(t0, mul2(r, f2(kSelLn2)), t0);
  const float2 s = mul2(t, rcp2(add2(t, f2(2.f)))), q = mul2(s, s);
  float2 p = fma2(q, f2(1.f / 15.f), f2(1.f / 13.f));
  p = fma2(q, p, f2(1.f / 11.f));
  p = fma2(q, p, f2(1.f / 9.f));
  p = fma2(q, p, f2(1.f / 7.f));
  p = fma2(q, p, f2(1.f / 5.f));
  p = fma2(q, p, f2(1.f / 3.f));
  // NaN is not below zero
  return fma2(f2(2.f), fma2(mul2(s, q), p, s), make_float2(v.x < 0.f ? 0.f : v.x, v.y < 0.f ? 0.f : v.y));
}
// The same of one value (one of a pair in its place: single tokens 15.5 us for 13.7).
__device__ __forceinline__ float softplus_f(float v) {
  const float w = fminf(fabsf(v), 128.f), e = w * -kLog2e, t0 = fast_exp2(e);
  const float r = fmaf(w, -kLog2eRest, fmaf(w, -kLog2e, -e)), t = fmaf(t0, r * kSelLn2, t0);
  const float s = t * rcp_fast(t + 2.f), q = s * s;
  float p = fmaf(q, 1.f / 15.f, 1.f / 13.f);
  p = fmaf(q, p, 1.f / 11.f);
  p = fmaf(q, p, 1.f / 9.f);
  p = fmaf(q, p, 1.f / 7.f);
  p = fmaf(q, p, 1.f / 5.f);
  p = fmaf(q, p, 1.f / 3.f);
  return fmaf(2.f, fmaf(s * q, p, s), v < 0.f ? 0.f : v);
}

// 1 / (1 + e^-v), within 2^-21; for v < 0 the exponent's rounding adds up to |v| 2^-23
__device__ __forceinline__ float2 sigmoid2(float2 v) {
  return rcp2(add2(exp2_2(mul2(v, f2(-kLog2e))), f2(1.f)));
}
__device__ __forceinline__ float sigmoid_f(float v) { return rcp_fast(1.f + fast_exp2(-v * kLog2e)); }

// ---------------------------------------------------------------------------
// geometry
// ---------------------------------------------------------------------------
struct SelSpan {  // rows of a chunk
  int64_t lo;
  int rows;
  int b, c;
};

__device__ __forceinline__ SelSpan sel_span(const SelArgs& a, int bc) {
  SelSpan s;
  s.b = bc / a.chunks;
  s.c = bc - s.b * a.chunks;
  const int64_t at = s.c * a.chunk;
  s.lo = (int64_t)s.b * a.T + at;
  s.rows = (int)min(a.chunk, a.T - at);
  return s;
}

struct SelSeq {
  int64_t lo, hi;
  int n;
};

// The sequence of row r (the last that starts at or in front of it).
__device__ __forceinline__ SelSeq seq_of(const SelArgs& a, int b, int64_t r) {
  if (!a.cu) return SelSeq{(int64_t)b * a.T, (int64_t)(b + 1) * a.T, b};
  int lo = 0, hi = a.n_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid] <= r) lo = mid; else hi = mid;
  }
  return SelSeq{a.cu[lo], a.cu[lo + 1], lo};
}

// The rows of a chunk at which the sequence of its row r begins and behind which it
// ends.
struct SelSides {
  int lo, hi;
  __device__ __forceinline__ SelSides(const SelArgs& a, const SelSpan& sp, int r) {
    const SelSeq s = seq_of(a, sp.b, sp.lo + r);
    lo = (int)max(s.lo - sp.lo, (int64_t)-1);
    hi = (int)min(s.hi - sp.lo, (int64_t)0x7fffffff);
  }
};

// Sequences that begin and end at rows r0 .. r0 + 15 (-1: none, kAbsent: no such row),
// by 16 threads.
constexpr int kAbsent = -2;
struct SelEdges {
  int begin[kSub], end[kSub];
};
__device__ __forceinline__ void mark_edges(const SelArgs& a, SelEdges& m, int b, int64_t r0, int64_t hi) {
  if (threadIdx.x < kSub) {
    const int64_t r = r0 + threadIdx.x;
    int bn = kAbsent, en = kAbsent;
    if (r < hi) {
      bn = en = -1;
      const SelSeq s = seq_of(a, b, r);
      if (r == s.lo) bn = s.n;
      if (r + 1 == s.hi) en = s.n;
    }
    m.begin[threadIdx.x] = bn;
    m.end[threadIdx.x] = en;
  }
}

// The barrier in front of a block's rows.  Whether they go by the rows that look for
// edges: where there are (`edge`), or, with REST, where a thread has an `odd` value.
template <bool REST>
__device__ __forceinline__ bool sync_or_mark(const SelArgs& a, SelEdges& m, bool odd, bool edge, const SelSpan& sp,
                                             int r0) {
  if constexpr (REST) {
    if (__syncthreads_or(odd) && !edge) {
      mark_edges(a, m, sp.b, sp.lo + r0, sp.lo + sp.rows);
      __syncthreads();
      edge = true;
    }
  } else {
    __syncthreads();
  }
  return edge;
}

// M neighbouring states of a channel, from n0 on, in an [..][D][N] array.
template <int M>
__device__ __forceinline__ void load_states(const float* p, int N, int n0, bool on, float2 (&h)[M / 2]) {
#pragma unroll
  for (int i = 0; i < M / 2; ++i) {
    h[i].x = p && on && n0 + 2 * i < N ? p[n0 + 2 * i] : 0.f;
    h[i].y = p && on && n0 + 2 * i + 1 < N ? p[n0 + 2 * i + 1] : 0.f;
  }
}
template <int M>
__device__ __forceinline__ void store_states(float* p, int N, int n0, bool on, const float2 (&h)[M / 2]) {
#pragma unroll
  for (int i = 0; i < M / 2; ++i) {
    if (on && n0 + 2 * i < N) p[n0 + 2 * i] = h[i].x;
    if (on && n0 + 2 * i + 1 < N) p[n0 + 2 * i + 1] = h[i].y;
  }
}
// The same in an [..][D][NP] array of this file, as one vector.
__device__ __forceinline__ void load_packed(const float* p, int NP, int n0, bool on, float2 (&h)[2]) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (on && n0 < NP) v = *reinterpret_cast<const float4*>(p + n0);
  h[0] = make_float2(v.x, v.y);
  h[1] = make_float2(v.z, v.w);
}
__device__ __forceinline__ void store_packed(float* p, int NP, int n0, bool on, const float2 (&h)[2]) {
  if (on && n0 < NP) *reinterpret_cast<float4*>(p + n0) = make_float4(h[0].x, h[0].y, h[1].x, h[1].y);
}

// States beyond the last, of the 2 M neighbouring ones from n0 on: zero.  They stay so by
// themselves while steps and inputs are finite; infinity times their zeros is NaN.
template <int M> __device__ __forceinline__ void clear_rest(int N, int n0, float2 (&h)[M]) {
#pragma unroll
  for (int i = 0; i < M; ++i) {
    if (n0 + 2 * i >= N) h[i].x = 0.f;
    if (n0 + 2 * i + 1 >= N) h[i].y = 0.f;
  }
}

// Sums that are not finite where one of the values is not.
__device__ __forceinline__ float sizes2(float2 x, float2 y) { return (fabsf(x.x) + fabsf(x.y)) + (fabsf(y.x) + fabsf(y.y)); }

// A thread's running sums of blocks of rows, four in its place of shared memory.
struct BlockSums {
  float4 v[kSelThreads];
  __device__ __forceinline__ void clear() { v[threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void add(float2 x, float2 y) {
    const float4 a = v[threadIdx.x];
    v[threadIdx.x] = make_float4(a.x + x.x, a.y + x.y, a.z + y.x, a.w + y.y);
  }
};

// Two neighbouring values in shared memory.
template <typename E> __device__ __forceinline__ float2 pair_at(const E* p) { return ld2<E>(p); }

// 16 rows of W columns of each of K tensors (those that are there) on their way into
// shared memory, one tensor after the other.  The 16-byte pieces are dealt out to
// the threads; a thread keeps its pieces' addresses, which move from block to block
// of 16 rows, in its place of shared memory.  What does not exist becomes zero.
template <typename E, int W, int K> struct RowCursor {
  static constexpr int VE = 16 / (int)sizeof(E), CPR = W / VE, PIECES = kSub * CPR;
  static constexpr int NS = (K * PIECES + kSelThreads - 1) / kSelThreads;
  static_assert(W % VE == 0 && (kSelThreads % PIECES == 0 || PIECES % kSelThreads == 0), "whole pieces");
  struct alignas(16) Piece {
    const char* p;
    int step;   // bytes from block to block
    int bytes;  // of the piece; -1: no tensor
  };
  Piece of[NS][kSelThreads];

  static __device__ __forceinline__ int row_of(int i) {
    return (threadIdx.x % PIECES) / CPR + (i * kSelThreads % PIECES) / CPR;
  }
  // Blocks from row r0 on, forward (way 1) or backward (-1).  Returns the bits of all
  // rows' addresses, of which the lowest says how they are aligned.
  __device__ __forceinline__ uint32_t start(const SelSource* src, int64_t r0, int64_t col, int ncols, int way) {
    uint32_t bits = 0u;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (src[k].p)
        bits |= (uint32_t)reinterpret_cast<uintptr_t>((const E*)src[k].p + col) | (uint32_t)(src[k].ld * sizeof(E));
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int k = (threadIdx.x + i * kSelThreads) / PIECES;
      Piece x{nullptr, 0, -1};
      if ((K * PIECES % kSelThreads == 0 || k < K) && src[k].p) {
        const int c = threadIdx.x % CPR * VE, n = max(0, min(ncols - c, VE));
        // a piece without a value reads nothing, from an address that exists and has the
        // alignment that was looked at (a group's first column may have another than column 0)
        x.p = (const char*)((const E*)src[k].p + col + (n ? (r0 + row_of(i)) * src[k].ld + c : 0));
        x.step = n ? (int)(way * kSub * src[k].ld * (int)sizeof(E)) : 0;
        x.bytes = n * (int)sizeof(E);
      }
      of[i][threadIdx.x] = x;
    }
    return bits;
  }
  // the next block, of which `rows` rows exist; `size`: of an asynchronous copy that
  // the rows' alignment allows (16, 8 or 4 bytes, 0: none)
  __device__ __forceinline__ void request(E* to, int rows, int size) {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const Piece x = of[i][threadIdx.x];
      if (x.bytes < 0) continue;
      E* dst = to + (threadIdx.x + i * kSelThreads) * VE;
      const int bytes = row_of(i) < rows ? x.bytes : 0;
      if (rows >= kSub && size == 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(x.p), "r"(bytes)
                     : "memory");
      } else if (bytes == 0) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(0u, 0u, 0u, 0u);
      } else if (size == 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(x.p), "r"(bytes)
                     : "memory");
      } else if (size == 8) {
#pragma unroll
        for (int b = 0; b < 16; b += 8)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(dst) + b),
                       "l"(x.p + (b < bytes ? b : 0)), "r"(max(0, min(bytes - b, 8)))
                       : "memory");
      } else if (size == 4) {
#pragma unroll
        for (int b = 0; b < 16; b += 4)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst) + b),
                       "l"(x.p + (b < bytes ? b : 0)), "r"(max(0, min(bytes - b, 4)))
                       : "memory");
      } else {
        const int n = bytes / (int)sizeof(E);
#pragma unroll
        for (int e = 0; e < VE; ++e) dst[e] = e < n ? ((const E*)x.p)[e] : from_f<E>(0.f);
      }
      of[i][threadIdx.x].p = x.p + x.step;
    }
  }
};

// The channels of a CTA (L lanes of four states for each in the forward, 2 L of
// two in the backward), and what a thread stages of them.
template <int L> struct SelTile {
  static constexpr int CH = kSelThreads / L;  // channels
  static constexpr int NL = 4 * L;            // states, padded
  static constexpr int PAIRS = CH / 2;        // pairs of channels: a thread stages one, in
  static constexpr int STEP = 2 * L;          // every STEP-th row
  static constexpr int BC_STEP = kSelThreads / (2 * NL), BC_ROWS = kHalf / BC_STEP < 1 ? 1 : kHalf / BC_STEP;
  static constexpr int PER = STEP < kSub ? kSub / STEP : 1, PER_HALF = STEP < kHalf ? kHalf / STEP : 1;
  int d0, nch, g, tile;
  int pc, pr;         // the pair's first channel, the first row
  __device__ __forceinline__ SelTile(const SelArgs& a, int tile_) : tile(tile_) {
    g = tile / a.tiles_per_group;
    const int dg = a.D / a.G, at = (tile - g * a.tiles_per_group) * CH;
    d0 = g * dg + at;
    nch = min(CH, dg - at);
    pc = 2 * (threadIdx.x % PAIRS);
    pr = threadIdx.x / PAIRS;
  }
  // a parameter's values of the staged pair (zero without it)
  __device__ __forceinline__ float2 pair_of(const float* p) const {
    return make_float2(p && pc < nch ? p[d0 + pc] : 0.f, p && pc + 1 < nch ? p[d0 + pc + 1] : 0.f);
  }
  // whether a staged pair can be stored as one word in contiguous [rows][D] results
  template <typename E> __device__ __forceinline__ bool whole(const void* p, int D) const {
    return pc + 1 < nch && (D & 1) == 0 && ((reinterpret_cast<uintptr_t>((const E*)p + d0 + pc)) & (2 * sizeof(E) - 1)) == 0;
  }
  template <typename E> __device__ __forceinline__ void store_pair(E* to, bool whole, float2 v) const {
    if (whole) {
      if constexpr (sizeof(E) == 4) *reinterpret_cast<float2*>(to) = v;
      else *reinterpret_cast<uint32_t*>(to) = pack2<E>(v.x, v.y);
    } else {
      if (pc < nch) to[0] = from_f<E>(v.x);
      if (pc + 1 < nch) to[1] = from_f<E>(v.y);
    }
  }
};

__device__ __forceinline__ int64_t block_states(const SelArgs& a, int b, int64_t r0) {
  return ((int64_t)b * a.subs + (r0 - (int64_t)b * a.T) / kSub) * a.D * a.NP;
}

// Values of 16 rows as they come from memory: x, dy (backward), z, and dt where it
// has their type.
template <typename T, int L, bool BWD> struct SelRaw {
  using S = SelTile<L>;
  static constexpr int V = kSub * S::CH, K = BWD ? 4 : 3;
  alignas(16) T tok[K * V];
  alignas(16) T vec[2 * kSub * S::NL];  // B, C
  __device__ __forceinline__ float2 x(int i) const { return pair_at(tok + i); }
  __device__ __forceinline__ float2 dy(int i) const { return pair_at(tok + V + i); }
  __device__ __forceinline__ float2 z(int i) const { return pair_at(tok + (K - 2) * V + i); }
  __device__ __forceinline__ float2 dt(int i) const { return pair_at(tok + (K - 1) * V + i); }
};

// Their copies.
template <typename T, int L, bool BWD> struct SelCopies {
  using S = SelTile<L>;
  using R = SelRaw<T, L, BWD>;
  RowCursor<T, S::CH, R::K> tok;
  RowCursor<T, S::NL, 2> vec;
};
template <typename T, int L, bool BWD, typename Shared>
__device__ __forceinline__ int start_copies(const SelArgs& a, const SelTile<L>& t, Shared& s, int64_t r0) {
  constexpr int way = BWD ? -1 : 1;
  uint32_t bits = s.copies.tok.start(a.tok, r0, t.d0, t.nch, way);
  bits |= s.copies.vec.start(a.vec, r0, (int64_t)t.g * a.N, a.N, way);
  if (a.dt_f32) bits |= s.dt32.cursor.start(&a.dt32, r0, t.d0, t.nch, way);
  return (bits & 15) == 0 ? 16 : (bits & 7) == 0 ? 8 : (bits & 3) == 0 ? 4 : 0;
}
template <typename Shared>
__device__ __forceinline__ void request_copies(const SelArgs& a, Shared& s, int at, int rows, int size) {
  s.copies.tok.request(s.raw[at].tok, rows, size);
  s.copies.vec.request(s.raw[at].vec, rows, size);
  if (a.dt_f32) s.dt32.cursor.request(s.dt32.v[at], rows, size);
  asm volatile("cp.async.commit_group;" ::: "memory");
}
// dt as fp32, of both blocks: the end of shared memory, left out where dt is not.
template <int L> struct SelDt32 {
  RowCursor<float, SelTile<L>::CH, 1> cursor;
  alignas(16) float v[2][kSub * SelTile<L>::CH];
};

__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// B or C of 16 rows as fp32.
template <typename T, int L> __device__ __forceinline__ void widen(float* to, const T* from) {
#pragma unroll
  for (int i = 0; i < (kSub * 2 * L + kSelThreads - 1) / kSelThreads; ++i) {
    const int at = 2 * (threadIdx.x + i * kSelThreads);
    if (kSub * 4 * L % (2 * kSelThreads) == 0 || at < kSub * 4 * L)
      *reinterpret_cast<float2*>(to + at) = pair_at(from + at);
  }
}

// Two fp32 values in a 64-bit register, as packed arithmetic takes them: pairs that
// come from shared memory as 64-bit words need no moves.
typedef unsigned long long pair64;
__device__ __forceinline__ pair64 pmul(pair64 a, pair64 b) {
  pair64 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ pair64 pfma(pair64 a, pair64 b, pair64 c) {
  pair64 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ pair64 to_pair(float2 v) {
  pair64 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(v.x), "f"(v.y));
  return d;
}
__device__ __forceinline__ float2 of_pair(pair64 v) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(v));
  return d;
}
__device__ __forceinline__ ulonglong2 two_pairs(const void* p) { return *reinterpret_cast<const ulonglong2*>(p); }

// The factor of a channel goes to both of its states: scalar operations, which need
// no second copy of it, where packed ones would.
__device__ __forceinline__ float2 scale2(float a, float2 x) { return make_float2(a * x.x, a * x.y); }
__device__ __forceinline__ float2 scale_add2(float a, float2 x, float2 y) {
  return make_float2(fmaf(a, x.x, y.x), fmaf(a, x.y, y.y));
}

__device__ __forceinline__ float2 lo2(float4 v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ float2 hi2(float4 v) { return make_float2(v.z, v.w); }

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
template <typename T, int L> struct SelFwdShared {
  using S = SelTile<L>;
  SelRaw<T, L, false> raw[2];
  alignas(16) float b[kSub * S::NL];
  alignas(16) float c[kSub * S::NL];
  alignas(16) float2 dd[kSub][S::CH];       // dt, dt x
  alignas(16) float y[kSub][kSelThreads];   // each lane's share of its channel's sum
  SelEdges edges;
  SelCopies<T, L, false> copies;
  SelDt32<L> dt32;
  static constexpr int without_dt32() { return (int)(sizeof(SelFwdShared) - sizeof(SelDt32<L>)); }
};

struct FwdLane {
  int l, mc, d;  // which of the channel's lanes, which channel
  bool on;
};

// 16 rows of one lane's states; LOCAL: only the states.  EDGE: rows with a sequence's
// begin or end, or with values that are not finite; REST: lanes hold states beyond the last.
template <bool LOCAL, bool EDGE, bool REST, typename T, int L>
__device__ __forceinline__ void fwd_rows(const SelArgs& a, SelFwdShared<T, L>& s, const FwdLane& t,
                                         const pair64 (&A2)[2], pair64 (&h)[2], float& dsum) {
  using S = SelTile<L>;
  constexpr int U = 4;  // rows whose decays and inputs are formed together
#pragma unroll 2
  for (int q = 0; q < kSub; q += U) {
    pair64 da[U][2], in[U][2];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const float2 dd = s.dd[q + j][t.mc];
      const float4 B = *reinterpret_cast<const float4*>(s.b + (q + j) * S::NL + 4 * t.l);
      da[j][0] = to_pair(exp2_2(scale2(dd.x, of_pair(A2[0]))));
      da[j][1] = to_pair(exp2_2(scale2(dd.x, of_pair(A2[1]))));
      in[j][0] = to_pair(scale2(dd.y, lo2(B)));
      in[j][1] = to_pair(scale2(dd.y, hi2(B)));
      if constexpr (LOCAL) dsum += dd.x;
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int r = q + j;
      if constexpr (EDGE) {
        const int n = s.edges.begin[r];
        if (n >= 0) {
          float2 v[2];
          load_states<4>(a.h0 ? a.h0 + ((int64_t)n * a.D + t.d) * a.N : nullptr, a.N, 4 * t.l, t.on, v);
          h[0] = to_pair(v[0]);
          h[1] = to_pair(v[1]);
        }
      }
      h[0] = pfma(da[j][0], h[0], in[j][0]);
      h[1] = pfma(da[j][1], h[1], in[j][1]);
      if constexpr (EDGE && REST) {
        float2 v[2] = {of_pair(h[0]), of_pair(h[1])};
        clear_rest(a.N, 4 * t.l, v);
        h[0] = to_pair(v[0]);
        h[1] = to_pair(v[1]);
      }
      if constexpr (!LOCAL) {
        const ulonglong2 C = two_pairs(s.c + r * S::NL + 4 * t.l);
        const float2 o = of_pair(pfma(h[1], C.y, pmul(h[0], C.x)));
        s.y[r][threadIdx.x] = o.x + o.y;
        if constexpr (EDGE) {
          const int n = s.edges.end[r];
          const float2 v[2] = {of_pair(h[0]), of_pair(h[1])};
          if (n >= 0 && a.ht) store_states<4>(a.ht + ((int64_t)n * a.D + t.d) * a.N, a.N, 4 * t.l, t.on, v);
        }
      }
    }
  }
}

// The sum of a channel's L shares.
template <int L> __device__ __forceinline__ float sum_shares(const float* p) {
  if constexpr (L == 2) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    return v.x + v.y;
  } else {
    float f = 0.f;
#pragma unroll
    for (int i = 0; i < L / 4; ++i) {
      const float4 v = reinterpret_cast<const float4*>(p)[i];
      f += (v.x + v.y) + (v.z + v.w);
    }
    return f;
  }
}

template <typename T, int L, bool REST, bool LOCAL>
__global__ void __launch_bounds__(kSelThreads) k_sel_fwd(const SelArgs a) {
  using S = SelTile<L>;
  extern __shared__ __align__(16) char raw_shared[];
  SelFwdShared<T, L>& s = *reinterpret_cast<SelFwdShared<T, L>*>(raw_shared);
  const int bc = blockIdx.x / a.tiles;
  const S t(a, blockIdx.x - bc * a.tiles);
  const SelSpan sp = sel_span(a, bc);
  if (LOCAL && sp.c + 1 == a.chunks) return;  // nothing follows the last
  const int size = start_copies<T, L, false>(a, t, s, sp.lo);
  request_copies(a, s, 0, sp.rows, size);
  const int mc = threadIdx.x / L;
  const FwdLane lane{(int)threadIdx.x % L, mc, t.d0 + mc, mc < t.nch};
  float2 rate[2], start[2] = {f2(0.f), f2(0.f)};
  load_states<4>(a.A + (int64_t)lane.d * a.N, a.N, 4 * lane.l, lane.on, rate);
  const pair64 A2[2] = {to_pair(mul2(rate[0], f2(kLog2e))), to_pair(mul2(rate[1], f2(kLog2e)))};
  float dsum = 0.f;
  const int64_t mine = (int64_t)lane.d * a.NP;
  if (!LOCAL && sp.c > 0)
    load_packed(a.carry + (int64_t)bc * a.D * a.NP + mine, a.NP, 4 * lane.l, lane.on, start);
  pair64 h[2] = {to_pair(start[0]), to_pair(start[1])};
  auto put_states = [&](float* to) {
    const float2 v[2] = {of_pair(h[0]), of_pair(h[1])};
    store_packed(to + mine, a.NP, 4 * lane.l, lane.on, v);
  };
  const float2 bias = t.pair_of(a.bias), skip = t.pair_of(a.Dk);
  const bool whole = !LOCAL && t.template whole<T>(a.y, a.D);
  T* out = (T*)a.y + (sp.lo + t.pr) * a.D + t.d0 + t.pc;
  float* keep = a.saved + block_states(a, sp.b, sp.lo);
  SelSides side(a, sp, 0);

  int at = 0;
  for (int r0 = 0; r0 < sp.rows; r0 += kSub, at ^= 1) {
    const SelRaw<T, L, false>& raw = s.raw[at];
    const bool edge = side.lo == r0 || side.hi <= r0 + kSub;
    const int rows = sp.rows - r0;  // that are left
    float most = 0.f;
    copies_done();
    __syncthreads();
    if (rows > kSub) request_copies(a, s, at ^ 1, rows - kSub, size);
#pragma unroll
    for (int i = 0; i < S::PER; ++i) {
      const int row = t.pr + i * S::STEP;
      if (S::STEP > kSub && row >= kSub) break;
      const int p = row * S::CH + t.pc;
      float2 d = add2((a.dt_f32 ? pair_at(s.dt32.v[at] + p) : raw.dt(p)), bias);
      if (a.softplus) d = softplus2(d);
      if (row >= rows) d = f2(0.f);  // rows behind the last leave the states as they are
      const float2 u = mul2(d, raw.x(p));
      *reinterpret_cast<float4*>(&s.dd[row][t.pc]) = make_float4(d.x, u.x, d.y, u.y);
      if constexpr (REST) most += sizes2(d, u);
    }
    widen<T, L>(s.b, raw.vec);
    if constexpr (!LOCAL) widen<T, L>(s.c, raw.vec + kSub * S::NL);
    if (edge) mark_edges(a, s.edges, sp.b, sp.lo + r0, sp.lo + sp.rows);
    if constexpr (!LOCAL)
      if (a.saved) {
        put_states(keep);
        keep += (int64_t)a.D * a.NP;
      }
    if (sync_or_mark<REST>(a, s.edges, !(most <= FLT_MAX), edge, sp, r0)) {
      fwd_rows<LOCAL, true, REST>(a, s, lane, A2, h, dsum);
      if (rows > kSub) side = SelSides(a, sp, r0 + kSub);
    } else {
      fwd_rows<LOCAL, false, REST>(a, s, lane, A2, h, dsum);
    }
    if constexpr (!LOCAL) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < S::PER; ++i) {
        const int row = t.pr + i * S::STEP;
        if (S::STEP > kSub && row >= kSub) break;
        const int p = row * S::CH + t.pc;
        const float* share = s.y[row] + t.pc * L;
        float2 y = make_float2(sum_shares<L>(share), sum_shares<L>(share + L));
        if (a.Dk) y = fma2(skip, raw.x(p), y);
        if (a.z) {
          const float2 z = raw.z(p);
          y = mul2(y, mul2(z, sigmoid2(z)));
        }
        if (row < rows) t.store_pair(out + (int64_t)i * S::STEP * a.D, whole, y);
      }
      out += (int64_t)kSub * a.D;
    }
  }
  if constexpr (LOCAL) {
    put_states(a.carry + (int64_t)bc * a.D * a.NP);
    if (lane.l == 0 && lane.on) a.decay[(int64_t)bc * a.D + lane.d] = dsum;
  }
}

// carry[b][c] from the state behind chunk c, started at zero, to the state in
// front of it (BACK: from the gradient in front of chunk c to the one behind it).
// A sequence that begins in a chunk keeps what is in front of it out.
template <bool BACK> __global__ void __launch_bounds__(256) k_sel_carry(const SelArgs a) {
  constexpr int U = 8;  // chunks whose values are on their way together
  __shared__ bool begins[kMostChunks];
  const int64_t per = (int64_t)a.D * a.NP, tiles = (per + 255) / 256;
  const int b = (int)(blockIdx.x / tiles);
  const int64_t at = (blockIdx.x - b * tiles) * 256 + threadIdx.x;
  const int64_t base = (int64_t)b * a.chunks;
  for (int c = threadIdx.x; c < a.chunks; c += 256) {
    const SelSpan sp = sel_span(a, (int)(base + c));
    begins[c] = seq_of(a, b, sp.lo + sp.rows - 1).lo >= sp.lo;
  }
  __syncthreads();
  if (at >= per) return;
  const int d = (int)(at / a.NP), n = (int)(at - (int64_t)d * a.NP);
  const float A2 = n < a.N ? a.A[(int64_t)d * a.N + n] * kLog2e : 0.f;
  float run = 0.f;
  for (int k0 = 0; k0 < a.chunks; k0 += U) {
    float own[U], dsum[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int c = BACK ? a.chunks - 1 - (k0 + i) : k0 + i;
      const bool used = k0 + i + 1 < a.chunks;  // the last chunk's is not written
      own[i] = used ? a.carry[(base + c) * per + at] : 0.f;
      dsum[i] = used ? a.decay[(base + c) * a.D + d] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int c = BACK ? a.chunks - 1 - (k0 + i) : k0 + i;
      if (k0 + i >= a.chunks) break;
      a.carry[(base + c) * per + at] = run;
      // nothing stays nothing, however large the factor, and infinity infinite, however small
      run = begins[c] || run == 0.f ? own[i]
            : fabsf(run) == INFINITY ? run + own[i] : fmaf(fast_exp2(dsum[i] * A2), run, own[i]);
    }
  }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
template <typename T, int L> struct SelBwdShared {
  using S = SelTile<L>;
  static constexpr int G = 2 * L;           // lanes of a channel
  SelRaw<T, L, true> raw[2];
  alignas(16) float b[kSub * S::NL];
  alignas(16) float c[kSub * S::NL];
  alignas(16) float2 dd[kSub][S::CH];       // dt, dt x
  alignas(16) float o[kSub][S::CH];         // dy silu(z)
  // shares of three sums over the states of a pair of channels: B e, A2 a h' e, and
  // C h, where neighbouring lanes have added theirs (one has the first channel's)
  alignas(16) float2 share[2][kHalf][S::PAIRS * G];
  alignas(16) float share_y[kHalf][S::PAIRS * G];
  float bc[kSelWarps][kHalf][2][2][8];      // dB, dC of a warp's channels: state 0 and 1 of each lane
  alignas(16) BlockSums sum_a, sum_d;        // dA; dD and ddt_bias of the staged pair
  alignas(8) float2 par[2][S::PAIRS];       // dt_bias and D of the pairs
  SelEdges edges;
  SelCopies<T, L, true> copies;
  SelDt32<L> dt32;
  static constexpr int without_dt32() { return (int)(sizeof(SelBwdShared) - sizeof(SelDt32<L>)); }
};

// Where a lane stands in the backward: two neighbouring channels, two states of
// each.  Lane 4 g + k of a warp has channels 2 k, 2 k + 1 of eight, as a tensor-core
// operand of 16 states by 8 channels has them; its states are the group l = g of
// eight groups, or of the warp's eight lanes-of-four several channel sets share
// (fewer than 16 states) or several warps make up the groups (more).
template <int L> struct BwdLane {
  static constexpr int G = 2 * L, SETS = G < 8 ? 8 / G : 1, BLOCKS = G > 8 ? G / 8 : 1;
  int l, mc, d, set;
  bool on[2];
  __device__ __forceinline__ BwdLane(const SelTile<L>& t) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2;
    set = G < 8 ? g / G : 0;
    l = G < 8 ? g % G : (warp % BLOCKS) * 8 + g;
    mc = ((warp / BLOCKS) * SETS + set) * 8 + 2 * (lane & 3);
    d = t.d0 + mc;
    on[0] = mc < t.nch;
    on[1] = mc + 1 < t.nch;
  }
  __device__ __forceinline__ void load(const float* p, int N, float2 (&v)[2]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float2 x[1];
      load_states<2>(p ? p + (int64_t)(d + i) * N : nullptr, N, 2 * l, on[i], x);
      v[i] = x[0];
    }
  }
  __device__ __forceinline__ void store(float* p, int N, const float2 (&v)[2]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 x[1] = {v[i]};
      store_states<2>(p + (int64_t)(d + i) * N, N, 2 * l, on[i], x);
    }
  }
  __device__ __forceinline__ void clear_rest(int N, float2& v) const {
    float2 x[1] = {v};
    gdn2::clear_rest(N, 2 * l, x);
    v = x[0];
  }
  __device__ __forceinline__ void load_packed(const float* p, int NP, float2 (&v)[2]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      v[i] = on[i] && 2 * l < NP ? *reinterpret_cast<const float2*>(p + (int64_t)(d + i) * NP + 2 * l) : f2(0.f);
  }
  __device__ __forceinline__ void store_packed(float* p, int NP, const float2 (&v)[2]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (on[i] && 2 * l < NP) *reinterpret_cast<float2*>(p + (int64_t)(d + i) * NP + 2 * l) = v[i];
  }
};

// d = A B from a zero start (m16n8k8, TF32).
__device__ __forceinline__ void mma_tf32_new(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// A value's upper 19 bits, a TF32 operand as it stands; of NaN those of the one that
// arithmetic gives stay NaN.
__device__ __forceinline__ uint32_t tf32_cut(float x) { return __float_as_uint(x) & 0xffffe000u; }

// Sums over a warp's eight channels (of each set) by the tensor core: A holds a
// value for each state and channel as the lanes have them, B the channels' factors
// in every column.  An operand is the sum of two TF32 values and three products are
// summed in fp32, whatever the results' type: shares that cancel leave digits that
// one TF32 operand (11 bits) does not have.  (One product, 8 x 4096 x 2048 x 16 in
// bf16: forward and backward 2.81 ms, three 3.23 ms.)  What the cuts leave (below 2^-20
// of a value, and of a product's second order) counts where the first product is
// finite: infinity minus itself is NaN.
__device__ __forceinline__ void sum_channels(float (&sum)[4], const float2 (&v)[2], float w0, float w1) {
  const float x[4] = {v[0].x, v[0].y, v[1].x, v[1].y};
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hi[i] = tf32_cut(x[i]);
    lo[i] = tf32_cut(x[i] - __uint_as_float(hi[i]));
  }
  const uint32_t h0 = tf32_cut(w0), h1 = tf32_cut(w1);
  float more[4];
  mma_tf32_new(sum, hi, h0, h1);
  mma_tf32_new(more, lo, h0, h1);
  mma_tf32(more, hi, tf32_cut(w0 - __uint_as_float(h0)), tf32_cut(w1 - __uint_as_float(h1)));
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (fabsf(sum[i]) <= FLT_MAX) sum[i] += more[i];
}

// What a row has for a lane's two channels and two states.
struct BwdRow {
  float d[2], u[2];  // dt, dt x
  template <typename T, int L>
  __device__ __forceinline__ void load(const SelBwdShared<T, L>& s, const BwdLane<L>& t, int r) {
    const float4 v = *reinterpret_cast<const float4*>(&s.dd[r][t.mc]);
    d[0] = v.x; u[0] = v.y; d[1] = v.z; u[1] = v.w;
  }
};

// One row's states from those in front of it; da and p: the decays, and the
// decayed states.
template <bool EDGE, bool REST, typename T, int L>
__device__ __forceinline__ void state_row(const SelArgs& a, const SelBwdShared<T, L>& s, const BwdLane<L>& t,
                                          int r, const BwdRow& x, const float2 (&A2)[2], float2 (&h)[2],
                                          float2 (&da)[2], float2 (&p)[2]) {
  if constexpr (EDGE) {
    const int n = s.edges.begin[r];
    if (n >= 0) t.load(a.h0 ? a.h0 + (int64_t)n * a.D * a.N : nullptr, a.N, h);
  }
  const float2 B = *reinterpret_cast<const float2*>(s.b + r * SelTile<L>::NL + 2 * t.l);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    da[i] = exp2_2(scale2(x.d[i], A2[i]));
    p[i] = mul2(da[i], h[i]);
    h[i] = scale_add2(x.u[i], B, p[i]);
    if constexpr (EDGE && REST) {
      t.clear_rest(a.N, da[i]);
      t.clear_rest(a.N, p[i]);
      t.clear_rest(a.N, h[i]);
    }
  }
}

// Four rows from q on: their states again, then back through them.
template <bool EDGE, bool REST, typename T, int L>
__device__ __forceinline__ void bwd_rows(const SelArgs& a, SelBwdShared<T, L>& s, const BwdLane<L>& t, int q,
                                         const float2 (&A2)[2], const float2 (&h0)[2], float2 (&e)[2],
                                         float2 (&dA)[2]) {
  using W = BwdLane<L>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, k = lane & 3;
  // the columns 2 k, 2 k + 1 of a product belong to the set k / (4 / SETS); with one
  // set all are equal, and two lanes write the same
  const int which = k & 1;  // 0: dB, 1: dC
  const bool writes = W::SETS == 1 || k / (4 / W::SETS) == t.set;
  float* const to_bc = &s.bc[warp][0][which][0][lane >> 2];
  float2 h[2] = {h0[0], h0[1]}, da[kHeld][2], p[kHeld][2];
  BwdRow x[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; ++j) x[j].load(s, t, q + j);
#pragma unroll
  for (int j = 0; j < kHeld; ++j) state_row<EDGE, REST>(a, s, t, q + j, x[j], A2, h, da[j], p[j]);
#pragma unroll
  for (int j = kHeld - 1; j >= 0; --j) {
    const int r = q + j, at = r & (kHalf - 1);
    const float2 B = *reinterpret_cast<const float2*>(s.b + r * SelTile<L>::NL + 2 * t.l);
    const float2 C = *reinterpret_cast<const float2*>(s.c + r * SelTile<L>::NL + 2 * t.l);
    const float2 o = *reinterpret_cast<const float2*>(&s.o[r][t.mc]);
    if constexpr (EDGE) {
      const int n = s.edges.end[r];
      if (n >= 0) t.load(a.dht ? a.dht + (int64_t)n * a.D * a.N : nullptr, a.N, e);
    }
    float2 hh[2], v[3];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      hh[i] = scale_add2(x[j].u[i], B, p[j][i]);
      e[i] = scale_add2(i ? o.y : o.x, C, e[i]);
      if constexpr (EDGE && REST) {
        t.clear_rest(a.N, hh[i]);
        t.clear_rest(a.N, e[i]);
      }
    }
    float sb[4], sc[4];
    sum_channels(sb, e, x[j].u[0], x[j].u[1]);
    sum_channels(sc, hh, o.x, o.y);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float2 g = mul2(p[j][i], e[i]);
      if constexpr (EDGE)  // an infinite state times the zero behind the last row is no share of dA
        if (s.edges.begin[r] == kAbsent) g = f2(0.f);
      (i ? v[0].y : v[0].x) = fmaf(hh[i].y, C.y, hh[i].x * C.x);
      (i ? v[1].y : v[1].x) = fmaf(e[i].y, B.y, e[i].x * B.x);
      (i ? v[2].y : v[2].x) = fmaf(g.y, A2[i].y, g.x * A2[i].x);
      dA[i] = scale_add2(x[j].d[i], g, dA[i]);
      e[i] = mul2(da[j][i], e[i]);
    }
    const int mine = (t.mc >> 1) * W::G + t.l;
    s.share[0][at][mine] = v[1];
    s.share[1][at][mine] = v[2];
    const bool odd = t.l & 1;
    s.share_y[at][mine] = (odd ? v[0].y : v[0].x) + __shfl_xor_sync(0xffffffffu, odd ? v[0].x : v[0].y, 4);
    if (writes) {
      to_bc[at * 32] = which ? sc[0] : sb[0];
      to_bc[at * 32 + 8] = which ? sc[2] : sb[2];
    }
    if constexpr (EDGE) {
      const int n = s.edges.begin[r];
      if (n >= 0) {
        if (a.dh0) t.store(a.dh0 + (int64_t)n * a.D * a.N, a.N, e);
        e[0] = e[1] = f2(0.f);
      }
    }
  }
}

// LOCAL: only e, from zero behind the chunk to what it is in front of it.
template <bool EDGE, bool REST, typename T, int L>
__device__ __forceinline__ void bwd_rows_local(const SelArgs& a, SelBwdShared<T, L>& s, const BwdLane<L>& t,
                                               const float2 (&A2)[2], float2 (&e)[2], float2& dsum) {
#pragma unroll 8
  for (int r = kSub - 1; r >= 0; --r) {
    const float2 C = *reinterpret_cast<const float2*>(s.c + r * SelTile<L>::NL + 2 * t.l);
    const float2 o = *reinterpret_cast<const float2*>(&s.o[r][t.mc]);
    const float4 v = *reinterpret_cast<const float4*>(&s.dd[r][t.mc]);
    if constexpr (EDGE) {
      const int n = s.edges.end[r];
      if (n >= 0) t.load(a.dht ? a.dht + (int64_t)n * a.D * a.N : nullptr, a.N, e);
    }
    e[0] = mul2(exp2_2(scale2(v.x, A2[0])), scale_add2(o.x, C, e[0]));
    e[1] = mul2(exp2_2(scale2(v.z, A2[1])), scale_add2(o.y, C, e[1]));
    dsum = add2(dsum, make_float2(v.x, v.z));
    if constexpr (EDGE && REST) {
      t.clear_rest(a.N, e[0]);
      t.clear_rest(a.N, e[1]);
    }
    if constexpr (EDGE)
      if (s.edges.begin[r] >= 0) e[0] = e[1] = f2(0.f);
  }
}

// The sum of the G shares of a pair; neighbours start at different places, which
// spreads them over the banks.
template <int G> __device__ __forceinline__ float2 sum_pairs(const float2* p, int pair) {
  float2 f = f2(0.f);
#pragma unroll
  for (int i = 0; i < G / 2; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(p + 2 * (i ^ ((pair >> 1) & (G / 2 - 1))));
    f = add2(f, add2(lo2(v), hi2(v)));
  }
  return f;
}

template <typename T, int L, bool REST, bool LOCAL>
__global__ void __launch_bounds__(kSelThreads, 4) k_sel_bwd(const SelArgs a) {
  using S = SelTile<L>;
  using W = BwdLane<L>;
  extern __shared__ __align__(16) char raw_shared[];
  SelBwdShared<T, L>& s = *reinterpret_cast<SelBwdShared<T, L>*>(raw_shared);
  const int bc = blockIdx.x / a.tiles;
  const S t(a, blockIdx.x - bc * a.tiles);
  const SelSpan sp = sel_span(a, bc);
  if (LOCAL && sp.c == 0) return;  // nothing is in front of the first
  const int last = (sp.rows - 1) / kSub * kSub;  // the last 16 rows' first
  const int size = start_copies<T, L, true>(a, t, s, sp.lo + last);
  request_copies(a, s, 0, sp.rows - last, size);
  const W lane(t);
  float2 A2[2], e[2] = {f2(0.f), f2(0.f)}, dsum = f2(0.f);
  lane.load(a.A, a.N, A2);
  A2[0] = mul2(A2[0], f2(kLog2e));
  A2[1] = mul2(A2[1], f2(kLog2e));
  const int64_t states = (int64_t)a.D * a.NP;
  if (!LOCAL && sp.c + 1 < a.chunks) lane.load_packed(a.carry + bc * states, a.NP, e);
  if (threadIdx.x < S::PAIRS) {
    s.par[0][threadIdx.x] = t.pair_of(a.bias);
    s.par[1][threadIdx.x] = t.pair_of(a.Dk);
  }
  s.sum_a.clear();
  s.sum_d.clear();
  SelSides side(a, sp, sp.rows - 1);
  bool whole = false, whole_dt = false;
  const float* keep = nullptr;
  int64_t out = 0;       // of the pair in the block's results
  float* to_part = nullptr;
  float2 dA[2] = {f2(0.f), f2(0.f)}, dd = f2(0.f), db = f2(0.f);
  int held = 0;          // blocks in these sums
  // what this thread adds up of the warps' dB and dC
  const int bc_v = threadIdx.x % (2 * S::NL), bc_row = threadIdx.x / (2 * S::NL);
  const int bc_n = bc_v % S::NL, bc_l = bc_n >> 1;
  const float* const from_bc =
      &s.bc[W::BLOCKS > 1 ? bc_l >> 3 : 0][bc_row][bc_v / S::NL][bc_n & 1][W::G < 8 ? bc_l : bc_l & 7];
  if constexpr (!LOCAL) {
    keep = a.saved + block_states(a, sp.b, sp.lo + last);
    out = (sp.lo + last + t.pr) * a.D + t.d0 + t.pc;
    to_part = a.part_bc + (((int64_t)t.tile * a.B * a.T + sp.lo + last + bc_row) * 2 + bc_v / S::NL) * a.N + bc_n;
    whole = t.template whole<T>(a.dx, a.D) && (!a.z || t.template whole<T>(a.dz, a.D));
    whole_dt = a.dt_f32 ? t.template whole<float>(a.ddt, a.D) : t.template whole<T>(a.ddt, a.D);
  }

  int at = 0;
  for (int r0 = last; r0 >= 0; r0 -= kSub, at ^= 1) {
    const SelRaw<T, L, true>& raw = s.raw[at];
    bool edge = side.lo >= r0 || side.hi <= r0 + kSub;
    const int rows = sp.rows - r0;  // from here on
    float most = 0.f;
    copies_done();
    __syncthreads();
    if (r0 > 0) request_copies(a, s, at ^ 1, kSub, size);
    float2 hs[kSub / kHeld][2];
    if constexpr (!LOCAL) {
      lane.load_packed(keep, a.NP, hs[0]);
      keep -= states;
    }
    const float2 bias = s.par[0][t.pc >> 1];
#pragma unroll
    for (int i = 0; i < S::PER; ++i) {
      const int row = t.pr + i * S::STEP;
      if (S::STEP > kSub && row >= kSub) break;
      const int p = row * S::CH + t.pc;
      float2 d = add2((a.dt_f32 ? pair_at(s.dt32.v[at] + p) : raw.dt(p)), bias);
      if (a.softplus) d = softplus2(d);
      if (row >= rows) d = f2(0.f);
      const float2 u = LOCAL ? d : mul2(d, raw.x(p));
      *reinterpret_cast<float4*>(&s.dd[row][t.pc]) = make_float4(d.x, u.x, d.y, u.y);
      float2 o = raw.dy(p);
      if (a.z) {
        const float2 z = raw.z(p);
        o = mul2(o, mul2(z, sigmoid2(z)));
      } else if constexpr (sizeof(T) == 4) {  // the one NaN that tf32_cut keeps
        if (o.x != o.x) o.x = __uint_as_float(0x7fffffffu);
        if (o.y != o.y) o.y = __uint_as_float(0x7fffffffu);
      }
      *reinterpret_cast<float2*>(&s.o[row][t.pc]) = o;
      if constexpr (REST) most += sizes2(u, o) + sizes2(d, f2(0.f));
    }
    if constexpr (!LOCAL) widen<T, L>(s.b, raw.vec);
    widen<T, L>(s.c, raw.vec + kSub * S::NL);
    if (edge) mark_edges(a, s.edges, sp.b, sp.lo + r0, sp.lo + sp.rows);
    edge = sync_or_mark<REST>(a, s.edges, !(most <= FLT_MAX), edge, sp, r0);
    if constexpr (LOCAL) {
      if (edge) bwd_rows_local<true, REST>(a, s, lane, A2, e, dsum);
      else bwd_rows_local<false, REST>(a, s, lane, A2, e, dsum);
    } else {
      // the states in front of every four rows
#pragma unroll
      for (int k = 1; k < kSub / kHeld; ++k) {
        float2 da[2], p[2];
        hs[k][0] = hs[k - 1][0];
        hs[k][1] = hs[k - 1][1];
#pragma unroll
        for (int r = (k - 1) * kHeld; r < k * kHeld; ++r) {
          BwdRow x;
          x.load(s, lane, r);
          if (edge) state_row<true, REST>(a, s, lane, r, x, A2, hs[k], da, p);
          else state_row<false, REST>(a, s, lane, r, x, A2, hs[k], da, p);
        }
      }
#pragma unroll 1
      for (int q = kHalf; q >= 0; q -= kHalf) {
#pragma unroll
        for (int k = kHalf / kHeld - 1; k >= 0; --k) {
          const float2 h[2] = {q ? hs[k + kHalf / kHeld][0] : hs[k][0], q ? hs[k + kHalf / kHeld][1] : hs[k][1]};
          if (edge) bwd_rows<true, REST>(a, s, lane, q + k * kHeld, A2, h, e, dA);
          else bwd_rows<false, REST>(a, s, lane, q + k * kHeld, A2, h, e, dA);
        }
        __syncthreads();
        const float2 bias = s.par[0][t.pc >> 1], skip = s.par[1][t.pc >> 1];
#pragma unroll
        for (int m = 0; m < S::PER_HALF; ++m) {
          const int j = t.pr + m * S::STEP;
          if (S::STEP > kHalf && j >= kHalf) break;
          const int row = q + j, p = row * S::CH + t.pc, pair = t.pc >> 1;
          if (row >= rows) break;
          const float2 sum[3] = {
              sum_pairs<W::G / 2>(reinterpret_cast<const float2*>(s.share_y[j] + pair * W::G), pair),
              sum_pairs<W::G>(s.share[0][j] + pair * W::G, pair),
              sum_pairs<W::G>(s.share[1][j] + pair * W::G, pair)};
          const float2 x = raw.x(p), pre = add2((a.dt_f32 ? pair_at(s.dt32.v[at] + p) : raw.dt(p)), bias);
          const float4 du = *reinterpret_cast<const float4*>(&s.dd[row][t.pc]);
          const float2 dt = make_float2(du.x, du.z);
          const float2 o = *reinterpret_cast<const float2*>(&s.o[row][t.pc]);
          float2 ddt = fma2(x, sum[1], mul2(sum[2], f2(kSelLn2)));
          if (a.softplus) ddt = mul2(ddt, sigmoid2(pre));
          const int64_t r = out + (q + m * S::STEP) * a.D;
          const float2 dx = mul2(dt, sum[1]);
          t.store_pair((T*)a.dx + r, whole, a.Dk ? fma2(skip, o, dx) : dx);
          if (a.dt_f32) t.store_pair((float*)a.ddt + r, whole_dt, ddt);
          else t.store_pair((T*)a.ddt + r, whole_dt, ddt);
          if (a.z) {
            const float2 z = raw.z(p), sig = sigmoid2(z), dy = raw.dy(p);
            // silu'(z) = sig + z sig (1 - sig)
            const float2 f = fma2(mul2(z, sig), add2(f2(1.f), neg2(sig)), sig);
            t.store_pair((T*)a.dz + r, whole, mul2(mul2(dy, a.Dk ? fma2(skip, x, sum[0]) : sum[0]), f));
          }
          dd = fma2(o, x, dd);
          db = add2(db, ddt);
        }
        // this CTA's share of dB and dC: a thread's state is the same for all rows
#pragma unroll
        for (int m = 0; m < S::BC_ROWS; ++m) {
          if (q + bc_row + m * S::BC_STEP >= rows || bc_n >= a.N) break;
          float f = 0.f;
#pragma unroll
          for (int w = 0; w < kSelWarps / W::BLOCKS; ++w)
#pragma unroll
            for (int k = 0; k < W::SETS; ++k)
              f += from_bc[(w * W::BLOCKS * kHalf + m * S::BC_STEP) * 32 + k * W::G];
          to_part[(q + m * S::BC_STEP) * 2 * a.N] = f;
        }
        if (q) __syncthreads();
      }
      out -= (int64_t)kSub * a.D;
      to_part -= kSub * 2 * a.N;
      if (++held == 16 || r0 == 0) {
        s.sum_a.add(dA[0], dA[1]);
        s.sum_d.add(dd, db);
        dA[0] = dA[1] = dd = db = f2(0.f);
        held = 0;
      }
    }
    if (edge && r0 > 0) side = SelSides(a, sp, r0 - 1);
  }
  if constexpr (LOCAL) {
    lane.store_packed(a.carry + bc * states, a.NP, e);
    if (lane.l == 0) {
      if (lane.on[0]) a.decay[(int64_t)bc * a.D + lane.d] = dsum.x;
      if (lane.on[1]) a.decay[(int64_t)bc * a.D + lane.d + 1] = dsum.y;
    }
  } else {
    const float4 f = s.sum_a.v[threadIdx.x];
    const float2 g[2] = {lo2(f), hi2(f)};
    lane.store_packed(a.part_a + bc * states, a.NP, g);
    __syncthreads();
    if (threadIdx.x < S::PAIRS) {  // threads PAIRS apart staged the same pair
      float4 f = s.sum_d.v[threadIdx.x];
#pragma unroll
      for (int i = 1; i < S::STEP; ++i) {
        const float4 v = s.sum_d.v[threadIdx.x + i * S::PAIRS];
        f = make_float4(f.x + v.x, f.y + v.y, f.z + v.z, f.w + v.w);
      }
      const int64_t n = (int64_t)a.B * a.chunks * a.D, to = (int64_t)bc * a.D + t.d0 + t.pc;
      if (t.pc < t.nch) {
        a.part_d[to] = f.x;
        a.part_d[n + to] = f.z;
      }
      if (t.pc + 1 < t.nch) {
        a.part_d[to + 1] = f.y;
        a.part_d[n + to + 1] = f.w;
      }
    }
  }
}

// dB and dC from the CTAs' shares, in their order.
template <typename T>
__global__ void __launch_bounds__(256) k_sel_vectors(const SelArgs a, T* dB, T* dC) {
  const int64_t rows = (int64_t)a.B * a.T, per = 2 * (int64_t)a.N;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // [G][row][2][N]
  if (i >= a.G * rows * per) return;
  const int64_t g = i / (rows * per), at = i - g * rows * per;
  const float* p = a.part_bc + g * a.tiles_per_group * rows * per + at;
  float s = 0.f;
#pragma unroll 8
  for (int k = 0; k < a.tiles_per_group; ++k) s += p[k * rows * per];
  const int64_t r = at / per;
  const int v = (int)(at - r * per), n = v % a.N;
  (v < a.N ? dB : dC)[(r * a.G + g) * a.N + n] = from_f<T>(s);
}

// dA, dD and ddt_bias from the chunks' shares.
__global__ void __launch_bounds__(256) k_sel_params(const SelArgs a, float* dA, float* dD, float* dbias) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t na = (int64_t)a.D * a.N, bc = (int64_t)a.B * a.chunks;
  double s = 0.;
  if (i < na) {
    const int64_t d = i / a.N, n = i - d * a.N;
    for (int64_t k = 0; k < bc; ++k) s += a.part_a[(k * a.D + d) * a.NP + n];
    dA[i] = (float)s;
  } else if (i < na + 2 * a.D) {
    const int64_t d = (i - na) % a.D;
    float* out = i - na < a.D ? dD : dbias;
    if (!out) return;
    const float* p = a.part_d + (i - na < a.D ? 0 : bc * a.D);
    for (int64_t k = 0; k < bc; ++k) s += p[k * a.D + d];
    out[d] = (float)s;
  }
}

// ---------------------------------------------------------------------------
// one token
// ---------------------------------------------------------------------------
__device__ __forceinline__ void load_four(const float* p, int N, int n0, bool vec, float2 (&h)[2]) {
  if (vec) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (n0 < N) v = *reinterpret_cast<const float4*>(p + n0);
    h[0] = make_float2(v.x, v.y);
    h[1] = make_float2(v.z, v.w);
  } else {
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = n0 + i < N ? p[n0 + i] : 0.f;
    h[0] = make_float2(f[0], f[1]);
    h[1] = make_float2(f[2], f[3]);
  }
}
__device__ __forceinline__ void store_four(float* p, int N, int n0, bool vec, const float2 (&h)[2]) {
  if (vec) {
    if (n0 < N) *reinterpret_cast<float4*>(p + n0) = make_float4(h[0].x, h[0].y, h[1].x, h[1].y);
  } else {
    const float f[4] = {h[0].x, h[0].y, h[1].x, h[1].y};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n0 + i < N) p[n0 + i] = f[i];
  }
}

// Every lane has four states of a channel.  What does not depend on the token's place
// in the pool is read first.  The time is that of short chains of reads: 64 tokens of
// 4096 channels of 16 states take 13.7 us (their states 5.5 us of traffic), 256 41.5 us
// at three quarters of the issue rate.  Two channels to a lane (half the instructions),
// four tokens to a CTA, and the next token's values on their way while one is worked
// on were no faster (45, 47 and 103 us for the 256, where this took 43).
template <typename T, int L>
__global__ void __launch_bounds__(kSelThreads) k_sel_step(const SelArgs a, float* state, int64_t stride,
                                                          int pool, const int32_t* idx) {
  const int64_t n = blockIdx.x;
  const int d = (int)(blockIdx.y + gridDim.y * blockIdx.z) * (kSelThreads / L) + threadIdx.x / L, l = threadIdx.x % L;
  const unsigned lanes = __ballot_sync(0xffffffffu, d < a.D);
  if (d >= a.D) return;  // all of a channel's lanes
  const int slot = idx ? idx[n] : (int)n;
  const bool vec = (a.N & 3) == 0 && ((reinterpret_cast<uintptr_t>(state) | (stride * 4) |
                                       reinterpret_cast<uintptr_t>(a.A)) & 15) == 0;
  const bool vec_bc = (a.N & 3) == 0 && ((reinterpret_cast<uintptr_t>(a.Bv) | reinterpret_cast<uintptr_t>(a.Cv) |
                                          ((a.ldb | a.ldc) * sizeof(T))) & (4 * sizeof(T) - 1)) == 0;
  const int left = a.N - 4 * l, at = (a.G > 1 ? d / (a.D / a.G) * a.N : 0) + 4 * l;
  const T* pb = (const T*)a.Bv + n * a.ldb + at;
  const T* pc = (const T*)a.Cv + n * a.ldc + at;
  const Raw<T, 4> B = vec_bc ? load_group<T, 4, true>(pb, left) : load_group<T, 4, false>(pb, left);
  const Raw<T, 4> C = vec_bc ? load_group<T, 4, true>(pc, left) : load_group<T, 4, false>(pc, left);
  const float x = to_f<T>(((const T*)a.x)[n * a.ldx + d]);
  float dt = a.dt_f32 ? ((const float*)a.dt)[n * a.lddt + d] : to_f<T>(((const T*)a.dt)[n * a.lddt + d]);
  const float z = a.z ? to_f<T>(((const T*)a.z)[n * a.ldz + d]) : 0.f;
  float2 A2[2], h[2];
  load_four(a.A + (int64_t)d * a.N, a.N, 4 * l, vec, A2);
  T* y = (T*)a.y + n * a.D + d;
  if (slot < 0 || slot >= pool) {
    if (l == 0) *y = from_f<T>(0.f);
    return;
  }
  float* p = state + slot * stride + (int64_t)d * a.N;
  load_four(p, a.N, 4 * l, vec, h);
  if (a.bias) dt += a.bias[d];
  if (a.softplus) dt = softplus_f(dt);
  float out = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 b = make_float2(raw_get(B, 2 * i), raw_get(B, 2 * i + 1));
    const float2 c = make_float2(raw_get(C, 2 * i), raw_get(C, 2 * i + 1));
    h[i] = fma2(exp2_2(mul2(f2(dt), mul2(A2[i], f2(kLog2e)))), h[i], mul2(f2(dt * x), b));
    if (left < 4) {  // beyond the last: infinity times zero is NaN
      if (2 * i >= left) h[i].x = 0.f;
      if (2 * i + 1 >= left) h[i].y = 0.f;
    }
    const float2 o = mul2(h[i], c);
    out += o.x + o.y;
  }
  store_four(p, a.N, 4 * l, vec, h);
#pragma unroll
  for (int o = L / 2; o > 0; o /= 2) out += __shfl_xor_sync(lanes, out, o);
  if (l == 0) {
    if (a.Dk) out = fmaf(a.Dk[d], x, out);
    if (a.z) out *= z * sigmoid_f(z);
    *y = from_f<T>(out);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int lanes_of(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

int check_sel(const gdn2_selective_problem* p, const char* fn) {
  if (!p) return fail(GDN2_ERR_INVALID, "%s: null problem", fn);
  if (p->B < 0 || p->T < 0 || p->D <= 0 || p->N <= 0 || p->G <= 0 || p->n_seqs < 0)
    return fail(GDN2_ERR_INVALID, "%s: needs B, T, n_seqs >= 0 and D, N, G > 0", fn);
  if (p->D % p->G)
    return fail(GDN2_ERR_INVALID, "%s: %d channels do not divide into %d groups", fn, p->D, p->G);
  if (p->N > 64) return fail(GDN2_ERR_UNSUPPORTED, "%s: up to 64 states are supported (got %d)", fn, p->N);
  if (!dtype_valid(p->dtype) || !dtype_valid(p->dt_dtype))
    return fail(GDN2_ERR_INVALID, "%s: unknown dtype %d / %d", fn, p->dtype, p->dt_dtype);
  if (p->dt_dtype != p->dtype && p->dt_dtype != GDN2_DTYPE_F32)
    return fail(GDN2_ERR_UNSUPPORTED, "%s: dt must be fp32 or have x's dtype", fn);
  if (p->cu_seqlens ? p->B != 1 : p->n_seqs != p->B)
    return fail(GDN2_ERR_INVALID, "%s: packed sequences need B = 1, others n_seqs = B", fn);
  const int64_t least = (int64_t)p->G * p->N, most = (int64_t)1 << 22;
  if (least > most || p->D > most) return fail(GDN2_ERR_UNSUPPORTED, "%s: rows are too wide", fn);
  const int64_t wide[] = {p->ld_x, p->ld_dt, p->ld_z, p->ld_dy};
  for (int64_t ld : wide)
    if (ld < p->D || ld > most)
      return fail(GDN2_ERR_INVALID, "%s: row strides must be D .. 2^22 elements (got %lld)", fn, (long long)ld);
  if (p->ld_b < least || p->ld_b > most || p->ld_c < least || p->ld_c > most)
    return fail(GDN2_ERR_INVALID, "%s: row strides of B and C must be G N .. 2^22 elements", fn);
  if (p->B && p->T > ((int64_t)1 << 40) / p->B)
    return fail(GDN2_ERR_UNSUPPORTED, "%s: too many rows", fn);
  if (p->T > 2147483647LL)
    return fail(GDN2_ERR_UNSUPPORTED, "%s: sequences are up to 2^31 - 1 rows", fn);
  if (p->T > 0 && p->B > 0 && p->n_seqs == 0)
    return fail(GDN2_ERR_INVALID, "%s: rows without a sequence in cu_seqlens", fn);
  return GDN2_OK;
}

struct SelPlan {
  int64_t chunk, subs;
  int chunks, tiles_per_group, tiles;
};

// Cuts the time axis into chunks of whole 16 rows where the CTAs of the channels
// and batch entries alone are fewer than two for each of 148 SMs (the extra
// launches cost two thirds of the forward and a fifth of the backward once more:
// 207 + 10 of 525 us and 228 + 10 of 1384 us at 65536 tokens x 512 channels); then as
// many chunks as give four for each, of 64 rows at least.  Both sides of the border, n x
// 8192 tokens x 2048 channels x 16 states, forward and backward: 256 CTAs 4.09 ms cut
// and 4.50 whole, 320 CTAs 5.50 and 5.31 (forward alone 1.00 and 0.96, 1.26 and 1.13).
SelPlan sel_plan(const gdn2_selective_problem* p) {
  SelPlan q;
  const int ch = kSelThreads / lanes_of(p->N);
  q.tiles_per_group = (p->D / p->G + ch - 1) / ch;
  q.tiles = q.tiles_per_group * p->G;
  q.subs = (p->T + kSub - 1) / kSub;
  q.chunk = std::max<int64_t>(q.subs, 1) * kSub;
  const int64_t ctas = (int64_t)q.tiles * std::max(p->B, 1);
  if (ctas < 2 * 148) {
    const int64_t want = (4 * 148 + ctas - 1) / ctas;
    const int64_t len = std::max<int64_t>((q.subs + want - 1) / want, 4);
    q.chunk = std::min(q.chunk, len * kSub);
  }
  q.chunks = (int)std::max<int64_t>((p->T + q.chunk - 1) / q.chunk, 1);
  return q;
}

struct SelWork {  // bytes of the workspace's sections
  size_t carry, decay, part_bc, part_a, part_d, total;
};

SelWork sel_work(const gdn2_selective_problem* p, const SelPlan& q, bool backward) {
  SelWork w{};
  const size_t np = (size_t)((p->N + 3) / 4 * 4), bc = (size_t)p->B * q.chunks;
  size_t off = 0;
  auto take = [&](size_t n) { const size_t at = off; off = align256(off + n * sizeof(float)); return at; };
  w.carry = take(q.chunks > 1 ? bc * p->D * np : 0);
  w.decay = take(q.chunks > 1 ? bc * p->D : 0);
  if (backward) {
    w.part_bc = take((size_t)q.tiles * p->B * p->T * 2 * p->N);
    w.part_a = take(bc * p->D * np);
    w.part_d = take(2 * bc * p->D);
  }
  w.total = off;
  return w;
}

SelArgs sel_args(const gdn2_selective_problem* p, const SelPlan& q) {
  SelArgs a{};
  a.B = p->B; a.D = p->D; a.G = p->G; a.N = p->N; a.NP = (p->N + 3) / 4 * 4; a.n_seqs = p->n_seqs;
  a.T = p->T; a.cu = p->cu_seqlens;
  a.ldx = p->ld_x; a.lddt = p->ld_dt; a.ldz = p->ld_z; a.ldb = p->ld_b; a.ldc = p->ld_c; a.lddy = p->ld_dy;
  a.dt_f32 = p->dt_dtype == GDN2_DTYPE_F32 && p->dtype != GDN2_DTYPE_F32; a.softplus = p->dt_softplus != 0;
  a.chunk = q.chunk; a.subs = q.subs; a.chunks = q.chunks;
  a.tiles_per_group = q.tiles_per_group; a.tiles = q.tiles;
  return a;
}

// The tensors that come in by rows; dy NULL in the forward.
void sel_sources(SelArgs& a, const void* x, const void* dy, const void* z, const void* dt, const void* Bv,
                 const void* Cv) {
  int k = 0;
  a.tok[k++] = SelSource{x, a.ldx};
  if (dy) a.tok[k++] = SelSource{dy, a.lddy};
  a.tok[k++] = SelSource{z, a.ldz};
  a.tok[k++] = SelSource{a.dt_f32 ? nullptr : dt, a.lddt};
  a.dt32 = SelSource{a.dt_f32 ? dt : nullptr, a.lddt};
  a.vec[0] = SelSource{Bv, a.ldb};
  a.vec[1] = SelSource{Cv, a.ldc};
}

// f(T{}, integral_constant<L>)
template <typename F> cudaError_t with_lanes(int dtype, int N, F&& f) {
  return with_dtype(dtype, [&](auto t) {
    switch (lanes_of(N)) {
      case 2: return f(t, std::integral_constant<int, 2>{});
      case 4: return f(t, std::integral_constant<int, 4>{});
      case 8: return f(t, std::integral_constant<int, 8>{});
      default: return f(t, std::integral_constant<int, 16>{});
    }
  });
}
// f(T{}, integral_constant<L>, bool_constant<REST>): whether lanes hold states beyond the
// last, which takes a look at every value (8 x 4096 x 2048 x 16, which does not need it,
// 3.37 ms with it and 3.22 without).
template <typename F> cudaError_t with_lanes_and_rest(int dtype, int N, F&& f) {
  return with_lanes(dtype, N, [&](auto t, auto lanes) {
    return N != 4 * lanes_of(N) ? f(t, lanes, std::true_type{}) : f(t, lanes, std::false_type{});
  });
}

// States of sequences without a token pass through: copied for all, where there
// can be such, in front of the kernels that write the others'.
cudaError_t pass_states(const gdn2_selective_problem* p, const float* from, float* to, cudaStream_t st) {
  const bool some = p->cu_seqlens || p->T == 0;
  const size_t bytes = (size_t)p->n_seqs * p->D * p->N * sizeof(float);
  if (!to || !some || !bytes) return cudaSuccess;
  return from ? cudaMemcpyAsync(to, from, bytes, cudaMemcpyDeviceToDevice, st)
              : cudaMemsetAsync(to, 0, bytes, st);
}

unsigned carry_grid(const SelArgs& a) {
  return (unsigned)((int64_t)a.B * (((int64_t)a.D * a.NP + 255) / 256));
}

template <typename K> cudaError_t allow_shared(K local, K full, int bytes) {
  const cudaError_t e = cudaFuncSetAttribute(full, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  return e == cudaSuccess ? cudaFuncSetAttribute(local, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) : e;
}

// What the element accesses of a call need: token tensors, dt, fp32 arrays.
template <typename... P>
int check_elements(const gdn2_selective_problem* p, const char* fn, const void* dt, const void* ddt, P... tok) {
  if (all_aligned(dtype_size(p->dtype), tok...) && all_aligned(dtype_size(p->dt_dtype), dt, ddt)) return GDN2_OK;
  return fail(GDN2_ERR_INVALID, "%s: a tensor is not aligned to its elements", fn);
}
template <typename... P> int check_words(const char* fn, P... f32) {
  return all_aligned(4, f32...) ? GDN2_OK : fail(GDN2_ERR_INVALID, "%s: an fp32 array is not aligned to 4 bytes", fn);
}

bool too_many(int64_t ctas) { return ctas > 2147483647LL; }

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

size_t gdn2_selective_saved_bytes(const gdn2_selective_problem* p) {
  if (check_sel(p, "gdn2_selective_saved_bytes")) return 0;
  const SelPlan q = sel_plan(p);
  return (size_t)p->B * q.subs * p->D * ((p->N + 3) / 4 * 4) * sizeof(float);
}

size_t gdn2_selective_workspace_bytes(const gdn2_selective_problem* p, int32_t backward) {
  if (check_sel(p, "gdn2_selective_workspace_bytes")) return 0;
  return sel_work(p, sel_plan(p), backward != 0).total;
}

int gdn2_selective_fwd(const gdn2_selective_problem* p, const void* x, const void* dt, const float* A,
                       const void* Bv, const void* Cv, const float* D, const void* z, const float* dt_bias,
                       const float* h0, void* y, float* ht, float* saved, void* workspace,
                       size_t workspace_bytes, void* stream) {
  const char* fn = "gdn2_selective_fwd";
  const int rc = check_sel(p, fn);
  if (rc) return rc;
  const SelPlan q = sel_plan(p);
  const SelWork w = sel_work(p, q, false);
  const cudaStream_t st = (cudaStream_t)stream;
  const int64_t ctas = (int64_t)p->B * q.chunks * q.tiles;
  if (too_many(ctas) || too_many((int64_t)p->B * q.chunks))
    return fail(GDN2_ERR_UNSUPPORTED, "%s: too many sequences", fn);
  const bool some = p->B > 0 && p->T > 0;
  if (some && (!x || !dt || !A || !Bv || !Cv || !y)) return fail(GDN2_ERR_INVALID, "%s: null pointer", fn);
  if (some && w.total && (!workspace || workspace_bytes < w.total))
    return fail(GDN2_ERR_WORKSPACE, "%s: needs a workspace of %zu bytes", fn, w.total);
  if (!aligned_to(workspace, 16) || !aligned_to(saved, 16))
    return fail(GDN2_ERR_INVALID, "%s: workspace and saved must start on 16-byte boundaries", fn);
  if (check_elements(p, fn, dt, nullptr, x, Bv, Cv, z, y) || check_words(fn, A, D, dt_bias, h0, ht, p->cu_seqlens))
    return GDN2_ERR_INVALID;
  cudaError_t e = pass_states(p, h0, ht, st);
  if (e != cudaSuccess) return cuda_status(e, fn);
  if (!some) return GDN2_OK;
  SelArgs a = sel_args(p, q);
  sel_sources(a, x, nullptr, z, dt, Bv, Cv);
  a.A = A; a.Dk = D; a.z = z; a.bias = dt_bias; a.h0 = h0;
  a.y = y; a.ht = ht; a.saved = saved;
  if (w.total) {
    a.carry = (float*)((char*)workspace + w.carry);
    a.decay = (float*)((char*)workspace + w.decay);
  }
  return cuda_status(with_lanes_and_rest(p->dtype, p->N, [&](auto t, auto lanes, auto rest) {
    using T = decltype(t);
    constexpr int L = decltype(lanes)::value;
    constexpr int most = (int)sizeof(SelFwdShared<T, L>);
    const int smem = a.dt_f32 ? most : SelFwdShared<T, L>::without_dt32();
    constexpr bool REST = decltype(rest)::value;
    auto local = k_sel_fwd<T, L, REST, true>;
    auto full = k_sel_fwd<T, L, REST, false>;
    cudaError_t e = allow_shared(local, full, most);
    if (e != cudaSuccess) return e;
    if (q.chunks > 1) {
      SelArgs b = a;  // the states need no z and no C
      b.tok[1].p = b.vec[1].p = nullptr;
      local<<<(unsigned)ctas, kSelThreads, smem, st>>>(b);
      k_sel_carry<false><<<carry_grid(a), 256, 0, st>>>(a);
    }
    full<<<(unsigned)ctas, kSelThreads, smem, st>>>(a);
    return cudaGetLastError();
  }), fn);
}

int gdn2_selective_bwd(const gdn2_selective_problem* p, const void* x, const void* dt, const float* A,
                       const void* Bv, const void* Cv, const float* D, const void* z, const float* dt_bias,
                       const float* h0, const float* saved, const void* dy, const float* dht, void* dx,
                       void* ddt, float* dA, void* dB, void* dC, float* dD, void* dz, float* ddt_bias,
                       float* dh0, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "gdn2_selective_bwd";
  const int rc = check_sel(p, fn);
  if (rc) return rc;
  const SelPlan q = sel_plan(p);
  const SelWork w = sel_work(p, q, true);
  const cudaStream_t st = (cudaStream_t)stream;
  const int64_t ctas = (int64_t)p->B * q.chunks * q.tiles, rows = (int64_t)p->B * p->T;
  const int64_t values = rows * p->G * 2 * p->N;
  if (too_many(ctas) || too_many((int64_t)p->B * q.chunks) || too_many(values / 256 + 1))
    return fail(GDN2_ERR_UNSUPPORTED, "%s: too many sequences or rows", fn);
  const bool some = rows > 0;
  if (some && (!x || !dt || !A || !Bv || !Cv || !saved || !dy || !dx || !ddt || !dA || !dB || !dC || (z && !dz)))
    return fail(GDN2_ERR_INVALID, "%s: null pointer", fn);
  if (some && (!workspace || workspace_bytes < w.total))
    return fail(GDN2_ERR_WORKSPACE, "%s: needs a workspace of %zu bytes", fn, w.total);
  if (!aligned_to(workspace, 16) || !aligned_to(saved, 16))
    return fail(GDN2_ERR_INVALID, "%s: workspace and saved must start on 16-byte boundaries", fn);
  if (check_elements(p, fn, dt, ddt, x, Bv, Cv, z, dy, dx, dB, dC, dz) ||
      check_words(fn, A, D, dt_bias, h0, dht, dA, dD, ddt_bias, dh0, p->cu_seqlens))
    return GDN2_ERR_INVALID;
  cudaError_t e = pass_states(p, dht, dh0, st);
  if (e != cudaSuccess) return cuda_status(e, fn);
  if (!some) {
    if (dA) e = cudaMemsetAsync(dA, 0, (size_t)p->D * p->N * sizeof(float), st);
    if (e == cudaSuccess && dD) e = cudaMemsetAsync(dD, 0, (size_t)p->D * sizeof(float), st);
    if (e == cudaSuccess && ddt_bias) e = cudaMemsetAsync(ddt_bias, 0, (size_t)p->D * sizeof(float), st);
    return cuda_status(e, fn);
  }
  SelArgs a = sel_args(p, q);
  sel_sources(a, x, dy, z, dt, Bv, Cv);
  a.A = A; a.Dk = D; a.z = z; a.bias = dt_bias; a.h0 = h0;
  a.saved = const_cast<float*>(saved); a.dht = dht;
  a.dx = dx; a.ddt = ddt; a.dz = dz; a.dh0 = dh0;
  char* ws = (char*)workspace;
  a.carry = (float*)(ws + w.carry); a.decay = (float*)(ws + w.decay);
  a.part_bc = (float*)(ws + w.part_bc); a.part_a = (float*)(ws + w.part_a); a.part_d = (float*)(ws + w.part_d);
  return cuda_status(with_lanes_and_rest(p->dtype, p->N, [&](auto t, auto lanes, auto rest) {
    using T = decltype(t);
    constexpr int L = decltype(lanes)::value;
    constexpr int most = (int)sizeof(SelBwdShared<T, L>);
    const int smem = a.dt_f32 ? most : SelBwdShared<T, L>::without_dt32();
    constexpr bool REST = decltype(rest)::value;
    auto local = k_sel_bwd<T, L, REST, true>;
    auto full = k_sel_bwd<T, L, REST, false>;
    cudaError_t e = allow_shared(local, full, most);
    if (e != cudaSuccess) return e;
    if (q.chunks > 1) {
      SelArgs b = a;  // the states' gradients need no x and no B
      b.tok[0].p = b.vec[0].p = nullptr;
      local<<<(unsigned)ctas, kSelThreads, smem, st>>>(b);
      k_sel_carry<true><<<carry_grid(a), 256, 0, st>>>(a);
    }
    full<<<(unsigned)ctas, kSelThreads, smem, st>>>(a);
    k_sel_vectors<T><<<(unsigned)((values + 255) / 256), 256, 0, st>>>(a, (T*)dB, (T*)dC);
    const int64_t n = (int64_t)a.D * (a.N + 2);
    k_sel_params<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a, dA, dD, ddt_bias);
    return cudaGetLastError();
  }), fn);
}

int gdn2_selective_step(const gdn2_selective_problem* p, const void* x, const void* dt, const float* A,
                        const void* Bv, const void* Cv, const float* D, const void* z, const float* dt_bias,
                        float* state, int64_t state_stride, int32_t pool, const int32_t* state_indices,
                        void* y, void* stream) {
  const char* fn = "gdn2_selective_step";
  const int rc = check_sel(p, fn);
  if (rc) return rc;
  if (p->T != 1 || p->cu_seqlens)
    return fail(GDN2_ERR_INVALID, "%s: takes one token for each of B sequences", fn);
  if (p->B == 0) return GDN2_OK;
  if (!x || !dt || !A || !Bv || !Cv || !state || !y) return fail(GDN2_ERR_INVALID, "%s: null pointer", fn);
  if (state_stride < (int64_t)p->D * p->N)
    return fail(GDN2_ERR_INVALID, "%s: a state takes %lld values, the stride is %lld", fn,
                (long long)p->D * p->N, (long long)state_stride);
  if (pool < 0 || (!state_indices && pool < p->B))
    return fail(GDN2_ERR_INVALID, "%s: %d sequences need as many states (got %d)", fn, p->B, pool);
  if (check_elements(p, fn, dt, nullptr, x, Bv, Cv, z, y) || check_words(fn, A, D, dt_bias, state, state_indices))
    return GDN2_ERR_INVALID;
  const int ch = kSelThreads / lanes_of(p->N), tiles = (p->D + ch - 1) / ch;
  const unsigned most = 65535u, deep = (tiles + most - 1) / most;
  const dim3 grid((unsigned)p->B, (tiles + deep - 1) / deep, deep);
  SelArgs a = sel_args(p, sel_plan(p));
  a.x = x; a.dt = dt; a.A = A; a.Bv = Bv; a.Cv = Cv; a.Dk = D; a.z = z; a.bias = dt_bias; a.y = y;
  const cudaStream_t st = (cudaStream_t)stream;
  return cuda_status(with_lanes(p->dtype, p->N, [&](auto t, auto lanes) {
    k_sel_step<decltype(t), decltype(lanes)::value>
        <<<grid, kSelThreads, 0, st>>>(a, state, state_stride, pool, state_indices);
    return cudaGetLastError();
  }), fn);
}

}  // extern "C"
