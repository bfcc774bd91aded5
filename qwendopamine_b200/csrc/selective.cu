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
// A channel takes L lanes with four states each, in registers from row to row;
// what a row needs of a channel (dt, dt x, o) and of a group (B, C) is formed
// once, 16 rows at a time, in shared memory.  Sums over a channel's lanes, and
// over a warp's channels for dB and dC, travel transposed: each step halves both
// the lanes that are apart and the values that a lane still holds.
//
// The time axis is cut where channels and sequences alone leave SMs idle: each
// chunk's end state is formed from a zero start, a second launch carries them from
// chunk to chunk (a chunk's decay is exp(A sum dt)), and the third starts every
// chunk from its state.  The backward does the same with e.  The forward keeps the
// state in front of every 16 rows; the backward forms the 16 rows' states again,
// eight at a time in registers.  dB and dC are summed over a CTA's channels in
// shared memory and over the CTAs by a launch of their own: every sum has a fixed
// order, equal inputs give equal bits.
#include "mma16.cuh"
#include "op_util.cuh"

#include <algorithm>

namespace gdn2 {
namespace {

constexpr int kSelThreads = 128;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSub = 16;   // rows of a block: one kept state for each
constexpr int kHalf = 8;   // rows whose states the backward holds at a time
constexpr float kSelLn2 = 0.6931471805599453f;

struct SelArgs {
  int B, D, G, N, NP, n_seqs;   // NP: N rounded up to 4
  int64_t T;
  const int32_t* cu;
  const void *x, *dt, *z, *Bv, *Cv;
  int64_t ldx, lddt, ldz, ldb, ldc;
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
  const void* dy;
  int64_t lddy;
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
// ln(1 + e^v) without loss for very negative v
__device__ __forceinline__ float softplus_f(float v) { return fmaxf(v, 0.f) + log1pf(expf(-fabsf(v))); }

// 1 / (1 + e^-v): exact functions where results are fp32, the hardware's where
// they are rounded to 16 bits (its errors are about 2^-21)
template <typename T> __device__ __forceinline__ float sigmoid_of(float v) {
  if constexpr (sizeof(T) == 4) return 1.f / (1.f + expf(-v));
  else return __fdividef(1.f, 1.f + __expf(-v));
}

// ---------------------------------------------------------------------------
// geometry
// ---------------------------------------------------------------------------
struct SelSpan {  // rows of a chunk, and the sequences they belong to
  int64_t lo, hi;
  int b, c;
};

__device__ __forceinline__ SelSpan sel_span(const SelArgs& a, int bc) {
  SelSpan s;
  s.b = bc / a.chunks;
  s.c = bc - s.b * a.chunks;
  const int64_t first = (int64_t)s.b * a.T;
  s.lo = first + s.c * a.chunk;
  s.hi = min(s.lo + a.chunk, first + a.T);
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

// Sequences that begin and end at rows r0 .. r0 + 15 (-1: none), by 16 threads.
struct SelEdges {
  int begin[kSub], end[kSub];
};
__device__ __forceinline__ void mark_edges(const SelArgs& a, SelEdges& m, int b, int64_t r0, int64_t hi) {
  if (threadIdx.x < kSub) {
    const int64_t r = r0 + threadIdx.x;
    int bn = -1, en = -1;
    if (r < hi) {
      const SelSeq s = seq_of(a, b, r);
      if (r == s.lo) bn = s.n;
      if (r + 1 == s.hi) en = s.n;
    }
    m.begin[threadIdx.x] = bn;
    m.end[threadIdx.x] = en;
  }
}

// Four states of a channel in an [..][D][N] array.
__device__ __forceinline__ void load_states(const float* p, int N, int n0, bool on, float2 (&h)[2]) {
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = p && on && n0 + i < N ? p[n0 + i] : 0.f;
  h[0] = make_float2(f[0], f[1]);
  h[1] = make_float2(f[2], f[3]);
}
__device__ __forceinline__ void store_states(float* p, int N, int n0, bool on, const float2 (&h)[2]) {
  const float f[4] = {h[0].x, h[0].y, h[1].x, h[1].y};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (on && n0 + i < N) p[n0 + i] = f[i];
}
// The same in an [..][D][NP] array of this file: one vector.
__device__ __forceinline__ void load_states4(const float* p, int NP, int n0, bool on, float2 (&h)[2]) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (on && n0 < NP) v = *reinterpret_cast<const float4*>(p + n0);
  h[0] = make_float2(v.x, v.y);
  h[1] = make_float2(v.z, v.w);
}
__device__ __forceinline__ void store_states4(float* p, int NP, int n0, bool on, const float2 (&h)[2]) {
  if (on && n0 < NP) *reinterpret_cast<float4*>(p + n0) = make_float4(h[0].x, h[0].y, h[1].x, h[1].y);
}

// R values of each of L lanes (neighbours) summed over the lanes: lane l gets
// the sum of value l % R.
template <int L, int R> __device__ __forceinline__ float sum_transposed(float (&v)[R], int l) {
#pragma unroll
  for (int o = R / 2; o > 0; o /= 2)
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const bool up = l & o;
      const float keep = up ? v[i + o] : v[i], send = up ? v[i] : v[i + o];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
#pragma unroll
  for (int o = R; o < L; o *= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  return v[0];
}

__device__ __forceinline__ float2 decay2(float dt, float2 A2) {
  const float2 y = mul2(f2(dt), A2);
  return make_float2(fast_exp2(y.x), fast_exp2(y.y));
}

// A running sum that keeps what rounding takes away.
struct LongSum {
  float hi = 0.f, lo = 0.f;
  __device__ __forceinline__ void add(float x) {
    const float s = hi + x, b = s - hi;
    lo += (hi - (s - b)) + (x - b);
    hi = s;
  }
  __device__ __forceinline__ float get() const { return hi + lo; }
};

template <typename T, int L> struct SelTile {
  static constexpr int CH = kSelThreads / L;  // channels of a CTA
  static constexpr int NL = 4 * L;            // states, padded
  static constexpr int PER = kSub / L;        // rows of a thread when it stages
  static constexpr int PAD = CH + 32 / L;     // row stride of what lanes write by row
  static constexpr int VPT = kSub * NL / kSelThreads;  // B (or C) values a thread stages
  int d0, nch, g, tile;
  int l, mc, d;       // as a lane: which of the channel's, which channel
  bool on;
  int sc, sr;         // when staging: channel, first row
  __device__ __forceinline__ SelTile(const SelArgs& a, int tile_) : tile(tile_) {
    g = tile / a.tiles_per_group;
    const int dg = a.D / a.G, at = (tile - g * a.tiles_per_group) * CH;
    d0 = g * dg + at;
    nch = min(CH, dg - at);
    l = threadIdx.x % L;
    mc = threadIdx.x / L;
    on = mc < nch;
    d = d0 + mc;
    sc = threadIdx.x % CH;
    sr = threadIdx.x / CH;
  }
  __device__ __forceinline__ void load_rates(const SelArgs& a, float2 (&A2)[2]) const {
    load_states(a.A + (int64_t)d * a.N, a.N, 4 * l, on, A2);
    A2[0] = mul2(A2[0], f2(kLog2e));
    A2[1] = mul2(A2[1], f2(kLog2e));
  }
  // B or C of 16 rows, zero where there is no state or row
  __device__ __forceinline__ void load_vectors(const SelArgs& a, const void* p, int64_t ld, int64_t r0,
                                               int64_t hi, float (&v)[VPT]) const {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int idx = threadIdx.x + i * kSelThreads, n = idx % NL;
      const int64_t r = r0 + idx / NL;
      v[i] = n < a.N && r < hi ? to_f<T>(((const T*)p)[r * ld + g * a.N + n]) : 0.f;
    }
  }
  __device__ __forceinline__ void put_vectors(float* s, const float (&v)[VPT]) const {
#pragma unroll
    for (int i = 0; i < VPT; ++i) s[threadIdx.x + i * kSelThreads] = v[i];
  }
  // a token tensor's values of this thread's channel and rows
  __device__ __forceinline__ void load_tokens(const void* p, bool f32, int64_t ld, int64_t r0, int64_t hi,
                                              float (&v)[PER]) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int64_t r = r0 + sr + L * i;
      const int64_t at = r * ld + d0 + sc;
      v[i] = 0.f;
      if (r < hi && sc < nch) v[i] = f32 ? ((const float*)p)[at] : to_f<T>(((const T*)p)[at]);
    }
  }
};

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
template <typename T, int L> struct SelFwdShared {
  using S = SelTile<T, L>;
  alignas(16) float b[kSub * S::NL];
  alignas(16) float c[kSub * S::NL];
  float2 dd[kSub][S::CH];       // dt, dt x
  float y[kSub][S::PAD];
  SelEdges edges;
};

// 16 rows of one lane's states; LOCAL: only the states.
template <typename T, int L, bool LOCAL, bool EDGE>
__device__ __forceinline__ void fwd_rows(const SelArgs& a, SelFwdShared<T, L>& s, const SelTile<T, L>& t,
                                         const float2 (&A2)[2], float2 (&h)[2], float& dsum) {
  using S = SelTile<T, L>;
#pragma unroll 1
  for (int q = 0; q < kSub; q += L) {
    float v[L];
#pragma unroll
    for (int j = 0; j < L; ++j) {
      const int r = q + j;
      const float2 dd = s.dd[r][t.mc];
      const float4 B = *reinterpret_cast<const float4*>(s.b + r * S::NL + 4 * t.l);
      if constexpr (EDGE) {
        const int n = s.edges.begin[r];
        if (n >= 0) {
          load_states(a.h0 ? a.h0 + ((int64_t)n * a.D + t.d) * a.N : nullptr, a.N, 4 * t.l, t.on, h);
        }
      }
      h[0] = fma2(decay2(dd.x, A2[0]), h[0], mul2(f2(dd.y), make_float2(B.x, B.y)));
      h[1] = fma2(decay2(dd.x, A2[1]), h[1], mul2(f2(dd.y), make_float2(B.z, B.w)));
      if constexpr (LOCAL) {
        dsum += dd.x;
      } else {
        const float4 C = *reinterpret_cast<const float4*>(s.c + r * S::NL + 4 * t.l);
        const float2 o = fma2(h[0], make_float2(C.x, C.y), mul2(h[1], make_float2(C.z, C.w)));
        v[j] = o.x + o.y;
        if constexpr (EDGE) {
          const int n = s.edges.end[r];
          if (n >= 0 && a.ht) store_states(a.ht + ((int64_t)n * a.D + t.d) * a.N, a.N, 4 * t.l, t.on, h);
        }
      }
    }
    if constexpr (!LOCAL) s.y[q + t.l][t.mc] = sum_transposed<L, L>(v, t.l);
  }
}

template <typename T, int L, bool LOCAL>
__global__ void __launch_bounds__(kSelThreads) k_sel_fwd(const SelArgs a) {
  using S = SelTile<T, L>;
  __shared__ SelFwdShared<T, L> s;
  const int bc = blockIdx.x / a.tiles;
  const S t(a, blockIdx.x - bc * a.tiles);
  const SelSpan sp = sel_span(a, bc);
  if (LOCAL && sp.c + 1 == a.chunks) return;  // nothing follows the last
  float2 A2[2], h[2];
  t.load_rates(a, A2);
  float dsum = 0.f;
  if (LOCAL || sp.c == 0) h[0] = h[1] = f2(0.f);
  else load_states4(a.carry + ((int64_t)bc * a.D + t.d) * a.NP, a.NP, 4 * t.l, t.on, h);
  const float bias = a.bias && t.sc < t.nch ? a.bias[t.d0 + t.sc] : 0.f;
  const float skip = a.Dk && t.sc < t.nch ? a.Dk[t.d0 + t.sc] : 0.f;
  SelSeq seq = seq_of(a, sp.b, sp.lo);

  float x[S::PER], dt[S::PER], z[S::PER], vb[S::VPT], vc[S::VPT];
  auto load = [&](int64_t r0) {
    t.load_tokens(a.x, false, a.ldx, r0, sp.hi, x);
    t.load_tokens(a.dt, a.dt_f32, a.lddt, r0, sp.hi, dt);
    t.load_vectors(a, a.Bv, a.ldb, r0, sp.hi, vb);
    if constexpr (!LOCAL) {
      if (a.z) t.load_tokens(a.z, false, a.ldz, r0, sp.hi, z);
      t.load_vectors(a, a.Cv, a.ldc, r0, sp.hi, vc);
    }
  };
  load(sp.lo);
  for (int64_t r0 = sp.lo; r0 < sp.hi; r0 += kSub) {
    const bool edge = seq.lo == r0 || seq.hi <= r0 + kSub;
    float x1[S::PER], z1[S::PER];
#pragma unroll
    for (int i = 0; i < S::PER; ++i) {
      float d = dt[i] + bias;
      if (a.softplus) d = softplus_f(d);
      if (r0 + t.sr + L * i >= sp.hi) d = 0.f;  // rows behind the last leave the states as they are
      s.dd[t.sr + L * i][t.sc] = make_float2(d, d * x[i]);
      x1[i] = x[i];
      z1[i] = z[i];
    }
    t.put_vectors(s.b, vb);
    if constexpr (!LOCAL) t.put_vectors(s.c, vc);
    if (edge) mark_edges(a, s.edges, sp.b, r0, sp.hi);
    __syncthreads();
    if (r0 + kSub < sp.hi) load(r0 + kSub);
    if constexpr (!LOCAL)
      if (a.saved)
        store_states4(a.saved + (((int64_t)sp.b * a.subs + (r0 - (int64_t)sp.b * a.T) / kSub) * a.D + t.d) * a.NP,
                      a.NP, 4 * t.l, t.on, h);
    if (edge) {
      fwd_rows<T, L, LOCAL, true>(a, s, t, A2, h, dsum);
      if (r0 + kSub < sp.hi) seq = seq_of(a, sp.b, r0 + kSub);
    } else {
      fwd_rows<T, L, LOCAL, false>(a, s, t, A2, h, dsum);
    }
    __syncthreads();
    if constexpr (!LOCAL) {
#pragma unroll
      for (int i = 0; i < S::PER; ++i) {
        const int64_t r = r0 + t.sr + L * i;
        float y = fmaf(skip, x1[i], s.y[t.sr + L * i][t.sc]);
        if (a.z) y *= z1[i] * sigmoid_of<T>(z1[i]);
        if (r < sp.hi && t.sc < t.nch) ((T*)a.y)[r * a.D + t.d0 + t.sc] = from_f<T>(y);
      }
    }
  }
  if constexpr (LOCAL) {
    store_states4(a.carry + ((int64_t)bc * a.D + t.d) * a.NP, a.NP, 4 * t.l, t.on, h);
    if (t.l == 0 && t.on) a.decay[(int64_t)bc * a.D + t.d] = dsum;
  }
}

// carry[b][c] from the state behind chunk c, started at zero, to the state in
// front of it (BACK: from the gradient in front of chunk c to the one behind it).
// A sequence that begins in a chunk keeps what is in front of it out.
template <bool BACK> __global__ void __launch_bounds__(256) k_sel_carry(const SelArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = (int64_t)a.D * a.NP;
  if (i >= a.B * per) return;
  const int b = (int)(i / per);
  const int64_t at = i - b * per;
  const int d = (int)(at / a.NP), n = (int)(at - (int64_t)d * a.NP);
  const float A2 = n < a.N ? a.A[(int64_t)d * a.N + n] * kLog2e : 0.f;
  float run = 0.f;
  const int64_t base = (int64_t)b * a.chunks;
  for (int k = 0; k < a.chunks; ++k) {
    const int c = BACK ? a.chunks - 1 - k : k;
    const SelSpan sp = sel_span(a, (int)(base + c));
    float* p = a.carry + (base + c) * per + at;
    const bool last = k + 1 == a.chunks;
    const float own = last ? 0.f : *p, dsum = last ? 0.f : a.decay[(base + c) * a.D + d];
    *p = run;
    const bool begins = seq_of(a, b, sp.hi - 1).lo >= sp.lo;
    run = begins ? own : fmaf(fast_exp2(dsum * A2), run, own);
  }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
template <typename T, int L> struct SelBwdShared {
  using S = SelTile<T, L>;
  alignas(16) float b[kSub * S::NL];
  alignas(16) float c[kSub * S::NL];
  float2 dd[kSub][S::CH];       // dt, dt x
  float o[kSub][S::CH];         // dy silu(z)
  float y[kSub][S::PAD], sb[kSub][S::PAD], sa[kSub][S::PAD];
  alignas(16) float bc[kSelWarps][kSub][2 * S::NL];  // dB, dC of a warp's channels
  float fold[2][kSelThreads];
  SelEdges edges;
};

// Eight values of each lane, four of dB and four of dC, summed over the channels
// of the warp (lanes L apart) into the warp's row of shared memory.
template <int L> __device__ __forceinline__ void sum_channels(float (&v)[8], float* row, int lane) {
  constexpr int CW = 32 / L, NL = 4 * L;       // channels of a warp
  constexpr int W = CW < 8 ? CW : 8;           // lanes that end with different values
  const int l = lane % L, w = lane / L;
  int first = 0;                               // of the values that this lane still holds
#pragma unroll
  for (int o = W / 2, n = 4; o > 0; o /= 2, n /= 2) {
    const bool up = w & o;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) {
        const float keep = up ? v[i + n] : v[i], send = up ? v[i] : v[i + n];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o * L);
      }
    first += up ? n : 0;
  }
  constexpr int left = 8 / W;
#pragma unroll
  for (int o = W; o < CW; o *= 2)
#pragma unroll
    for (int i = 0; i < left; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o * L);
  if (w < W) {
#pragma unroll
    for (int i = 0; i < left; ++i) {
      const int at = first + i;
      row[(at >> 2) * NL + 4 * l + (at & 3)] = v[i];
    }
  }
}

// One row's states from those in front of it.
template <bool EDGE, typename T, int L>
__device__ __forceinline__ void state_row(const SelArgs& a, const SelBwdShared<T, L>& s, const SelTile<T, L>& t,
                                          int r, const float2 (&A2)[2], float2 (&h)[2], float2 (&da)[2],
                                          float2 (&p)[2]) {
  using S = SelTile<T, L>;
  const float2 dd = s.dd[r][t.mc];
  const float4 B = *reinterpret_cast<const float4*>(s.b + r * S::NL + 4 * t.l);
  if constexpr (EDGE) {
    const int n = s.edges.begin[r];
    if (n >= 0)
      load_states(a.h0 ? a.h0 + ((int64_t)n * a.D + t.d) * a.N : nullptr, a.N, 4 * t.l, t.on, h);
  }
  da[0] = decay2(dd.x, A2[0]);
  da[1] = decay2(dd.x, A2[1]);
  p[0] = mul2(da[0], h[0]);
  p[1] = mul2(da[1], h[1]);
  h[0] = fma2(f2(dd.y), make_float2(B.x, B.y), p[0]);
  h[1] = fma2(f2(dd.y), make_float2(B.z, B.w), p[1]);
}

template <bool EDGE, typename T, int L>
__device__ __forceinline__ void bwd_half(const SelArgs& a, SelBwdShared<T, L>& s, const SelTile<T, L>& t, int q,
                                         const float2 (&A2)[2], float2 (&h)[2], float2 (&e)[2],
                                         float2 (&dA)[2]) {
  using S = SelTile<T, L>;
  constexpr int R = L < kHalf ? L : kHalf;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float2 da[kHalf][2], p[kHalf][2];
#pragma unroll
  for (int j = 0; j < kHalf; ++j) state_row<EDGE>(a, s, t, q + j, A2, h, da[j], p[j]);
#pragma unroll
  for (int k = kHalf - R; k >= 0; k -= R) {
    float vy[R], vb[R], va[R];
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      const int j = k + i, r = q + j;
      const float2 dd = s.dd[r][t.mc];
      const float o = s.o[r][t.mc];
      const float4 B = *reinterpret_cast<const float4*>(s.b + r * S::NL + 4 * t.l);
      const float4 C = *reinterpret_cast<const float4*>(s.c + r * S::NL + 4 * t.l);
      const float2 B2[2] = {make_float2(B.x, B.y), make_float2(B.z, B.w)};
      const float2 C2[2] = {make_float2(C.x, C.y), make_float2(C.z, C.w)};
      if constexpr (EDGE) {
        const int n = s.edges.end[r];
        if (n >= 0)
          load_states(a.dht ? a.dht + ((int64_t)n * a.D + t.d) * a.N : nullptr, a.N, 4 * t.l, t.on, e);
      }
      float v[8];
      float2 sy, sb, sa;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float2 hh = fma2(f2(dd.y), B2[u], p[j][u]);
        e[u] = fma2(f2(o), C2[u], e[u]);
        const float2 dC = mul2(f2(o), hh), dB = mul2(f2(dd.y), e[u]);
        v[2 * u] = dB.x; v[2 * u + 1] = dB.y;
        v[4 + 2 * u] = dC.x; v[5 + 2 * u] = dC.y;
        const float2 g = mul2(p[j][u], e[u]);
        sy = u ? fma2(hh, C2[u], sy) : mul2(hh, C2[u]);
        sb = u ? fma2(e[u], B2[u], sb) : mul2(e[u], B2[u]);
        sa = u ? fma2(g, A2[u], sa) : mul2(g, A2[u]);
        dA[u] = fma2(f2(dd.x), g, dA[u]);
        e[u] = mul2(da[j][u], e[u]);
      }
      vy[i] = sy.x + sy.y;
      vb[i] = sb.x + sb.y;
      va[i] = sa.x + sa.y;
      if constexpr (EDGE) {
        const int n = s.edges.begin[r];
        if (n >= 0) {
          if (a.dh0) store_states(a.dh0 + ((int64_t)n * a.D + t.d) * a.N, a.N, 4 * t.l, t.on, e);
          e[0] = e[1] = f2(0.f);
        }
      }
      sum_channels<L>(v, s.bc[warp][r], lane);
    }
    const float ry = sum_transposed<L, R>(vy, t.l), rb = sum_transposed<L, R>(vb, t.l);
    const float ra = sum_transposed<L, R>(va, t.l);
    if (t.l < R) {
      const int r = q + k + t.l;
      s.y[r][t.mc] = ry;
      s.sb[r][t.mc] = rb;
      s.sa[r][t.mc] = ra;
    }
  }
}

template <bool EDGE, typename T, int L>
__device__ __forceinline__ void bwd_rows(const SelArgs& a, SelBwdShared<T, L>& s, const SelTile<T, L>& t,
                                         const float2 (&A2)[2], const float2 (&h0)[2], float2 (&e)[2],
                                         float2 (&dA)[2]) {
  float2 h[2] = {h0[0], h0[1]}, da[2], p[2];
#pragma unroll 2
  for (int r = 0; r < kHalf; ++r) state_row<EDGE>(a, s, t, r, A2, h, da, p);
  bwd_half<EDGE>(a, s, t, kHalf, A2, h, e, dA);
  h[0] = h0[0];
  h[1] = h0[1];
  bwd_half<EDGE>(a, s, t, 0, A2, h, e, dA);
}

// LOCAL: only e, from zero behind the chunk to what it is in front of it.
template <bool EDGE, typename T, int L>
__device__ __forceinline__ void bwd_rows_local(const SelArgs& a, SelBwdShared<T, L>& s, const SelTile<T, L>& t,
                                               const float2 (&A2)[2], float2 (&e)[2], float& dsum) {
  using S = SelTile<T, L>;
#pragma unroll 4
  for (int r = kSub - 1; r >= 0; --r) {
    const float2 dd = s.dd[r][t.mc];
    const float o = s.o[r][t.mc];
    const float4 C = *reinterpret_cast<const float4*>(s.c + r * S::NL + 4 * t.l);
    if constexpr (EDGE) {
      const int n = s.edges.end[r];
      if (n >= 0)
        load_states(a.dht ? a.dht + ((int64_t)n * a.D + t.d) * a.N : nullptr, a.N, 4 * t.l, t.on, e);
    }
    e[0] = mul2(decay2(dd.x, A2[0]), fma2(f2(o), make_float2(C.x, C.y), e[0]));
    e[1] = mul2(decay2(dd.x, A2[1]), fma2(f2(o), make_float2(C.z, C.w), e[1]));
    dsum += dd.x;
    if constexpr (EDGE)
      if (s.edges.begin[r] >= 0) e[0] = e[1] = f2(0.f);
  }
}

template <typename T, int L, bool LOCAL>
__global__ void __launch_bounds__(kSelThreads, LOCAL ? 4 : 3) k_sel_bwd(const SelArgs a) {
  using S = SelTile<T, L>;
  extern __shared__ __align__(16) char raw_shared[];
  SelBwdShared<T, L>& s = *reinterpret_cast<SelBwdShared<T, L>*>(raw_shared);
  const int bc = blockIdx.x / a.tiles;
  const S t(a, blockIdx.x - bc * a.tiles);
  const SelSpan sp = sel_span(a, bc);
  if (LOCAL && sp.c == 0) return;  // nothing is in front of the first
  float2 A2[2], e[2];
  t.load_rates(a, A2);
  float dsum = 0.f;
  if (LOCAL || sp.c + 1 == a.chunks) e[0] = e[1] = f2(0.f);
  else load_states4(a.carry + ((int64_t)bc * a.D + t.d) * a.NP, a.NP, 4 * t.l, t.on, e);
  const float bias = a.bias && t.sc < t.nch ? a.bias[t.d0 + t.sc] : 0.f;
  const float skip = a.Dk && t.sc < t.nch ? a.Dk[t.d0 + t.sc] : 0.f;
  LongSum sum_a[4], sum_d, sum_bias;
  SelSeq seq = seq_of(a, sp.b, sp.hi - 1);

  const int64_t n_sub = (sp.hi - sp.lo + kSub - 1) / kSub;
  for (int64_t k = n_sub - 1; k >= 0; --k) {
    const int64_t r0 = sp.lo + k * kSub;
    const bool edge = seq.lo >= r0 || seq.hi <= r0 + kSub;
    float x[S::PER], pre[S::PER], dy[S::PER], z[S::PER];
    {
      float vb[S::VPT], vc[S::VPT];
      t.load_tokens(a.x, false, a.ldx, r0, sp.hi, x);
      t.load_tokens(a.dt, a.dt_f32, a.lddt, r0, sp.hi, pre);
      t.load_tokens(a.dy, false, a.lddy, r0, sp.hi, dy);
      if (a.z) t.load_tokens(a.z, false, a.ldz, r0, sp.hi, z);
      if constexpr (!LOCAL) t.load_vectors(a, a.Bv, a.ldb, r0, sp.hi, vb);
      t.load_vectors(a, a.Cv, a.ldc, r0, sp.hi, vc);
      if constexpr (!LOCAL) t.put_vectors(s.b, vb);
      t.put_vectors(s.c, vc);
    }
    float2 h0[2];
    if constexpr (!LOCAL)
      load_states4(a.saved + (((int64_t)sp.b * a.subs + (r0 - (int64_t)sp.b * a.T) / kSub) * a.D + t.d) * a.NP,
                   a.NP, 4 * t.l, t.on, h0);
    float dt[S::PER], sig[S::PER];
#pragma unroll
    for (int i = 0; i < S::PER; ++i) {
      pre[i] += bias;
      dt[i] = a.softplus ? softplus_f(pre[i]) : pre[i];
      if (r0 + t.sr + L * i >= sp.hi) dt[i] = 0.f;
      s.dd[t.sr + L * i][t.sc] = make_float2(dt[i], dt[i] * x[i]);
      float o = dy[i];
      if (a.z) {
        sig[i] = sigmoid_of<T>(z[i]);
        o *= z[i] * sig[i];
      }
      s.o[t.sr + L * i][t.sc] = o;
    }
    if (edge) mark_edges(a, s.edges, sp.b, r0, sp.hi);
    __syncthreads();
    if constexpr (LOCAL) {
      if (edge) bwd_rows_local<true>(a, s, t, A2, e, dsum);
      else bwd_rows_local<false>(a, s, t, A2, e, dsum);
    } else {
      float2 dA[2] = {f2(0.f), f2(0.f)};
      if (edge) bwd_rows<true>(a, s, t, A2, h0, e, dA);
      else bwd_rows<false>(a, s, t, A2, h0, e, dA);
      sum_a[0].add(dA[0].x);
      sum_a[1].add(dA[0].y);
      sum_a[2].add(dA[1].x);
      sum_a[3].add(dA[1].y);
    }
    if (edge && r0 > sp.lo) seq = seq_of(a, sp.b, r0 - 1);
    __syncthreads();
    if constexpr (!LOCAL) {
      float dd = 0.f, db = 0.f;
#pragma unroll
      for (int i = 0; i < S::PER; ++i) {
        const int rr = t.sr + L * i;
        const int64_t r = r0 + rr;
        const float sb = s.sb[rr][t.sc], sa = s.sa[rr][t.sc] * kSelLn2, o = s.o[rr][t.sc];
        float ddt = fmaf(x[i], sb, sa);
        if (a.softplus) ddt *= sigmoid_of<float>(pre[i]);
        if (r < sp.hi && t.sc < t.nch) {
          const int64_t at = r * a.D + t.d0 + t.sc;
          ((T*)a.dx)[at] = from_f<T>(fmaf(dt[i], sb, skip * o));
          if (a.dt_f32) ((float*)a.ddt)[at] = ddt;
          else ((T*)a.ddt)[at] = from_f<T>(ddt);
          if (a.z) {
            const float y = fmaf(skip, x[i], s.y[rr][t.sc]);
            ((T*)a.dz)[at] = from_f<T>(dy[i] * y * sig[i] * fmaf(z[i], 1.f - sig[i], 1.f));
          }
          dd = fmaf(o, x[i], dd);
          db += ddt;
        }
      }
      sum_d.add(dd);
      sum_bias.add(db);
      // this CTA's share of dB and dC
      for (int i = threadIdx.x; i < kSub * 2 * S::NL; i += kSelThreads) {
        const int rr = i / (2 * S::NL), v = i % (2 * S::NL), n = v % S::NL;
        if (r0 + rr >= sp.hi || n >= a.N) continue;
        float f = s.bc[0][rr][v];
#pragma unroll
        for (int w = 1; w < kSelWarps; ++w) f += s.bc[w][rr][v];
        a.part_bc[(((int64_t)t.tile * a.B * a.T + r0 + rr) * 2 + v / S::NL) * a.N + n] = f;
      }
    }
  }
  if constexpr (LOCAL) {
    store_states4(a.carry + ((int64_t)bc * a.D + t.d) * a.NP, a.NP, 4 * t.l, t.on, e);
    if (t.l == 0 && t.on) a.decay[(int64_t)bc * a.D + t.d] = dsum;
  } else {
    const float2 g[2] = {make_float2(sum_a[0].get(), sum_a[1].get()),
                         make_float2(sum_a[2].get(), sum_a[3].get())};
    store_states4(a.part_a + ((int64_t)bc * a.D + t.d) * a.NP, a.NP, 4 * t.l, t.on, g);
    s.fold[0][threadIdx.x] = sum_d.get();
    s.fold[1][threadIdx.x] = sum_bias.get();
    __syncthreads();
    if (threadIdx.x < t.nch) {
      float x = 0.f, y = 0.f;
#pragma unroll
      for (int i = 0; i < L; ++i) {
        x += s.fold[0][threadIdx.x + i * S::CH];
        y += s.fold[1][threadIdx.x + i * S::CH];
      }
      const int64_t n = (int64_t)a.B * a.chunks * a.D, at = (int64_t)bc * a.D + t.d0 + threadIdx.x;
      a.part_d[at] = x;
      a.part_d[n + at] = y;
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
// Every lane has four states of a channel.
template <typename T, int L>
__global__ void __launch_bounds__(kSelThreads) k_sel_step(const SelArgs a, float* state, int64_t stride,
                                                          int pool, const int32_t* idx) {
  constexpr int CH = kSelThreads / L;
  const int tiles = (a.D + CH - 1) / CH;
  const int n = blockIdx.x / tiles, d = (blockIdx.x - n * tiles) * CH + threadIdx.x / L, l = threadIdx.x % L;
  const bool on = d < a.D;
  const int slot = idx ? idx[n] : n;
  if (slot < 0 || slot >= pool) {
    if (on && l == 0) ((T*)a.y)[(int64_t)n * a.D + d] = from_f<T>(0.f);
    return;
  }
  float2 h[2] = {f2(0.f), f2(0.f)}, A2[2], B[2], C[2];
  float* p = state + slot * stride + (int64_t)d * a.N;
  const bool vec = (a.N & 3) == 0 && ((reinterpret_cast<uintptr_t>(state) | (stride * 4)) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(a.A) & 15) == 0;
  float x = 0.f, dt = 0.f;
  if (on) {
    if (vec) {
      load_states4(p, a.N, 4 * l, true, h);
      load_states4(a.A + (int64_t)d * a.N, a.N, 4 * l, true, A2);
    } else {
      load_states(p, a.N, 4 * l, true, h);
      load_states(a.A + (int64_t)d * a.N, a.N, 4 * l, true, A2);
    }
    x = to_f<T>(((const T*)a.x)[n * a.ldx + d]);
    dt = a.dt_f32 ? ((const float*)a.dt)[n * a.lddt + d] : to_f<T>(((const T*)a.dt)[n * a.lddt + d]);
    if (a.bias) dt += a.bias[d];
    if (a.softplus) dt = softplus_f(dt);
  } else {
    A2[0] = A2[1] = f2(0.f);
  }
  const int g = on ? d / (a.D / a.G) : 0;
  float b[4], c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = on && 4 * l + i < a.N;
    b[i] = in ? to_f<T>(((const T*)a.Bv)[n * a.ldb + g * a.N + 4 * l + i]) : 0.f;
    c[i] = in ? to_f<T>(((const T*)a.Cv)[n * a.ldc + g * a.N + 4 * l + i]) : 0.f;
  }
  float out = 0.f;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    B[u] = make_float2(b[2 * u], b[2 * u + 1]);
    C[u] = make_float2(c[2 * u], c[2 * u + 1]);
    h[u] = fma2(decay2(dt, mul2(A2[u], f2(kLog2e))), h[u], mul2(f2(dt * x), B[u]));
    const float2 o = mul2(h[u], C[u]);
    out += o.x + o.y;
  }
  if (on) {
    if (vec) store_states4(p, a.N, 4 * l, true, h);
    else store_states(p, a.N, 4 * l, true, h);
  }
#pragma unroll
  for (int o = L / 2; o > 0; o /= 2) out += __shfl_xor_sync(0xffffffffu, out, o);
  if (on && l == 0) {
    if (a.Dk) out = fmaf(a.Dk[d], x, out);
    if (a.z) {
      const float z = to_f<T>(((const T*)a.z)[n * a.ldz + d]);
      out *= z * sigmoid_of<T>(z);
    }
    ((T*)a.y)[(int64_t)n * a.D + d] = from_f<T>(out);
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
  if (p->T > (int64_t)1 << 40 || (p->B && p->T > ((int64_t)1 << 40) / p->B))
    return fail(GDN2_ERR_UNSUPPORTED, "%s: too many rows", fn);
  if (p->cu_seqlens && p->T > 2147483647LL)
    return fail(GDN2_ERR_UNSUPPORTED, "%s: packed rows are up to 2^31 - 1", fn);
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
// launches cost three quarters of the forward once more); then as many chunks as
// give four for each, of 64 rows at least.
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
  a.dt_f32 = p->dt_dtype == GDN2_DTYPE_F32; a.softplus = p->dt_softplus != 0;
  a.chunk = q.chunk; a.subs = q.subs; a.chunks = q.chunks;
  a.tiles_per_group = q.tiles_per_group; a.tiles = q.tiles;
  return a;
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

// States of sequences without a token pass through: copied for all, where there
// can be such, in front of the kernels that write the others'.
cudaError_t pass_states(const gdn2_selective_problem* p, const float* from, float* to, cudaStream_t st) {
  const bool some = p->cu_seqlens || p->T == 0;
  const size_t bytes = (size_t)p->n_seqs * p->D * p->N * sizeof(float);
  if (!to || !some || !bytes) return cudaSuccess;
  return from ? cudaMemcpyAsync(to, from, bytes, cudaMemcpyDeviceToDevice, st)
              : cudaMemsetAsync(to, 0, bytes, st);
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
  cudaError_t e = pass_states(p, h0, ht, st);
  if (e != cudaSuccess) return cuda_status(e, fn);
  if (!some) return GDN2_OK;
  SelArgs a = sel_args(p, q);
  a.x = x; a.dt = dt; a.A = A; a.Bv = Bv; a.Cv = Cv; a.Dk = D; a.z = z; a.bias = dt_bias; a.h0 = h0;
  a.y = y; a.ht = ht; a.saved = saved;
  if (w.total) {
    a.carry = (float*)((char*)workspace + w.carry);
    a.decay = (float*)((char*)workspace + w.decay);
  }
  return cuda_status(with_lanes(p->dtype, p->N, [&](auto t, auto lanes) {
    using T = decltype(t);
    constexpr int L = decltype(lanes)::value;
    if (q.chunks > 1) {
      k_sel_fwd<T, L, true><<<(unsigned)ctas, kSelThreads, 0, st>>>(a);
      const int64_t n = (int64_t)a.B * a.D * a.NP;
      k_sel_carry<false><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a);
    }
    k_sel_fwd<T, L, false><<<(unsigned)ctas, kSelThreads, 0, st>>>(a);
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
  cudaError_t e = pass_states(p, dht, dh0, st);
  if (e != cudaSuccess) return cuda_status(e, fn);
  if (!some) {
    if (dA) e = cudaMemsetAsync(dA, 0, (size_t)p->D * p->N * sizeof(float), st);
    if (e == cudaSuccess && dD) e = cudaMemsetAsync(dD, 0, (size_t)p->D * sizeof(float), st);
    if (e == cudaSuccess && ddt_bias) e = cudaMemsetAsync(ddt_bias, 0, (size_t)p->D * sizeof(float), st);
    return cuda_status(e, fn);
  }
  SelArgs a = sel_args(p, q);
  a.x = x; a.dt = dt; a.A = A; a.Bv = Bv; a.Cv = Cv; a.Dk = D; a.z = z; a.bias = dt_bias; a.h0 = h0;
  a.saved = const_cast<float*>(saved); a.dy = dy; a.dht = dht;
  a.dx = dx; a.ddt = ddt; a.dz = dz; a.dh0 = dh0;
  char* ws = (char*)workspace;
  a.carry = (float*)(ws + w.carry); a.decay = (float*)(ws + w.decay);
  a.part_bc = (float*)(ws + w.part_bc); a.part_a = (float*)(ws + w.part_a); a.part_d = (float*)(ws + w.part_d);
  return cuda_status(with_lanes(p->dtype, p->N, [&](auto t, auto lanes) {
    using T = decltype(t);
    constexpr int L = decltype(lanes)::value;
    constexpr int smem = (int)sizeof(SelBwdShared<T, L>);
    auto local = k_sel_bwd<T, L, true>;
    auto full = k_sel_bwd<T, L, false>;
    cudaError_t e = cudaFuncSetAttribute(full, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(local, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (q.chunks > 1) {
      local<<<(unsigned)ctas, kSelThreads, smem, st>>>(a);
      const int64_t n = (int64_t)a.B * a.D * a.NP;
      k_sel_carry<true><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a);
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
  const int ch = kSelThreads / lanes_of(p->N);
  const int64_t ctas = (int64_t)p->B * ((p->D + ch - 1) / ch);
  if (too_many(ctas)) return fail(GDN2_ERR_UNSUPPORTED, "%s: too many sequences", fn);
  SelArgs a = sel_args(p, sel_plan(p));
  a.x = x; a.dt = dt; a.A = A; a.Bv = Bv; a.Cv = Cv; a.Dk = D; a.z = z; a.bias = dt_bias; a.y = y;
  const cudaStream_t st = (cudaStream_t)stream;
  return cuda_status(with_lanes(p->dtype, p->N, [&](auto t, auto lanes) {
    k_sel_step<decltype(t), decltype(lanes)::value>
        <<<(unsigned)ctas, kSelThreads, 0, st>>>(a, state, state_stride, pool, state_indices);
    return cudaGetLastError();
  }), fn);
}

}  // extern "C"
