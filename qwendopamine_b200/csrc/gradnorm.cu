// gradnorm.cu -- the norm of many gradients taken together, the coefficient that
// clips it, and the clipping in place.
//
//   norm = sqrt(sum g^2)  or  max |g|,   coef = min(1, max_norm / (norm + 1e-6))
//
// Each CTA sums a chunk of one tensor into a double; a second launch of one CTA
// adds those in a fixed order, so equal inputs give equal bits.  A thread adds
// the squares of up to 64 values in fp32 and those sums in fp64: an error of a few
// 2^-24 that does not grow with the number of values.  Squares leave fp32's range
// for values above 2^64 or below 2^-75, which 16-bit gradients can hold: where a
// thread's fp32 sum is outside [2^-80, finite] it forms the same sum in fp64 from the
// values that it still has.  The largest magnitude is found on the bit patterns, where NaN
// is above infinity.
//
// Bound: HBM, one read of the gradients (and one more read and a write where
// they are scaled).  What it needs is bytes in flight: eight 16-byte vectors for
// each of 1024 threads of an SM (433 M values in bf16 129 us a call, 6.7 TB/s; 121 M
// clipped in place 126 us, two reads and a write, the second read partly from L2).
//
// The tensors' addresses travel in the kernel's parameters: no table in device
// memory, no copy before the launch.
#include "mma16.cuh"
#include "op_util.cuh"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <memory>
#include <new>

namespace gdn2 {
namespace {

constexpr int kGradThreads = 256;
constexpr int kGradUnroll = 8;       // vectors of a thread in flight
constexpr int kGradTensors = 256;    // of one launch (5.4 KB of parameters)
constexpr int kGradChunks = 4096;    // partial sums beyond one for each tensor
constexpr int64_t kGradLeast = 16 << 10;  // bytes of a chunk, at least

struct GradTensors {
  char* data[kGradTensors];
  int64_t numel[kGradTensors];
  uint32_t first[kGradTensors];  // first chunk of each tensor
  uint8_t dtype[kGradTensors];
  int n;
  int64_t chunk;  // bytes of a CTA, a multiple of 16
};

struct Span {  // a CTA's share of a tensor
  char* data;
  int64_t n;  // elements
  int dtype;
};

__device__ __forceinline__ Span span_of(const GradTensors& ts) {
  int lo = 0, hi = ts.n;  // the last tensor whose first chunk is not after this one
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (ts.first[mid] <= blockIdx.x) lo = mid; else hi = mid;
  }
  const int dt = ts.dtype[lo];
  const int64_t per = dt == GDN2_DTYPE_F32 ? ts.chunk / 4 : ts.chunk / 2;
  const int64_t at = (int64_t)(blockIdx.x - ts.first[lo]) * per;
  return Span{ts.data[lo] + at * (dt == GDN2_DTYPE_F32 ? 4 : 2), min(per, ts.numel[lo] - at), dt};
}

// Values of a span in front of its first 16-byte boundary and behind its last.
template <typename T, typename F> __device__ __forceinline__ void ragged_ends(T* p, int64_t n, F&& f) {
  constexpr int VE = 16 / (int)sizeof(T);
  const int64_t head = min(n, (int64_t)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
  const int tail = (int)((n - head) % VE);
  if (threadIdx.x < head) f(p + threadIdx.x);
  else if (threadIdx.x >= 32 && threadIdx.x - 32 < tail) f(p + n - tail + (threadIdx.x - 32));
}

// ---------------------------------------------------------------------------
// partial sums
// ---------------------------------------------------------------------------
template <typename T, int N> __device__ __forceinline__ float2 value_pair(const Raw<T, N>& r, int i) {
  if constexpr (sizeof(T) == 4)
    return make_float2(__uint_as_float(r.u[2 * i]), __uint_as_float(r.u[2 * i + 1]));
  else
    return unpack2<T>(r.u[i]);
}

template <typename T> struct SquareSum {
  static constexpr int VE = 16 / (int)sizeof(T);
  double total = 0.;
  __device__ __forceinline__ void one(T x) {
    const double d = to_f<T>(x);
    total += d * d;
  }
  __device__ __forceinline__ void many(const Raw<T, VE> (&v)[kGradUnroll]) {
    float2 s[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u)
#pragma unroll
      for (int i = 0; i < VE / 2; ++i) {
        const float2 x = value_pair(v[u], i);
        s[i & 1] = fma2(x, x, s[i & 1]);
      }
    const float2 t = add2(s[0], s[1]);
    const float sum = t.x + t.y;
    if (sum >= 0x1p-80f && sum <= FLT_MAX) {
      total += sum;
      return;
    }
    uint32_t some = 0u;  // rare, but for gradients that are zero
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) some |= v[u].u[i];
    if ((some & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu)) == 0u) return;
#pragma unroll 1
    for (int u = 0; u < kGradUnroll; ++u) {
      // indexed by a variable, the vectors would live in local memory
      Raw<T, VE> w = v[0];
#pragma unroll
      for (int q = 1; q < kGradUnroll; ++q)
        if (q == u) w = v[q];
#pragma unroll
      for (int i = 0; i < VE / 2; ++i) {
        const float2 x = value_pair(w, i);
        total += (double)x.x * x.x + (double)x.y * x.y;
      }
    }
  }
  __device__ __forceinline__ double result() const { return total; }
  static __device__ __forceinline__ double join(double a, double b) { return a + b; }
};

template <typename T> struct LargestMagnitude {
  static constexpr int VE = 16 / (int)sizeof(T);
  uint32_t most = 0u;  // bit patterns: one of 32 bits, or two of 16
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4) return max(a, b);
    else return __vmaxu2(a, b);
  }
  __device__ __forceinline__ void one(T x) {
    uint32_t bits;
    if constexpr (sizeof(T) == 4) bits = __float_as_uint(x) & 0x7fffffffu;
    else bits = *reinterpret_cast<const unsigned short*>(&x) & 0x7fffu;
    most = larger(most, bits);
  }
  __device__ __forceinline__ void many(const Raw<T, VE> (&v)[kGradUnroll]) {
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        most = larger(most, v[u].u[i] & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu));
  }
  __device__ __forceinline__ double result() const {
    if constexpr (sizeof(T) == 4) {
      return (double)__uint_as_float(most);
    } else {
      const float2 x = unpack2<T>(most);
      return join(x.x, x.y);
    }
  }
  static __device__ __forceinline__ double join(double a, double b) { return b > a || b != b ? b : a; }
};

// The threads' values joined in a fixed order; the result in thread 0.
template <typename J, int THREADS>
__device__ __forceinline__ double join_cta(double x, J&& join) {
  __shared__ double part[THREADS / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = join(x, __shfl_down_sync(0xffffffffu, x, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int i = 1; i < THREADS / 32; ++i) x = join(x, part[i]);
  return x;
}

template <typename T, typename S> __device__ __forceinline__ double sum_span(T* p, int64_t n) {
  constexpr int VE = S::VE;
  S s;
  ragged_ends(p, n, [&](const T* x) { s.one(*x); });
  const int64_t head = min(n, (int64_t)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
  const T* q = p + head;
  const int nv = (int)((n - head) / VE);  // a chunk is far below 2^31 vectors
  for (int j = threadIdx.x; j < nv; j += kGradThreads * kGradUnroll) {
    Raw<T, VE> v[kGradUnroll];
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u)
      v[u] = j + u * kGradThreads < nv ? load_raw<T, VE>(q + (int64_t)(j + u * kGradThreads) * VE)
                                       : raw_zero<T, VE>();
    s.many(v);
  }
  return s.result();
}

template <bool MAX>
__global__ void __launch_bounds__(kGradThreads, 4)
    k_grad_partial(const __grid_constant__ GradTensors ts, double* partial) {
  const Span s = span_of(ts);
  double x = 0.;
  auto of = [&](auto t) {
    using T = decltype(t);
    if constexpr (MAX) return sum_span<T, LargestMagnitude<T>>((T*)s.data, s.n);
    else return sum_span<T, SquareSum<T>>((T*)s.data, s.n);
  };
  if (s.dtype == GDN2_DTYPE_F32) x = of(float{});
  else if (s.dtype == GDN2_DTYPE_BF16) x = of(__nv_bfloat16{});
  else x = of(__half{});
  auto join = [](double a, double b) {
    return MAX ? LargestMagnitude<float>::join(a, b) : SquareSum<float>::join(a, b);
  };
  x = join_cta<decltype(join)&, kGradThreads>(x, join);
  if (threadIdx.x == 0) partial[blockIdx.x] = x;
}

constexpr int kFinishThreads = 512;

// out: the norm, the coefficient that clips it, and 1 where it is not finite.
template <bool MAX>
__global__ void __launch_bounds__(kFinishThreads)
    k_grad_finish(const double* partial, int n, double max_norm, float* out) {
  auto join = [](double a, double b) {
    return MAX ? LargestMagnitude<float>::join(a, b) : SquareSum<float>::join(a, b);
  };
  double x = 0.;
  for (int i = threadIdx.x; i < n; i += kFinishThreads) x = join(x, partial[i]);
  x = join_cta<decltype(join)&, kFinishThreads>(x, join);
  if (threadIdx.x != 0) return;
  const double norm = MAX ? x : sqrt(x);
  const float f = (float)norm;
  const bool finite = f <= FLT_MAX;
  out[0] = f;
  // max_norm < 0 stands for none; a norm that is not finite has no coefficient
  out[1] = finite && max_norm >= 0. ? (float)fmin(1., max_norm / (norm + 1e-6)) : 1.f;
  out[2] = finite ? 0.f : 1.f;
}

// ---------------------------------------------------------------------------
// scaling
// ---------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ void scale_span(T* p, int64_t n, float c) {
  constexpr int VE = 16 / (int)sizeof(T);
  ragged_ends(p, n, [&](T* x) { *x = from_f<T>(to_f<T>(*x) * c); });
  const int64_t head = min(n, (int64_t)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
  uint4* q = reinterpret_cast<uint4*>(p + head);
  const int nv = (int)((n - head) / VE);
  for (int j = threadIdx.x; j < nv; j += kGradThreads * kGradUnroll) {
    Raw<T, VE> v[kGradUnroll];
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u)
      if (j + u * kGradThreads < nv) {
        const uint4 x = q[j + u * kGradThreads];
        v[u].u[0] = x.x; v[u].u[1] = x.y; v[u].u[2] = x.z; v[u].u[3] = x.w;
      }
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u)
      if (j + u * kGradThreads < nv) {
        float f[VE];
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) {
          const float2 x = mul2(value_pair(v[u], i), make_float2(c, c));
          f[2 * i] = x.x;
          f[2 * i + 1] = x.y;
        }
        store_raw<T, VE>(reinterpret_cast<T*>(q + j + u * kGradThreads), raw_from<T, VE>(f));
      }
  }
}

__global__ void __launch_bounds__(kGradThreads, 4)
    k_grad_scale(const __grid_constant__ GradTensors ts, const float* coef) {
  const float c = *coef;
  if (c == 1.f) return;  // nothing to clip: the gradients stay as they are
  const Span s = span_of(ts);
  if (s.dtype == GDN2_DTYPE_F32) scale_span((float*)s.data, s.n, c);
  else if (s.dtype == GDN2_DTYPE_BF16) scale_span((__nv_bfloat16*)s.data, s.n, c);
  else scale_span((__half*)s.data, s.n, c);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int64_t grad_bytes(const gdn2_grad_tensor& t) { return t.numel * (int64_t)dtype_size((int)t.dtype); }

int check_grads(const gdn2_grad_tensor* tensors, int32_t n, const char* fn, int64_t* total) {
  if (n < 0 || (n > 0 && !tensors)) return fail(GDN2_ERR_INVALID, "%s: null tensors", fn);
  *total = 0;
  for (int i = 0; i < n; ++i) {
    const gdn2_grad_tensor& t = tensors[i];
    if (t.numel < 0) return fail(GDN2_ERR_INVALID, "%s: tensor %d: negative size", fn, i);
    if (t.numel > ((int64_t)1 << 42))
      return fail(GDN2_ERR_UNSUPPORTED, "%s: tensor %d is too large", fn, i);
    if (t.dtype < 0 || t.dtype > 2 || !dtype_valid((int)t.dtype))
      return fail(GDN2_ERR_INVALID, "%s: tensor %d: unknown dtype %lld", fn, i, (long long)t.dtype);
    if (t.numel == 0) continue;
    if (!t.data) return fail(GDN2_ERR_INVALID, "%s: tensor %d: null pointer", fn, i);
    if (!aligned_to(t.data, dtype_size((int)t.dtype)))
      return fail(GDN2_ERR_INVALID, "%s: tensor %d: not aligned to its elements", fn, i);
    *total += grad_bytes(t);
    if (*total > ((int64_t)1 << 44)) return fail(GDN2_ERR_UNSUPPORTED, "%s: too many values", fn);
  }
  return GDN2_OK;
}

// Bytes of a chunk: 16 KB, doubled until they are at most kGradChunks in all
// beyond the one that each tensor has anyway.
int64_t grad_chunk(int64_t total) {
  int64_t chunk = kGradLeast;
  while (total / chunk > kGradChunks) chunk *= 2;
  return chunk;
}

// Tensors that share memory would be scaled twice, at the same time.
int check_apart(const gdn2_grad_tensor* tensors, int32_t n, const char* fn) {
  struct Range { uintptr_t lo, hi; };
  std::unique_ptr<Range[]> r(new (std::nothrow) Range[n]);
  if (!r) return fail(GDN2_ERR_INVALID, "%s: out of host memory", fn);
  int m = 0;
  for (int i = 0; i < n; ++i)
    if (tensors[i].numel) {
      const uintptr_t lo = reinterpret_cast<uintptr_t>(tensors[i].data);
      r[m++] = Range{lo, lo + (uintptr_t)grad_bytes(tensors[i])};
    }
  std::sort(r.get(), r.get() + m, [](const Range& a, const Range& b) { return a.lo < b.lo; });
  for (int i = 1; i < m; ++i)
    if (r[i].lo < r[i - 1].hi) return fail(GDN2_ERR_INVALID, "%s: tensors overlap in memory", fn);
  return GDN2_OK;
}

// f(table, chunks of it, chunks before it) for the tensors in tables.
template <typename F>
cudaError_t for_tables(const gdn2_grad_tensor* tensors, int32_t n, int64_t chunk, F&& f) {
  GradTensors ts;
  ts.chunk = chunk;
  int64_t before = 0;
  for (int i = 0; i < n;) {
    ts.n = 0;
    int64_t chunks = 0;
    for (; i < n && ts.n < kGradTensors; ++i) {
      if (tensors[i].numel == 0) continue;
      ts.data[ts.n] = (char*)tensors[i].data;
      ts.numel[ts.n] = tensors[i].numel;
      ts.dtype[ts.n] = (uint8_t)tensors[i].dtype;
      ts.first[ts.n++] = (uint32_t)chunks;
      chunks += (grad_bytes(tensors[i]) + chunk - 1) / chunk;
    }
    if (!chunks) continue;
    const cudaError_t e = f(ts, (unsigned)chunks, before);
    if (e != cudaSuccess) return e;
    before += chunks;
  }
  return cudaSuccess;
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

size_t gdn2_grad_norm_workspace_bytes(int32_t n) {
  return n < 0 ? 0 : sizeof(double) * ((size_t)kGradChunks + (size_t)n);
}

int gdn2_grad_norm(const gdn2_grad_problem* p, const gdn2_grad_tensor* tensors, int32_t n,
                   float* out, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "gdn2_grad_norm";
  if (!p || !out) return fail(GDN2_ERR_INVALID, "%s: null pointer", fn);
  if (p->norm_type != 0 && p->norm_type != 2)
    return fail(GDN2_ERR_INVALID, "%s: norm_type must be 2 or 0 (largest magnitude); got %d", fn,
                p->norm_type);
  if (p->max_norm != p->max_norm) return fail(GDN2_ERR_INVALID, "%s: max_norm is NaN", fn);
  int64_t total = 0;
  const int rc = check_grads(tensors, n, fn, &total);
  if (rc) return rc;
  if (!workspace || workspace_bytes < gdn2_grad_norm_workspace_bytes(n))
    return fail(GDN2_ERR_WORKSPACE, "%s: needs a workspace of %zu bytes", fn,
                gdn2_grad_norm_workspace_bytes(n));
  if (!aligned_to(workspace, 8) || !aligned_to(out, 4))
    return fail(GDN2_ERR_INVALID, "%s: the workspace must start on an 8-byte boundary, the results on a 4-byte one",
                fn);
  double* partial = (double*)workspace;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool most = p->norm_type == 0;
  int64_t parts = 0;
  cudaError_t e = for_tables(tensors, n, grad_chunk(total),
                             [&](const GradTensors& ts, unsigned chunks, int64_t before) {
    if (most) k_grad_partial<true><<<chunks, kGradThreads, 0, st>>>(ts, partial + before);
    else k_grad_partial<false><<<chunks, kGradThreads, 0, st>>>(ts, partial + before);
    parts = before + chunks;
    return cudaGetLastError();
  });
  if (e != cudaSuccess) return cuda_status(e, fn);
  if (most) k_grad_finish<true><<<1, kFinishThreads, 0, st>>>(partial, (int)parts, p->max_norm, out);
  else k_grad_finish<false><<<1, kFinishThreads, 0, st>>>(partial, (int)parts, p->max_norm, out);
  return cuda_status(cudaGetLastError(), fn);
}

int gdn2_grad_scale(const gdn2_grad_tensor* tensors, int32_t n, const float* coef, void* stream) {
  const char* fn = "gdn2_grad_scale";
  int64_t total = 0;
  int rc = check_grads(tensors, n, fn, &total);
  if (rc) return rc;
  if (total == 0) return GDN2_OK;
  rc = check_apart(tensors, n, fn);
  if (rc) return rc;
  if (!coef || !aligned_to(coef, 4))
    return fail(GDN2_ERR_INVALID, "%s: the coefficient is null or not aligned to 4 bytes", fn);
  const cudaStream_t st = (cudaStream_t)stream;
  return cuda_status(for_tables(tensors, n, grad_chunk(total),
                                [&](const GradTensors& ts, unsigned chunks, int64_t) {
    k_grad_scale<<<chunks, kGradThreads, 0, st>>>(ts, coef);
    return cudaGetLastError();
  }), fn);
}

}  // extern "C"
