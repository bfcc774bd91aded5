// op_util.cuh -- helpers shared by the operators around the GDN-2 mixer
// (scan.cu, selective.cu, logprob.cu, sample.cu, adamw.cu, gradnorm.cu): error
// reporting at the C entries, element groups of a row with or without vector
// access, rows as aligned vectors, ordered keys of values, and dtype dispatch.
#pragma once

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <type_traits>

#include "../../include/gdn2_b200.h"

#include "common.cuh"

namespace gdn2 {
int set_error(int code, const char* msg);       // abi.cu: the per-thread last error
cudaError_t fault_word(unsigned int** ptr);     // state_tc.cu: the per-device fault word
namespace {

inline int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return set_error(code, buf);
}

inline int cuda_status(cudaError_t e, const char* where) {
  if (e == cudaSuccess) return GDN2_OK;
  return fail(GDN2_ERR_CUDA, "%s: CUDA error %d (%s)", where, (int)e, cudaGetErrorString(e));
}

inline bool dtype_valid(int dt) {
  return dt == GDN2_DTYPE_F32 || dt == GDN2_DTYPE_BF16 || dt == GDN2_DTYPE_F16;
}

inline size_t dtype_size(int dt) { return dt == GDN2_DTYPE_F32 ? 4 : 2; }

inline bool aligned_to(const void* p, size_t n) {
  return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

// Whether all of the pointers (NULL among them) are on multiples of n bytes.
template <typename... P> bool all_aligned(size_t n, P... p) { return (aligned_to(p, n) && ...); }

// f(T{}) with the element type of `dtype`.
template <typename F> cudaError_t with_dtype(int dtype, F&& f) {
  switch (dtype) {
    case GDN2_DTYPE_F32: return f(float{});
    case GDN2_DTYPE_BF16: return f(__nv_bfloat16{});
    default: return f(__half{});
  }
}

// N consecutive elements of T as raw 32-bit words (N * sizeof(T) is 4, 8 or a
// multiple of 16 bytes), kept packed until they are used.
template <typename T, int N> struct Raw {
  static constexpr int kWords = N * (int)sizeof(T) / 4;
  static_assert(kWords == 1 || kWords == 2 || kWords % 4 == 0, "vector width");
  uint32_t u[kWords];
};

template <typename T, int N> __device__ __forceinline__ Raw<T, N> raw_zero() {
  Raw<T, N> r;
#pragma unroll
  for (int i = 0; i < Raw<T, N>::kWords; ++i) r.u[i] = 0u;
  return r;
}

template <typename T, int N> __device__ __forceinline__ Raw<T, N> load_raw(const T* p) {
  Raw<T, N> r;
  constexpr int W = Raw<T, N>::kWords;
  if constexpr (W == 1) {
    r.u[0] = __ldg(reinterpret_cast<const unsigned int*>(p));
  } else if constexpr (W == 2) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    r.u[0] = v.x; r.u[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
      r.u[4 * i] = v.x; r.u[4 * i + 1] = v.y; r.u[4 * i + 2] = v.z; r.u[4 * i + 3] = v.w;
    }
  }
  return r;
}

template <typename T, int N> __device__ __forceinline__ void store_raw(T* p, const Raw<T, N>& r) {
  constexpr int W = Raw<T, N>::kWords;
  if constexpr (W == 1) {
    *reinterpret_cast<unsigned int*>(p) = r.u[0];
  } else if constexpr (W == 2) {
    *reinterpret_cast<uint2*>(p) = make_uint2(r.u[0], r.u[1]);
  } else {
#pragma unroll
    for (int i = 0; i < W / 4; ++i)
      reinterpret_cast<uint4*>(p)[i] =
          make_uint4(r.u[4 * i], r.u[4 * i + 1], r.u[4 * i + 2], r.u[4 * i + 3]);
  }
}

template <typename T, int N> __device__ __forceinline__ float raw_get(const Raw<T, N>& r, int i) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(r.u[i]);
  } else {
    const uint32_t w = r.u[i >> 1];
    const unsigned short h = (unsigned short)((i & 1) ? (w >> 16) : (w & 0xffffu));
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      return __uint_as_float((uint32_t)h << 16);
    else
      return __half2float(__ushort_as_half(h));
  }
}

template <typename T, int N>
__device__ __forceinline__ Raw<T, N> raw_from(const float (&f)[N]) {
  Raw<T, N> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) r.u[i] = __float_as_uint(f[i]);
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      r.u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      r.u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return r;
}

// N elements at p of which the first `n` exist (the rest read as zero): one
// vector access when VEC, element accesses otherwise.
template <typename T, int N, bool VEC>
__device__ __forceinline__ Raw<T, N> load_group(const T* p, int n) {
  if (n <= 0) return raw_zero<T, N>();
  if constexpr (VEC) {
    return load_raw<T, N>(p);
  } else {
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = i < n ? to_f<T>(p[i]) : 0.f;
    return raw_from<T, N>(f);
  }
}

template <typename T, int N, bool VEC>
__device__ __forceinline__ void store_group(T* p, const float (&f)[N], int n) {
  if (n <= 0) return;
  if constexpr (VEC) {
    store_raw<T, N>(p, raw_from<T, N>(f));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = from_f<T>(f[i]);
  }
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

}  // namespace
}  // namespace gdn2
