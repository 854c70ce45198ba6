// Eight adjacent elements of a row as floats: one 16-byte access (two for fp32).
#pragma once
#include "../../include/castle_b200.h"
#include "sm100.cuh"

namespace castle {

template <typename T> struct Raw8 { uint4 q[sizeof(T) / 2]; };   // as they lie

template <typename T> __device__ __forceinline__ void load8(const T* p, float* v) {
  uint4 q = *reinterpret_cast<const uint4*>(p);
  const uint32_t* u = &q.x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float2 f = Elem<T>::unpack2(u[j]);
    v[2 * j] = f.x; v[2 * j + 1] = f.y;
  }
}
template <> __device__ __forceinline__ void load8<float>(const float* p, float* v) {
  float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float* v) {
  uint4 q;
  q.x = Elem<T>::pack2(v[0], v[1]); q.y = Elem<T>::pack2(v[2], v[3]);
  q.z = Elem<T>::pack2(v[4], v[5]); q.w = Elem<T>::pack2(v[6], v[7]);
  *reinterpret_cast<uint4*>(p) = q;
}
template <> __device__ __forceinline__ void store8<float>(float* p, const float* v) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// One element as a float and back.
template <typename T> __device__ __forceinline__ float load1(const T* p) { return Elem<T>::to_f(*p); }
template <> __device__ __forceinline__ float load1<float>(const float* p) { return *p; }
template <typename T> __device__ __forceinline__ void store1(T* p, float v) { *p = Elem<T>::from_f(v); }
template <> __device__ __forceinline__ void store1<float>(float* p, float v) { *p = v; }

// Eight columns of a row per thread out of a stretch of 8 * THREADS that THREADS threads cover together: adjacent ones in one
// access (VEC: rows of a multiple of eight elements at 16-byte boundaries), else every THREADS-th, so that a warp's single
// accesses are adjacent.  Columns from `dim` on read as `fill` and are not written.
template <int THREADS, bool VEC> __device__ __forceinline__ int column8(int stretch, int thread, int j) {
  return stretch * 8 * THREADS + (VEC ? thread * 8 + j : j * THREADS + thread);
}
template <typename T, int THREADS, bool VEC>
__device__ __forceinline__ void load_columns8(const T* row, int stretch, int thread, int dim, float* v, float fill = 0.f) {
  if constexpr (VEC) {
    const int c = column8<THREADS, true>(stretch, thread, 0);
    if (c < dim) {
      load8<T>(row + c, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = fill;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column8<THREADS, false>(stretch, thread, j);
      v[j] = c < dim ? load1<T>(row + c) : fill;
    }
  }
}
template <typename T, int THREADS, bool VEC>
__device__ __forceinline__ void store_columns8(T* row, int stretch, int thread, int dim, const float* v) {
  if constexpr (VEC) {
    const int c = column8<THREADS, true>(stretch, thread, 0);
    if (c < dim) store8<T>(row + c, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column8<THREADS, false>(stretch, thread, j);
      if (c < dim) store1<T>(row + c, v[j]);
    }
  }
}

// Whether rows of `dim` elements, `stride` apart, at two addresses can be taken eight elements at a time.
inline bool vec_rows(int dtype, int dim, int64_t stride, const void* a, const void* b) {
  return dim % 8 == 0 && stride * (dtype == CASTLE_F32 ? 4 : 2) % 16 == 0 && (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) % 16 == 0;
}
// f called with a value of the type that `dtype` names
template <typename F> inline auto by_type(int dtype, F&& f) {
  return dtype == CASTLE_BF16 ? f(__nv_bfloat16()) : dtype == CASTLE_F16 ? f(__half()) : f(float());
}

}  // namespace castle
