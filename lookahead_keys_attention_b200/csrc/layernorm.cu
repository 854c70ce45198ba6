// Layer norm, forward and backward, with the reduction of the weight's and the bias's gradient.
//
//   m = mean x, r = 1 / sqrt(mean (x - m)^2 + eps), h = (x - m) r, y = h w + b
//   g = dy w;  dx = r (g - mean g - h mean(g h));  dw = sum over rows dy h;  db = sum over rows dy
//
// All sums are fp32; the variance is taken from the centred values (a second pass over registers, none over memory), since
// mean x^2 - m^2 loses everything where a row's offset is large.
//
// Both directions are bound by memory: x in and y out; x and dy in and dx out.  A row is held in the registers of a group of
// threads (16 elements each; 32 to 512 threads, up to 8192 columns), so it is read once.  In the backward the groups of a CTA
// take rows in turn, the next one on its way meanwhile, and keep their share of dw and db in registers; a CTA leaves one fp32
// row of each, and a last launch adds these in a fixed order.  Wider rows, and calls that want only some of the gradients, take
// a pass per result that reads its rows from memory (or cache) as often as it needs them.
#include <type_traits>

#include "common.cuh"
#include "vec.cuh"

namespace castle {

constexpr int kLnThreads = 256;

// Two sums over the THREADS threads of a group; `s` is the group's: 2 x 2 x (THREADS / 32) floats, used in turn.
template <int THREADS>
__device__ __forceinline__ float2 group_sum2(float a, float b, float2* s, int turn, int group) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if constexpr (THREADS > 32) {
    constexpr int W = THREADS / 32;
    const int warp = (threadIdx.x % THREADS) >> 5;
    float2* mine = s + turn * W;
    if ((threadIdx.x & 31) == 0) mine[warp] = make_float2(a, b);
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(THREADS) : "memory");
    a = b = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) { a += mine[k].x; b += mine[k].y; }
  }
  return make_float2(a, b);
}

template <int THREADS> constexpr int kLnBlock = THREADS > kLnThreads ? THREADS : kLnThreads;

template <typename T, bool VEC, int THREADS, int NV>
__global__ void __launch_bounds__(kLnBlock<THREADS>) castle_layernorm_fwd_kernel(const T* __restrict__ x, int64_t stride, const T* __restrict__ w,
                                                                                 const T* __restrict__ b, float eps, T* __restrict__ y,
                                                                                 float2* __restrict__ stats, int64_t rows, int dim) {
  constexpr int GROUPS = kLnBlock<THREADS> / THREADS;
  __shared__ float2 s[GROUPS][2 * (THREADS / 32)];
  const int group = threadIdx.x / THREADS, t = threadIdx.x % THREADS;
  const int64_t r = (int64_t)blockIdx.x * GROUPS + group;
  if (r >= rows) return;
  float v[NV][8], sum = 0.f, sq = 0.f;
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    load_columns8<T, THREADS, VEC>(x + r * stride, q, t, dim, v[q]);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += v[q][j];
  }
  const float mean = group_sum2<THREADS>(sum, 0.f, s[group], 0, group).x / (float)dim;
#pragma unroll
  for (int q = 0; q < NV; ++q)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = column8<THREADS, VEC>(q, t, j) < dim;
      v[q][j] = in ? v[q][j] - mean : 0.f;
      sq = fmaf(v[q][j], v[q][j], sq);
    }
  const float rstd = rsqrtf(group_sum2<THREADS>(sq, 0.f, s[group], 1, group).x / (float)dim + eps);
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    float g[8], c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { g[j] = 1.f; c[j] = 0.f; }
    if (w) load_columns8<T, THREADS, VEC>(w, q, t, dim, g);
    if (b) load_columns8<T, THREADS, VEC>(b, q, t, dim, c);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[q][j] = fmaf(v[q][j] * rstd, g[j], c[j]);
    store_columns8<T, THREADS, VEC>(y + r * dim, q, t, dim, v[q]);
  }
  if (stats && t == 0) stats[r] = make_float2(mean, rstd);
}

// Rows of any width: a CTA per row, read three times (the second and third time from the caches).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kLnThreads) castle_layernorm_fwd_wide_kernel(const T* __restrict__ x, int64_t stride, const T* __restrict__ w,
                                                                               const T* __restrict__ b, float eps, T* __restrict__ y,
                                                                               float2* __restrict__ stats, int dim) {
  __shared__ float2 s[2 * (kLnThreads / 32)];
  const int t = threadIdx.x, n = (dim + 8 * kLnThreads - 1) / (8 * kLnThreads);
  const int64_t r = blockIdx.x;
  float sum = 0.f, sq = 0.f, v[8];
  for (int q = 0; q < n; ++q) {
    load_columns8<T, kLnThreads, VEC>(x + r * stride, q, t, dim, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += v[j];
  }
  const float mean = group_sum2<kLnThreads>(sum, 0.f, s, 0, 0).x / (float)dim;
  for (int q = 0; q < n; ++q) {
    load_columns8<T, kLnThreads, VEC>(x + r * stride, q, t, dim, v, mean);
#pragma unroll
    for (int j = 0; j < 8; ++j) sq = fmaf(v[j] - mean, v[j] - mean, sq);
  }
  const float rstd = rsqrtf(group_sum2<kLnThreads>(sq, 0.f, s, 1, 0).x / (float)dim + eps);
  for (int q = 0; q < n; ++q) {
    float g[8], c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { g[j] = 1.f; c[j] = 0.f; }
    load_columns8<T, kLnThreads, VEC>(x + r * stride, q, t, dim, v);
    if (w) load_columns8<T, kLnThreads, VEC>(w, q, t, dim, g);
    if (b) load_columns8<T, kLnThreads, VEC>(b, q, t, dim, c);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fmaf((v[j] - mean) * rstd, g[j], c[j]);
    store_columns8<T, kLnThreads, VEC>(y + r * dim, q, t, dim, v);
  }
  if (stats && t == 0) stats[r] = make_float2(mean, rstd);
}

// dx alone, rows of any width.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kLnThreads) castle_layernorm_dx_kernel(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t stride,
                                                                         const T* __restrict__ w, const float2* __restrict__ stats, T* __restrict__ dx, int dim) {
  __shared__ float2 s[2 * (kLnThreads / 32)];
  const int t = threadIdx.x, n = (dim + 8 * kLnThreads - 1) / (8 * kLnThreads);
  const int64_t r = blockIdx.x;
  const float2 st = stats[r];
  float sg = 0.f, sgh = 0.f, a[8], v[8], g[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) g[j] = 1.f;
  auto load = [&](int q) {
    load_columns8<T, kLnThreads, VEC>(dy + r * dy_stride, q, t, dim, a);
    load_columns8<T, kLnThreads, VEC>(x + r * stride, q, t, dim, v, st.x);
    if (w) load_columns8<T, kLnThreads, VEC>(w, q, t, dim, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) { a[j] *= g[j]; v[j] = (v[j] - st.x) * st.y; }
  };
  for (int q = 0; q < n; ++q) {
    load(q);
#pragma unroll
    for (int j = 0; j < 8; ++j) { sg += a[j]; sgh = fmaf(a[j], v[j], sgh); }
  }
  const float2 sums = group_sum2<kLnThreads>(sg, sgh, s, 0, 0);
  const float mg = sums.x / (float)dim, mgh = sums.y / (float)dim;
  for (int q = 0; q < n; ++q) {
    load(q);
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = st.y * (a[j] - mg - v[j] * mgh);
    store_columns8<T, kLnThreads, VEC>(dx + r * dim, q, t, dim, a);
  }
}

// dw and db alone: partial[block.y][0 or 1][column] over the block's rows; a warp's lanes cover 256 columns, eight warps share the rows.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kLnThreads) castle_layernorm_dw_kernel(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t stride,
                                                                         const float2* __restrict__ stats, float* __restrict__ partial, int64_t rows, int dim,
                                                                         int rows_per_block) {
  constexpr int NW = kLnThreads / 32;
  __shared__ float s[NW][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, slab = blockIdx.x;
  const int64_t r0 = (int64_t)blockIdx.y * rows_per_block, r1 = min(rows, r0 + rows_per_block);
  float dw[8], db[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) dw[j] = db[j] = 0.f;
#pragma unroll 4
  for (int64_t r = r0 + warp; r < r1; r += NW) {
    float a[8], v[8];
    const float2 st = stats[r];
    load_columns8<T, 32, VEC>(dy + r * dy_stride, slab, lane, dim, a);
    load_columns8<T, 32, VEC>(x + r * stride, slab, lane, dim, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      dw[j] = fmaf(a[j], (v[j] - st.x) * st.y, dw[j]);
      db[j] += a[j];
    }
  }
  for (int side = 0; side < 2; ++side) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) s[warp][column8<32, VEC>(0, lane, j)] = side == 0 ? dw[j] : db[j];
    __syncthreads();
    const int col = slab * 256 + threadIdx.x;
    if (col < dim) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) t += s[k][threadIdx.x];
      partial[((int64_t)blockIdx.y * 2 + side) * dim + col] = t;
    }
  }
}

// All gradients in one pass over dy and x.
template <typename T, bool VEC, int THREADS, int NV>
__global__ void __launch_bounds__(kLnBlock<THREADS>, THREADS > kLnThreads ? 1 : 2)
    castle_layernorm_bwd_kernel(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t stride, const T* __restrict__ w,
                                const float2* __restrict__ stats, T* __restrict__ dx, float* __restrict__ partial, int64_t rows, int dim) {
  constexpr int GROUPS = kLnBlock<THREADS> / THREADS, COLS = THREADS * NV * 8;
  __shared__ float2 s[GROUPS][2 * (THREADS / 32)];
  __shared__ float add[GROUPS > 1 ? GROUPS * COLS : 1];
  const int group = threadIdx.x / THREADS, t = threadIdx.x % THREADS;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  float dw[NV][8], db[NV][8];
  alignas(16) T na[NV][8], nv[NV][8];   // the next row as it lies
  float2 nst = make_float2(0.f, 0.f);
#pragma unroll
  for (int q = 0; q < NV; ++q)
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[q][j] = db[q][j] = 0.f;
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      if constexpr (VEC) {
        const int c = column8<THREADS, true>(q, t, 0);
        if (c < dim) {
          *reinterpret_cast<Raw8<T>*>(na[q]) = *reinterpret_cast<const Raw8<T>*>(dy + r * dy_stride + c);
          *reinterpret_cast<Raw8<T>*>(nv[q]) = *reinterpret_cast<const Raw8<T>*>(x + r * stride + c);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = column8<THREADS, false>(q, t, j);
          if (c < dim) { na[q][j] = dy[r * dy_stride + c]; nv[q][j] = x[r * stride + c]; }
        }
      }
    }
    nst = stats[r];
  };
  int64_t r = (int64_t)blockIdx.x * GROUPS + group;
  if (r < rows) fetch(r);
  for (int turn = 0; r < rows; r += step, turn ^= 1) {
    float a[NV][8], h[NV][8], sg = 0.f, sgh = 0.f;
    const float2 st = nst;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      float g[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = 1.f;
      if (w) load_columns8<T, THREADS, VEC>(w, q, t, dim, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool in = column8<THREADS, VEC>(q, t, j) < dim;
        const float d = in ? load1<T>(&na[q][j]) : 0.f;
        h[q][j] = in ? (load1<T>(&nv[q][j]) - st.x) * st.y : 0.f;
        dw[q][j] = fmaf(d, h[q][j], dw[q][j]);
        db[q][j] += d;
        a[q][j] = d * g[j];
        sg += a[q][j];
        sgh = fmaf(a[q][j], h[q][j], sgh);
      }
    }
    if (r + step < rows) fetch(r + step);
    const float2 sums = group_sum2<THREADS>(sg, sgh, s[group], turn, group);
    const float mg = sums.x / (float)dim, mgh = sums.y / (float)dim;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
#pragma unroll
      for (int j = 0; j < 8; ++j) a[q][j] = st.y * (a[q][j] - mg - h[q][j] * mgh);
      store_columns8<T, THREADS, VEC>(dx + r * dim, q, t, dim, a[q]);
    }
  }
  // the groups' sums, in order
  for (int side = 0; side < 2; ++side) {
    if constexpr (GROUPS > 1) {
      __syncthreads();
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int j = 0; j < 8; ++j) add[group * COLS + column8<THREADS, VEC>(q, t, j)] = side == 0 ? dw[q][j] : db[q][j];
      __syncthreads();
      for (int col = threadIdx.x; col < COLS && col < dim; col += kLnBlock<THREADS>) {
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) sum += add[k * COLS + col];
        partial[((int64_t)blockIdx.x * 2 + side) * dim + col] = sum;
      }
    } else {
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int col = column8<THREADS, VEC>(q, t, j);
          if (col < dim) partial[((int64_t)blockIdx.x * 2 + side) * dim + col] = side == 0 ? dw[q][j] : db[q][j];
        }
    }
  }
}

// blockIdx.y 0: dw, 1: db.  32 columns per block, 8 threads of each adding every eighth part, in a fixed order.
template <typename T>
__global__ void __launch_bounds__(kLnThreads) castle_layernorm_sum_kernel(const float* __restrict__ partial, T* __restrict__ dw, T* __restrict__ db, int parts, int dim) {
  __shared__ float s[8][32];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), k0 = threadIdx.x >> 5;
  T* out = blockIdx.y == 0 ? dw : db;
  overlap_wait();
  if (!out) return;
  float t = 0.f;
  if (col < dim) {
#pragma unroll 8
    for (int k = k0; k < parts; k += 8) t += partial[((int64_t)k * 2 + blockIdx.y) * dim + col];
  }
  s[k0][threadIdx.x & 31] = t;
  __syncthreads();
  if (threadIdx.x < 32 && col < dim) {
#pragma unroll
    for (int k = 1; k < 8; ++k) t += s[k][threadIdx.x];
    store1<T>(out + col, t);
  }
}

static int ln_check(const char* who, int32_t dtype, int64_t rows, int32_t dim) {
  if (dtype < CASTLE_BF16 || dtype > CASTLE_F32) return reject("%s: unknown dtype", who);
  if (rows <= 0 || rows > 2147483647 || dim <= 0 || dim > (1 << 24)) return reject("%s: %lld rows, dim %d not supported", who, (long long)rows, dim);
  return 0;
}

constexpr int kLnWhole = 8192;   // widest row that a group's registers hold

// CTAs of the backward's one pass, or row ranges of dw's own: two per SM, but no more than there are rows for.
static int ln_parts(int64_t rows, int dim) {
  const int64_t most = dim > 4096 ? 148 : 296, have = (rows + 7) / 8;
  return (int)(have < most ? have : most);
}

// f<THREADS, NV>() with the group that holds a row of `dim` columns, 16 or (up to 256) 8 elements a thread
template <typename F> static void ln_group(int dim, F&& f) {
  using std::integral_constant;
  if (dim <= 256) f(integral_constant<int, 32>(), integral_constant<int, 1>());
  else if (dim <= 512) f(integral_constant<int, 32>(), integral_constant<int, 2>());
  else if (dim <= 1024) f(integral_constant<int, 64>(), integral_constant<int, 2>());
  else if (dim <= 2048) f(integral_constant<int, 128>(), integral_constant<int, 2>());
  else if (dim <= 4096) f(integral_constant<int, 256>(), integral_constant<int, 2>());
  else f(integral_constant<int, 512>(), integral_constant<int, 2>());
}

template <typename T, bool VEC>
static cudaError_t ln_fwd(int64_t rows, int dim, const T* x, int64_t stride, const T* w, const T* b, float eps, T* y, float2* stats, cudaStream_t st) {
  if (dim > kLnWhole) {
    castle_layernorm_fwd_wide_kernel<T, VEC><<<(unsigned)rows, kLnThreads, 0, st>>>(x, stride, w, b, eps, y, stats, dim);
  } else {
    ln_group(dim, [&](auto threads, auto nv) {
      constexpr int TH = decltype(threads)::value, G = kLnBlock<TH> / TH;
      castle_layernorm_fwd_kernel<T, VEC, TH, decltype(nv)::value><<<(unsigned)((rows + G - 1) / G), kLnBlock<TH>, 0, st>>>(x, stride, w, b, eps, y, stats, rows, dim);
    });
  }
  return cudaGetLastError();
}

template <typename T, bool VEC>
static cudaError_t ln_bwd(int64_t rows, int dim, const T* dy, int64_t dy_stride, const T* x, int64_t stride, const T* w, const float2* stats, T* dx, T* dw, T* db,
                          float* ws, cudaStream_t st) {
  const int parts = ln_parts(rows, dim);
  const bool params = dw || db;
  if (dx && params && dim <= kLnWhole) {
    ln_group(dim, [&](auto threads, auto nv) {
      constexpr int TH = decltype(threads)::value;
      castle_layernorm_bwd_kernel<T, VEC, TH, decltype(nv)::value><<<parts, kLnBlock<TH>, 0, st>>>(dy, dy_stride, x, stride, w, stats, dx, ws, rows, dim);
    });
  } else {
    if (dx) castle_layernorm_dx_kernel<T, VEC><<<(unsigned)rows, kLnThreads, 0, st>>>(dy, dy_stride, x, stride, w, stats, dx, dim);
    if (params)
      castle_layernorm_dw_kernel<T, VEC><<<dim3((dim + 255) / 256, parts), kLnThreads, 0, st>>>(dy, dy_stride, x, stride, stats, ws, rows, dim, (int)((rows + parts - 1) / parts));
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !params) return e;
  return launch_kernel(castle_layernorm_sum_kernel<T>, dim3((dim + 31) / 32, 2), kLnThreads, 0, st, true, (const float*)ws, dw, db, parts, dim);
}

}  // namespace castle

using namespace castle;

extern "C" int castle_layernorm_fwd(int32_t dtype, int64_t rows, int32_t dim, const void* x, int64_t row_stride, const void* weight, const void* bias, float eps,
                                    void* y, float* stats, void* stream) {
  if (int rc = ln_check("castle_layernorm_fwd", dtype, rows, dim)) return rc;
  const int es = elem_size(dtype);
  if (!x || !y || row_stride < 0 || ((uintptr_t)x | (uintptr_t)y | (uintptr_t)weight | (uintptr_t)bias) % es || (uintptr_t)stats % 8)
    return reject("castle_layernorm_fwd: x and y (aligned to their elements), a stride of at least 0 and stats at a multiple of 8 bytes are needed");
  const bool vec = vec_rows(dtype, dim, row_stride, x, y) && ((uintptr_t)weight | (uintptr_t)bias) % 16 == 0;
  const cudaError_t e = by_type(dtype, [&](auto t) {
    using T = decltype(t);
    return (vec ? ln_fwd<T, true> : ln_fwd<T, false>)(rows, dim, (const T*)x, row_stride, (const T*)weight, (const T*)bias, eps, (T*)y, (float2*)stats, (cudaStream_t)stream);
  });
  return e == cudaSuccess ? 0 : cuda_fail(e, "castle_layernorm_fwd launch");
}

extern "C" size_t castle_layernorm_bwd_workspace_bytes(int64_t rows, int32_t dim) {
  return rows <= 0 || dim <= 0 ? 0 : (size_t)ln_parts(rows, dim) * 2 * dim * sizeof(float);
}

extern "C" int castle_layernorm_bwd(int32_t dtype, int64_t rows, int32_t dim, const void* dy, int64_t dy_stride, const void* x, int64_t row_stride, const void* weight,
                                    const float* stats, void* dx, void* dweight, void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = ln_check("castle_layernorm_bwd", dtype, rows, dim)) return rc;
  const int es = elem_size(dtype);
  if (!dy || !x || !stats || dy_stride < 0 || row_stride < 0 ||
      ((uintptr_t)dy | (uintptr_t)x | (uintptr_t)weight | (uintptr_t)dx | (uintptr_t)dweight | (uintptr_t)dbias) % es || (uintptr_t)stats % 8)
    return reject("castle_layernorm_bwd: dy, x (aligned to their elements, strides of at least 0) and stats at a multiple of 8 bytes are needed");
  if ((dweight || dbias) && (!workspace || (uintptr_t)workspace % 4 || workspace_bytes < castle_layernorm_bwd_workspace_bytes(rows, dim)))
    return reject("castle_layernorm_bwd: workspace too small");
  const bool vec = vec_rows(dtype, dim, row_stride, x, dx) && vec_rows(dtype, dim, dy_stride, dy, weight);
  const cudaError_t e = by_type(dtype, [&](auto t) {
    using T = decltype(t);
    return (vec ? ln_bwd<T, true> : ln_bwd<T, false>)(rows, dim, (const T*)dy, dy_stride, (const T*)x, row_stride, (const T*)weight, (const float2*)stats, (T*)dx,
                                                     (T*)dweight, (T*)dbias, (float*)workspace, (cudaStream_t)stream);
  });
  return e == cudaSuccess ? 0 : cuda_fail(e, "castle_layernorm_bwd launch");
}
