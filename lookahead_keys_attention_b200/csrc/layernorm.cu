// Layer norm, forward and backward, with the reduction of the weight's and the bias's gradient.
//
//   m = mean x, r = 1 / sqrt(mean (x - m)^2 + eps), h = (x - m) r, y = h w + b
//   g = dy w;  dx = r (g - mean g - h mean(g h));  dw = sum over rows dy h;  db = sum over rows dy
//
// All sums are fp32; the variance is taken from the centred values (a second pass over registers, none over memory), since
// mean x^2 - m^2 loses everything where a row's offset is large.
//
// Both directions should be bound by memory (x in and y out; x and dy in and dx out), but 4096 columns of bf16 at 6.5 TB/s leave an SM
// some seven instructions per element: one kernel per row with single arithmetic was bound by instruction issue (32768 rows: 135
// and 174 us, where the bytes take 82 and 123).  So groups of threads (16 elements each, 32 in the widest forward; 32 to 512 threads) stay and take rows in
// turn: the weight (and bias) is unpacked once, arithmetic is on packed pairs, and the rows ahead are on their way into shared memory,
// each thread's columns into places of its own (asynchronous copies that it alone waits for, so nothing has to be synchronised).
// The backward's groups keep their share of dw and db in registers; a CTA leaves one fp32 row of each, and a last launch adds
// these in a fixed order.  Wider rows, and calls that want no dx, take a pass per result that reads its rows from memory (or
// cache) as often as it needs them.
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

// The columns of one thread: NV stretches of eight, as pairs.
template <int NV> struct LnRow { float2 v[NV][4]; };

// Which of them there are: whole stretches (VEC), or single ones.
template <int THREADS, bool VEC> __device__ __forceinline__ bool has_column(int q, int t, int j, int dim) {
  return column8<THREADS, VEC>(q, t, VEC ? 0 : j) < dim;
}

// Rows of COUNT tensors (x, or x and dy) a few ahead of their use: VEC through shared memory, single elements at the time of use.
constexpr int ln_ahead(size_t row_bytes) { return row_bytes * 4 <= 98304 ? 4 : row_bytes * 3 <= 98304 ? 3 : row_bytes * 2 <= 131072 ? 2 : 1; }
template <typename T, bool VEC, int THREADS, int NV, int COUNT> struct LnRows {
  static constexpr int BLOCK = kLnBlock<THREADS>, PARTS = sizeof(Raw8<T>) / 16;
  static constexpr size_t kRow = VEC ? (size_t)COUNT * NV * BLOCK * sizeof(Raw8<T>) : 0;
  static constexpr int AHEAD = VEC ? ln_ahead(kRow) : 1;
  static constexpr size_t kBytes = kRow * AHEAD;
  const T* base[COUNT];
  int64_t stride[COUNT], rows, step;
  uint4* ring;   // [row ahead][tensor][stretch][16-byte part][thread]
  int dim, t, slot;

  __device__ __forceinline__ uint4* place(int s, int which, int q, int part) const { return ring + (((s * COUNT + which) * NV + q) * PARTS + part) * BLOCK + threadIdx.x; }
  __device__ __forceinline__ void fetch(int64_t r, int s) const {
    if constexpr (VEC) {
      if (r < rows) {
#pragma unroll
        for (int q = 0; q < NV; ++q) {
          const int c = column8<THREADS, true>(q, t, 0);
          if (c < dim) {
#pragma unroll
            for (int i = 0; i < COUNT; ++i)
#pragma unroll
              for (int k = 0; k < PARTS; ++k)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(place(s, i, q, k))),
                             "l"(base[i] + r * stride[i] + c + k * (16 / (int)sizeof(T))) : "memory");
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");   // also of nothing, so that groups can be counted
    }
  }
  __device__ __forceinline__ void begin(int64_t r) {
    slot = 0;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) fetch(r + k * step, k);
  }
  // Row r, and the row AHEAD further on is sent for.  Columns that are not there are zero.
  __device__ __forceinline__ void take(int64_t r, LnRow<NV>* out) {
    if constexpr (VEC) asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
#pragma unroll
      for (int q = 0; q < NV; ++q) {
        float f[8];
        if constexpr (VEC) {
          alignas(16) T raw[8];
#pragma unroll
          for (int k = 0; k < PARTS; ++k) reinterpret_cast<uint4*>(raw)[k] = *place(slot, i, q, k);
          load8<T>(raw, f);
          if (!has_column<THREADS, true>(q, t, 0, dim)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = 0.f;
          }
        } else {
          load_columns8<T, THREADS, false>(base[i] + r * stride[i], q, t, dim, f);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) out[i].v[q][j] = make_float2(f[2 * j], f[2 * j + 1]);
      }
    fetch(r + AHEAD * step, slot);
    slot = slot + 1 == AHEAD ? 0 : slot + 1;
  }
};

template <typename T, bool VEC, int THREADS, int NV>
__device__ __forceinline__ void ln_param(const T* p, float none, int t, int dim, LnRow<NV>& out) {
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    float f[8];
    if (p) {
      load_columns8<T, THREADS, VEC>(p, q, t, dim, f);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = none;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) out.v[q][j] = make_float2(f[2 * j], f[2 * j + 1]);
  }
}

template <typename T, bool VEC, int THREADS, int NV>
__device__ __forceinline__ void ln_store(T* row, int t, int dim, const LnRow<NV>& v) {
#pragma unroll
  for (int q = 0; q < NV; ++q) store_columns8<T, THREADS, VEC>(row, q, t, dim, reinterpret_cast<const float*>(v.v[q]));
}

// Columns that are not there become zero again after something was added to them.
template <int THREADS, bool VEC, int NV> __device__ __forceinline__ void ln_clear(int t, int dim, LnRow<NV>& v) {
#pragma unroll
  for (int q = 0; q < NV; ++q)
    if (VEC ? !has_column<THREADS, true>(q, t, 0, dim) : !has_column<THREADS, false>(q, t, 7, dim)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!has_column<THREADS, VEC>(q, t, 2 * j, dim)) v.v[q][j].x = 0.f;
        if (!has_column<THREADS, VEC>(q, t, 2 * j + 1, dim)) v.v[q][j].y = 0.f;
      }
    }
}

// Blocks of an SM.  Rows of more than 4096 columns: two of 256 threads with 32 elements each wait less for each other's sums than one of 512 with 16
// (15063 rows of 8192 in bf16 78 us / 105, of 4824 62 / 97; 8000 of 5000 in fp32 82 / 98).  The registers that this leaves hold all but 8 to 48 bytes a thread
// where single elements are read, with 32 elements 124 to 140; of the backward's, two blocks as well, 56 to 60.
template <int NV> constexpr int kLnFwdBlocks = NV > 2 ? 2 : 3;
template <typename T, bool VEC, int THREADS, int NV>
__global__ void __launch_bounds__(kLnBlock<THREADS>, kLnFwdBlocks<NV>) castle_layernorm_fwd_kernel(
    const T* __restrict__ x, int64_t stride, const T* __restrict__ w, const T* __restrict__ b, float eps, T* __restrict__ y, float2* __restrict__ stats, int64_t rows,
    int dim) {
  constexpr int GROUPS = kLnBlock<THREADS> / THREADS;
  __shared__ float2 s[GROUPS][2 * (THREADS / 32)];
  extern __shared__ __align__(16) uint4 ring[];
  const int group = threadIdx.x / THREADS, t = threadIdx.x % THREADS;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  int64_t r = (int64_t)blockIdx.x * GROUPS + group;
  LnRows<T, VEC, THREADS, NV, 1> in{{x}, {stride}, rows, step, ring, dim, t, 0};
  in.begin(r);
  LnRow<NV> g, c, v;
  ln_param<T, VEC, THREADS, NV>(w, 1.f, t, dim, g);
  ln_param<T, VEC, THREADS, NV>(b, 0.f, t, dim, c);
  const float over = 1.f / (float)dim;
  for (; r < rows; r += step) {
    in.take(r, &v);
    float2 sum = make_float2(0.f, 0.f), sq = sum;
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = add2(sum, v.v[q][j]);
    const float mean = group_sum2<THREADS>(sum.x + sum.y, 0.f, s[group], 0, group).x * over;
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) v.v[q][j] = add2(v.v[q][j], splat(-mean));
    ln_clear<THREADS, VEC, NV>(t, dim, v);
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) sq = fma2(v.v[q][j], v.v[q][j], sq);
    const float rstd = rsqrtf(group_sum2<THREADS>(sq.x + sq.y, 0.f, s[group], 1, group).x * over + eps);
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) v.v[q][j] = fma2(mul2(v.v[q][j], splat(rstd)), g.v[q][j], c.v[q][j]);
    ln_store<T, VEC, THREADS, NV>(y + r * dim, t, dim, v);
    if (stats && t == 0) stats[r] = make_float2(mean, rstd);
  }
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

// dx, rows of any width.
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

// All gradients in one pass over dy and x, or dx alone (`partial` NULL: a thread's sums cost less than a pass without them in another kernel, 46882 x 256 in fp32 40 us, there 127).
template <typename T, bool VEC, int THREADS, int NV>
__global__ void __launch_bounds__(kLnBlock<THREADS>, THREADS > kLnThreads ? 1 : 2)
    castle_layernorm_bwd_kernel(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t stride, const T* __restrict__ w,
                                const float2* __restrict__ stats, T* __restrict__ dx, float* __restrict__ partial, int64_t rows, int dim) {
  constexpr int GROUPS = kLnBlock<THREADS> / THREADS, COLS = THREADS * NV * 8;
  __shared__ float2 s[GROUPS][2 * (THREADS / 32)];
  __shared__ float add[GROUPS > 1 ? GROUPS * COLS : 1];
  extern __shared__ __align__(16) uint4 ring[];
  const int group = threadIdx.x / THREADS, t = threadIdx.x % THREADS;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  int64_t r = (int64_t)blockIdx.x * GROUPS + group;
  LnRows<T, VEC, THREADS, NV, 2> in{{x, dy}, {stride, dy_stride}, rows, step, ring, dim, t, 0};
  in.begin(r);
  LnRow<NV> g, dw, db;
  ln_param<T, VEC, THREADS, NV>(w, 1.f, t, dim, g);
#pragma unroll
  for (int q = 0; q < NV; ++q)
#pragma unroll
    for (int j = 0; j < 4; ++j) dw.v[q][j] = db.v[q][j] = make_float2(0.f, 0.f);
  float2 next = r < rows ? stats[r] : make_float2(0.f, 0.f);
  const float over = 1.f / (float)dim;
  for (int turn = 0; r < rows; r += step, turn ^= 1) {
    LnRow<NV> v[2];   // x, then h; dy, then dy w
    const float2 st = next;
    if (r + step < rows) next = stats[r + step];
    in.take(r, v);
    float2 sg = make_float2(0.f, 0.f), sgh = sg;
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 h = mul2(add2(v[0].v[q][j], splat(-st.x)), splat(st.y)), d = v[1].v[q][j];   // (dy is zero where there is no column)
        dw.v[q][j] = fma2(d, h, dw.v[q][j]);
        db.v[q][j] = add2(db.v[q][j], d);
        const float2 a = mul2(d, g.v[q][j]);
        sg = add2(sg, a);
        sgh = fma2(a, h, sgh);
        v[0].v[q][j] = h;
        v[1].v[q][j] = a;
      }
    const float2 sums = group_sum2<THREADS>(sg.x + sg.y, sgh.x + sgh.y, s[group], turn, group);
    const float2 mg = splat(-sums.x * over), mgh = splat(-sums.y * over);
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[1].v[q][j] = mul2(fma2(v[0].v[q][j], mgh, add2(v[1].v[q][j], mg)), splat(st.y));
    ln_store<T, VEC, THREADS, NV>(dx + r * dim, t, dim, v[1]);
  }
  if (!partial) return;   // dx alone
  // the groups' sums, in order
  for (int side = 0; side < 2; ++side) {
    if constexpr (GROUPS > 1) {
      __syncthreads();
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int j = 0; j < 8; ++j) add[group * COLS + column8<THREADS, VEC>(q, t, j)] = reinterpret_cast<const float*>(side == 0 ? dw.v[q] : db.v[q])[j];
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
          if (col < dim) partial[((int64_t)blockIdx.x * 2 + side) * dim + col] = reinterpret_cast<const float*>(side == 0 ? dw.v[q] : db.v[q])[j];
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
  const int64_t most = dim > 4096 ? 148 : 296, have = (rows + 3) / 4;
  return (int)(have < most ? have : most);
}

// f(THREADS, NV) with the group that holds a row of `dim` columns, 8 NV elements a thread; rows beyond 4096 columns have WIDE threads of 8 WIDE_NV elements.
template <int WIDE, int WIDE_NV, typename F> static cudaError_t ln_group(int dim, F&& f) {
  using std::integral_constant;
  if (dim <= 256) return f(integral_constant<int, 32>(), integral_constant<int, 1>());
  if (dim <= 512) return f(integral_constant<int, 32>(), integral_constant<int, 2>());
  if (dim <= 1024) return f(integral_constant<int, 64>(), integral_constant<int, 2>());
  if (dim <= 2048) return f(integral_constant<int, 128>(), integral_constant<int, 2>());
  if (dim <= 4096) return f(integral_constant<int, 256>(), integral_constant<int, 2>());
  return f(integral_constant<int, WIDE>(), integral_constant<int, WIDE_NV>());
}
template <typename K, typename... A> static cudaError_t ln_launch(K kernel, int64_t grid, int threads, size_t ring, cudaStream_t st, A... args) {
  if (ring > 16384) {   // (beside up to 17 KB of the kernel's own)
    const cudaError_t e = allow_smem(kernel, (int)ring);
    if (e != cudaSuccess) return e;
  }
  kernel<<<(unsigned)grid, threads, ring, st>>>(args...);
  return cudaGetLastError();
}

template <typename T, bool VEC>
static cudaError_t ln_fwd(int64_t rows, int dim, const T* x, int64_t stride, const T* w, const T* b, float eps, T* y, float2* stats, cudaStream_t st) {
  if (dim > kLnWhole) {
    castle_layernorm_fwd_wide_kernel<T, VEC><<<(unsigned)rows, kLnThreads, 0, st>>>(x, stride, w, b, eps, y, stats, dim);
    return cudaGetLastError();
  }
  return ln_group<256, 4>(dim, [&](auto threads, auto nv) {
    constexpr int TH = decltype(threads)::value, NV = decltype(nv)::value, G = kLnBlock<TH> / TH;
    const int64_t have = (rows + G - 1) / G, most = 148 * kLnFwdBlocks<NV>;
    return ln_launch(castle_layernorm_fwd_kernel<T, VEC, TH, NV>, have < most ? have : most, kLnBlock<TH>, LnRows<T, VEC, TH, NV, 1>::kBytes, st, x, stride, w, b, eps, y,
                     stats, rows, dim);
  });
}

template <typename T, bool VEC>
static cudaError_t ln_bwd(int64_t rows, int dim, const T* dy, int64_t dy_stride, const T* x, int64_t stride, const T* w, const float2* stats, T* dx, T* dw, T* db,
                          float* ws, cudaStream_t st) {
  const int parts = ln_parts(rows, dim);
  const bool params = dw || db;
  if (dx && dim <= kLnWhole) {
    const cudaError_t e = ln_group<512, 2>(dim, [&](auto threads, auto nv) {
      constexpr int TH = decltype(threads)::value, NV = decltype(nv)::value;
      return ln_launch(castle_layernorm_bwd_kernel<T, VEC, TH, NV>, parts, kLnBlock<TH>, LnRows<T, VEC, TH, NV, 2>::kBytes, st, dy, dy_stride, x, stride, w, stats, dx,
                       params ? ws : (float*)nullptr, rows, dim);
    });
    if (e != cudaSuccess) return e;
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
