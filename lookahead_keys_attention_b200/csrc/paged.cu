// Cached single-token CASTLE step over caches in pages, for sequences of different lengths (HBM-bound).
//
// For each sequence b with L = lengths[b] positions, and each head (rows of d, scale s):
//
//     a_k = sigmoid(s qu_k . ku)      U_k <- round(U_k + a_k vu)      S_k = s qc . kc_k - silu(s qc . U_k)      k < L
//     S_L = s qc . kc_new             out = softmax(S) . (vc, vc_new)
//
// and row L is appended to the four caches (a zero row to U).  A row is in page table[b][k / page], at place k % page of it.  qu, kc and
// vc rows never change once they are written, so sequences may share their pages; U's are one sequence's own, hence a table of their own.
//
// The lengths are known to the device alone, so every CTA works out the same plan from them: the rows of all (sequence, head) pairs are
// tiles of kRows, laid end to end, and cut into `pieces` of equal size whatever the pairs' ends.  CTA i takes pieces i, i + grid, ...: all
// CTAs have the same work, and at any time neighbouring ones read neighbouring memory.  A pair inside one piece is finished by its CTA;
// one that is cut leaves a partial (maximum, sum, weighted values) per piece, and the CTA that leaves the last one joins them in order.
#include <algorithm>
#include "common.cuh"
#include "decode_row.cuh"
#include "vec.cuh"

namespace castle {

constexpr int kPagedThreads = 128, kPagedWarps = kPagedThreads / 32;
constexpr int kPagedCtas = 4;                       // per SM
constexpr int kPagedGrid = 148 * kPagedCtas;
constexpr int kPagedMaxBatch = 4096;
constexpr int kPagedPieceTiles = 64, kPagedMaxRounds = 32;   // tiles of a piece; pieces of a CTA

// Rows of a tile: 4 KB of each cache, at least 16.
template <typename T, int D> struct PagedRows { static constexpr int fit = 4096 / (D * (int)sizeof(T)), value = fit > 16 ? fit : 16; };
static int paged_rows(int dtype, int d) { return std::max(16, 4096 / (d * elem_size(dtype))); }

struct PagedParams {
  castle_tensor_t qc, kc, vc, qu, ku, vu, out;
  castle_pages_t U, quc, kcc, vcc;
  const int32_t *u_table, *table, *lengths;
  int64_t u_table_stride, table_stride;
  int B, H, page_shift, capacity;   // capacity: positions that the tables have places for
  int u_pages, pages;
  float scale;
  RotaryParams rot;
  float* part;                      // [2 per piece][2 + D]
  uint32_t* counters;               // [B * H], zero
  int32_t* status;
};

// Where a pair's rows lie and what a piece has of them.
struct PagedSegment {
  int b, h, length, tile0, tiles, all;   // tiles [tile0, tile0 + tiles) of the pair's `all`
  int64_t first;                         // the pair's first tile among all pairs' tiles
};
struct PagedPlan {
  int64_t tiles;   // of all pairs
  int pieces;
};

// start[b] = tiles before sequence b, for the whole CTA; a sequence without positions has a tile without rows (its new row is attended to),
// one that is not there (length < 0) or does not fit has none.
template <int THREADS> __device__ __forceinline__ PagedPlan paged_plan(const PagedParams& p, int rows, int* start) {
  __shared__ int warp_sum[THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0;
  for (int b0 = 0; b0 < p.B; b0 += THREADS) {
    const int b = b0 + threadIdx.x;
    const int length = b < p.B ? p.lengths[b] : -1;
    int n = length < 0 || length >= p.capacity ? 0 : max(1, (length + rows - 1) / rows) * p.H;
    const int own = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int below = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += below;
    }
    if (lane == 31) warp_sum[warp] = n;
    __syncthreads();
    int ahead = before, total = before;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) ahead += warp_sum[w];
      total += warp_sum[w];
    }
    if (b < p.B) start[b] = ahead + n - own;
    before = total;
    __syncthreads();
  }
  if (threadIdx.x == 0) start[p.B] = before;
  __syncthreads();
  PagedPlan plan;
  plan.tiles = before;
  // two tiles at least, where there is less than that for every CTA; else equal shares of at most kPagedPieceTiles
  plan.pieces = before <= 2 * kPagedGrid ? (before + 1) / 2
                                         : kPagedGrid * min(kPagedMaxRounds, (before - 1) / (kPagedGrid * kPagedPieceTiles) + 1);
  return plan;
}
__device__ __forceinline__ int64_t piece_begin(const PagedPlan& plan, int piece) { return piece * plan.tiles / plan.pieces; }
__device__ __forceinline__ int piece_of(const PagedPlan& plan, int64_t tile) { return (int)(((tile + 1) * plan.pieces - 1) / plan.tiles); }

// The part of a pair that begins at tile `at` and ends with the pair or before `end`.
__device__ __forceinline__ PagedSegment paged_segment(const PagedParams& p, const int* start, int64_t at, int64_t end) {
  int lo = 0, hi = p.B;   // start[lo] <= at < start[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= at) lo = mid; else hi = mid;
  }
  PagedSegment s;
  s.b = lo;
  s.length = p.lengths[lo];
  s.all = (start[lo + 1] - start[lo]) / p.H;
  const int in = (int)at - start[lo];
  s.h = in / s.all;
  s.tile0 = in - s.h * s.all;
  s.tiles = (int)min((int64_t)(s.all - s.tile0), end - at);
  s.first = at - s.tile0;
  return s;
}

template <typename T> __device__ __forceinline__ T* page_row(const castle_pages_t& t, int page, int h, int row, int d) {
  return reinterpret_cast<T*>(t.ptr) + page * t.stride_page + h * t.stride_h + (int64_t)row * d;
}
template <typename T> __device__ __forceinline__ T* new_row(const castle_tensor_t& t, int b, int h) {
  return reinterpret_cast<T*>(t.ptr) + b * t.stride_b + h * t.stride_h;
}
template <typename T> __device__ __forceinline__ void paged_store_out(const PagedParams& p, int b, int h, int c, float v) { store1<T>(new_row<T>(p.out, b, h) + c, v); }

// What a thread has summed up of its rows.
template <int VEC> struct Softmax {
  float m, l, acc[VEC];
  __device__ __forceinline__ void clear() {
    m = -INFINITY; l = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
  }
  __device__ __forceinline__ void add(float s, const float* v) {
    const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.f : mn;   // (scores of minus infinity alone weigh nothing)
    const float corr = __expf(m - ref), pe = __expf(s - ref);
    l = l * corr + pe;
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = acc[i] * corr + pe * v[i];
    m = mn;
  }
};

// Joins the parts of a pair: D columns x (threads / D) groups of parts.
template <typename T, int D> __device__ __forceinline__ void paged_join(const PagedParams& p, const PagedPlan& plan, const PagedSegment& s, int first_piece, int parts) {
  constexpr int G = kPagedThreads / D;
  __shared__ float s_red[2][kPagedWarps], s_sum[G][D];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto part = [&](int i) { return p.part + (int64_t)(2 * (first_piece + i) + (i == 0 ? 1 : 0)) * (2 + D); };
  float mm = -INFINITY;
  for (int i = tid; i < parts; i += kPagedThreads) mm = fmaxf(mm, __ldcg(part(i)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  if (lane == 0) s_red[0][warp] = mm;
  group_sync(1);
#pragma unroll
  for (int w = 0; w < kPagedWarps; ++w) mm = fmaxf(mm, s_red[0][w]);
  const float ref = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f;
  for (int i = tid; i < parts; i += kPagedThreads) ll += __ldcg(part(i) + 1) * __expf(__ldcg(part(i)) - ref);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, o);
  if (lane == 0) s_red[1][warp] = ll;
  const int c = tid % D, g = tid / D;
  float a = 0.f;
#pragma unroll 8
  for (int i = g; i < parts; i += G) a += __ldcg(part(i) + 2 + c) * __expf(__ldcg(part(i)) - ref);
  s_sum[g][c] = a;
  group_sync(1);
  ll = 0.f;
#pragma unroll
  for (int w = 0; w < kPagedWarps; ++w) ll += s_red[1][w];
  if (g == 0) {
#pragma unroll
    for (int k = 1; k < G; ++k) a += s_sum[k][c];
    paged_store_out<T>(p, s.b, s.h, c, a / ll);
  }
  group_sync(1);
}

// The end of a segment: the lane groups of a warp, then the warps; the result, or a partial and, if it is the pair's last, the join.
template <typename T, int D>
__device__ __forceinline__ void paged_finish(const PagedParams& p, const PagedPlan& plan, const PagedSegment& s, int piece, Softmax<Vec<T>::N>& x) {
  constexpr int VEC = Vec<T>::N, LPR = D / VEC;
  __shared__ float s_m[kPagedWarps], s_l[kPagedWarps], s_acc[kPagedWarps][D];
  __shared__ bool s_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane % LPR, grp = lane / LPR;
#pragma unroll
  for (int o = LPR; o < 32; o <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, x.m, o), l2 = __shfl_xor_sync(0xffffffffu, x.l, o);
    const float mn = fmaxf(x.m, m2), ref = mn == -INFINITY ? 0.f : mn;
    const float c1 = __expf(x.m - ref), c2 = __expf(m2 - ref);
    x.l = x.l * c1 + l2 * c2;
#pragma unroll
    for (int i = 0; i < VEC; ++i) x.acc[i] = x.acc[i] * c1 + __shfl_xor_sync(0xffffffffu, x.acc[i], o) * c2;
    x.m = mn;
  }
  if (grp == 0) {
    if (sub == 0) { s_m[warp] = x.m; s_l[warp] = x.l; }
#pragma unroll
    for (int i = 0; i < VEC; ++i) s_acc[warp][sub * VEC + i] = x.acc[i];
  }
  group_sync(1);
  const bool whole = s.tiles == s.all;
  if (threadIdx.x < D) {
    float mm = -INFINITY, ll = 0.f, aa = 0.f;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) mm = fmaxf(mm, s_m[w]);
    const float ref = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) {
      const float c = __expf(s_m[w] - ref);
      ll += s_l[w] * c;
      aa += s_acc[w][threadIdx.x] * c;
    }
    if (whole) {
      paged_store_out<T>(p, s.b, s.h, threadIdx.x, aa / ll);
    } else {
      float* dst = p.part + (int64_t)(2 * piece + (s.tile0 == 0 ? 1 : 0)) * (2 + D);
      if (threadIdx.x == 0) { dst[0] = mm; dst[1] = ll; }
      dst[2 + threadIdx.x] = aa;
    }
  }
  if (whole) {
    group_sync(1);   // before the next segment writes s_m, s_acc
    return;
  }
  __threadfence();
  group_sync(1);
  const int first = piece_of(plan, s.first), parts = piece_of(plan, s.first + s.all - 1) - first + 1;
  if (threadIdx.x == 0) {
    uint32_t* counter = p.counters + s.b * p.H + s.h;
    s_last = atomicAdd(counter, 1u) == (uint32_t)parts - 1;
    if (s_last) *counter = 0;   // ready for the next launch
  }
  group_sync(1);
  if (!s_last) return;
  __threadfence();
  paged_join<T, D>(p, plan, s, first, parts);
}

// Sequences without tiles: zeros where there is none, NaN (and a status) where the length has no places in the tables.
template <typename T, int D> __device__ __forceinline__ void paged_outside(const PagedParams& p) {
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    const int length = p.lengths[b];
    if (length >= 0 && length < p.capacity) continue;
    for (int i = threadIdx.x; i < p.H * D; i += blockDim.x) paged_store_out<T>(p, b, i / D, i % D, length < 0 ? 0.f : __int_as_float(0x7fc00000));
    if (length >= 0 && threadIdx.x == 0) atomicOr(p.status, CASTLE_STATUS_BAD_INDEX);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kPagedThreads, kPagedCtas) castle_paged_step_kernel(const PagedParams p) {
  constexpr int VEC = Vec<T>::N, LPR = D / VEC, RPW = 32 / LPR, ROWS = PagedRows<T, D>::value;
  extern __shared__ __align__(16) int start[];
  overlap_next();
  overlap_wait();
  const PagedPlan plan = paged_plan<kPagedThreads>(p, ROWS, start);
  paged_outside<T, D>(p);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane % LPR, grp = lane / LPR, col = sub * VEC, mask = (1 << p.page_shift) - 1;
  for (int piece = blockIdx.x; piece < plan.pieces; piece += gridDim.x) {
    const int64_t end = piece_begin(plan, piece + 1);
    for (int64_t at = piece_begin(plan, piece); at < end;) {
      const PagedSegment s = paged_segment(p, start, at, end);
      at += s.tiles;
      const int32_t *ut = p.u_table + s.b * p.u_table_stride, *kt = p.table + s.b * p.table_stride;
      RotaryParams rot = p.rot;
      rot.position0 = (float)s.length;
      float qcv[VEC], kuv[VEC], vuv[VEC];
      Vec<T>::load(new_row<T>(p.qc, s.b, s.h) + col, qcv);
      Vec<T>::load(new_row<T>(p.ku, s.b, s.h) + col, kuv);
      Vec<T>::load(new_row<T>(p.vu, s.b, s.h) + col, vuv);
      rotate_new<T>(rot, col, qcv, kuv, vuv);
#pragma unroll
      for (int i = 0; i < VEC; ++i) { qcv[i] *= p.scale; kuv[i] *= p.scale; }
      Softmax<VEC> x;
      x.clear();
      bool bad = false;
      const int r_end = min(s.length, (s.tile0 + s.tiles) * ROWS);
      for (int base = s.tile0 * ROWS + warp * RPW; base < r_end; base += RPW * kPagedWarps) {   // (uniform in the warp)
        const int r = base + grp;
        bool live = r < r_end;
        float quv[VEC], uv[VEC], kv[VEC], vv[VEC];
        T* u = nullptr;
        if (live) {
          const int up = ut[r >> p.page_shift], kp = kt[r >> p.page_shift];
          if ((uint32_t)up >= (uint32_t)p.u_pages || (uint32_t)kp >= (uint32_t)p.pages) {
            bad = true;
            live = false;
          } else {
            const int in = r & mask;
            u = page_row<T>(p.U, up, s.h, in, D) + col;
            Vec<T>::load(page_row<T>(p.quc, kp, s.h, in, D) + col, quv);
            Vec<T>::load(u, uv);
            Vec<T>::load(page_row<T>(p.kcc, kp, s.h, in, D) + col, kv);
            Vec<T>::load(page_row<T>(p.vcc, kp, s.h, in, D) + col, vv);
          }
        }
        float z = 0.f, sc = 0.f, su = 0.f;
        if (live) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) z += quv[i] * kuv[i];
        }
        z = group_sum<LPR>(z);
        const float a = sigmoid_f(z);
        if (live) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) uv[i] += a * vuv[i];
          Vec<T>::round(uv);
          Vec<T>::store(u, uv);
#pragma unroll
          for (int i = 0; i < VEC; ++i) { sc += qcv[i] * kv[i]; su += qcv[i] * uv[i]; }
        }
        sc = group_sum<LPR>(sc);
        su = group_sum<LPR>(su);
        if (live) x.add(sc - su * sigmoid_f(su), vv);
      }
      if (s.tile0 + s.tiles == s.all && warp == 0) {   // the appended row; its U is zero, so its score is qc . kc_new alone
        float kn[VEC], vn[VEC], qn[VEC], zero[VEC];
        Vec<T>::load(new_row<T>(p.kc, s.b, s.h) + col, kn);
        Vec<T>::load(new_row<T>(p.vc, s.b, s.h) + col, vn);
        Vec<T>::load(new_row<T>(p.qu, s.b, s.h) + col, qn);
        rotate_new<T>(rot, col, kn, qn, nullptr);
#pragma unroll
        for (int i = 0; i < VEC; ++i) zero[i] = 0.f;
        const int up = ut[s.length >> p.page_shift], kp = kt[s.length >> p.page_shift], in = s.length & mask;
        const bool there = (uint32_t)up < (uint32_t)p.u_pages && (uint32_t)kp < (uint32_t)p.pages;
        bad |= !there;
        if (grp == 0 && there) {
          Vec<T>::store(page_row<T>(p.kcc, kp, s.h, in, D) + col, kn);
          Vec<T>::store(page_row<T>(p.vcc, kp, s.h, in, D) + col, vn);
          Vec<T>::store(page_row<T>(p.quc, kp, s.h, in, D) + col, qn);
          Vec<T>::store(page_row<T>(p.U, up, s.h, in, D) + col, zero);
        }
        float sc = 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) sc += qcv[i] * kn[i];
        sc = group_sum<LPR>(sc);
        if (grp == 0) x.add(sc, vn);
      }
      if (bad) {
        x.l = __int_as_float(0x7fc00000);
        atomicOr(p.status, CASTLE_STATUS_BAD_INDEX);
      }
      paged_finish<T, D>(p, plan, s, piece, x);
    }
  }
}

template <typename T, int D> static int launch_paged(const PagedParams& p, cudaStream_t st) {
  const size_t smem = (size_t)(p.B + 1) * sizeof(int);
  ev_start(CASTLE_KERNEL_DECODE, st);
  const cudaError_t e = launch_kernel(castle_paged_step_kernel<T, D>, dim3(kPagedGrid), kPagedThreads, smem, st, false, p);
  if (e != cudaSuccess) return cuda_fail(e, "castle_paged_decode_step launch");
  ev_stop(CASTLE_KERNEL_DECODE, st);
  return 0;
}
template <typename T> static int launch_paged_d(const PagedParams& p, int D, cudaStream_t st) {
  switch (D) {
    case 16: return launch_paged<T, 16>(p, st);
    case 32: return launch_paged<T, 32>(p, st);
    case 64: return launch_paged<T, 64>(p, st);
    default: return launch_paged<T, 128>(p, st);
  }
}

// Tiles of all pairs if every sequence filled its places; -1 where they or the sizes are out of range.
static int64_t paged_most_tiles(const castle_problem_t* p, int32_t page_size, int32_t table_width) {
  if (!p || p->batch <= 0 || p->batch > kPagedMaxBatch || p->heads <= 0 || page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) || table_width <= 0) return -1;
  if (p->dtype < CASTLE_BF16 || p->dtype > CASTLE_F32 || (p->dim_head != 16 && p->dim_head != 32 && p->dim_head != 64 && p->dim_head != 128)) return -1;
  const int64_t capacity = (int64_t)table_width * page_size, rows = paged_rows(p->dtype, p->dim_head);
  const int64_t pairs = (int64_t)p->batch * p->heads;
  if (capacity > INT32_MAX - 1024 || pairs > INT32_MAX) return -1;
  const int64_t each = (capacity + rows - 1) / rows;
  return each > INT32_MAX / pairs ? -1 : each * pairs;
}
// The most pieces that a call with so many tiles or fewer has (their number grows with the tiles').
static int64_t paged_most_pieces(int64_t tiles) {
  return tiles <= 2 * kPagedGrid ? (tiles + 1) / 2 : kPagedGrid * std::min<int64_t>(kPagedMaxRounds, (tiles - 1) / (kPagedGrid * kPagedPieceTiles) + 1);
}

}  // namespace castle

using namespace castle;

extern "C" size_t castle_paged_decode_workspace_bytes(const castle_problem_t* p, int32_t page_size, int32_t table_width) {
  const int64_t tiles = paged_most_tiles(p, page_size, table_width);
  return tiles < 0 ? 0 : (size_t)paged_most_pieces(tiles) * 2 * (2 + p->dim_head) * sizeof(float);
}

extern "C" int castle_paged_decode_step(const castle_problem_t* p, int32_t page_size, int32_t u_pages, int32_t pages, const castle_tensor_t* qc_new,
                                        const castle_tensor_t* kc_new, const castle_tensor_t* vc_new, const castle_tensor_t* qu_new, const castle_tensor_t* ku_new,
                                        const castle_tensor_t* vu_new, const castle_pages_t* u_cache, const castle_pages_t* qu_cache, const castle_pages_t* kc_cache,
                                        const castle_pages_t* vc_cache, const int32_t* u_table, int64_t u_table_stride, const int32_t* table, int64_t table_stride,
                                        int32_t table_width, const int32_t* lengths, const castle_tensor_t* out, const castle_rotary_t* rotary, uint32_t* counters,
                                        void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  const char* who = "castle_paged_decode_step";
  if (!p) return reject("%s: null problem", who);
  if (p->batch <= 0 || p->batch > kPagedMaxBatch || p->heads <= 0) return reject("%s: 1 to %d sequences and at least one head expected", who, kPagedMaxBatch);
  if (p->dtype < CASTLE_BF16 || p->dtype > CASTLE_F32) return reject("%s: unknown dtype %d", who, p->dtype);
  if (p->dim_head != 16 && p->dim_head != 32 && p->dim_head != 64 && p->dim_head != 128) return reject("%s: dim_head %d not supported (16, 32, 64, 128)", who, p->dim_head);
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return reject("%s: page size %d is not a power of two from 16 to 1024", who, page_size);
  if (u_pages <= 0 || pages <= 0 || table_width <= 0) return reject("%s: empty pools or tables", who);
  if (paged_most_tiles(p, page_size, table_width) < 0) return reject("%s: %d sequences x %d heads x %d pages are too many positions", who, p->batch, p->heads, table_width);
  if (!u_table || !table || !lengths || !counters || !status) return reject("%s: null table, lengths, counters or status", who);
  if (((uintptr_t)u_table | (uintptr_t)table | (uintptr_t)lengths | (uintptr_t)counters | (uintptr_t)status | (uintptr_t)workspace) % 4)
    return reject("%s: tables, lengths, counters, workspace and status must be 4-byte aligned", who);
  if (u_table_stride < 0 || table_stride < 0) return reject("%s: negative table strides", who);
  int rc = 0;
  const castle_tensor_t* ts[7] = {qc_new, kc_new, vc_new, qu_new, ku_new, vu_new, out};
  const char* names[7] = {"qc_new", "kc_new", "vc_new", "qu_new", "ku_new", "vu_new", "out"};
  for (int i = 0; i < 7; ++i)
    if (!tensor_ok(ts[i], p->dtype, names[i], &rc)) return rc;
  const castle_pages_t* ps[4] = {u_cache, qu_cache, kc_cache, vc_cache};
  const char* page_names[4] = {"u_cache", "qu_cache", "kc_cache", "vc_cache"};
  const int es = elem_size(p->dtype);
  for (int i = 0; i < 4; ++i) {
    if (!ps[i] || !ps[i]->ptr) return reject("%s: null tensor", page_names[i]);
    if ((uintptr_t)ps[i]->ptr % 16 || ps[i]->stride_page * es % 16 || ps[i]->stride_h * es % 16)
      return reject("%s: the base pointer and the strides must be multiples of 16 bytes", page_names[i]);
  }
  const size_t bytes = castle_paged_decode_workspace_bytes(p, page_size, table_width);
  if (!workspace || workspace_bytes < bytes) return reject("%s: workspace too small (%zu < %zu bytes)", who, workspace_bytes, bytes);
  PagedParams q;
  q.qc = *qc_new; q.kc = *kc_new; q.vc = *vc_new; q.qu = *qu_new; q.ku = *ku_new; q.vu = *vu_new; q.out = *out;
  q.U = *u_cache; q.quc = *qu_cache; q.kcc = *kc_cache; q.vcc = *vc_cache;
  q.u_table = u_table; q.table = table; q.lengths = lengths; q.u_table_stride = u_table_stride; q.table_stride = table_stride;
  q.B = p->batch; q.H = p->heads; q.capacity = table_width * page_size; q.u_pages = u_pages; q.pages = pages; q.scale = p->scale;
  q.page_shift = 0;
  while ((1 << q.page_shift) < page_size) ++q.page_shift;
  q.rot = RotaryParams{nullptr, CASTLE_F32, 0, 0.f};
  if (rotary && rotary->freqs) {
    if (rotary->dtype < CASTLE_BF16 || rotary->dtype > CASTLE_F32) return reject("%s: unknown rotary dtype", who);
    q.rot = RotaryParams{rotary->freqs, rotary->dtype, rotary->inverse, 0.f};
  }
  q.part = (float*)workspace; q.counters = counters; q.status = status;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (p->dtype) {
    case CASTLE_BF16: return launch_paged_d<__nv_bfloat16>(q, p->dim_head, st);
    case CASTLE_F16: return launch_paged_d<__half>(q, p->dim_head, st);
    default: return launch_paged_d<float>(q, p->dim_head, st);
  }
}
