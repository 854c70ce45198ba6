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
// tiles of a few rows, laid end to end, and cut into pieces of equal size, one for each CTA of a wave, whatever the pairs' ends.  A pair
// inside one piece is finished by its CTA; one that is cut leaves a partial (maximum, sum, weighted values) per piece, and the CTA that
// leaves the last one joins them in order.  (Pieces of at most n tiles instead, several of them to a CTA, n = 16 / 32 / 64 / 128, us of
// a step: 64 ragged sequences of 8.2 thousand positions on average, 16 heads of 128 bf16, 2478 / 2055 / 1864 / 1807, one piece each 1754;
// one sequence of 131071, 16 heads of 128 fp16, 1218 / 688 / 561 / 484, one piece each 446: the ends cost more than neighbouring CTAs gain
// that read neighbouring memory.  Pages in random order or one behind the other: no difference.)
#include <algorithm>
#include "common.cuh"
#include "decode_row.cuh"
#include "vec.cuh"

namespace castle {

constexpr int kPagedThreads = 128, kPagedWarps = kPagedThreads / 32;
constexpr int kPagedCtas = 4, kPagedSms = 148;       // CTAs of an SM at most
constexpr int kPagedSmem = 228 * 1024, kPagedStatic = 3 * 1024 + 512;   // an SM's shared memory; a CTA's beside the dynamic part, the system's 1 KB included
constexpr int kPagedMaxBatch = 4096;

// Rows of a tile: 4 KB of each cache, at least 8.
template <typename T, int D> struct PagedRows { static constexpr int fit = 4096 / (D * (int)sizeof(T)), value = fit > 8 ? fit : 8; };
static int paged_rows(int dtype, int d) { return std::max(8, 4096 / (d * elem_size(dtype))); }

struct PagedParams {
  castle_tensor_t qc, kc, vc, qu, ku, vu, out;
  castle_pages_t U, quc, kcc, vcc;
  const int32_t *u_table, *table, *lengths;
  int64_t u_table_stride, table_stride;
  int B, H, page_shift, capacity;   // capacity: positions that the tables have places for
  int u_pages, pages;
  float scale;
  RotaryParams rot;
  float* part;                      // [2 per piece][4 + D]: D sums, the maximum, the sum of the weights
  uint32_t* counters;               // [B * H], zero
  int32_t* status;
  uint32_t row_polls;               // of a wait for rows, see castle_selftest_paged_polls
};

// Where a pair's rows lie and what a piece has of them.
struct PagedSegment {
  int b, h, length, tile0, tiles, all;   // tiles [tile0, tile0 + tiles) of the pair's `all`
  int first, next;                       // the pair's first tile among all pairs' units; where the piece goes on
};
struct PagedPlan {   // pieces of `each` units, the first `more` of them of one more
  int pieces, each, more;
};
// A pair counts as its tiles and kPagedPair units ahead of them, for its new rows and its end.  us of a step with 0 / 1 / 2 / 3 / 4 of them,
// bf16: 256 sequences of 40 positions on average, 16 heads of 128, 69.6 / 56.2 / 56.1 / 57.3 / 60.1; 256 of 300 273 / 271 / 269 / 273 / 273; 16 of up to 1024, 8
// heads of 64, 13.3 / 12.4 / 11.7 / 11.6 / 11.9.
constexpr int kPagedPair = 2;

// start[b] = units before sequence b, and the lengths, for the whole CTA; a sequence without positions has a tile without rows (its new row is attended to),
// one that is not there (length < 0) or does not fit has none.
template <int THREADS> __device__ __forceinline__ PagedPlan paged_plan(const PagedParams& p, int rows, int* start, int* lengths) {
  __shared__ int warp_sum[THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0;
  for (int b0 = 0; b0 < p.B; b0 += THREADS) {
    const int b = b0 + threadIdx.x;
    const int length = b < p.B ? p.lengths[b] : -1;
    int n = length < 0 || length >= p.capacity ? 0 : (max(1, (length + rows - 1) / rows) + kPagedPair) * p.H;
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
    if (b < p.B) { start[b] = ahead + n - own; lengths[b] = length; }
    before = total;
    __syncthreads();
  }
  if (threadIdx.x == 0) start[p.B] = before;
  __syncthreads();
  PagedPlan plan;
  plan.pieces = min((int)gridDim.x, before);
  plan.each = plan.pieces > 0 ? before / plan.pieces : 0;
  plan.more = before - plan.each * plan.pieces;
  return plan;
}
__device__ __forceinline__ int piece_begin(const PagedPlan& plan, int piece) { return piece * plan.each + min(piece, plan.more); }
__device__ __forceinline__ int piece_of(const PagedPlan& plan, int tile) {
  const int large = plan.more * (plan.each + 1);
  return tile < large ? tile / (plan.each + 1) : plan.more + (tile - large) / plan.each;
}

// The part of a pair that begins at tile `at` and ends with the pair or before `end`.
template <int ROWS> __device__ __forceinline__ PagedSegment paged_segment(const PagedParams& p, const int* start, const int* lengths, int at, int end) {
  int lo = 0, hi = p.B;   // start[lo] <= at < start[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= at) lo = mid; else hi = mid;
  }
  PagedSegment s;
  s.b = lo;
  s.length = lengths[lo];
  s.all = max(1, (s.length + ROWS - 1) / ROWS);
  const int pair = s.all + kPagedPair, in = at - start[lo];
  s.h = in / pair;
  const int from = in - s.h * pair - kPagedPair, to = min(s.all, from + end - at);   // in the pair's tiles; below zero: in front of them
  s.tile0 = max(0, from);
  s.tiles = max(0, to - s.tile0);
  s.first = at - from;
  s.next = s.first + to;
  return s;
}

template <typename T> __device__ __forceinline__ T* page_row(const castle_pages_t& t, int page, int h, int row, int d) {
  return reinterpret_cast<T*>(t.ptr) + page * t.stride_page + h * t.stride_h + (int64_t)row * d;
}
template <typename T> __device__ __forceinline__ T* new_row(const castle_tensor_t& t, int b, int h) {
  return reinterpret_cast<T*>(t.ptr) + b * t.stride_b + h * t.stride_h;
}
template <typename T> __device__ __forceinline__ void paged_store_out(const PagedParams& p, int b, int h, int c, float v) { store1<T>(new_row<T>(p.out, b, h) + c, v); }

__device__ __forceinline__ float sigmoid_fast(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }   // (2 units of the last place of fp32)

// 16 bytes of a row as pairs of floats.
template <typename T> struct Pairs {
  static constexpr int N = 4;
  static __device__ __forceinline__ void load(const T* p, float2* v) { unpack(*reinterpret_cast<const uint4*>(p), v); }
  static __device__ __forceinline__ void unpack(uint4 q, float2* v) {
    v[0] = Elem<T>::unpack2(q.x); v[1] = Elem<T>::unpack2(q.y); v[2] = Elem<T>::unpack2(q.z); v[3] = Elem<T>::unpack2(q.w);
  }
  // rounds v to what is stored, so that the score's lookahead key is the one that is kept
  static __device__ __forceinline__ uint4 round(float2* v) {
    const uint4 q = make_uint4(Elem<T>::pack2(v[0].x, v[0].y), Elem<T>::pack2(v[1].x, v[1].y), Elem<T>::pack2(v[2].x, v[2].y), Elem<T>::pack2(v[3].x, v[3].y));
    unpack(q, v);
    return q;
  }
};
template <> struct Pairs<float> {
  static constexpr int N = 2;
  static __device__ __forceinline__ void load(const float* p, float2* v) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = make_float2(q.x, q.y); v[1] = make_float2(q.z, q.w);
  }
  static __device__ __forceinline__ uint4 round(float2* v) {
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
  }
};
template <int N> __device__ __forceinline__ float dot(const float2* a, const float2* b) {
  float2 s = mul2(a[0], b[0]), t = mul2(a[1], b[1]);
#pragma unroll
  for (int i = 2; i < N; i += 2) { s = fma2(a[i], b[i], s); t = fma2(a[i + 1], b[i + 1], t); }
  s = add2(s, t);
  return s.x + s.y;
}
// Of two rows that the same LPR lanes share: even lanes get the sum of a, odd ones that of b.
template <int LPR> __device__ __forceinline__ float sum_of_two(float a, float b, bool odd) {
  float v = (odd ? b : a) + __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
#pragma unroll
  for (int o = 2; o < LPR; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a thread has summed up of its rows.
template <int N> struct Softmax {
  float m, l;
  float2 acc[N];
};

__device__ __forceinline__ uint32_t count_release(uint32_t* counter) {
  uint32_t before;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
  return before;
}

// Joins the parts of a pair: D / 4 columns x groups of parts, each thread four columns.
template <typename T, int D> __device__ __forceinline__ void paged_join(const PagedParams& p, const PagedSegment& s, int first_piece, int parts, float* buffer) {
  constexpr int L = D / 4, G = kPagedThreads / L;
  float(*s_sum)[D + 4] = reinterpret_cast<float(*)[D + 4]>(buffer);   // [G][D + 4]: and a group's maximum and sum of weights
  const int tid = threadIdx.x, c = tid % L * 4, g = tid / L;
  float m = -INFINITY, l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = g; i < parts; i += G) {
    const float* part = p.part + (int64_t)(2 * (first_piece + i) + (i == 0 ? 1 : 0)) * (4 + D);
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(part + D));
    const float4 v = __ldcg(reinterpret_cast<const float4*>(part + c));
    const float mn = fmaxf(m, ml.x), ref = mn == -INFINITY ? 0.f : mn, w0 = __expf(m - ref), w = __expf(ml.x - ref);
    m = mn;
    l = l * w0 + ml.y * w;
    a.x = a.x * w0 + v.x * w; a.y = a.y * w0 + v.y * w; a.z = a.z * w0 + v.z * w; a.w = a.w * w0 + v.w * w;
  }
  *reinterpret_cast<float4*>(&s_sum[g][c]) = a;
  if (c == 0) { s_sum[g][D] = m; s_sum[g][D + 1] = l; }
  group_sync(1);
  if (tid < D) {
    float mm = -INFINITY, sum = 0.f, total = 0.f;
#pragma unroll
    for (int k = 0; k < G; ++k) mm = fmaxf(mm, s_sum[k][D]);
    const float ref = mm == -INFINITY ? 0.f : mm;
#pragma unroll 4
    for (int k = 0; k < G; ++k) {
      const float w = __expf(s_sum[k][D] - ref);
      sum += s_sum[k][tid] * w;
      total += s_sum[k][D + 1] * w;
    }
    paged_store_out<T>(p, s.b, s.h, tid, sum / total);
  }
  group_sync(1);
}

// The end of a segment: the lane groups of a warp, then the warps; the result, or a partial and, if it is the pair's last, the join.
template <typename T, int D>
__device__ __forceinline__ void paged_finish(const PagedParams& p, const PagedPlan& plan, const PagedSegment& s, int piece, Softmax<Pairs<T>::N>& x) {
  constexpr int N = Pairs<T>::N, VEC = 2 * N, LPR = D / VEC;
  __shared__ float s_m[kPagedWarps], s_l[kPagedWarps];
  constexpr int G = 4 * kPagedThreads / D;
  __shared__ __align__(16) float buffer[G * (D + 4) > kPagedWarps * D ? G * (D + 4) : kPagedWarps * D];
  float(*s_acc)[D] = reinterpret_cast<float(*)[D]>(buffer);
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
    for (int i = 0; i < N; ++i) {
      x.acc[i].x = x.acc[i].x * c1 + __shfl_xor_sync(0xffffffffu, x.acc[i].x, o) * c2;
      x.acc[i].y = x.acc[i].y * c1 + __shfl_xor_sync(0xffffffffu, x.acc[i].y, o) * c2;
    }
    x.m = mn;
  }
  if (grp == 0) {
    if (sub == 0) { s_m[warp] = x.m; s_l[warp] = x.l; }
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<float2*>(&s_acc[warp][sub * VEC + 2 * i]) = x.acc[i];
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
      float* dst = p.part + (int64_t)(2 * piece + (s.tile0 == 0 ? 1 : 0)) * (4 + D);
      if (threadIdx.x == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(mm, ll);
      dst[threadIdx.x] = aa;
    }
  }
  if (whole) {
    group_sync(1);   // before the next segment writes s_m, s_acc
    return;
  }
  group_sync(1);
  const int first = piece_of(plan, s.first), parts = piece_of(plan, s.first + s.all - 1) - first + 1;
  if (threadIdx.x == 0) {
    uint32_t* counter = p.counters + s.b * p.H + s.h;
    s_last = count_release(counter) == (uint32_t)parts - 1;   // (the barrier puts the other threads' stores before it, and their loads behind it)
    if (s_last) *counter = 0;   // ready for the next launch
  }
  group_sync(1);
  if (!s_last) return;
  paged_join<T, D>(p, s, first, parts, buffer);
}

// Sequences without tiles: zeros where there is none, NaN (and a status) where the length has no places in the tables.  By a warp.
template <typename T, int D> __device__ __forceinline__ void paged_outside(const PagedParams& p, const int* lengths) {
  const int lane = threadIdx.x & 31;
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    const int length = lengths[b];
    if (length >= 0 && length < p.capacity) continue;
    for (int i = lane; i < p.H * D; i += 32) paged_store_out<T>(p, b, i / D, i % D, length < 0 ? 0.f : __int_as_float(0x7fc00000));
    if (length >= 0 && lane == 0) atomicOr(p.status, CASTLE_STATUS_BAD_INDEX);
  }
}

// The caches' rows come as bulk asynchronous copies into a ring of shared-memory stages, a tile of all four caches each, issued by a warp
// of its own: its lanes look a tile's pages up (a tile ahead) and issue a copy each, (page of the tile, cache), and it goes on from piece to
// piece without waiting for the ends of the softmaxes.  The other warps take the same walk through pieces and segments.
constexpr int kPagedStages = 3, kPagedTilePages = 8;   // a tile of 128 rows over pages of 16
template <typename T, int D> constexpr uint32_t kPagedTensor = PagedRows<T, D>::value * D * sizeof(T);   // a cache's part of a stage

template <typename T, int D>
__global__ void __launch_bounds__(kPagedThreads + 32, kPagedCtas) castle_paged_step_kernel(const __grid_constant__ PagedParams p) {
  constexpr int VEC = Vec<T>::N, N = VEC / 2, LPR = D / VEC, RPW = 32 / LPR, ROWS = PagedRows<T, D>::value, HALF = RPW * kPagedWarps;
  static_assert(ROWS == 2 * HALF, "two rows of a tile for each thread");
  constexpr uint32_t ROWB = D * sizeof(T), TENB = kPagedTensor<T, D>;
  static_assert(ROWS / 16 <= kPagedTilePages && 4 * kPagedTilePages <= 32, "a lane for each copy of a tile");
  extern __shared__ __align__(128) uint8_t smem[];                             // [stage][qu, U, kc, vc][row][D], [2][new qc, ku, vu, kc, vc, qu][D], the plan
  int *start = reinterpret_cast<int*>(smem + kPagedStages * 4 * TENB + 2 * 6 * ROWB), *lengths = start + p.B + 1;
  __shared__ uint64_t full[kPagedStages], empty[kPagedStages], new_full[2], new_place[2], new_empty[2];
  __shared__ T* s_new[2][4];                                                   // where a pair's rows are appended to qu, U, kc, vc; null: outside the pools
  __shared__ T* s_u[kPagedStages][kPagedTilePages];                            // where a stage's rows of U are, null where one of their pages is outside its pool
  __shared__ int abort_flag;
  volatile int* abortp = &abort_flag;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kPagedStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], kPagedWarps); }
    for (int i = 0; i < 2; ++i) { mbar_init(&new_full[i], 1); mbar_init(&new_place[i], 1); mbar_init(&new_empty[i], kPagedWarps); }
    mbar_fence_init();
    abort_flag = 0;
  }
  overlap_next();
  overlap_wait();
  const PagedPlan plan = paged_plan<kPagedThreads + 32>(p, ROWS, start, lengths);     // (its barriers cover the initialisation too)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int piece = blockIdx.x, begin = piece < plan.pieces ? piece_begin(plan, piece) : 0, end = piece < plan.pieces ? piece_begin(plan, piece + 1) : 0;
  int count = 0, segments = 0;                                                 // stages and segments so far
  if (warp == kPagedWarps) {
    const int which = lane & 3, nth = lane >> 2, page_size = 1 << p.page_shift;
    bool over = false;   // a wait of this CTA ran out: what was waited for has not ended, so nothing more is fetched and no barrier is arrived at again
    for (int at = begin; at < end && !over;) {
      const PagedSegment s = paged_segment<ROWS>(p, start, lengths, at, end);
      at = s.next;
      if (s.tiles == 0) continue;
      const int32_t* table = which == 1 ? p.u_table + s.b * p.u_table_stride : p.table + s.b * p.table_stride;
      const castle_pages_t pool = which == 0 ? p.quc : which == 1 ? p.U : which == 2 ? p.kcc : p.vcc;
      const int r_end = min(s.length, (s.tile0 + s.tiles) * ROWS);
      auto look_up = [&](int r0) {                                           // the page of this lane's copy, of the tile that begins with row r0
        const int r = r0 + nth * page_size;
        return r < min(r_end, r0 + ROWS) ? __ldg(table + (r >> p.page_shift)) : -1;
      };
      int page = look_up(s.tile0 * ROWS);
      const int last = __ldg(table + (s.length >> p.page_shift)), slot = segments & 1;   // (the new rows need not wait for the pages)
      if (segments >= 2) mbar_wait(&new_empty[slot], (uint32_t)((segments >> 1) - 1) & 1, abortp);
      if ((over = __any_sync(0xffffffffu, *abortp != 0))) break;
      {
        const castle_tensor_t t = lane == 0 ? p.qc : lane == 1 ? p.ku : lane == 2 ? p.vu : lane == 3 ? p.kc : lane == 4 ? p.vc : p.qu;
        if (lane == 0) mbar_expect_tx(&new_full[slot], 6 * ROWB);
        __syncwarp();
        if (lane < 6) bulk_g2s(smem + kPagedStages * 4 * TENB + (slot * 6 + lane) * ROWB, new_row<T>(t, s.b, s.h), ROWB, &new_full[slot]);
        ++segments;
      }
      for (int r0 = s.tile0 * ROWS; r0 < r_end; r0 += ROWS, ++count) {
        const int st = count % kPagedStages, next = look_up(r0 + ROWS);
        if (count >= kPagedStages) mbar_wait(&empty[st], (uint32_t)(count / kPagedStages - 1) & 1, abortp);
        if ((over = __any_sync(0xffffffffu, *abortp != 0))) break;
        const int r = r0 + nth * page_size, rows = min(min(page_size, ROWS), r_end - r);   // of this lane's copy
        const bool mine = nth * page_size < ROWS && rows > 0;
        const bool good = (uint32_t)page < (uint32_t)(which == 1 ? p.u_pages : p.pages);
        const uint32_t all = __ballot_sync(0xffffffffu, good);
        const bool copy = mine && (all >> (lane & ~3) & 15u) == 15u;
        const uint32_t bytes = copy ? rows * ROWB : 0, sum = __reduce_add_sync(0xffffffffu, bytes);
        T* rows_at = page_row<T>(pool, copy ? page : 0, s.h, r & (page_size - 1), D);
        if (mine && which == 1) s_u[st][nth] = copy ? rows_at : nullptr;
        __syncwarp();
        if (lane == 0) mbar_expect_tx(&full[st], sum);
        __syncwarp();
        if (copy) bulk_g2s(smem + st * 4 * TENB + which * TENB + nth * page_size * ROWB, rows_at, bytes, &full[st]);
        page = next;
      }
      if (over) break;
      const uint32_t good = __ballot_sync(0xffffffffu, (uint32_t)last < (uint32_t)(which == 1 ? p.u_pages : p.pages));
      if (lane < 4) s_new[slot][lane] = (good & 15u) == 15u ? page_row<T>(pool, last, s.h, s.length & (page_size - 1), D) : nullptr;
      __syncwarp();
      if (lane == 0) mbar_arrive(&new_place[slot]);
    }
    paged_outside<T, D>(p, lengths);
    // Its own last copies have ended when it leaves, whoever else waited for them or gave up.
    for (int i = max(0, count - kPagedStages); i < count; ++i) mbar_drain(&full[i % kPagedStages], (uint32_t)(i / kPagedStages) & 1);
    for (int i = max(0, segments - 2); i < segments; ++i) mbar_drain(&new_full[i & 1], (uint32_t)(i >> 1) & 1);
    return;
  }
  const int sub = lane % LPR, grp = lane / LPR, col = sub * VEC, mask = (1 << p.page_shift) - 1, row = warp * RPW + grp;
  const bool odd = lane & 1;
  bool there = true;   // until a wait of this warp has run out: its later ones would see the phases of others, so that it makes none and stores nothing any more
  {
    for (int at = begin; at < end;) {
      const PagedSegment s = paged_segment<ROWS>(p, start, lengths, at, end);
      at = s.next;
      if (s.tiles == 0) continue;
      const int slot = segments & 1;
      const uint32_t turn = (uint32_t)(segments++ >> 1) & 1;
      there = there && !mbar_wait_failed(&new_full[slot], turn, abortp);
      const T* rows = reinterpret_cast<const T*>(smem + kPagedStages * 4 * TENB + slot * 6 * ROWB) + col;
      RotaryParams rot = p.rot;
      rot.position0 = (float)s.length;
      float qcv[VEC], kuv[VEC], vuv[VEC];
      Vec<T>::load(rows, qcv);
      Vec<T>::load(rows + D, kuv);
      Vec<T>::load(rows + 2 * D, vuv);
      rotate_new<T>(rot, col, qcv, kuv, vuv);
      float2 qc[N], ku[N], vu[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        qc[i] = make_float2(qcv[2 * i] * p.scale, qcv[2 * i + 1] * p.scale);
        ku[i] = make_float2(kuv[2 * i] * p.scale, kuv[2 * i + 1] * p.scale);
        vu[i] = make_float2(vuv[2 * i], vuv[2 * i + 1]);
      }
      Softmax<N> x;
      x.m = -INFINITY; x.l = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) x.acc[i] = make_float2(0.f, 0.f);
      bool bad = false;
      const int r_end = min(s.length, (s.tile0 + s.tiles) * ROWS);
      for (int r0 = s.tile0 * ROWS; r0 < r_end; r0 += ROWS, ++count) {
        const int st = count % kPagedStages;
        // A wait that ran out means that the stage never arrived: U is persistent state, so nothing computed from it may be stored.
        there = there && !mbar_wait_failed(&full[st], (uint32_t)(count / kPagedStages) & 1, abortp, p.row_polls);
        // A thread has two rows, side by side: each is a chain of dot products, shuffles and exponentials, which is the time where few warps are
        // resident.  The lanes of a row share them out: even ones sum up the first row's products and work out its gate, odd ones the second's.
        const T* src = reinterpret_cast<const T*>(smem + st * 4 * TENB) + row * D + col;
        T* u[2];
        float z[2], sc[2], su[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int in = row + k * HALF;   // row of the tile
          u[k] = nullptr;
          if (there && in < r_end - r0) {
            u[k] = s_u[st][in >> p.page_shift];
            bad |= u[k] == nullptr;
            if (u[k]) u[k] += (in & mask) * D + col;
          }
          float2 q[N];
          Pairs<T>::load(src + k * HALF * D, q);
          z[k] = dot<N>(q, ku);
        }
        const float gate = sigmoid_fast(sum_of_two<LPR>(z[0], z[1], odd)), other_gate = __shfl_xor_sync(0xffffffffu, gate, 1);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float2 v[N], kk[N];
          Pairs<T>::load(src + (ROWS + k * HALF) * D, v);
          const float2 a = splat(odd == (k == 1) ? gate : other_gate);
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] = fma2(a, vu[i], v[i]);
          const uint4 kept = Pairs<T>::round(v);
          if (u[k]) *reinterpret_cast<uint4*>(u[k]) = kept;
          su[k] = dot<N>(v, qc);
          Pairs<T>::load(src + (2 * ROWS + k * HALF) * D, kk);
          sc[k] = dot<N>(kk, qc);
        }
        const float sum_u = sum_of_two<LPR>(su[0], su[1], odd), sum_c = sum_of_two<LPR>(sc[0], sc[1], odd);
        const float score = sum_c - sum_u * sigmoid_fast(sum_u), other = __shfl_xor_sync(0xffffffffu, score, 1);
        const float s0 = u[0] ? (odd ? other : score) : -INFINITY, s1 = u[1] ? (odd ? score : other) : -INFINITY;
        const float best = fmaxf(x.m, fmaxf(s0, s1)), ref = best == -INFINITY ? 0.f : best;   // (scores of minus infinity alone weigh nothing)
        const float corr = __expf(x.m - ref), w[2] = {__expf(s0 - ref), __expf(s1 - ref)};
        x.m = best;
        x.l *= corr;
#pragma unroll
        for (int i = 0; i < N; ++i) x.acc[i] = mul2(x.acc[i], splat(corr));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (!u[k]) continue;
          float2 v[N];
          Pairs<T>::load(src + (3 * ROWS + k * HALF) * D, v);
          x.l += w[k];
#pragma unroll
          for (int i = 0; i < N; ++i) x.acc[i] = fma2(splat(w[k]), v[i], x.acc[i]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
      }
      if (s.tile0 + s.tiles == s.all && warp == 0) {   // the appended row; its U is zero, so its score is qc . kc_new alone
        float kn[VEC], vn[VEC], qn[VEC];
        Vec<T>::load(rows + 3 * D, kn);
        Vec<T>::load(rows + 4 * D, vn);
        Vec<T>::load(rows + 5 * D, qn);
        rotate_new<T>(rot, col, kn, qn, nullptr);
        there = there && !mbar_wait_failed(&new_place[slot], turn, abortp);
        bad |= there && s_new[slot][0] == nullptr;
        if (grp == 0 && there && s_new[slot][0]) {   // (rows that arrived before a wait that ran out are rewritten and this one is not: such a sequence's caches are void)
          Vec<T>::store(s_new[slot][0] + col, qn);
          *reinterpret_cast<uint4*>(s_new[slot][1] + col) = make_uint4(0, 0, 0, 0);
          Vec<T>::store(s_new[slot][2] + col, kn);
          Vec<T>::store(s_new[slot][3] + col, vn);
        }
        float sc = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) sc += qc[i].x * kn[2 * i] + qc[i].y * kn[2 * i + 1];
        sc = group_sum<LPR>(sc);
        if (grp == 0) {
          const float best = fmaxf(x.m, sc), ref = best == -INFINITY ? 0.f : best, corr = __expf(x.m - ref), w = __expf(sc - ref);
          x.m = best;
          x.l = x.l * corr + w;
#pragma unroll
          for (int i = 0; i < N; ++i) x.acc[i] = make_float2(x.acc[i].x * corr + w * vn[2 * i], x.acc[i].y * corr + w * vn[2 * i + 1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&new_empty[slot]);
      if (bad || !there) x.l = __int_as_float(0x7fc00000);   // (a mean of some of the rows would look like a result)
      if (bad) atomicOr(p.status, CASTLE_STATUS_BAD_INDEX);
      paged_finish<T, D>(p, plan, s, piece, x);
    }
  }
  if (threadIdx.x == 0 && abort_flag) atomicOr(p.status, CASTLE_STATUS_WAIT_TIMEOUT);
}

static thread_local uint32_t paged_row_polls = kWaitPollLimit;   // (for the tests)

template <typename T, int D> static int launch_paged(const PagedParams& p, cudaStream_t st) {
  constexpr size_t fixed = kPagedStages * 4 * kPagedTensor<T, D> + 2 * 6 * D * sizeof(T);
  const size_t smem = fixed + (size_t)(2 * p.B + 1) * sizeof(int);
  // as many CTAs as are resident together: a second wave of them would take as long as the first (a batch of some hundreds needs room for its plan)
  const int ctas = (int)std::min<size_t>(kPagedCtas, kPagedSmem / (smem + kPagedStatic));
  cudaError_t e = allow_smem(castle_paged_step_kernel<T, D>, (int)(fixed + (2 * kPagedMaxBatch + 1) * sizeof(int)));
  if (e != cudaSuccess) return cuda_fail(e, "castle_paged_decode_step attribute");
  ev_start(CASTLE_KERNEL_DECODE, st);
  e = launch_kernel(castle_paged_step_kernel<T, D>, dim3(kPagedSms * ctas), kPagedThreads + 32, smem, st, true, p);
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

// Units of all pairs if every sequence filled its places; -1 where they or the sizes are out of range.
static int64_t paged_most_units(const castle_problem_t* p, int32_t page_size, int32_t table_width) {
  if (!p || p->batch <= 0 || p->batch > kPagedMaxBatch || p->heads <= 0 || page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) || table_width <= 0) return -1;
  if (p->dtype < CASTLE_BF16 || p->dtype > CASTLE_F32 || (p->dim_head != 16 && p->dim_head != 32 && p->dim_head != 64 && p->dim_head != 128)) return -1;
  const int64_t capacity = (int64_t)table_width * page_size, rows = paged_rows(p->dtype, p->dim_head);
  const int64_t pairs = (int64_t)p->batch * p->heads;
  if (capacity > INT32_MAX - 1024 || pairs > INT32_MAX) return -1;
  const int64_t each = (capacity + rows - 1) / rows + kPagedPair;
  return each > INT32_MAX / pairs ? -1 : each * pairs;
}

}  // namespace castle

using namespace castle;

extern "C" size_t castle_paged_decode_workspace_bytes(const castle_problem_t* p, int32_t page_size, int32_t table_width) {
  const int64_t units = paged_most_units(p, page_size, table_width);
  return units < 0 ? 0 : (size_t)std::min<int64_t>(kPagedSms * kPagedCtas, units) * 2 * (4 + p->dim_head) * sizeof(float);
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
  if (paged_most_units(p, page_size, table_width) < 0) return reject("%s: %d sequences x %d heads x %d pages are too many positions", who, p->batch, p->heads, table_width);
  if (!u_table || !table || !lengths || !counters || !status) return reject("%s: null table, lengths, counters or status", who);
  if (((uintptr_t)u_table | (uintptr_t)table | (uintptr_t)lengths | (uintptr_t)counters | (uintptr_t)status) % 4 || (uintptr_t)workspace % 16)
    return reject("%s: tables, lengths, counters and status must be 4-byte aligned, the workspace 16-byte", who);
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
  q.part = (float*)workspace; q.counters = counters; q.status = status; q.row_polls = paged_row_polls;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (p->dtype) {
    case CASTLE_BF16: return launch_paged_d<__nv_bfloat16>(q, p->dim_head, st);
    case CASTLE_F16: return launch_paged_d<__half>(q, p->dim_head, st);
    default: return launch_paged_d<float>(q, p->dim_head, st);
  }
}

extern "C" int castle_selftest_paged_polls(int32_t limit) {
  if (limit < -1 || limit > 65536) return reject("castle_selftest_paged_polls: -1 or 0..65536 polls expected");
  paged_row_polls = limit < 0 ? kWaitPollLimit : (uint32_t)limit;
  return 0;
}
