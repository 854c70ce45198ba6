// Lookup of tokens in a table of rows, scaled, and the table's gradient.
//
//   y[i] = scale W[t_i]                       dW[v] = scale sum over i with t_i = v of dy[i]
//
// Both are bound by memory: a row read and a row written per token; in the gradient a row read per token and the whole table
// written, zero rows included.  The gradient needs the tokens of each row together.  A sort brings them there: it is stable,
// so a row's gradients are added in the order of their positions, in fp32, and the result is the same from call to call
// (atomic additions into the rows would be in arrival order, would need an fp32 table and a pass to round it).
//
// Sort, two launches.  A row has one of 128 owners (or 256 and so on: as many as one's counters need), its number modulo theirs.  First,
// 128 CTAs take a slice of the tokens each and put it in the order of the owners; then a CTA per owner takes its part of every slice and puts
// these in the order of its rows.  Where an owner begins in the whole list is the sum of where it begins in the slices, so CTAs of a launch
// need nothing of one another, and a row that takes all the tokens is no special case.  Both count per warp and key, tokens shared out among
// the warps in contiguous parts, and sums of these give every (key, warp) its place; a second reading puts the tokens there, lanes
// with the same key in the order of the lanes.  The list is in the order (owner, row): tokenisers give frequent tokens low
// numbers, and owners of neighbouring rows would be as unequal as the tokens are.  (One launch, in which each owner read all tokens: 38 us
// for 65536 of them, 108 for 200000.)
//
// Sums: the sorted list is cut into chunks of `piece` entries; a warp takes a chunk's sums in a slab of 256 columns and writes a row when
// its entries end.  (A warp per row instead took 600 us for 65536 tokens with the frequencies of text in 131072 rows of 2048; one per
// sixteen rows 383: the frequent rows are neighbours.)  A row of more entries than a chunk leaves its parts' sums in scratch, which a
// third launch adds in order.
#include "common.cuh"
#include "vec.cuh"

namespace castle {

constexpr int kEmbThreads = 256, kBinThreads = 512, kBinWarps = kBinThreads / 32, kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kSlices = 128, kWarpSlices = kSlices / kSortWarps;
constexpr int kSortRows = 1536;    // most rows of an owner: 32 counters of 4 bytes each
constexpr int kMaxOwners = 2048;   // 16 counters each
constexpr int64_t kMostTokens = 1 << 30, kMostRows = (int64_t)kSortRows * kMaxOwners;   // places in the list, and a chunk behind the last, are 32 bits

template <typename I> __device__ __forceinline__ int64_t token_at(const void* t, int64_t i) { return (int64_t)static_cast<const I*>(t)[i]; }

// A warp takes a stretch of 4 x 256 columns of a token's row.
template <typename T, typename I, bool VEC>
__global__ void __launch_bounds__(kEmbThreads) castle_embedding_fwd_kernel(const void* __restrict__ tokens, const T* __restrict__ w, int64_t row_stride,
                                                                           float scale, T* __restrict__ y, int64_t n, int64_t vocab, int dim, int slabs,
                                                                           int32_t* status) {
  const int64_t item = (int64_t)blockIdx.x * (kEmbThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= n * slabs) return;
  const int64_t i = slabs == 1 ? item : item / slabs;
  const int slab = (int)(item - i * slabs);
  const int64_t t = token_at<I>(tokens, i);
  const bool ok = t >= 0 && t < vocab;
  if (!ok && slab == 0 && lane == 0) atomicOr(status, CASTLE_STATUS_BAD_INDEX);
  const T* row = w + (ok ? t : 0) * row_stride;
  float v[4][8];
#pragma unroll
  for (int q = 0; q < 4; ++q) load_columns8<T, 32, VEC>(row, slab * 4 + q, lane, dim, v[q]);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[q][j] = ok ? v[q][j] * scale : __int_as_float(0x7fffffff);
    store_columns8<T, 32, VEC>(y + i * dim, slab * 4 + q, lane, dim, v[q]);
  }
}

// The sorted list's order of rows: row v is number (v mod owners) * per + v / owners, owners = 2^shift, per = rows of an owner.
struct EmbOrder {
  int shift, per;
  __host__ __device__ __forceinline__ int owners() const { return 1 << shift; }
  __device__ __forceinline__ int number(int row) const { return (row & (owners() - 1)) * per + (row >> shift); }
  __device__ __forceinline__ int64_t row(int number) const { return ((int64_t)(number % per) << shift) + number / per; }
};

constexpr uint32_t kNoRow = 0xffffffffu;
// A token as a row's number in the table; kNoRow: outside of it (`bad`), or the padding's.
template <typename I> __device__ __forceinline__ uint32_t token_row(const void* tokens, int64_t i, uint32_t vocab, uint32_t padding, bool& bad) {
  uint32_t t;
  bool in;
  if constexpr (sizeof(I) == 8) {
    const uint2 w = static_cast<const uint2*>(tokens)[i];
    t = w.x;
    in = w.y == 0 && t < vocab;
  } else {
    t = static_cast<const uint32_t*>(tokens)[i];
    in = t < vocab;
  }
  bad |= !in;
  return in && t != padding ? t : kNoRow;
}

// Counters [warp][key] of a CTA of WARPS warps become the places where each (key, warp) begins, from `base` on; begin(key, place) is called for
// every key.  Returns the end.
template <int WARPS, typename F> __device__ __forceinline__ int places(int32_t* count, int keys, int base, int32_t* warp_sums, F&& begin) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int k0 = 0; k0 < keys; k0 += WARPS * 32) {
    const int key = k0 + tid;
    int total = 0;
    if (key < keys)
      for (int w = 0; w < WARPS; ++w) total += count[w * keys + key];
    int scan = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += up;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = scan;
    __syncthreads();
    int at = base + scan - total, all = 0;
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) at += warp_sums[w];
      all += warp_sums[w];
    }
    if (key < keys) {
      begin(key, at);
      for (int w = 0; w < WARPS; ++w) {
        const int c = count[w * keys + key];
        count[w * keys + key] = at;
        at += c;
      }
    }
    base += all;
  }
  __syncthreads();
  return base;
}
// The place of a lane's entry with `key` (-1: none) behind those of its warp before it; by a whole warp.
__device__ __forceinline__ int next_place(int32_t* mine, int key, int lane) {
  const unsigned peers = __match_any_sync(0xffffffffu, key);
  const int at = key >= 0 ? mine[key] : 0, rank = __popc(peers & ((1u << lane) - 1));
  __syncwarp();
  if (key >= 0 && rank == 0) mine[key] = at + __popc(peers);
  __syncwarp();
  return at + rank;
}

// A slice in the order of the owners: bins[slice * length ..] as (row of the owner, position); begins[slice][owner] where each begins in it.
template <typename I>
__global__ void __launch_bounds__(kBinThreads) castle_token_bin_kernel(const void* __restrict__ tokens, int64_t n, int length, uint32_t vocab, uint32_t padding,
                                                                       EmbOrder order, int2* __restrict__ bins, int32_t* __restrict__ begins, int32_t* long_count,
                                                                       int32_t* status) {
  extern __shared__ int32_t count[];   // [warp][owner]
  __shared__ int32_t warp_sums[kBinWarps];
  if (blockIdx.x == 0 && threadIdx.x == 0) *long_count = 0;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, owners = order.owners();
  const int64_t s0 = (int64_t)blockIdx.x * length, s1 = min(n, s0 + length);
  const int share = (length + kBinThreads - 1) / kBinThreads * 32;
  const int64_t i0 = min(s1, s0 + warp * share), i1 = min(s1, i0 + share);
  for (int k = tid; k < kBinWarps * owners; k += kBinThreads) count[k] = 0;
  __syncthreads();
  int32_t* mine = count + warp * owners;
  bool bad = false;
#pragma unroll 4
  for (int64_t i = i0 + lane; i < i1; i += 32) {
    const uint32_t t = token_row<I>(tokens, i, vocab, padding, bad);
    if (t != kNoRow) atomicAdd(&mine[t & (owners - 1)], 1);
  }
  if (bad) atomicOr(status, CASTLE_STATUS_BAD_INDEX);
  __syncthreads();
  int32_t* out = begins + (int64_t)blockIdx.x * (owners + 1);
  const int end = places<kBinWarps>(count, owners, 0, warp_sums, [&](int owner, int at) { out[owner] = at; });
  if (tid == 0) out[owners] = end;
#pragma unroll 4
  for (int64_t i = i0; i < i1; i += 32) {
    const uint32_t t = i + lane < i1 ? token_row<I>(tokens, i + lane, vocab, padding, bad) : kNoRow;
    const int at = next_place(mine, t != kNoRow ? (int)(t & (owners - 1)) : -1, lane);
    if (t != kNoRow) bins[s0 + at] = make_int2((int)(t >> order.shift), (int)(i + lane));
  }
}

// An owner's entries of all slices in the order of its rows.  start[k] = number of tokens (with a row of their own) in rows before number
// k; sorted[start[k] .. start[k + 1]) the positions of row k's, in order; row_of[e] the number of entry e's row.
__global__ void __launch_bounds__(kSortThreads) castle_token_sort_kernel(const int2* __restrict__ bins, const int32_t* __restrict__ begins, int length, EmbOrder order,
                                                                         int32_t* __restrict__ start, int32_t* __restrict__ sorted, int32_t* __restrict__ row_of) {
  extern __shared__ int32_t count[];   // [warp][row]
  __shared__ int32_t warp_sums[kSortWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rows = order.per, me = blockIdx.x, owners = order.owners();
  for (int k = tid; k < kSortWarps * rows; k += kSortThreads) count[k] = 0;
  overlap_wait();
  // lane j < kWarpSlices: where the owner's entries of the warp's slice j lie, and how many there are up to its end
  int first = 0, upto = 0;
  if (lane < kWarpSlices) {
    const int32_t* b = begins + (int64_t)(warp * kWarpSlices + lane) * (owners + 1) + me;
    first = b[0];
    upto = b[1] - b[0];
  }
  int below = lane < kWarpSlices ? first : 0;
#pragma unroll
  for (int o = 1; o < kWarpSlices; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += up;
    below += __shfl_xor_sync(0xffffffffu, below, o);
  }
  const int all = __shfl_sync(0xffffffffu, upto, kWarpSlices - 1);
  auto entry = [&](int e) {   // of the warp's, by a whole warp; any beyond the last is not used
    int slice = 0, before = 0;
#pragma unroll
    for (int j = 0; j + 1 < kWarpSlices; ++j) {
      const int end = __shfl_sync(0xffffffffu, upto, j);
      if (e >= end) { slice = j + 1; before = end; }
    }
    const int at = __shfl_sync(0xffffffffu, first, slice) + e - before;
    return e < all ? bins[(int64_t)(warp * kWarpSlices + slice) * length + at] : make_int2(-1, 0);
  };
  if (lane == 0) warp_sums[warp] = below;
  __syncthreads();
  int base = 0;
  for (int k = 0; k < kSortWarps; ++k) base += warp_sums[k];
  int32_t* mine = count + warp * rows;
  for (int e0 = 0; e0 < all; e0 += 32) {
    const int2 v = entry(e0 + lane);
    if (v.x >= 0) atomicAdd(&mine[v.x], 1);
  }
  __syncthreads();
  const int end = places<kSortWarps>(count, rows, base, warp_sums, [&](int row, int at) { start[(int64_t)me * rows + row] = at; });
  if (tid == 0 && me == owners - 1) start[(int64_t)owners * rows] = end;
  for (int e0 = 0; e0 < all; e0 += 32) {
    const int2 v = entry(e0 + lane);
    const int at = next_place(mine, v.x, lane);
    if (v.x >= 0) {
      sorted[at] = v.y;
      row_of[at] = me * rows + v.x;
    }
  }
}

struct EmbGrad {
  const int32_t *start, *sorted, *row_of;
  float* partial;   // [chunk][2][dim]: of the run that the chunk begins in, and of another one that it ends in
  EmbOrder order;
  int numbers;      // of rows in the sorted list's order: owners * per
  int64_t vocab, dy_stride;
  int dim, slabs, piece, chunks, sum_blocks;
  float scale;
  int32_t *longs, *long_count;   // chunks in which a row of more than a chunk begins, in any order
};

// Eight rows of dy, a lane's columns of each, as they lie until they are added, with nothing to wait for in between (65536 x 1023 in bf16 into
// 50000 rows: 109 us, each element converted on arrival 342).
template <typename T, bool VEC> struct EmbBatch {
  Raw8<T> raw[VEC ? 8 : 1];
  T one[VEC ? 1 : 8][8];
  __device__ __forceinline__ void load(int u, const T* row, int slab, int lane, int dim) {
    if constexpr (VEC) {
      const int c = column8<32, true>(slab, lane, 0);
      raw[u] = c < dim ? *reinterpret_cast<const Raw8<T>*>(row + c) : Raw8<T>{};
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) one[u][j] = row[min(column8<32, false>(slab, lane, j), dim - 1)];   // (sums of columns that are not there go nowhere)
    }
  }
  __device__ __forceinline__ void add(int u, float* acc) const {
    float f[8];
    if constexpr (VEC) {
      load8<T>(reinterpret_cast<const T*>(&raw[u]), f);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = load1<T>(&one[u][j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += f[j];
  }
};

// Entries [a, b) of the sorted list in order, eight rows of dy on their way at a time; next(row) is called (by the whole warp) before
// an entry is added to acc.
template <typename T, bool VEC, typename F>
__device__ __forceinline__ void walk_entries(const EmbGrad& p, const T* __restrict__ dy, int a, int b, int slab, int lane, float* acc, F&& next) {
  for (int k0 = a; k0 < b; k0 += 32) {
    const int left = min(32, b - k0);
    const int at = lane < left ? p.sorted[k0 + lane] : 0, row = lane < left ? p.row_of[k0 + lane] : 0;
    for (int k = 0; k < left; k += 8) {
      EmbBatch<T, VEC> batch;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int64_t i = __shfl_sync(0xffffffffu, at, min(k + u, left - 1));
        if (k + u < left) batch.load(u, dy + i * p.dy_stride, slab, lane, p.dim);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int r = __shfl_sync(0xffffffffu, row, min(k + u, left - 1));
        if (k + u < left) {
          next(r);
          batch.add(u, acc);
        }
      }
    }
  }
}

// Blocks [0, sum_blocks), a warp each: the sums of a chunk's entries in a slab of columns.  A short row (up to `piece` entries, the length
// of a chunk) belongs to the chunk in which it begins, of a longer one each chunk sums its part.  The other blocks: zeros for rows without
// entries, four threads a row: bulk copies of a buffer of zeros (VEC; stores of the warps took 67 us for 200 MB beside 25 MB of sums).
constexpr int kZeros = 1024, kZeroRows = kEmbThreads / 4;
template <typename T, bool VEC>
__global__ void __launch_bounds__(kEmbThreads) castle_embedding_bwd_kernel(const EmbGrad p, const T* __restrict__ dy, T* __restrict__ dw) {
  __shared__ __align__(128) uint4 zeros[VEC ? kZeros / 16 : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if ((int)blockIdx.x < p.sum_blocks) {
    const int64_t item = (int64_t)blockIdx.x * (kEmbThreads / 32) + warp;
    overlap_wait();
    const int c = (int)(item / p.slabs), slab = (int)(item % p.slabs), total = p.start[p.numbers];
    const int64_t a64 = (int64_t)c * p.piece;
    if (a64 >= total) return;
    const int a = (int)a64, b = min(total, a + p.piece);
    float acc[8];
    auto clear = [&] {
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = 0.f;
    };
    clear();
    auto part = [&](int from, int to, int side) {   // of a long row
      walk_entries<T, VEC>(p, dy, from, to, slab, lane, acc, [](int) {});
      store_columns8<float, 32, VEC>(p.partial + ((int64_t)c * 2 + side) * p.dim, slab, lane, p.dim, acc);
      clear();
    };
    const int first = p.row_of[a], last = p.row_of[b - 1];
    const int f0 = p.start[first], f1 = p.start[first + 1], l0 = p.start[last], l1 = p.start[last + 1];
    int from = a, to = l1;
    if (f1 - f0 > p.piece) {
      from = min(b, f1);
      part(a, from, 0);
    } else if (f0 < a) {
      from = f1;
    }
    if (l1 - l0 > p.piece) {
      to = l0;
      if (l0 >= from) part(l0, b, 1);
      if (l0 >= a && slab == 0 && lane == 0) p.longs[atomicAdd(p.long_count, 1)] = c;
    }
    if (from >= to) return;
    int row = p.row_of[from];
    auto store = [&](int next) {
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] *= p.scale;
      store_columns8<T, 32, VEC>(dw + p.order.row(row) * p.dim, slab, lane, p.dim, acc);
      clear();
      row = next;
    };
    walk_entries<T, VEC>(p, dy, from, to, slab, lane, acc, [&](int next) {
      if (next != row) store(next);
    });
    store(0);
    return;
  }
  const int64_t row = (int64_t)(blockIdx.x - p.sum_blocks) * kZeroRows + threadIdx.x / 4;
  if constexpr (VEC) {
    if (threadIdx.x < kZeros / 16) zeros[threadIdx.x] = make_uint4(0u, 0u, 0u, 0u);
    fence_async_smem();
    __syncthreads();
  }
  overlap_wait();
  bool none = false;
  if (row < p.vocab) {
    const int number = p.order.number((int)row);
    none = p.start[number] == p.start[number + 1];
  }
  if constexpr (VEC) {
    if (none) {
      char* out = reinterpret_cast<char*>(dw + row * p.dim);
      const int bytes = p.dim * (int)sizeof(T);
      for (int o = (threadIdx.x & 3) * kZeros; o < bytes; o += 4 * kZeros) bulk_s2g(out + o, zeros, min(kZeros, bytes - o));
      bulk_commit();
      bulk_wait_read0();
    }
  } else {
    const float zero[8] = {};
    for (unsigned left = __ballot_sync(0xffffffffu, none) & 0x11111111u; left; left &= left - 1) {
      T* out = dw + (row - lane / 4 + __ffs(left) / 4) * p.dim;
      for (int q = 0; q < p.slabs; ++q) store_columns8<T, 32, false>(out, q, lane, p.dim, zero);
    }
  }
}

// A CTA per slab of a long row: the sums of its pieces, eight shares of them in order.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kEmbThreads) castle_embedding_join_kernel(const EmbGrad p, T* __restrict__ dw) {
  __shared__ float s[kEmbThreads / 32][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  overlap_wait();
  const int64_t items = (int64_t)*p.long_count * p.slabs;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int c = p.longs[item / p.slabs], slab = (int)(item % p.slabs), a = c * p.piece, b = min(p.start[p.numbers], a + p.piece);
    const int row = p.row_of[b - 1], r0 = p.start[row], r1 = p.start[row + 1];
    const int parts = (r1 - 1) / p.piece - c + 1, share = (parts + 7) / 8, k1 = min(parts, (warp + 1) * share);
    float acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.f;
#pragma unroll 4
    for (int k = warp * share; k < k1; ++k) {
      float v[8];
      const int side = k == 0 && r0 > a;   // in its first chunk the row is the one that the chunk ends in, unless it is the first, too
      load_columns8<float, 32, VEC>(p.partial + ((int64_t)(c + k) * 2 + side) * p.dim, slab, lane, p.dim, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += v[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s[warp][j * 32 + lane] = acc[j];
    __syncthreads();
    if (warp == 0) {
      for (int k = 1; k < kEmbThreads / 32; ++k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += s[k][j * 32 + lane];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] *= p.scale;
      store_columns8<T, 32, VEC>(dw + p.order.row(row) * p.dim, slab, lane, p.dim, acc);
    }
    __syncthreads();
  }
}

// Entries of a chunk: as many as leave some sixteen warps per SM with one, 16 to 64.
static int emb_piece(int64_t n, int dim) {
  const int64_t slabs = (dim + 255) / 256;
  int piece = 16;
  while (piece < 64 && n * slabs / piece > 148 * 16) piece *= 2;
  return piece;
}

static EmbOrder emb_order(int64_t vocab) {
  EmbOrder o{7, 0};
  while (((vocab - 1) >> o.shift) + 1 > kSortRows) ++o.shift;
  o.per = (int)((vocab - 1) >> o.shift) + 1;
  return o;
}

static int emb_slice(int64_t n) { return (int)((n + kSlices - 1) / kSlices); }

struct EmbScratch { size_t start, sorted, row_of, bins, begins, longs, partial, bytes; };
static EmbScratch emb_scratch(int64_t n, int64_t vocab, int dim) {
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  const int piece = emb_piece(n, dim);
  EmbScratch s;
  s.start = 0;
  const EmbOrder order = emb_order(vocab);
  s.sorted = up(((size_t)order.owners() * order.per + 1) * 4);
  s.row_of = s.sorted + up((size_t)n * 4);
  s.bins = s.row_of + up((size_t)n * 4);
  s.begins = s.bins + up((size_t)emb_slice(n) * kSlices * sizeof(int2));
  s.longs = s.begins + up((size_t)kSlices * (order.owners() + 1) * 4);
  s.partial = s.longs + up(((size_t)((n + piece - 1) / piece) + 1) * 4);
  s.bytes = s.partial + (size_t)((n + piece - 1) / piece) * 2 * dim * 4;
  return s;
}

static int emb_check(const char* who, int32_t dtype, int32_t index_bytes, int64_t tokens, int64_t vocab, int32_t dim, const void* index, int64_t stride,
                     const int32_t* status) {
  if (dtype < CASTLE_BF16 || dtype > CASTLE_F32) return reject("%s: unknown dtype", who);
  if (index_bytes != 4 && index_bytes != 8) return reject("%s: tokens must be 32- or 64-bit integers", who);
  if (tokens <= 0 || tokens > kMostTokens || vocab <= 0 || vocab > kMostRows || dim <= 0 || dim > (1 << 24))
    return reject("%s: %lld tokens, vocabulary %lld, dim %d not supported", who, (long long)tokens, (long long)vocab, dim);
  if (!index || (uintptr_t)index % index_bytes || !status) return reject("%s: tokens (aligned to their size) and a status word are needed", who);
  if (stride < 0) return reject("%s: negative strides are not supported", who);
  return 0;
}

template <typename T, bool VEC>
static cudaError_t emb_bwd(const EmbGrad& p, const T* dy, T* dw, cudaStream_t st) {
  const int64_t blocks = p.sum_blocks + (p.vocab + kZeroRows - 1) / kZeroRows;
  const cudaError_t e = launch_kernel(castle_embedding_bwd_kernel<T, VEC>, dim3((unsigned)blocks), kEmbThreads, 0, st, true, p, dy, dw);
  if (e != cudaSuccess) return e;
  const int64_t most = (int64_t)p.chunks * p.slabs;
  return launch_kernel(castle_embedding_join_kernel<T, VEC>, dim3((unsigned)(most < 148 * 4 ? most : 148 * 4)), kEmbThreads, 0, st, true, p, dw);
}

}  // namespace castle

using namespace castle;

extern "C" int castle_embedding_fwd(int32_t dtype, int32_t index_bytes, int64_t tokens, int64_t vocab, int32_t dim, const void* index, const void* weight,
                                    int64_t row_stride, float scale, void* y, int32_t* status, void* stream) {
  if (int rc = emb_check("castle_embedding_fwd", dtype, index_bytes, tokens, vocab, dim, index, row_stride, status)) return rc;
  const int es = elem_size(dtype), slabs = (dim + 1023) / 1024;
  if (!weight || !y || ((uintptr_t)weight | (uintptr_t)y) % es) return reject("castle_embedding_fwd: weight and y must be aligned to their elements");
  const int64_t blocks = (tokens * slabs + 7) / 8;
  if (blocks > 2147483647) return reject("castle_embedding_fwd: too many tokens");
  const cudaStream_t st = (cudaStream_t)stream;
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kernel) {
      kernel<<<(unsigned)blocks, kEmbThreads, 0, st>>>(index, (const T*)weight, row_stride, scale, (T*)y, tokens, vocab, dim, slabs, status);
      return 0;
    };
    if (vec_rows(dtype, dim, row_stride, weight, y))
      return index_bytes == 8 ? go(castle_embedding_fwd_kernel<T, int64_t, true>) : go(castle_embedding_fwd_kernel<T, int32_t, true>);
    return index_bytes == 8 ? go(castle_embedding_fwd_kernel<T, int64_t, false>) : go(castle_embedding_fwd_kernel<T, int32_t, false>);
  });
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : cuda_fail(e, "castle_embedding_fwd launch");
}

extern "C" size_t castle_embedding_bwd_workspace_bytes(int64_t tokens, int64_t vocab, int32_t dim) {
  return tokens <= 0 || tokens > kMostTokens || vocab <= 0 || vocab > kMostRows || dim <= 0 ? 0 : emb_scratch(tokens, vocab, dim).bytes;
}

extern "C" int castle_embedding_bwd(int32_t dtype, int32_t index_bytes, int64_t tokens, int64_t vocab, int32_t dim, const void* index, int64_t padding_idx,
                                    const void* dy, int64_t dy_stride, float scale, void* dweight, void* workspace, size_t workspace_bytes,
                                    int32_t* status, void* stream) {
  if (int rc = emb_check("castle_embedding_bwd", dtype, index_bytes, tokens, vocab, dim, index, dy_stride, status)) return rc;
  const int es = elem_size(dtype);
  if (!dy || !dweight || ((uintptr_t)dy | (uintptr_t)dweight) % es) return reject("castle_embedding_bwd: dy and dweight must be aligned to their elements");
  if (padding_idx < -1 || padding_idx >= vocab)   // (the kernels compare 32 bits)
    return reject("castle_embedding_bwd: padding_idx %lld is neither a row of the table nor -1", (long long)padding_idx);
  const EmbScratch s = emb_scratch(tokens, vocab, dim);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < s.bytes) return reject("castle_embedding_bwd: workspace too small or not 16-byte aligned");
  EmbGrad p;
  char* ws = static_cast<char*>(workspace);
  int32_t *start = (int32_t*)(ws + s.start), *sorted = (int32_t*)(ws + s.sorted), *row_of = (int32_t*)(ws + s.row_of);
  p.start = start; p.sorted = sorted; p.row_of = row_of; p.partial = (float*)(ws + s.partial);
  p.order = emb_order(vocab); p.numbers = p.order.owners() * p.order.per;
  p.vocab = vocab; p.dy_stride = dy_stride; p.dim = dim; p.slabs = (dim + 255) / 256; p.piece = emb_piece(tokens, dim);
  p.chunks = (int)((tokens + p.piece - 1) / p.piece); p.scale = scale;
  p.longs = (int32_t*)(ws + s.longs); p.long_count = p.longs + p.chunks;
  p.sum_blocks = (int)(((int64_t)p.chunks * p.slabs + 7) / 8);
  if ((int64_t)p.chunks * p.slabs > 2000000000) return reject("castle_embedding_bwd: too many tokens for the width");
  const cudaStream_t st = (cudaStream_t)stream;
  const int slice = emb_slice(tokens), bin_smem = p.order.owners() * kBinWarps * 4, sort_smem = p.order.per * kSortWarps * 4;
  int2* bins = (int2*)(ws + s.bins);
  int32_t* begins = (int32_t*)(ws + s.begins);
  auto bin = [&](auto kernel) {
    const cudaError_t e = allow_smem(kernel, kMaxOwners * kBinWarps * 4);
    if (e != cudaSuccess) return e;
    kernel<<<kSlices, kBinThreads, bin_smem, st>>>(index, tokens, slice, (uint32_t)vocab, padding_idx < 0 ? kNoRow : (uint32_t)padding_idx, p.order, bins, begins, p.long_count, status);
    return cudaGetLastError();
  };
  cudaError_t e = index_bytes == 8 ? bin(castle_token_bin_kernel<int64_t>) : bin(castle_token_bin_kernel<int32_t>);
  if (e == cudaSuccess) e = allow_smem(castle_token_sort_kernel, kSortRows * kSortWarps * 4);
  if (e == cudaSuccess)
    e = launch_kernel(castle_token_sort_kernel, dim3(p.order.owners()), kSortThreads, sort_smem, st, true, (const int2*)bins, (const int32_t*)begins, slice, p.order, start,
                      sorted, row_of);
  if (e == cudaSuccess)
    by_type(dtype, [&](auto t) {
      using T = decltype(t);
      e = vec_rows(dtype, dim, dy_stride, dy, dweight) ? emb_bwd<T, true>(p, (const T*)dy, (T*)dweight, st) : emb_bwd<T, false>(p, (const T*)dy, (T*)dweight, st);
      return 0;
    });
  return e == cudaSuccess ? 0 : cuda_fail(e, "castle_embedding_bwd launch");
}
