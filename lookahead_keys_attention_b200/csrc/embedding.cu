// Lookup of tokens in a table of rows, scaled, and the table's gradient.
//
//   y[i] = scale W[t_i]                       dW[v] = scale sum over i with t_i = v of dy[i]
//
// Both are bound by memory: a row read and a row written per token; in the gradient a row read per token and the whole table
// written, zero rows included.  The gradient needs the tokens of each row together.  A sort brings them there: it is stable,
// so a row's gradients are added in the order of their positions, in fp32, and the result is the same from call to call
// (atomic additions into the rows would be in arrival order, would need an fp32 table and a pass to round it).
//
// Sort, one launch: a CTA owns a range of rows and reads all tokens, in as many contiguous shares as it has warps.  It counts the
// tokens of smaller rows (where its part of the sorted list begins) and, per warp, those of each of its own; sums of these
// give every (row, warp) its place, and a second reading puts the positions there, lanes with the same token in the order of the
// lanes.  CTAs need nothing of one another, and a row that takes all the tokens is no special case.
//
// Sums: the sorted list is cut into chunks of `piece` entries; a warp takes a chunk's sums in a slab of 256 columns and writes a row when
// its entries end.  (A warp per row instead took 600 us for 65536 tokens with the frequencies of text in 131072 rows of 2048; one per
// sixteen rows 383: the frequent rows are neighbours.)  A row of more entries than a chunk leaves its parts' sums in scratch, which a
// third launch adds in order.
#include "common.cuh"
#include "vec.cuh"

namespace castle {

constexpr int kEmbThreads = 256, kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kSortRows = 1536;   // most rows of a CTA: 32 counters of 4 bytes each
constexpr int kSortBatch = 8;     // tokens that a lane has on their way
constexpr int kSortSeen = 8;      // words of 32 x 32 tokens each per warp: the second reading of up to 262144 tokens skips what the first knows

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

// start[v] = number of tokens (with a row of their own) below v; sorted[start[v] .. start[v + 1]) the positions of v's, in order;
// row_of[k] the token of entry k.
template <typename I>
__global__ void __launch_bounds__(kSortThreads) castle_token_sort_kernel(const void* __restrict__ tokens, int64_t n, int64_t vocab, int64_t padding, int rows,
                                                                         int32_t* __restrict__ start, int32_t* __restrict__ sorted,
                                                                         int32_t* __restrict__ row_of, int32_t* status) {
  extern __shared__ int32_t count[];   // [warp][row]
  __shared__ uint32_t seen[kSortWarps][kSortSeen];   // bit k: of the warp's share, 32 tokens from 32 k on, one is in the range
  __shared__ int32_t warp_sums[kSortWarps + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t lo = (int64_t)blockIdx.x * rows;
  const int own = (int)min((int64_t)rows, vocab - lo);
  const int64_t share = ((n + kSortWarps - 1) / kSortWarps + 31) / 32 * 32, i0 = warp * share, i1 = min(n, i0 + share);
  for (int k = tid; k < kSortWarps * rows; k += kSortThreads) count[k] = 0;
  const bool skip = share <= 1024 * kSortSeen;
  if (lane < kSortSeen) seen[warp][lane] = 0;
  __syncthreads();
  int32_t* mine = count + warp * rows;
  int below = 0;
  bool bad = false;
  for (int64_t i = i0; i < i1; i += 32 * kSortBatch) {
    int64_t t[kSortBatch];
    unsigned hits = 0;
#pragma unroll
    for (int u = 0; u < kSortBatch; ++u) t[u] = i + u * 32 + lane < i1 ? token_at<I>(tokens, i + u * 32 + lane) : padding;
#pragma unroll
    for (int u = 0; u < kSortBatch; ++u) {
      const bool in = i + u * 32 + lane < i1, ok = t[u] >= 0 && t[u] < vocab;
      bad |= in && !ok;
      if (in && ok && t[u] != padding) {
        below += t[u] < lo;
        if (t[u] >= lo && t[u] < lo + own) {
          atomicAdd(&mine[t[u] - lo], 1);
          hits |= 1u << u;
        }
      }
    }
    hits = __reduce_or_sync(0xffffffffu, hits);
    if (skip && hits && lane == 0) {
      const int k = (int)((i - i0) / 32);   // a multiple of the batch, which divides 32
      seen[warp][k / 32] |= hits << (k % 32);
    }
  }
  if (blockIdx.x == 0 && bad) atomicOr(status, CASTLE_STATUS_BAD_INDEX);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) below += __shfl_xor_sync(0xffffffffu, below, o);
  if (lane == 0) warp_sums[warp] = below;
  __syncthreads();
  int base = 0;
  for (int k = 0; k < kSortWarps; ++k) base += warp_sums[k];
  // where each row of the range begins, 1024 rows at a time
  for (int r0 = 0; r0 < own; r0 += kSortThreads) {
    const int r = r0 + tid;
    int total = 0;
    if (r < own)
      for (int k = 0; k < kSortWarps; ++k) total += count[k * rows + r];
    int scan = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += up;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = scan;
    __syncthreads();
    int before = base + scan - total, all = 0;
    for (int k = 0; k < kSortWarps; ++k) {
      if (k < warp) before += warp_sums[k];
      all += warp_sums[k];
    }
    if (r < own) {
      start[lo + r] = before;
      int at = before;
      for (int k = 0; k < kSortWarps; ++k) {
        const int c = count[k * rows + r];
        count[k * rows + r] = at;
        at += c;
      }
    }
    base += all;
  }
  if (tid == 0 && lo + own == vocab) start[vocab] = base;
  __syncthreads();
  for (int64_t i = i0; i < i1; i += 32 * kSortBatch) {
    int local[kSortBatch];
    unsigned look = ~0u;
    if (skip) look = seen[warp][(i - i0) / 1024] >> ((i - i0) / 32 % 32);
    if (!(look & ((1u << kSortBatch) - 1))) continue;
#pragma unroll
    for (int u = 0; u < kSortBatch; ++u) {
      const int64_t k = i + u * 32 + lane, t = k < i1 && (look >> u & 1) ? token_at<I>(tokens, k) : -1;
      local[u] = t >= lo && t < lo + own && t != padding ? (int)(t - lo) : -1;
    }
#pragma unroll
    for (int u = 0; u < kSortBatch; ++u) {
      const bool hit = local[u] >= 0;
      if (!__any_sync(0xffffffffu, hit)) continue;
      const unsigned peers = __match_any_sync(0xffffffffu, local[u]);
      const int at = hit ? mine[local[u]] : 0;
      __syncwarp();
      if (hit) {
        const int rank = __popc(peers & ((1u << lane) - 1));
        if (rank == 0) mine[local[u]] = at + __popc(peers);
        sorted[at + rank] = (int32_t)(i + u * 32 + lane);
        row_of[at + rank] = (int32_t)(lo + local[u]);
      }
      __syncwarp();
    }
  }
}

struct EmbGrad {
  const int32_t *start, *sorted, *row_of;
  float* partial;   // [chunk][2][dim]: of the run that the chunk begins in, and of another one that it ends in
  int64_t vocab, dy_stride;
  int dim, slabs, piece, chunks, group;
  float scale;
};

// Eight rows of dy, a lane's columns of each, as they lie until they are added.
template <typename T, bool VEC> struct EmbBatch {
  Raw8<T> raw[VEC ? 8 : 1];
  float v[VEC ? 1 : 8][8];
  __device__ __forceinline__ void load(int u, const T* row, int slab, int lane, int dim) {
    if constexpr (VEC) {
      const int c = column8<32, true>(slab, lane, 0);
      raw[u] = c < dim ? *reinterpret_cast<const Raw8<T>*>(row + c) : Raw8<T>{};
    } else {
      load_columns8<T, 32, false>(row, slab, lane, dim, v[u]);
    }
  }
  __device__ __forceinline__ void add(int u, float* acc) const {
    float f[8];
    if constexpr (VEC) load8<T>(reinterpret_cast<const T*>(&raw[u]), f);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += VEC ? f[j] : v[VEC ? 0 : u][j];
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

// Warps [0, chunks * slabs): the sums of a chunk's entries in a slab of columns.  A short row (up to `piece` entries, the length of
// a chunk) belongs to the chunk in which it begins, of a longer one each chunk sums its part.  The others: zeros for rows without entries.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kEmbThreads) castle_embedding_bwd_kernel(const EmbGrad p, const T* __restrict__ dy, T* __restrict__ dw) {
  const int lane = threadIdx.x & 31;
  int64_t item = (int64_t)blockIdx.x * (kEmbThreads / 32) + (threadIdx.x >> 5);
  overlap_wait();
  const int64_t pieces = (int64_t)p.chunks * p.slabs;
  float acc[8];
  auto clear = [&] {
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.f;
  };
  clear();
  if (item < pieces) {
    const int c = (int)(item / p.slabs), slab = (int)(item % p.slabs), total = p.start[p.vocab];
    const int a = c * p.piece, b = min(total, a + p.piece);
    if (a >= b) return;
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
    }
    if (from >= to) return;
    int row = p.row_of[from];
    auto store = [&](int next) {
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] *= p.scale;
      store_columns8<T, 32, VEC>(dw + (int64_t)row * p.dim, slab, lane, p.dim, acc);
      clear();
      row = next;
    };
    walk_entries<T, VEC>(p, dy, from, to, slab, lane, acc, [&](int next) {
      if (next != row) store(next);
    });
    store(0);
    return;
  }
  item -= pieces;
  const int wide = (p.slabs + 3) / 4;   // four slabs at a time
  const int64_t row0 = item / wide * p.group;
  const int slab = (int)(item % wide) * 4;
  if (row0 >= p.vocab) return;
  const int rows = (int)min((int64_t)p.group, p.vocab - row0);
  const int begin = p.start[row0 + min(lane, rows)], count = __shfl_down_sync(0xffffffffu, begin, 1) - begin;   // of row row0 + lane
  for (unsigned none = __ballot_sync(0xffffffffu, lane < rows && count == 0); none; none &= none - 1) {
    T* out = dw + (row0 + __ffs(none) - 1) * p.dim;
#pragma unroll
    for (int q = 0; q < 4; ++q) store_columns8<T, 32, VEC>(out, slab + q, lane, p.dim, acc);
  }
}

// A CTA per chunk and slab: if a long row begins in the chunk, the sums of its pieces, eight shares of them in order.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kEmbThreads) castle_embedding_join_kernel(const EmbGrad p, T* __restrict__ dw) {
  __shared__ float s[kEmbThreads / 32][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x, slab = blockIdx.y;
  overlap_wait();
  const int total = p.start[p.vocab], a = c * p.piece, b = min(total, a + p.piece);
  if (a >= b) return;
  const int row = p.row_of[b - 1], r0 = p.start[row], r1 = p.start[row + 1];
  if (r0 < a || r1 - r0 <= p.piece) return;
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
  if (warp > 0) return;
  for (int k = 1; k < kEmbThreads / 32; ++k) {
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += s[k][j * 32 + lane];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] *= p.scale;
  store_columns8<T, 32, VEC>(dw + (int64_t)row * p.dim, slab, lane, p.dim, acc);
}

// Entries of a chunk: as many as leave some sixteen warps per SM with one, 16 to 64.
static int emb_piece(int64_t n, int dim) {
  const int64_t slabs = (dim + 255) / 256;
  int piece = 16;
  while (piece < 64 && n * slabs / piece > 148 * 16) piece *= 2;
  return piece;
}

struct EmbScratch { size_t start, sorted, row_of, partial, bytes; };
static EmbScratch emb_scratch(int64_t n, int64_t vocab, int dim) {
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  const int piece = emb_piece(n, dim);
  EmbScratch s;
  s.start = 0;
  s.sorted = up((size_t)(vocab + 1) * 4);
  s.row_of = s.sorted + up((size_t)n * 4);
  s.partial = s.row_of + up((size_t)n * 4);
  s.bytes = s.partial + (size_t)((n + piece - 1) / piece) * 2 * dim * 4;
  return s;
}

static int emb_check(const char* who, int32_t dtype, int32_t index_bytes, int64_t tokens, int64_t vocab, int32_t dim, const void* index, int64_t stride,
                     const int32_t* status) {
  if (dtype < CASTLE_BF16 || dtype > CASTLE_F32) return reject("%s: unknown dtype", who);
  if (index_bytes != 4 && index_bytes != 8) return reject("%s: tokens must be 32- or 64-bit integers", who);
  if (tokens <= 0 || tokens > 2147483647 || vocab <= 0 || vocab > 2147483646 || dim <= 0 || dim > (1 << 24))
    return reject("%s: %lld tokens, vocabulary %lld, dim %d not supported", who, (long long)tokens, (long long)vocab, dim);
  if (!index || (uintptr_t)index % index_bytes || !status) return reject("%s: tokens (aligned to their size) and a status word are needed", who);
  if (stride < 0) return reject("%s: negative strides are not supported", who);
  return 0;
}

template <typename T, bool VEC>
static cudaError_t emb_bwd(const EmbGrad& p, const T* dy, T* dw, cudaStream_t st) {
  const int64_t warps = (int64_t)p.chunks * p.slabs + (p.vocab + p.group - 1) / p.group * ((p.slabs + 3) / 4);
  const cudaError_t e = launch_kernel(castle_embedding_bwd_kernel<T, VEC>, dim3((unsigned)((warps + 7) / 8)), kEmbThreads, 0, st, true, p, dy, dw);
  return e != cudaSuccess ? e : launch_kernel(castle_embedding_join_kernel<T, VEC>, dim3(p.chunks, p.slabs), kEmbThreads, 0, st, true, p, dw);
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
  return tokens <= 0 || vocab <= 0 || dim <= 0 ? 0 : emb_scratch(tokens, vocab, dim).bytes;
}

extern "C" int castle_embedding_bwd(int32_t dtype, int32_t index_bytes, int64_t tokens, int64_t vocab, int32_t dim, const void* index, int64_t padding_idx,
                                    const void* dy, int64_t dy_stride, float scale, void* dweight, void* workspace, size_t workspace_bytes,
                                    int32_t* status, void* stream) {
  if (int rc = emb_check("castle_embedding_bwd", dtype, index_bytes, tokens, vocab, dim, index, dy_stride, status)) return rc;
  const int es = elem_size(dtype);
  if (!dy || !dweight || ((uintptr_t)dy | (uintptr_t)dweight) % es) return reject("castle_embedding_bwd: dy and dweight must be aligned to their elements");
  const EmbScratch s = emb_scratch(tokens, vocab, dim);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < s.bytes) return reject("castle_embedding_bwd: workspace too small or not 16-byte aligned");
  EmbGrad p;
  char* ws = static_cast<char*>(workspace);
  int32_t *start = (int32_t*)(ws + s.start), *sorted = (int32_t*)(ws + s.sorted), *row_of = (int32_t*)(ws + s.row_of);
  p.start = start; p.sorted = sorted; p.row_of = row_of; p.partial = (float*)(ws + s.partial);
  p.vocab = vocab; p.dy_stride = dy_stride; p.dim = dim; p.slabs = (dim + 255) / 256; p.piece = emb_piece(tokens, dim);
  p.chunks = (int)((tokens + p.piece - 1) / p.piece); p.scale = scale;
  p.group = 1;   // rows that a warp looks through for empty ones: as many as leave some sixteen warps per SM, 16 at most
  while (p.group < 16 && vocab * ((p.slabs + 3) / 4) / p.group > 148 * 16) p.group *= 2;
  if (p.slabs > 65535 || ((int64_t)p.chunks + vocab) * p.slabs / 8 > 2147483646) return reject("castle_embedding_bwd: too many rows");
  // a CTA per SM, of at most kSortRows rows
  int64_t ranges = vocab < 148 ? vocab : 148;
  if ((vocab + ranges - 1) / ranges > kSortRows) ranges = (vocab + kSortRows - 1) / kSortRows;
  const int rows = (int)((vocab + ranges - 1) / ranges);
  const unsigned grid = (unsigned)((vocab + rows - 1) / rows);
  const int smem = rows * kSortWarps * 4;
  const cudaStream_t st = (cudaStream_t)stream;
  auto sort = [&](auto kernel) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortRows * kSortWarps * 4);
    if (e != cudaSuccess) return e;
    kernel<<<grid, kSortThreads, smem, st>>>(index, tokens, vocab, padding_idx, rows, start, sorted, row_of, status);
    return cudaGetLastError();
  };
  cudaError_t e = index_bytes == 8 ? sort(castle_token_sort_kernel<int64_t>) : sort(castle_token_sort_kernel<int32_t>);
  if (e == cudaSuccess)
    by_type(dtype, [&](auto t) {
      using T = decltype(t);
      e = vec_rows(dtype, dim, dy_stride, dy, dweight) ? emb_bwd<T, true>(p, (const T*)dy, (T*)dweight, st) : emb_bwd<T, false>(p, (const T*)dy, (T*)dweight, st);
      return 0;
    });
  return e == cudaSuccess ? 0 : cuda_fail(e, "castle_embedding_bwd launch");
}
