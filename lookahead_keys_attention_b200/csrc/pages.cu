// Pages of a cache: copies inside pools (a fork's, a compaction's), and a prompt's rows into pages.  Both read and write each byte once;
// what bounds them is HBM, and for a few pages a launch.
#include <algorithm>
#include <new>
#include <vector>
#include "common.cuh"
#include "sm100.cuh"

namespace castle {

constexpr int kCopyThreads = 256, kCopyLoads = 4, kCopyChunk = kCopyThreads * kCopyLoads * 16;   // bytes of a CTA

// Which pages, by kernel argument: a host list needs no copy to the device of its own, and is read when the call returns.
constexpr int kCopyPools = 24, kCopyPairs = 400;
struct CopyPool { uint8_t* ptr; int64_t stride_page, stride_block; };
struct CopyParams {
  int64_t block_bytes;
  int chunks;                      // of a block
  CopyPool pool[kCopyPools];
  int32_t source[kCopyPairs], target[kCopyPairs];
};
static_assert(sizeof(CopyParams) <= 4096, "a kernel's arguments");

__global__ void __launch_bounds__(kCopyThreads) castle_copy_pages_kernel(const __grid_constant__ CopyParams p) {
  const CopyPool pool = p.pool[blockIdx.z];
  const int64_t block = blockIdx.x / p.chunks, begin = (int64_t)(blockIdx.x % p.chunks) * kCopyChunk;
  const int64_t bytes = min(p.block_bytes - begin, (int64_t)kCopyChunk);
  const uint8_t* src = pool.ptr + p.source[blockIdx.y] * pool.stride_page + block * pool.stride_block + begin;
  uint8_t* dst = pool.ptr + p.target[blockIdx.y] * pool.stride_page + block * pool.stride_block + begin;
  uint4 v[kCopyLoads];
#pragma unroll
  for (int i = 0; i < kCopyLoads; ++i) {
    const int64_t at = (int64_t)(i * kCopyThreads + threadIdx.x) * 16;
    if (at < bytes) v[i] = *reinterpret_cast<const uint4*>(src + at);
  }
#pragma unroll
  for (int i = 0; i < kCopyLoads; ++i) {
    const int64_t at = (int64_t)(i * kCopyThreads + threadIdx.x) * 16;
    if (at < bytes) *reinterpret_cast<uint4*>(dst + at) = v[i];
  }
}

// A set of pages, on the host: places of a table that is at most half full, one behind the other from where a page's number leads.  (Of the standard
// library's sets a call with 1000 pairs took 47 us.)
class PageSet {
 public:
  explicit PageSet(int64_t count) {
    while (((int64_t)1 << bits_) < 2 * count) ++bits_;
    places_.assign((size_t)1 << bits_, -1);
  }
  bool insert(int32_t page) {
    size_t at = find(page);
    if (places_[at] == page) return false;
    places_[at] = page;
    return true;
  }
  bool has(int32_t page) const { return places_[find(page)] == page; }

 private:
  size_t find(int32_t page) const {   // the page's place, or the free one where it would be
    size_t at = (size_t)(((uint64_t)(uint32_t)page * 0x9e3779b97f4a7c15ull) >> (64 - bits_));
    while (places_[at] != -1 && places_[at] != page) at = (at + 1) & (places_.size() - 1);
    return at;
  }
  int bits_ = 1;
  std::vector<int32_t> places_;
};

struct WriteParams {
  castle_tensor_t src[4];          // U, qu, kc, vc
  castle_pages_t dst[4];
  const int32_t *u_table, *table, *lengths;
  int64_t u_table_stride, table_stride;
  int H, N, page_shift, capacity, u_pages, pages;
  int es, lanes, tiles;            // bytes of an element, 16-byte vectors of a row, CTAs of a pair
  int32_t* status;
};

// Grid: (pair, tile of rows), four caches.  A thread copies 16-byte vectors, kCopyLoads on their way.
__global__ void __launch_bounds__(kCopyThreads) castle_write_pages_kernel(const WriteParams p) {
  const int which = blockIdx.y, pair = blockIdx.x / p.tiles, tile = blockIdx.x % p.tiles, b = pair / p.H, h = pair % p.H;
  const int length = p.lengths[b];
  if (length > p.N || length > p.capacity) {
    if (threadIdx.x == 0) atomicOr(p.status, CASTLE_STATUS_BAD_INDEX);
    return;
  }
  const int rows = kCopyThreads * kCopyLoads / p.lanes;   // of a tile
  const int32_t* table = which == 0 ? p.u_table + b * p.u_table_stride : p.table + b * p.table_stride;
  const uint32_t pages = which == 0 ? p.u_pages : p.pages;
  const castle_tensor_t s = p.src[which];
  const castle_pages_t d = p.dst[which];
  const uint8_t* src = static_cast<const uint8_t*>(s.ptr) + (b * s.stride_b + h * s.stride_h) * p.es;
  uint8_t* dst = static_cast<uint8_t*>(d.ptr) + h * d.stride_h * p.es;
  uint4 v[kCopyLoads];
  int page[kCopyLoads];
#pragma unroll
  for (int i = 0; i < kCopyLoads; ++i) {
    const int e = i * kCopyThreads + threadIdx.x, in = e / p.lanes, r = tile * rows + in;
    page[i] = -1;
    if (in < rows && r < length) {
      v[i] = *reinterpret_cast<const uint4*>(src + r * s.stride_n * p.es + e % p.lanes * 16);
      page[i] = table[r >> p.page_shift];
      if ((uint32_t)page[i] >= pages) {
        page[i] = -1;
        atomicOr(p.status, CASTLE_STATUS_BAD_INDEX);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kCopyLoads; ++i) {
    const int e = i * kCopyThreads + threadIdx.x, r = tile * rows + e / p.lanes;
    if (page[i] >= 0)
      *reinterpret_cast<uint4*>(dst + page[i] * d.stride_page * p.es + ((int64_t)(r & ((1 << p.page_shift) - 1)) * p.lanes + e % p.lanes) * 16) = v[i];
  }
}

}  // namespace castle

using namespace castle;

extern "C" int castle_copy_pages(int32_t pools, void* const* ptr, const int64_t* stride_page, const int64_t* stride_block, int64_t blocks, int64_t block_bytes,
                                 int64_t pages, const int32_t* source, const int32_t* target, int64_t count, void* stream) {
  const char* who = "castle_copy_pages";
  if (pools < 0 || count < 0 || blocks <= 0 || block_bytes <= 0 || pages < 0) return reject("%s: negative or empty sizes", who);
  if (pools == 0 || count == 0) return 0;
  if (!ptr || !stride_page || !stride_block || !source || !target) return reject("%s: null arrays", who);
  if (block_bytes % 16) return reject("%s: blocks of %lld bytes are not multiples of 16", who, (long long)block_bytes);
  const int64_t chunks = (block_bytes + kCopyChunk - 1) / kCopyChunk;
  if (blocks > INT32_MAX / chunks) return reject("%s: pages of %lld x %lld bytes are too large", who, (long long)blocks, (long long)block_bytes);
  for (int32_t k = 0; k < pools; ++k) {
    if (!ptr[k] || (uintptr_t)ptr[k] % 16) return reject("%s: pool %d is null or not 16-byte aligned", who, k);
    if (stride_page[k] % 16 || stride_block[k] % 16) return reject("%s: the strides of pool %d are not multiples of 16 bytes", who, k);
    for (int32_t j = 0; j < k; ++j)
      if (ptr[j] == ptr[k]) return reject("%s: pool %d is pool %d again", who, k, j);
  }
  try {
    PageSet targets(count);
    for (int64_t i = 0; i < count; ++i) {
      if (source[i] < 0 || source[i] >= pages || target[i] < 0 || target[i] >= pages)
        return reject("%s: pair %lld (%d to %d) is outside the %lld pages", who, (long long)i, source[i], target[i], (long long)pages);
      if (!targets.insert(target[i])) return reject("%s: page %d is a target twice", who, target[i]);
    }
    for (int64_t i = 0; i < count; ++i)
      if (targets.has(source[i])) return reject("%s: page %d is a target and a source", who, source[i]);
  } catch (const std::bad_alloc&) {
    return reject("%s: out of host memory", who);
  }
  CopyParams q;
  q.block_bytes = block_bytes;
  q.chunks = (int)chunks;
  for (int32_t k0 = 0; k0 < pools; k0 += kCopyPools) {
    const int nk = std::min(pools - k0, kCopyPools);
    for (int k = 0; k < nk; ++k) q.pool[k] = {static_cast<uint8_t*>(ptr[k0 + k]), stride_page[k0 + k], stride_block[k0 + k]};
    for (int64_t i0 = 0; i0 < count; i0 += kCopyPairs) {
      const int n = (int)std::min<int64_t>(count - i0, kCopyPairs);
      std::copy(source + i0, source + i0 + n, q.source);
      std::copy(target + i0, target + i0 + n, q.target);
      const cudaError_t e = launch_kernel(castle_copy_pages_kernel, dim3((unsigned)(blocks * chunks), n, nk), kCopyThreads, 0, (cudaStream_t)stream, false, q);
      if (e != cudaSuccess) return cuda_fail(e, "castle_copy_pages launch");
    }
  }
  return 0;
}

extern "C" int castle_write_pages(const castle_problem_t* p, int32_t page_size, int32_t u_pages, int32_t pages, const castle_tensor_t* u, const castle_tensor_t* qu,
                                  const castle_tensor_t* kc, const castle_tensor_t* vc, const castle_pages_t* u_cache, const castle_pages_t* qu_cache,
                                  const castle_pages_t* kc_cache, const castle_pages_t* vc_cache, const int32_t* u_table, int64_t u_table_stride, const int32_t* table,
                                  int64_t table_stride, int32_t table_width, const int32_t* lengths, int32_t* status, void* stream) {
  const char* who = "castle_write_pages";
  if (!p || p->batch <= 0 || p->heads <= 0 || p->seq_len <= 0) return reject("%s: null problem, or no sequences, heads or positions", who);
  if (p->dtype < CASTLE_BF16 || p->dtype > CASTLE_F32) return reject("%s: unknown dtype %d", who, p->dtype);
  const int es = elem_size(p->dtype);
  if (p->dim_head <= 0 || p->dim_head * es % 16 || p->dim_head * es > 16 * kCopyThreads * kCopyLoads) return reject("%s: dim_head %d not supported", who, p->dim_head);
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return reject("%s: page size %d is not a power of two from 16 to 1024", who, page_size);
  if (u_pages <= 0 || pages <= 0 || table_width <= 0) return reject("%s: empty pools or tables", who);
  if ((int64_t)table_width * page_size > INT32_MAX - 1024) return reject("%s: %d pages of %d positions are too many", who, table_width, page_size);
  if (p->seq_len > INT32_MAX - 1024) return reject("%s: %d positions are too many", who, p->seq_len);   // (a tile's rows past the last one are counted in 32 bits)
  if (!u_table || !table || !lengths || !status) return reject("%s: null table, lengths or status", who);
  if (((uintptr_t)u_table | (uintptr_t)table | (uintptr_t)lengths | (uintptr_t)status) % 4) return reject("%s: tables, lengths and status must be 4-byte aligned", who);
  if (u_table_stride < 0 || table_stride < 0) return reject("%s: negative table strides", who);
  WriteParams q;
  int rc = 0;
  const castle_tensor_t* src[4] = {u, qu, kc, vc};
  const castle_pages_t* dst[4] = {u_cache, qu_cache, kc_cache, vc_cache};
  const char* names[4] = {"u", "qu", "kc", "vc"};
  for (int i = 0; i < 4; ++i) {
    if (!tensor_ok(src[i], p->dtype, names[i], &rc)) return rc;
    if (!dst[i] || !dst[i]->ptr || (uintptr_t)dst[i]->ptr % 16 || dst[i]->stride_page * es % 16 || dst[i]->stride_h * es % 16)
      return reject("%s: the pages of %s are null, or their address or strides not multiples of 16 bytes", who, names[i]);
    q.src[i] = *src[i];
    q.dst[i] = *dst[i];
  }
  q.u_table = u_table; q.table = table; q.lengths = lengths; q.u_table_stride = u_table_stride; q.table_stride = table_stride;
  q.H = p->heads; q.N = p->seq_len; q.capacity = table_width * page_size; q.u_pages = u_pages; q.pages = pages; q.status = status;
  q.page_shift = 0;
  while ((1 << q.page_shift) < page_size) ++q.page_shift;
  q.es = es;
  q.lanes = p->dim_head * es / 16;
  const int64_t rows = kCopyThreads * kCopyLoads / q.lanes, tiles = (p->seq_len + rows - 1) / rows, pairs = (int64_t)p->batch * p->heads;
  if (pairs > INT32_MAX / tiles) return reject("%s: %d sequences x %d heads x %d positions are too many", who, p->batch, p->heads, p->seq_len);
  q.tiles = (int)tiles;
  const cudaError_t e = launch_kernel(castle_write_pages_kernel, dim3((unsigned)(pairs * tiles), 4), kCopyThreads, 0, (cudaStream_t)stream, false, q);
  return e == cudaSuccess ? 0 : cuda_fail(e, "castle_write_pages launch");
}
