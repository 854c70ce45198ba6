// y = x W^T with weights of 4 bits, for the rows of prompts and batches of them (16-bit types; linear_4bit.cu has the few rows of tokens).
//
// A CTA owns 128 weight rows and up to 256 rows of x (and where that leaves SMs without a tile, a share of K: the CTAs of a cluster add up their results through
// each other's shared memory, in order).  The weights are the first operand of its tcgen05 products and come from tensor memory:
// a thread owns a weight row, loads the 64 bytes of its codes for 128 k, unpacks and scales them, and stores the pairs to its lane, so that the weights at
// full width are never in memory of any kind but that.  The rows of x come by TMA into shared memory, the results are formed in 128 x 256
// fp32 accumulators.  A weight is (code - zero) * scale, rounded to the rows' type (with zero points that are no whole numbers, code - zero
// is rounded as well), as the products' operands have to be.
//
// What bounds it: the products, 4 cycles a column of x and step of 128 k, as long as the tile has some 100 columns; below that the unpacking, some 256
// operations a thread and step, by three groups of four warps in turn.
#include <algorithm>
#include "common.cuh"
#include "linear_4bit_plan.cuh"
#include "sm100.cuh"
#include "vec.cuh"

namespace castle {

// Twelve warps unpack, three groups of four in turn; one loads x, one issues the products.  A stage is 128 k of both operands and has one barrier for them:
// a wait costs the issuing thread some 280 cycles even where it is over, and with a barrier for x and two for halves of the weights the products waited for
// it (777 x 4096 -> 4096 54 us).  The stages are a multiple of the groups, so that a stage is always the same group's: a wait sees only the parity of
// a phase, and a group that came to a stage on every fourth use of three took the phase before last for the last one.
constexpr int kTileGroups = 3, kTileWarps = 4 * kTileGroups, kTileThreads = 32 * (kTileWarps + 2), kTileMaxStages = 6;
constexpr uint32_t kTileSmem = 3 * 2 * 256 * 128;   // three stages of 256 rows of x, or six of 128
constexpr int64_t kTileLaunchRows = 65535 * 32;      // of a launch: a grid's second dimension and the fewest rows of a tile

struct Linear4TileParams {
  const uint4* codes;
  const void *scales, *zeros;
  void* y;
  int rows, K, N, blocks, shift, groups, bn;   // bn: rows of x in a tile, a multiple of 16
  int ks;                                              // CTAs of a cluster, which share K out
  int stages;                                          // six up to 128 rows, three above: tensor memory has bn and 64 columns a stage, rounded up
  bool vec_groups;                                     // eight groups of a row can be loaded at once
  int32_t* status;
  uint32_t mask, bits;                                 // Pair's: as constants the and and the or became an operation each
};

// Eight codes of a word as four pairs of weights.
template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static constexpr int at = 3;
  static constexpr uint32_t mask = 0x00780078u, bits = 0x41804180u;   // 16 + code: the code at the top of the mantissa
  static __device__ __forceinline__ type splat(float v) { return __float2bfloat162_rn(v); }
};
template <> struct Pair<__half> {
  using type = __half2;
  static constexpr int at = 6;
  static constexpr uint32_t mask = 0x03c003c0u, bits = 0x4c004c00u;
  static __device__ __forceinline__ type splat(float v) { return __float2half2_rn(v); }
};
template <typename T, bool ZEROS>
__device__ __forceinline__ void unpack_word(uint32_t w, typename Pair<T>::type scale, typename Pair<T>::type zero, uint32_t mask, uint32_t bits, uint32_t* out) {
  using P = Pair<T>;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int right = 4 * i - P::at;
    uint32_t v = right >= 0 ? w >> right : w << -right;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(v), "r"(mask), "r"(bits));   // v & mask | bits
    typename P::type d = __hsub2(*reinterpret_cast<const typename P::type*>(&v), P::splat(ZEROS ? 16.f : 24.f));   // exact
    if constexpr (ZEROS) d = __hsub2(d, zero);
    d = __hmul2(d, scale);
    out[i] = *reinterpret_cast<const uint32_t*>(&d);
  }
}

template <typename T, bool ZEROS>
__global__ void __launch_bounds__(kTileThreads, 1) castle_linear_4bit_tile_kernel(const __grid_constant__ Linear4TileParams p, const __grid_constant__ CUtensorMap m_x) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t full[kTileMaxStages], free_[kTileMaxStages], done;
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_flag;
  volatile int* abortp = &abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = p.ks > 1 ? (int)cluster_rank() : 0, all = (p.K + 127) / 128;
  const int n0 = blockIdx.x / p.ks * 128, r0 = blockIdx.y * p.bn;
  const int first = all * rank / p.ks, chunks = all * (rank + 1) / p.ks - first;   // this CTA's steps of 128 k
  const uint32_t panel = (uint32_t)p.bn * 128;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kTileMaxStages; ++i) { mbar_init(&full[i], 5); mbar_init(&free_[i], 1); }   // four warps' weights and x
    mbar_init(&done, 1);
    mbar_fence_init();
    abort_flag = 0;
  }
  if (warp == 0) { tmem_alloc(&tmem_base_s, 512); tmem_relinquish(); }
  tc_fence_before();
  overlap_next();
  overlap_wait();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s, weights = tmem + (p.stages == 3 ? 256 : 128);   // columns from 0 on: the results; from `weights` on: the stages of the weights
  if (warp == kTileWarps) {
    if (elect_one()) {
      int c = 0;
      for (int s = 0, turn = 0; c < chunks; ++c) {
        if (turn > 0) mbar_wait(&free_[s], (uint32_t)(turn - 1) & 1, abortp);
        if (*abortp) break;
        mbar_expect_tx(&full[s], 2 * panel);
        uint8_t* x = smem + s * 2 * panel;
        tma_load_4d(x, &m_x, &full[s], (first + c) * 128, r0, 0, 0);
        tma_load_4d(x + panel, &m_x, &full[s], (first + c) * 128 + 64, r0, 0, 0);
        if (++s == p.stages) { s = 0; ++turn; }
      }
      // What is on its way arrives before this thread leaves, whoever else waits for it or gave up.  (Where a wait ran out the weights of a stage may be missing, and
      // these end with their polls.)
      for (int i = max(0, c - p.stages); i < c; ++i) mbar_drain(&full[i % p.stages], (uint32_t)(i / p.stages) & 1);
    }
  } else if (warp == kTileWarps + 1) {
    if (elect_one()) {
      const uint32_t idesc = make_idesc(128, p.bn, Elem<T>::fmt, false, false, false);
      for (int c = 0, s = 0, turn = 0; c < chunks; ++c) {
        mbar_wait(&full[s], (uint32_t)turn & 1, abortp);
        if (*abortp) break;
        tc_fence_after();
        const uint64_t x = desc_kmajor(smem_u32(smem) + s * 2 * panel);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          mma_ts(tmem, weights + s * 64 + k * 8, x + (uint64_t)(((k >> 2) * panel + 32 * (k & 3)) >> 4), idesc, c > 0 || k > 0);
        mma_commit(&free_[s]);
        if (++s == p.stages) { s = 0; ++turn; }
      }
      mma_commit(&done);   // (also after an abort: whatever was issued has ended then)
    }
  } else {
    // ---- a weight row for each thread of a group of four warps, the groups in turn
    const int group = warp >> 2, m = (warp & 3) * 32 + lane;
    const int n = min(n0 + m, p.N - 1);
    const uint4* codes = p.codes + (int64_t)(n >> 4) * p.blocks * 128 + (int64_t)first * 64 + (n >> 3 & 1) * 32 + (n & 7) * 4;
    const T *scales = reinterpret_cast<const T*>(p.scales) + (int64_t)n * p.groups, *zeros = reinterpret_cast<const T*>(p.zeros) + (int64_t)n * p.groups;
    const uint32_t at = weights + ((uint32_t)((warp & 3) * 32) << 16);
    uint4 next[4];             // the codes of this group's next step
    // Scales and zero points eight groups of the row at a time, the next eight on their way: single ones of 32 rows are 32 lines of the cache each,
    // which was the time (777 x 4096 -> 4096, groups of 64: 50 us, with zero points 79).
    uint4 scale8, next_scale8, zero8, next_zero8;
    int window = first * 4 >> p.shift >> 3;
    auto load8 = [&](const T* row, int w) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (p.vec_groups) {
        if (w * 8 < p.groups) v = __ldg(reinterpret_cast<const uint4*>(row + w * 8));
      } else {
        uint32_t* u = &v.x;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (w * 8 + i < p.groups) u[i / 2] |= (uint32_t) * reinterpret_cast<const uint16_t*>(row + w * 8 + i) << (16 * (i & 1));
      }
      return v;
    };
    scale8 = load8(scales, window);
    next_scale8 = load8(scales, window + 1);
    if constexpr (ZEROS) { zero8 = load8(zeros, window); next_zero8 = load8(zeros, window + 1); }
    auto pick = [&](const uint4& v, int g) {   // element g of eight, twice
      const uint32_t w = g & 4 ? (g & 2 ? v.w : v.z) : (g & 2 ? v.y : v.x), r = __byte_perm(w, w, g & 1 ? 0x3232 : 0x1010);
      return *reinterpret_cast<const typename Pair<T>::type*>(&r);
    };
    auto fetch = [&](int c) {
      if (c >= chunks) return;
#pragma unroll
      for (int t = 0; t < 4; ++t) next[t] = __ldg(codes + (int64_t)c * 64 + t);
    };
    fetch(group);
    for (int c = group, s = group, turn = 0; c < chunks; c += kTileGroups) {
      const uint4 q[4] = {next[0], next[1], next[2], next[3]};
      while ((first + c) * 4 >> p.shift >> 3 > window) {   // (a step's four stretches of 32 k are in one window)
        ++window;
        scale8 = next_scale8;
        next_scale8 = load8(scales, window + 1);
        if constexpr (ZEROS) { zero8 = next_zero8; next_zero8 = load8(zeros, window + 1); }
      }
      fetch(c + kTileGroups);
      // (a wait that ran out: the stage may be in use, and its barrier takes no second arrival in a phase)
      if (turn > 0 && mbar_wait_failed(&free_[s], (uint32_t)(turn - 1) & 1, abortp)) break;
      tc_fence_after();
#pragma unroll
      for (int j = 0; j < 4; ++j) {   // 32 k, 16 columns
        uint32_t v[16];
        const int g = ((first + c) * 4 + j) >> p.shift & 7;
        const typename Pair<T>::type scale = pick(scale8, g), zero = ZEROS ? pick(zero8, g) : scale;
#pragma unroll
        for (int t = 0; t < 4; ++t) unpack_word<T, ZEROS>(j == 0 ? q[t].x : j == 1 ? q[t].y : j == 2 ? q[t].z : q[t].w, scale, zero, p.mask, p.bits, v + t * 4);
        tmem_st16(at + s * 64 + j * 16, v);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[s]);
      s += kTileGroups;
      if (s >= p.stages) { s -= p.stages; ++turn; }
    }
    // ---- the results: a thread has some of its weight row's columns, the lanes of a warp adjacent elements of y's rows
    mbar_wait(&done, 0, abortp);
    if (*abortp) mbar_drain(&done, 0);   // tensor memory is not given back under products that are still in flight
    __syncwarp();
    tc_fence_after();
    if (*abortp == 0) {
      T* y = reinterpret_cast<T*>(p.y) + n0 + m;
      float* part = reinterpret_cast<float*>(smem) + m;   // [row of x][weight row], over the stages
      for (int c0 = group * 32; c0 < p.bn; c0 += 32 * kTileGroups) {
        float v[32];
        tmem_ld32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + c0, v);
        tmem_ld_wait();
        if (p.ks > 1) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (c0 + i < p.bn) part[(c0 + i) * 128] = v[i];
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (c0 + i < p.bn && r0 + c0 + i < p.rows && n0 + m < p.N) y[(int64_t)(r0 + c0 + i) * p.N] = Elem<T>::from_f(v[i]);
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
    __syncwarp();
  }
  if (p.ks > 1) {   // the CTAs' shares of K, in order; each adds up some of the rows of x
    cluster_sync();
    const int count = min(p.bn, p.rows - r0) * 128;
    for (int e = rank * kTileThreads + threadIdx.x; e < count; e += p.ks * kTileThreads) {
      float sum = 0.f;
      for (int r = 0; r < p.ks; ++r) sum += cluster_load(reinterpret_cast<const float*>(smem) + e, r);
      const int n = n0 + (e & 127);
      if (n < p.N) reinterpret_cast<T*>(p.y)[(int64_t)(r0 + (e >> 7)) * p.N + n] = Elem<T>::from_f(sum);
    }
    __syncwarp();
    cluster_sync();
  }
  if (threadIdx.x == 0 && abort_flag) atomicOr(p.status, CASTLE_STATUS_WAIT_TIMEOUT);
}

}  // namespace castle

using namespace castle;

extern "C" int castle_linear_4bit_tile(int32_t dtype, int64_t rows, int32_t in_features, int64_t out_features, int32_t group, const void* x, int64_t row_stride,
                                       const void* codes, const void* scales, const void* zeros, void* y, int32_t* status, void* stream) {
  const char* who = "castle_linear_4bit_tile";
  if (dtype != CASTLE_BF16 && dtype != CASTLE_F16) return reject("%s: bf16 or fp16 expected", who);
  if (rows <= 0 || rows > INT32_MAX / 2 || in_features <= 0 || in_features > (1 << 24) || out_features <= 0 || out_features > INT32_MAX / 2)
    return reject("%s: %lld rows of %d -> %lld not supported", who, (long long)rows, in_features, (long long)out_features);
  if (group < 32 || group > (1 << 24) || (group & (group - 1))) return reject("%s: group size %d is not a power of two from 32 up", who, group);
  if (!x || !codes || !scales || !y || !status) return reject("%s: null tensor", who);
  if (((uintptr_t)x | (uintptr_t)codes) % 16 || row_stride * 2 % 16 || row_stride < in_features) return reject("%s: rows and codes must be 16-byte aligned, rows of a multiple of 16 bytes", who);
  if (((uintptr_t)scales | (uintptr_t)zeros | (uintptr_t)y) % 2 || (uintptr_t)status % 4) return reject("%s: scales, zero points and results must be aligned to their type", who);
  Linear4TileParams whole{static_cast<const uint4*>(codes), scales, zeros, y, (int)rows, in_features, (int)out_features, (in_features + 255) / 256, 0, (in_features + group - 1) / group, 0, 1, 0, false, status};
  whole.vec_groups = whole.groups % 8 == 0 && ((uintptr_t)scales | (uintptr_t)zeros) % 16 == 0;
  while ((32 << whole.shift) < group) ++whole.shift;
  const int64_t n_tiles = (out_features + 127) / 128;
  whole.mask = dtype == CASTLE_BF16 ? Pair<__nv_bfloat16>::mask : Pair<__half>::mask;
  whole.bits = dtype == CASTLE_BF16 ? Pair<__nv_bfloat16>::bits : Pair<__half>::bits;
  auto launch = [&](auto kernel) {
    for (int64_t done = 0; done < rows; done += kTileLaunchRows) {
      Linear4TileParams p = whole;
      p.rows = (int)std::min(rows - done, kTileLaunchRows);
      p.y = static_cast<char*>(y) + done * out_features * 2;
      const TilePlan plan = linear_4bit_tile_plan(p.rows, in_features, out_features);
      p.bn = plan.bn;
      p.ks = plan.ks;
      p.stages = p.bn <= 128 ? 6 : 3;
      CUtensorMap m_x;
      const castle_tensor_t t{static_cast<char*>(const_cast<void*>(x)) + done * row_stride * 2, p.rows * row_stride, p.rows * row_stride, row_stride};
      if (const int rc = make_tmap_16bit(&m_x, &t, dtype, 1, 1, p.rows, in_features, p.bn, "x")) return rc;
      cudaError_t e = allow_smem(kernel, kTileSmem + 1024);
      cudaLaunchConfig_t c = {};
      cudaLaunchAttribute attr[2];
      attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[0].val.programmaticStreamSerializationAllowed = 1;
      attr[1].id = cudaLaunchAttributeClusterDimension;
      attr[1].val.clusterDim = {(unsigned)p.ks, 1, 1};
      c.gridDim = dim3((unsigned)(n_tiles * p.ks), (unsigned)((p.rows + p.bn - 1) / p.bn)); c.blockDim = dim3(kTileThreads);
      c.dynamicSmemBytes = kTileSmem + 1024; c.stream = (cudaStream_t)stream; c.attrs = attr; c.numAttrs = p.ks > 1 ? 2 : 1;
      if (e == cudaSuccess) e = cudaLaunchKernelEx(&c, kernel, p, m_x);
      if (e != cudaSuccess) return cuda_fail(e, "castle_linear_4bit_tile launch");
    }
    return 0;
  };
  if (dtype == CASTLE_BF16) return zeros ? launch(castle_linear_4bit_tile_kernel<__nv_bfloat16, true>) : launch(castle_linear_4bit_tile_kernel<__nv_bfloat16, false>);
  return zeros ? launch(castle_linear_4bit_tile_kernel<__half, true>) : launch(castle_linear_4bit_tile_kernel<__half, false>);
}
