// Cross entropy of a linear head, forward and backward, without its logits.
//
//   z = x W^T,   loss_i = log sum_v exp z_iv - z_it,   G_iv = c_i (exp(z_iv - lse_i) - [v = t_i]),   dx = G W,   dW = G^T x
//
// with c_i the upstream gradient of row i's loss.  Rows whose target is to be ignored take no part: the others are counted and,
// where any are ignored, gathered into adjacent rows first, so that work goes with their number and whatever an ignored row holds
// (NaN, say) reaches nothing.  How many rows there are is known on the device only; the products read it there.
//
//   castle_ce_rows_kernel    the rows that take part: their number, their places, targets, coefficients; their gathered copies
//   castle_ce_kernel<kLse>   tiles of z; each leaves (max, sum of exponentials) of its part of every row
//   castle_ce_join_kernel    these parts together: lse, the losses and their sum
//   castle_ce_kernel<kGrad>  tiles of z again, and from them G in the operands' type, for a piece of the vocabulary
//   castle_ce_kernel<kDx>    dx += G W of the piece (fp32 sums in scratch if there are several pieces, or shares of a long sum)
//   castle_ce_kernel<kDw>    dW of the piece
//
// The four products are one kernel: CTAs that stay, one per SM, with a warp that loads tiles by TMA, a warp that issues the tensor
// cores' products (128 x 256 of the result, 64 of the contraction at a time), and eight warps that work on a finished tile in one
// half of tensor memory while the next one is summed in the other.  All sums, the logits and the statistics are fp32.
//
// fp32 tensors: every value is the sum of three bf16 ones (8 bits each: 24), and a product is the six largest of the nine products
// of such parts (what is left out is 2^-24 of it), the smallest first.  So the same kernels serve, with six times the steps.
//
// The tensor cores cut what they add to an accumulator, always towards zero, so a long sum is off by some 2^-24 per addition (197 rows
// of 512, fp32: losses 3.3e-6 off, gradients of longer sums 1.7e-5, where fp32 arithmetic has 2e-7).  Where the result has 32 bits
// (the logits' statistics, and everything of fp32 tensors), accumulators are therefore emptied every `flush` steps into sums that
// the working warps keep in registers.
//
// G in 16 bits: c_i is taken in units of a power of two that leaves G below 2^15 (the unit is multiplied back in fp32 at the
// end), so that fp16 keeps probabilities down to 2^-28 in full precision; rounding G is off by half a step of the type, as
// rounding the logits' gradient is where logits are tensors of that type.
#include <type_traits>

#include "common.cuh"
#include "vec.cuh"

namespace castle {

enum CeMode { kLse, kGrad, kDx, kDw };

constexpr int kCeM = 128, kCeN = 256, kCeK = 64, kCeStages = 4, kCeThreads = 320;
constexpr uint32_t kCeA = kCeM * kCeK * 2, kCeB = kCeN * kCeK * 2, kCeStage = kCeA + kCeB;
constexpr uint32_t kCeStaging = 8 * 4096;   // kGrad: 32 rows x 64 columns of each working warp
constexpr size_t kCeSmem = kCeStages * kCeStage + kCeStaging + 1024;
constexpr int64_t kCeScratch = (int64_t)1 << 30;   // bytes that a piece of the vocabulary may take
// Steps between emptyings: of a 16-bit operand's logits (32 additions in the tensor cores), of fp32's parts (24).  197 x 512 in
// fp32: TBD
constexpr int kCeFlush = 8, kCeFlushF32 = 1, kCeNoFlush = 1 << 30;
constexpr float kCeUnit = 16384.f;                 // of G: |c| < 2 units

struct CeHead {          // at the start of the workspace, written by castle_ce_rows_kernel
  int rows;              // that take part
  int gathered;          // whether they lie in the copy
  int bad;               // targets outside the vocabulary
  unsigned done;         // CTAs of the join that have ended
  float unit;            // of G, multiplied back into dx and dW
};
struct CeRow { int target; float lse, coef; int row; };   // of the rows that take part, in order; row: in the caller's tensors

__constant__ const int8_t kTermA[6] = {2, 0, 1, 1, 0, 0}, kTermB[6] = {0, 2, 1, 0, 1, 0};   // one term: the last

// ------------------------------------------------------------------------------------------------ rows that take part
struct CeRowsParams {
  const int64_t* targets;
  const void* x;
  const float *lse, *dloss;   // backward; NULL in the forward
  int64_t n, vocab, ignore, x_stride, copy_rows;
  int dim, pitch, planes, rows_per_cta, mean, each;
  bool copy_always;
  CeHead* head;
  CeRow* rows;
  uint16_t* copy;             // [plane][copy_rows][pitch]
  void* dx;                   // rows that take no part become zero; NULL: none wanted
  float *loss, *lse_out;      // forward: loss of each row (NULL unless wanted) and lse
  int32_t* status;
};

__device__ __forceinline__ int block_sum(int v, int* s) {   // of 1024 threads
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  int t = 0;
  for (int k = 0; k < 32; ++k) t += s[k];
  return t;
}

// One value as one 16-bit number, or as three whose sum it is.
template <typename T> struct CePlanes {
  static constexpr int count = 1;
  using Op = T;
  static __device__ __forceinline__ void split(float v, float* p) { p[0] = v; }
};
template <> struct CePlanes<float> {
  static constexpr int count = 3;
  using Op = __nv_bfloat16;
  static __device__ __forceinline__ void split(float v, float* p) {
    p[0] = __bfloat162float(__float2bfloat16_rn(v));
    const float r = v - p[0];
    p[1] = isfinite(p[0]) ? __bfloat162float(__float2bfloat16_rn(r)) : 0.f;   // an infinity is its first part alone
    p[2] = isfinite(p[0]) ? r - p[1] : 0.f;
  }
};
// A row into its planes, by a warp; columns from dim to pitch are zero.
template <typename T>
__device__ __forceinline__ void copy_row(const T* src, uint16_t* dst, int64_t plane, int dim, int pitch, int lane) {
  using Op = typename CePlanes<T>::Op;
  constexpr int P = CePlanes<T>::count;
  const bool vec = P == 1 && dim % 8 == 0 && reinterpret_cast<uintptr_t>(src) % 16 == 0;
  if (vec) {
#pragma unroll 4
    for (int c = lane * 8; c < dim; c += 256) *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(src + c);
    return;
  }
  for (int c = lane * 2; c < pitch; c += 64) {
    float a[P], b[P];
    CePlanes<T>::split(c < dim ? load1<T>(src + c) : 0.f, a);
    CePlanes<T>::split(c + 1 < dim ? load1<T>(src + c + 1) : 0.f, b);
#pragma unroll
    for (int p = 0; p < P; ++p) *reinterpret_cast<uint32_t*>(dst + p * plane + c) = Elem<Op>::pack2(a[p], b[p]);
  }
}

// Every CTA reads all targets (and, in a backward with a gradient per row, these), so it needs nothing of the others.
template <typename T>
__global__ void __launch_bounds__(1024, 1) castle_ce_rows_kernel(const CeRowsParams p) {
  __shared__ int s[32];
  __shared__ float sf[32];
  __shared__ int place[1024];   // of a row in the gathered order, -1: it takes no part
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r0 = (int64_t)blockIdx.x * p.rows_per_cta, r1 = min(p.n, r0 + p.rows_per_cta);
  overlap_wait();
  int before = 0, all = 0, ignored = 0;
  float most = 0.f;
#pragma unroll 4
  for (int64_t i = tid; i < p.n; i += 1024) {
    const int64_t t = p.targets[i];
    const bool on = t != p.ignore && t >= 0 && t < p.vocab;
    ignored += t == p.ignore;
    all += on;
    before += on && i < r0;
    if (p.each && on) {
      const float g = fabsf(p.dloss[i]);
      if (g < INFINITY) most = fmaxf(most, g);
    }
  }
  before = block_sum(before, s);
  all = block_sum(all, s);
  ignored = block_sum(ignored, s);
  float g_one = 0.f, unit = 1.f;
  if (p.dloss) {
    if (p.each) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (lane == 0) sf[warp] = most;
      __syncthreads();
      for (int k = 0; k < 32; ++k) most = fmaxf(most, sf[k]);
    } else {
      g_one = p.dloss[0];
      if (p.mean) g_one /= (float)(p.n - ignored);
      if (fabsf(g_one) < INFINITY) most = fabsf(g_one);
    }
    if (most > 0.f) unit = __uint_as_float(max(__float_as_uint(most) & 0x7f800000u, 0x00800000u));   // its power of two
  }
  const bool gather = all < p.n;
  if (blockIdx.x == 0 && tid == 0) {
    CeHead h;
    h.rows = all;
    h.gathered = gather || p.copy_always;
    h.bad = (int)(p.n - ignored) - all;
    h.done = 0;
    h.unit = unit * (1.f / kCeUnit);
    *p.head = h;
    if (h.bad) atomicOr(p.status, CASTLE_STATUS_BAD_INDEX);
  }
  for (int64_t i0 = r0; i0 < r1; i0 += 1024) {   // the CTA's own rows, 1024 at a time
    const int64_t i = i0 + tid;
    int64_t t = -1;
    bool on = false, skip = true;
    if (i < r1) {
      t = p.targets[i];
      skip = t == p.ignore;
      on = !skip && t >= 0 && t < p.vocab;
    }
    const unsigned vote = __ballot_sync(0xffffffffu, on);
    __syncthreads();
    if (lane == 0) s[warp] = __popc(vote);
    __syncthreads();
    int at = before, total = 0;
    for (int k = 0; k < 32; ++k) {
      if (k < warp) at += s[k];
      total += s[k];
    }
    at += __popc(vote & ((1u << lane) - 1));
    before += total;
    place[tid] = on ? at : -1;
    if (on) {
      CeRow r;
      r.target = (int)t;
      r.row = (int)i;
      r.lse = p.lse ? p.lse[i] : 0.f;
      r.coef = p.dloss ? (p.each ? p.dloss[i] : g_one) / unit * kCeUnit : 0.f;
      p.rows[at] = r;
    } else if (i < r1 && p.lse_out) {
      const float none = skip ? 0.f : __int_as_float(0x7fffffff);
      p.lse_out[i] = none;
      if (p.loss) p.loss[i] = none;
    }
    __syncthreads();
    if (gather || p.copy_always) {
      const int64_t plane = p.copy_rows * p.pitch;
      const int have = (int)min((int64_t)1024, r1 - i0);
      for (int k = warp; k < have; k += 32) {
        const T* src = static_cast<const T*>(p.x) + (i0 + k) * p.x_stride;
        if (place[k] >= 0) {
          copy_row<T>(src, p.copy + (int64_t)place[k] * p.pitch, plane, p.dim, p.pitch, lane);
        } else if (p.dx) {
          T* row = static_cast<T*>(p.dx) + (i0 + k) * p.dim;
          for (int c = lane; c < p.dim; c += 32) store1<T>(row + c, 0.f);
        }
      }
    }
  }
  // what the contraction over rows reads behind the last one
  if ((gather || p.copy_always) && blockIdx.x == gridDim.x - 1) {
    const int64_t plane = p.copy_rows * p.pitch;
    const int64_t end = min(p.copy_rows, ((int64_t)all + kCeK - 1) / kCeK * kCeK);
    for (int64_t k = all + warp; k < end; k += 32)
      for (int q = 0; q < p.planes; ++q)
        for (int c = lane; c < p.pitch; c += 32) p.copy[q * plane + k * p.pitch + c] = 0;
  }
}

// Rows of the weight into their planes, a warp each.
template <typename T>
__global__ void __launch_bounds__(256) castle_ce_split_kernel(const T* __restrict__ w, int64_t stride, uint16_t* __restrict__ out, int64_t rows, int dim, int pitch) {
  const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  overlap_wait();
  if (r < rows) copy_row<T>(w + r * stride, out + r * pitch, rows * pitch, dim, pitch, threadIdx.x & 31);
}

// ------------------------------------------------------------------------------------------------ the products
struct CeProduct {
  const CeHead* head;
  const CeRow* rows;
  int m, n, k;           // of the result and the contraction; m (kDw: k) is the number of rows that take part instead
  int b_row0;            // where the piece begins in B's rows (kLse, kGrad: along n, kDx: along k)
  int vocab0, vocab;     // the piece's first column of z, and how many there are (kLse, kGrad)
  int terms, splits, group;
  int flush;             // steps after which an accumulator is emptied
  // kLse
  float2* parts;         // [2 per tile of n][parts_ld]
  float* target_logit;
  int64_t parts_ld;
  // kDx, kDw
  void* out;             // (rows, ld)
  float* slab;           // [split][slab_rows][slab_ld] instead of out, if not NULL
  int64_t ld, slab_rows, slab_ld, out_row0;
  bool vec, add;         // out can be stored 16 bytes at a time; the slab's values are added to
  int32_t* status;
};

template <CeMode MODE> struct CeTiles {
  int tiles_m, tiles_n, steps, total, group;   // steps: of 64 of the contraction, all shares and terms
  int per;                                      // steps of a share
  __device__ __forceinline__ CeTiles(const CeProduct& p, int rows) {
    tiles_m = ((MODE == kDw ? p.m : rows) + kCeM - 1) / kCeM;
    tiles_n = (p.n + kCeN - 1) / kCeN;
    steps = ((MODE == kDw ? rows : p.k) + kCeK - 1) / kCeK;
    per = (steps + p.splits - 1) / p.splits;
    total = tiles_m * tiles_n * p.splits;
    group = min(p.group, max(tiles_m, 1));
  }
  // Tiles in bands of `group` tiles of rows, down the rows first: CTAs that run together share rows of both operands.
  __device__ __forceinline__ void at(int t, int& m, int& n, int& split) const {
    const int plane = tiles_m * tiles_n;
    split = t / plane;
    t -= split * plane;
    const int band = t / (group * tiles_n), first = band * group, high = min(group, tiles_m - first);
    t -= band * group * tiles_n;
    n = t / high;
    m = first + t - n * high;
  }
  __device__ __forceinline__ int begin(int split) const { return min(steps, split * per); }
  __device__ __forceinline__ int end(int split) const { return min(steps, (split + 1) * per); }
};

// T: the operands' type, OUT: the result's (kDx, kDw) or the caller's (kGrad: float means three planes of G).
template <typename T, typename OUT, CeMode MODE>
__global__ void __launch_bounds__(kCeThreads) castle_ce_kernel(const CeProduct p, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_copy,
                                                               const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_g) {
  constexpr bool A_MN = MODE == kDw, B_MN = MODE == kDx || MODE == kDw;
  constexpr bool REG = MODE == kLse || CePlanes<OUT>::count > 1;   // accumulators are emptied into registers on the way
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t bar_full[kCeStages], bar_free[kCeStages], bar_done[2], bar_read[2], bar_end;
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < kCeStages; ++s) { mbar_init(&bar_full[s], 1); mbar_init(&bar_free[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&bar_done[s], 1); mbar_init(&bar_read[s], 8); }
    mbar_init(&bar_end, 1);
    mbar_fence_init();
    abort_flag = 0;
    tma_prefetch_desc(&map_a); tma_prefetch_desc(&map_b);
  }
  if (warp == 1) { tmem_alloc(&tmem_base_s, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;
  volatile int* abortp = &abort_flag;
  overlap_wait();
  const CeHead head = *p.head;
  const CeTiles<MODE> tiles(p, head.rows);
  const int first = blockIdx.x, stride = gridDim.x;

  if (warp == 0) {
    if (elect_one()) {
      const bool copy = head.gathered;
      const CUtensorMap* ma = MODE != kDx && MODE != kDw && copy ? &map_copy : &map_a;
      const CUtensorMap* mb = MODE == kDw && copy ? &map_copy : &map_b;
      int it = 0;
      for (int t = first; t < tiles.total && !*abortp; t += stride) {
        int m, n, split;
        tiles.at(t, m, n, split);
        const int m0 = m * kCeM, n0 = n * kCeN;
        for (int ks = tiles.begin(split); ks < tiles.end(split); ++ks) {
          for (int term = 6 - p.terms; term < 6; ++term, ++it) {
            const int s = it % kCeStages, k = ks * kCeK, pa = kTermA[term], pb = kTermB[term];
            if (!mbar_wait_ok<true>(&bar_free[s], ((uint32_t)(it / kCeStages) & 1u) ^ 1u, abortp)) { ks = tiles.end(split); break; }
            uint8_t *a = smem + s * kCeStage, *b = a + kCeA;
            mbar_expect_tx(&bar_full[s], kCeStage);
            if (A_MN) {
              tma_load_4d(a, ma, &bar_full[s], m0, k, pa, 0);
              tma_load_4d(a + kCeA / 2, ma, &bar_full[s], m0 + 64, k, pa, 0);
            } else {
              tma_load_4d(a, ma, &bar_full[s], k, m0, pa, 0);
            }
            if (B_MN) {
#pragma unroll
              for (int j = 0; j < 4; ++j) tma_load_4d(b + j * (kCeB / 4), mb, &bar_full[s], n0 + j * 64, k + (MODE == kDx ? p.b_row0 : 0), pb, 0);
            } else {
              tma_load_4d(b, mb, &bar_full[s], k, p.b_row0 + n0, pb, 0);
            }
          }
        }
      }
      // a copy that nobody waited for (after an abort) must not arrive in another CTA's shared memory
      if (*abortp)
        for (int j = max(0, it - kCeStages); j < it; ++j) mbar_drain(&bar_full[j % kCeStages], (uint32_t)(j / kCeStages) & 1u);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      int it = 0, turn = 0;
      for (int t = first; t < tiles.total && !*abortp; t += stride) {
        int m, n, split;
        tiles.at(t, m, n, split);
        const int cols = min(kCeN, (p.n - n * kCeN + 15) / 16 * 16);
        const uint32_t idesc = make_idesc(kCeM, 16, Elem<T>::fmt, A_MN, B_MN, false) + ((uint32_t)((cols - 16) >> 3) << 17);
        for (int k0 = tiles.begin(split); k0 < tiles.end(split) && !*abortp; k0 += p.flush, ++turn) {
          const int acc = turn & 1, steps = min(p.flush, tiles.end(split) - k0) * p.terms;
          const uint32_t d = tmem + acc * kCeN;
          if (!mbar_wait_ok<true>(&bar_read[acc], ((uint32_t)(turn >> 1) & 1u) ^ 1u, abortp)) break;
          tc_fence_after();
          for (int j = 0; j < steps; ++j, ++it) {
            const int s = it % kCeStages;
            if (!mbar_wait_ok<true>(&bar_full[s], (uint32_t)(it / kCeStages) & 1u, abortp)) break;
            tc_fence_after();
            const uint32_t a = smem_u32(smem) + s * kCeStage, b = a + kCeA;
            const uint64_t da = A_MN ? desc_mnmajor(a, kCeA / 2) : desc_kmajor(a), db = B_MN ? desc_mnmajor(b, kCeB / 4) : desc_kmajor(b);
#pragma unroll
            for (int q = 0; q < kCeK / 16; ++q)
              mma_ss(d, da + (uint64_t)(((A_MN ? 2048 : 32) * q) >> 4), db + (uint64_t)(((B_MN ? 2048 : 32) * q) >> 4), idesc, j > 0 || q > 0);
            mma_commit(&bar_free[s]);
          }
          mma_commit(&bar_done[acc]);
        }
      }
      mma_commit(&bar_end);   // all products have read their operands
      mbar_drain(&bar_end, 0);
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    uint8_t* staging = smem + kCeStages * kCeStage + (warp - 2) * 4096;
    int turn = 0;
    bool over = false;
    for (int t = first; t < tiles.total && !over; t += stride) {
      int m, n, split;
      tiles.at(t, m, n, split);
      const int row = m * kCeM + quarter * 32 + lane, c_base = n * kCeN + half * 128;
      const int cols = min(128, p.n - c_base);   // that there are; columns from `cols` rounded up to 16 on were not computed
      const uint32_t src = tmem + half * 128 + lanes;
      const int k_end = tiles.end(split);
      int k0 = tiles.begin(split);
      const bool empty = k_end <= k0;
      float sums[REG ? 128 : 1];
      if constexpr (REG) {
#pragma unroll
        for (int j = 0; j < 128; ++j) sums[j] = 0.f;
        for (; k0 < k_end; k0 += p.flush, ++turn) {
          if (mbar_wait_failed(&bar_done[turn & 1], (uint32_t)(turn >> 1) & 1u, abortp)) { over = true; break; }
          tc_fence_after();
#pragma unroll
          for (int c0 = 0; c0 < 128; c0 += 16) {   // (32 at a time spill)
            if (c0 >= cols) break;
            float v[16];
            tmem_ld16(src + (turn & 1) * kCeN + c0, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) sums[c0 + j] += v[j];
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_read[turn & 1]);
        }
        if (over) break;
      } else if (!empty) {
        if (mbar_wait_failed(&bar_done[turn & 1], (uint32_t)(turn >> 1) & 1u, abortp)) break;
        tc_fence_after();
      }
      // values [c0, c0 + COUNT) of the thread's half row
      auto take = [&](auto count, int c0, float* v) {
        constexpr int COUNT = decltype(count)::value;
        if constexpr (REG) {
#pragma unroll
          for (int j = 0; j < COUNT; ++j) v[j] = sums[c0 + j];
        } else {
#pragma unroll
          for (int j = 0; j < COUNT; j += 32) tmem_ld32(src + (turn & 1) * kCeN + c0 + j, v + j);
          tmem_ld_wait();
        }
      };
      auto release = [&] {   // the accumulator has been read
        if constexpr (!REG) {
          if (empty) return;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_read[turn & 1]);
        }
      };
      constexpr float kLog2e = 1.4426950408889634f;
      if constexpr (MODE == kLse) {
        const bool on = row < head.rows;
        const int target = on ? p.rows[row].target - p.vocab0 - c_base : -1;
        float best = -INFINITY, sum = 0.f;
#pragma unroll
        for (int c0 = 0; c0 < 128; c0 += 32) {
          if (c0 >= cols) break;
          float v[32];
          take(std::integral_constant<int, 32>(), c0, v);
          if (c0 + 32 > cols) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = c0 + j < cols ? v[j] : -INFINITY;
          }
          float top = best;
#pragma unroll
          for (int j = 0; j < 32; ++j) top = fmaxf(top, v[j]);
          if (target >= c0 && target < c0 + 32) {
            float z = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) z = c0 + j == target ? v[j] : z;
            p.target_logit[row] = z;
          }
          __syncwarp();
          const float zero = top == -INFINITY ? 0.f : top;
          float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 d = mul2(add2(make_float2(v[j], v[j + 1]), splat(-zero)), splat(kLog2e));
            s2 = add2(s2, make_float2(ex2_approx(d.x), ex2_approx(d.y)));
          }
          sum = fmaf(sum, ex2_approx((best - zero) * kLog2e), s2.x + s2.y);
          best = top;
        }
        if (on) p.parts[(int64_t)(n * 2 + half) * p.parts_ld + row] = make_float2(best, sum);
      } else if constexpr (MODE == kGrad) {
        CeRow r;
        r.target = -1; r.lse = 0.f; r.coef = 0.f; r.row = 0;
        if (row < head.rows) r = p.rows[row];
        const int target = r.target - p.vocab0 - c_base;
        constexpr int PLANES = CePlanes<OUT>::count;
#pragma unroll
        for (int c0 = 0; c0 < 128; c0 += 64) {
          if (c0 >= cols) break;
          float v[64];
          take(std::integral_constant<int, 64>(), c0, v);
          if (c0 + 64 >= cols) release();
#pragma unroll
          for (int j = 0; j < 64; j += 2) {
            const float2 d = mul2(add2(make_float2(v[j], v[j + 1]), splat(-r.lse)), splat(kLog2e));
            v[j] = ex2_approx(d.x);
            v[j + 1] = ex2_approx(d.y);
          }
          if (target >= c0 && target < c0 + 64) {
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = c0 + j == target ? v[j] - 1.f : v[j];
          }
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] = r.coef == 0.f ? 0.f : v[j] * r.coef;
#pragma unroll
          for (int q = 0; q < PLANES; ++q) {
            if (lane == 0) bulk_wait_read0();   // what was stored from here before has left
            __syncwarp();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float w[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                float parts[PLANES];
                CePlanes<OUT>::split(v[h * 32 + j], parts);
                w[j] = parts[q];
              }
              store_row32<T>(staging, 4096, lane, h * 32, w);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_4d(&map_g, staging, c_base + c0, m * kCeM + quarter * 32, q, 0);
              bulk_commit();
            }
          }
        }
        if (cols <= 0) release();   // a half without columns
      } else {
        const float unit = head.unit;
        const bool on = row < (MODE == kDw ? p.m : head.rows);
        const int64_t to = MODE == kDw ? p.out_row0 + row : on ? p.rows[row].row : 0;
#pragma unroll
        for (int c0 = 0; c0 < 128; c0 += 32) {
          if (c0 >= cols) break;
          float v[32];
          if (empty) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0.f;
          } else {
            take(std::integral_constant<int, 32>(), c0, v);
          }
          const int col = c_base + c0, have = min(32, cols - c0);
          if (!on) {
          } else if (p.slab) {
            float* out = p.slab + ((int64_t)split * p.slab_rows + row) * p.slab_ld + col;
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              if (j < have) {
                float4 o = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                if (p.add) {
                  const float4 old = *reinterpret_cast<const float4*>(out + j);
                  o.x += old.x; o.y += old.y; o.z += old.z; o.w += old.w;
                }
                *reinterpret_cast<float4*>(out + j) = o;
              }
          } else {
            OUT* out = static_cast<OUT*>(p.out) + to * p.ld + col;
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= unit;
            if (p.vec) {
#pragma unroll
              for (int j = 0; j < 32; j += 8)
                if (j < have) store8<OUT>(out + j, v + j);
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (j < have) store1<OUT>(out + j, v[j]);
            }
          }
          __syncwarp();
        }
        release();
      }
      if (!REG && !empty) ++turn;
    }
    if (MODE == kGrad && lane == 0) bulk_wait_read0();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
  if (tid == 0 && abort_flag) atomicOr(p.status, CASTLE_STATUS_WAIT_TIMEOUT);
}

// The shares of a long sum, or the sums over the pieces of the vocabulary, added in order and rounded.
struct CeSum {
  const CeHead* head;
  const CeRow* rows;      // dx: where each row goes; NULL: rows [0, m) of out
  const float* slab;
  int64_t slab_rows, slab_ld, ld, m;
  void* out;
  int n, splits;
};
template <typename OUT>
__global__ void __launch_bounds__(256) castle_ce_sum_kernel(const CeSum p) {
  overlap_wait();
  const int64_t m = p.rows ? p.head->rows : p.m;
  const float unit = p.head->unit;
  const int quads = (p.n + 3) / 4;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < m * quads; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / quads;
    const int col = (int)(i - row * quads) * 4;
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < p.splits; ++s) {
      const float4 v = *reinterpret_cast<const float4*>(p.slab + (s * p.slab_rows + row) * p.slab_ld + col);
      t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w;
    }
    const float v[4] = {t.x, t.y, t.z, t.w};
    OUT* out = static_cast<OUT*>(p.out) + (p.rows ? (int64_t)p.rows[row].row : row) * p.ld + col;
    if (p.ld % 4 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0) {
      if constexpr (sizeof(OUT) == 4) *reinterpret_cast<float4*>(out) = make_float4(v[0] * unit, v[1] * unit, v[2] * unit, v[3] * unit);
      else *reinterpret_cast<uint2*>(out) = make_uint2(Elem<OUT>::pack2(v[0] * unit, v[1] * unit), Elem<OUT>::pack2(v[2] * unit, v[3] * unit));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < p.n) store1<OUT>(out + j, v[j] * unit);
    }
  }
}

// ------------------------------------------------------------------------------------------------ the losses
struct CeJoin {
  CeHead* head;
  const CeRow* rows;
  const float2* parts;
  float2* running;        // (max, sum) of the pieces before
  const float* target_logit;
  double* sums;           // of a CTA's losses
  float *lse, *loss;
  int64_t parts_ld;
  int parts_n;
  bool begin, end, each, mean;
};
// ROWS rows of a CTA, 256 / ROWS threads for each.
template <int ROWS>
__global__ void __launch_bounds__(256) castle_ce_join_kernel(const CeJoin p) {
  constexpr int LANES = 256 / ROWS;
  __shared__ float2 s[LANES][ROWS];
  __shared__ double total;
  __shared__ bool last;
  const int r = threadIdx.x % ROWS, l = threadIdx.x / ROWS;
  const int64_t row = (int64_t)blockIdx.x * ROWS + r;
  overlap_wait();
  const int rows = p.head->rows;
  float best = -INFINITY, sum = 0.f;
  auto join = [&](float2 o) {
    const float top = fmaxf(best, o.x), zero = top == -INFINITY ? 0.f : top;
    sum = sum * __expf(best - zero) + o.y * __expf(o.x - zero);
    best = top;
  };
  if (row < rows) {
    if (!p.begin && l == 0) join(p.running[row]);
#pragma unroll 4
    for (int k = l; k < p.parts_n; k += LANES) join(p.parts[(int64_t)k * p.parts_ld + row]);
  }
  s[l][r] = make_float2(best, sum);
  __syncthreads();
  double loss = 0.0;
  if (l == 0 && row < rows) {
    for (int k = 1; k < LANES; ++k) join(s[k][r]);
    if (!p.end) {
      p.running[row] = make_float2(best, sum);
    } else {
      const float lse = best + logf(sum);
      const int to = p.rows[row].row;
      p.lse[to] = lse;
      const float one = (best - p.target_logit[row]) + logf(sum);
      loss = one;
      if (p.each) p.loss[to] = one;
    }
  }
  if (!p.end || p.each) return;
  // the CTA's sum, and by the last CTA all CTAs', in a fixed order
  __shared__ double ds[ROWS];
  if (l == 0) ds[r] = loss;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int k = 0; k < ROWS; ++k) t += ds[k];
    p.sums[blockIdx.x] = t;
    __threadfence();
    last = atomicAdd(&p.head->done, 1u) + 1 == gridDim.x;
    __threadfence();
  }
  __syncthreads();
  if (!last) return;
  __shared__ double all[256];
  double t = 0.0;
  for (int k = threadIdx.x; k < (int)gridDim.x; k += 256) t += __ldcg(p.sums + k);
  all[threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    total = 0.0;
    for (int k = 0; k < 256; ++k) total += all[k];
    if (p.mean) total /= (double)rows;
    p.loss[0] = p.head->bad ? __int_as_float(0x7fffffff) : (float)total;
  }
}

// ------------------------------------------------------------------------------------------------ host
struct CePlan {
  int planes, terms, pitch, piece_fwd, piece_bwd, parts_per_piece;
  bool copy_x, copy_w;        // operands are laid out anew: fp32, or rows that TMA cannot read
  int64_t copy_rows, g_rows;
  int dx_splits, dw_splits, pieces;
  size_t rows, copy, wcopy, parts, running, logit, sums, g, slab_dx, slab_dw, bytes;   // offsets
};

static int ce_splits(int64_t tiles, int64_t steps) {   // shares of a long sum where the tiles alone leave SMs idle, of 16 steps at least
  if (tiles >= 148) return 1;
  const int64_t want = 148 / tiles, most = steps / 16;
  const int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 32 ? 32 : s);
}

static CePlan ce_plan(int dtype, int64_t n, int dim, int64_t vocab, bool x_ok, bool w_ok, bool backward) {
  CePlan q{};
  auto up = [](int64_t v, int64_t to) { return (v + to - 1) / to * to; };
  const bool f32 = dtype == CASTLE_F32;
  q.planes = f32 ? 3 : 1;
  q.terms = f32 ? 6 : 1;
  q.pitch = (int)up(dim, 8);
  q.copy_x = f32 || !x_ok;
  q.copy_w = f32 || !w_ok;
  q.copy_rows = up(n, kCeK);
  q.g_rows = up(n, kCeM);
  const int64_t w_row = q.copy_w ? (int64_t)q.planes * q.pitch * 2 : 0;
  auto piece = [&](int64_t per_column) {
    int64_t v = kCeScratch / (per_column > 0 ? per_column : 1) / kCeN * kCeN;
    if (v < kCeN) v = kCeN;
    return (int)(v < vocab ? v : vocab);
  };
  q.piece_fwd = piece(w_row + q.copy_rows / 16);
  q.piece_bwd = piece(w_row + q.planes * q.g_rows * 2);
  q.pieces = (int)((vocab + q.piece_bwd - 1) / q.piece_bwd);
  size_t at = 1024;   // behind the CeHead
  auto take = [&](size_t bytes) { const size_t o = at; at += up((int64_t)bytes, 1024); return o; };
  q.rows = take((size_t)n * sizeof(CeRow));
  q.copy = take((size_t)q.planes * q.copy_rows * q.pitch * 2);
  const int64_t most = backward ? q.piece_bwd : q.piece_fwd;
  q.wcopy = take(q.copy_w ? (size_t)most * w_row : 0);
  if (!backward) {
    q.parts_per_piece = 2 * (int)((q.piece_fwd + kCeN - 1) / kCeN);
    q.parts = take((size_t)q.parts_per_piece * q.copy_rows * sizeof(float2));
    q.running = take((size_t)n * sizeof(float2));
    q.logit = take((size_t)n * sizeof(float));
    q.sums = take((size_t)((n + 7) / 8) * sizeof(double));
  } else {
    const int64_t g_pitch = up(q.piece_bwd, 8);
    q.g = take((size_t)q.planes * q.g_rows * g_pitch * 2);
    const int64_t tiles_d = (dim + kCeN - 1) / kCeN;
    q.dx_splits = ce_splits((n + kCeM - 1) / kCeM * tiles_d, (int64_t)q.piece_bwd / kCeK * q.terms);
    q.dw_splits = ce_splits(((int64_t)q.piece_bwd + kCeM - 1) / kCeM * tiles_d, n / kCeK * q.terms);
    const int64_t slab_ld = up(dim, 4);
    q.slab_dx = take(q.dx_splits > 1 || q.pieces > 1 ? (size_t)q.dx_splits * n * slab_ld * 4 : 0);
    q.slab_dw = take(q.dw_splits > 1 ? (size_t)q.dw_splits * q.piece_bwd * slab_ld * 4 : 0);
  }
  q.bytes = at;
  return q;
}

static int ce_check(const char* who, int32_t dtype, int64_t rows, int32_t dim, int64_t vocab, const void* x, int64_t xs, const void* w, int64_t ws,
                    const int64_t* targets, int32_t reduction, const int32_t* status) {
  if (dtype < CASTLE_BF16 || dtype > CASTLE_F32) return reject("%s: unknown dtype", who);
  if (rows <= 0 || rows > (1 << 30) || vocab <= 0 || vocab > (1 << 30) || dim <= 0 || dim > (1 << 20))
    return reject("%s: %lld rows, vocabulary %lld, dim %d not supported", who, (long long)rows, (long long)vocab, dim);
  if (reduction < 0 || reduction > 2) return reject("%s: unknown reduction", who);
  if (!x || !w || ((uintptr_t)x | (uintptr_t)w) % elem_size(dtype) || xs < 0 || ws < 0)
    return reject("%s: x and weight (aligned to their elements, strides of at least 0) are needed", who);
  if (!targets || (uintptr_t)targets % 8 || !status) return reject("%s: targets (64-bit) and a status word are needed", who);
  return 0;
}

// Whether TMA can read rows of 16-bit elements where they lie.
static bool ce_tma_rows(int dtype, int64_t rows, int dim, const void* p, int64_t stride) {
  return dtype != CASTLE_F32 && dim % 8 == 0 && (uintptr_t)p % 16 == 0 && (rows == 1 || (stride >= dim && stride % 8 == 0));
}

// 16-bit rows in `planes` planes, boxes of box_rows x 64.
static int ce_map(CUtensorMap* m, const void* p, int op, int64_t rows, int cols, int64_t pitch, int64_t plane, int planes, int box_rows, const char* what) {
  const castle_tensor_t t{const_cast<void*>(p), 0, plane, pitch};
  return make_tmap_16bit(m, &t, op, 1, planes, (int)rows, cols, box_rows, what);
}

template <typename T, typename OUT, CeMode MODE>
static cudaError_t ce_launch(const CeProduct& p, int64_t most_tiles, const CUtensorMap& a, const CUtensorMap& copy, const CUtensorMap& b, const CUtensorMap& g,
                             cudaStream_t st) {
  auto kernel = castle_ce_kernel<T, OUT, MODE>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kCeSmem);
  if (e != cudaSuccess) return e;
  return launch_kernel(kernel, dim3((unsigned)(most_tiles < 148 ? most_tiles : 148)), kCeThreads, kCeSmem, st, true, p, a, copy, b, g);
}

static int ce_rows_per_cta(int64_t n) {   // a CTA per SM, at least 32 rows each
  const int64_t r = (n + 147) / 148;
  return (int)(r < 32 ? 32 : r);
}

struct CeCall {
  int dtype, dim;
  int64_t n, vocab, xs, ws;
  const void *x, *w;
  const int64_t* targets;
  int64_t ignore;
  int reduction;
  char* work;
  int32_t* status;
  cudaStream_t st;
};

template <typename OUT>
static cudaError_t ce_rows(const CeCall& c, const CePlan& q, const float* lse, const float* dloss, void* dx, float* loss, float* lse_out) {
  CeRowsParams r{};
  r.targets = c.targets; r.x = c.x; r.lse = lse; r.dloss = dloss; r.n = c.n; r.vocab = c.vocab; r.ignore = c.ignore; r.x_stride = c.xs;
  r.copy_rows = q.copy_rows; r.dim = c.dim; r.pitch = q.pitch; r.planes = q.planes; r.rows_per_cta = ce_rows_per_cta(c.n);
  r.mean = c.reduction == CASTLE_REDUCE_MEAN; r.each = dloss && c.reduction == CASTLE_REDUCE_NONE; r.copy_always = q.copy_x;
  r.head = (CeHead*)c.work; r.rows = (CeRow*)(c.work + q.rows); r.copy = (uint16_t*)(c.work + q.copy); r.dx = dx; r.loss = loss; r.lse_out = lse_out;
  r.status = c.status;
  const unsigned grid = (unsigned)((c.n + r.rows_per_cta - 1) / r.rows_per_cta);
  return launch_kernel(castle_ce_rows_kernel<OUT>, dim3(grid), 1024, 0, c.st, true, r);
}

// The weight's rows [v0, v0 + count) laid out anew, if they have to be.
template <typename OUT>
static cudaError_t ce_weight(const CeCall& c, const CePlan& q, int64_t v0, int64_t count) {
  if (!q.copy_w) return cudaSuccess;
  return launch_kernel(castle_ce_split_kernel<OUT>, dim3((unsigned)((count + 7) / 8)), 256, 0, c.st, true, (const OUT*)c.w + v0 * c.ws, c.ws,
                       (uint16_t*)(c.work + q.wcopy), count, c.dim, q.pitch);
}

#define CE_TRY(call) do { if (int rc_ = (call)) return rc_; } while (0)
#define CE_CUDA(call, what) do { const cudaError_t e_ = (call); if (e_ != cudaSuccess) return cuda_fail(e_, what); } while (0)

// Maps over x, over its copy and over the weight (or the piece's copy) with the boxes that a product reads.
static int ce_x_maps(const CeCall& c, const CePlan& q, int op, int box_rows, CUtensorMap* x, CUtensorMap* copy) {
  const int64_t plane = q.copy_rows * q.pitch;
  CE_TRY(ce_map(copy, c.work + q.copy, op, q.copy_rows, q.pitch, q.pitch, plane, q.planes, box_rows, "castle_linear_ce: copy of x"));
  if (q.copy_x) { *x = *copy; return 0; }
  return ce_map(x, c.x, op, c.n, c.dim, c.n == 1 ? c.dim : c.xs, 0, 1, box_rows, "castle_linear_ce: x");
}
static int ce_w_map(const CeCall& c, const CePlan& q, int op, int64_t count, int box_rows, CUtensorMap* w) {
  if (q.copy_w) return ce_map(w, c.work + q.wcopy, op, count, q.pitch, q.pitch, count * q.pitch, q.planes, box_rows, "castle_linear_ce: copy of the weight");
  return ce_map(w, c.w, op, c.vocab, c.dim, c.vocab == 1 ? c.dim : c.ws, 0, 1, box_rows, "castle_linear_ce: weight");
}

template <typename OUT>
static int ce_forward(const CeCall& c, const CePlan& q, float* loss, float* lse) {
  using T = typename CePlanes<OUT>::Op;
  const int op = c.dtype == CASTLE_F16 ? CASTLE_F16 : CASTLE_BF16;
  const bool each = c.reduction == CASTLE_REDUCE_NONE;
  CE_CUDA(ce_rows<OUT>(c, q, nullptr, nullptr, nullptr, each ? loss : nullptr, lse), "castle_linear_ce_fwd launch");
  CUtensorMap x, copy, w;
  CE_TRY(ce_x_maps(c, q, op, kCeM, &x, &copy));
  const int64_t tiles_m = (c.n + kCeM - 1) / kCeM;
  for (int64_t v0 = 0; v0 < c.vocab; v0 += q.piece_fwd) {
    const int64_t count = c.vocab - v0 < q.piece_fwd ? c.vocab - v0 : q.piece_fwd;
    const int tiles_n = (int)((count + kCeN - 1) / kCeN);
    CE_CUDA(ce_weight<OUT>(c, q, v0, count), "castle_linear_ce_fwd launch");
    CE_TRY(ce_w_map(c, q, op, count, kCeN, &w));
    CeProduct p{};
    p.head = (const CeHead*)c.work; p.rows = (const CeRow*)(c.work + q.rows); p.n = (int)count; p.k = q.pitch; p.b_row0 = q.copy_w ? 0 : (int)v0;
    p.vocab0 = (int)v0; p.vocab = (int)c.vocab; p.terms = q.terms; p.splits = 1; p.group = 32;
    p.flush = q.terms > 1 ? kCeFlushF32 : kCeFlush;
    p.parts = (float2*)(c.work + q.parts); p.parts_ld = q.copy_rows; p.target_logit = (float*)(c.work + q.logit); p.status = c.status;
    CE_CUDA((ce_launch<T, OUT, kLse>(p, tiles_m * tiles_n, x, copy, w, w, c.st)), "castle_linear_ce_fwd launch");
    CeJoin j{};
    j.head = (CeHead*)c.work; j.rows = p.rows; j.parts = p.parts; j.running = (float2*)(c.work + q.running); j.target_logit = p.target_logit;
    j.sums = (double*)(c.work + q.sums); j.lse = lse; j.loss = loss; j.parts_ld = q.copy_rows; j.parts_n = 2 * tiles_n;
    j.begin = v0 == 0; j.end = v0 + count == c.vocab; j.each = each; j.mean = c.reduction == CASTLE_REDUCE_MEAN;
    // few rows: a warp each; many: neighbouring threads on neighbouring rows
    if (c.n >= 4096) CE_CUDA(launch_kernel(castle_ce_join_kernel<32>, dim3((unsigned)((c.n + 31) / 32)), 256, 0, c.st, true, j), "castle_linear_ce_fwd launch");
    else CE_CUDA(launch_kernel(castle_ce_join_kernel<8>, dim3((unsigned)((c.n + 7) / 8)), 256, 0, c.st, true, j), "castle_linear_ce_fwd launch");
  }
  return 0;
}

template <typename OUT>
static int ce_backward(const CeCall& c, const CePlan& q, const float* lse, const float* dloss, void* dx, void* dw) {
  using T = typename CePlanes<OUT>::Op;
  const char* what = "castle_linear_ce_bwd launch";
  const int op = c.dtype == CASTLE_F16 ? CASTLE_F16 : CASTLE_BF16;
  const int64_t tiles_m = (c.n + kCeM - 1) / kCeM, slab_ld = (c.dim + 3) / 4 * 4;
  const int tiles_d = (c.dim + kCeN - 1) / kCeN, es = elem_size(c.dtype);
  CE_CUDA(ce_rows<OUT>(c, q, lse, dloss, dx, nullptr, nullptr), what);
  CUtensorMap x, copy, xk, copyk, w, wk, g, ga, gt;
  CE_TRY(ce_x_maps(c, q, op, kCeM, &x, &copy));
  CE_TRY(ce_x_maps(c, q, op, kCeK, &xk, &copyk));
  CeProduct base{};
  base.head = (const CeHead*)c.work; base.rows = (const CeRow*)(c.work + q.rows); base.terms = q.terms; base.flush = q.terms > 1 ? kCeFlushF32 : kCeNoFlush; base.splits = 1; base.group = 32; base.status = c.status;
  base.vocab = (int)c.vocab; base.ld = c.dim;
  auto sum = [&](int splits, int64_t rows, int64_t slab_rows, bool by_row, const float* slab, void* out) {
    CeSum s{};
    s.head = base.head; s.rows = by_row ? base.rows : nullptr; s.slab = slab; s.slab_rows = slab_rows; s.slab_ld = slab_ld; s.ld = c.dim; s.m = rows; s.out = out;
    s.n = c.dim; s.splits = splits;
    const int64_t blocks = (rows * (slab_ld / 4) + 255) / 256;
    return launch_kernel(castle_ce_sum_kernel<OUT>, dim3((unsigned)(blocks < 148 * 8 ? blocks : 148 * 8)), 256, 0, c.st, true, s);
  };
  for (int64_t v0 = 0; v0 < c.vocab; v0 += q.piece_bwd) {
    const int64_t count = c.vocab - v0 < q.piece_bwd ? c.vocab - v0 : q.piece_bwd, pitch = (count + 7) / 8 * 8;
    uint16_t* gp = (uint16_t*)(c.work + q.g);
    CE_CUDA(ce_weight<OUT>(c, q, v0, count), what);
    CE_TRY(ce_w_map(c, q, op, count, kCeN, &w));
    CE_TRY(ce_w_map(c, q, op, count, kCeK, &wk));
    CE_TRY(ce_map(&g, gp, op, q.g_rows, (int)count, pitch, q.g_rows * pitch, q.planes, 32, "castle_linear_ce: logits' gradient"));
    CE_TRY(ce_map(&ga, gp, op, q.g_rows, (int)count, pitch, q.g_rows * pitch, q.planes, kCeM, "castle_linear_ce: logits' gradient"));
    CE_TRY(ce_map(&gt, gp, op, q.g_rows, (int)count, pitch, q.g_rows * pitch, q.planes, kCeK, "castle_linear_ce: logits' gradient"));
    CeProduct p = base;
    p.n = (int)count; p.k = q.pitch; p.b_row0 = q.copy_w ? 0 : (int)v0; p.vocab0 = (int)v0;
    CE_CUDA((ce_launch<T, OUT, kGrad>(p, tiles_m * ((count + kCeN - 1) / kCeN), x, copy, w, g, c.st)), what);
    if (dx) {
      p = base;
      p.n = c.dim; p.k = (int)count; p.b_row0 = q.copy_w ? 0 : (int)v0; p.out = dx; p.splits = q.dx_splits; p.group = 16;
      p.vec = c.dim % 8 == 0 && (uintptr_t)dx % 16 == 0;
      if (q.dx_splits > 1 || q.pieces > 1) { p.slab = (float*)(c.work + q.slab_dx); p.slab_rows = c.n; p.slab_ld = slab_ld; p.add = v0 > 0; }
      CE_CUDA((ce_launch<T, OUT, kDx>(p, tiles_m * tiles_d * p.splits, ga, ga, wk, wk, c.st)), what);
      if (p.slab && v0 + count == c.vocab) CE_CUDA(sum(p.splits, c.n, c.n, true, p.slab, dx), what);
    }
    if (dw) {
      p = base;
      p.m = (int)count; p.n = c.dim; p.out = dw; p.out_row0 = v0; p.splits = q.dw_splits; p.group = 16;
      p.vec = c.dim % 8 == 0 && (uintptr_t)dw % 16 == 0;
      if (q.dw_splits > 1) { p.slab = (float*)(c.work + q.slab_dw); p.slab_rows = q.piece_bwd; p.slab_ld = slab_ld; }
      CE_CUDA((ce_launch<T, OUT, kDw>(p, (count + kCeM - 1) / kCeM * tiles_d * p.splits, gt, copyk, xk, xk, c.st)), what);
      if (p.slab) CE_CUDA(sum(p.splits, count, p.slab_rows, false, p.slab, static_cast<char*>(dw) + v0 * c.dim * es), what);
    }
  }
  return 0;
}

}  // namespace castle

using namespace castle;

extern "C" size_t castle_linear_ce_workspace_bytes(int32_t dtype, int64_t rows, int32_t dim, int64_t vocab, int32_t backward) {
  if (dtype < CASTLE_BF16 || dtype > CASTLE_F32 || rows <= 0 || rows > (1 << 30) || dim <= 0 || dim > (1 << 20) || vocab <= 0 || vocab > (1 << 30)) return 0;
  const size_t direct = ce_plan(dtype, rows, dim, vocab, true, true, backward != 0).bytes, copied = ce_plan(dtype, rows, dim, vocab, false, false, backward != 0).bytes;
  return direct > copied ? direct : copied;
}

static int ce_call(const char* who, CeCall& c, CePlan& q, int32_t dtype, int64_t rows, int32_t dim, int64_t vocab, const void* x, int64_t x_stride, const void* weight,
                   int64_t w_stride, const int64_t* targets, int64_t ignore_index, int32_t reduction, void* workspace, size_t workspace_bytes, int32_t* status,
                   void* stream, bool backward) {
  if (int rc = ce_check(who, dtype, rows, dim, vocab, x, x_stride, weight, w_stride, targets, reduction, status)) return rc;
  q = ce_plan(dtype, rows, dim, vocab, ce_tma_rows(dtype, rows, dim, x, x_stride), ce_tma_rows(dtype, vocab, dim, weight, w_stride), backward);
  if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < castle_linear_ce_workspace_bytes(dtype, rows, dim, vocab, backward)) return reject("%s: workspace too small or not 256-byte aligned", who);
  c = CeCall{dtype, dim, rows, vocab, x_stride, w_stride, x, weight, targets, ignore_index, reduction, static_cast<char*>(workspace), status, (cudaStream_t)stream};
  return 0;
}

extern "C" int castle_linear_ce_fwd(int32_t dtype, int64_t rows, int32_t dim, int64_t vocab, const void* x, int64_t x_stride, const void* weight, int64_t w_stride,
                                    const int64_t* targets, int64_t ignore_index, int32_t reduction, float* loss, float* lse, void* workspace,
                                    size_t workspace_bytes, int32_t* status, void* stream) {
  CeCall c;
  CePlan q;
  if (int rc = ce_call("castle_linear_ce_fwd", c, q, dtype, rows, dim, vocab, x, x_stride, weight, w_stride, targets, ignore_index, reduction, workspace,
                       workspace_bytes, status, stream, false)) return rc;
  if (!loss || !lse || ((uintptr_t)loss | (uintptr_t)lse) % 4) return reject("castle_linear_ce_fwd: loss and lse are needed");
  return by_type(dtype, [&](auto t) { return ce_forward<decltype(t)>(c, q, loss, lse); });
}

extern "C" int castle_linear_ce_bwd(int32_t dtype, int64_t rows, int32_t dim, int64_t vocab, const void* x, int64_t x_stride, const void* weight, int64_t w_stride,
                                    const int64_t* targets, int64_t ignore_index, int32_t reduction, const float* lse, const float* dloss, void* dx, void* dweight,
                                    void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  CeCall c;
  CePlan q;
  if (int rc = ce_call("castle_linear_ce_bwd", c, q, dtype, rows, dim, vocab, x, x_stride, weight, w_stride, targets, ignore_index, reduction, workspace,
                       workspace_bytes, status, stream, true)) return rc;
  if (!lse || !dloss || ((uintptr_t)lse | (uintptr_t)dloss) % 4 || ((uintptr_t)dx | (uintptr_t)dweight) % elem_size(dtype))
    return reject("castle_linear_ce_bwd: lse, dloss and results aligned to their elements are needed");
  if (!dx && !dweight) return 0;
  return by_type(dtype, [&](auto t) { return ce_backward<decltype(t)>(c, q, lse, dloss, dx, dweight); });
}
