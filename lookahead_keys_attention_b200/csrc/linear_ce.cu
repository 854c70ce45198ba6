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
//   castle_ce_kernel<kDx>    dx += G W of the piece (fp32 sums in scratch if there are several pieces)
//   castle_ce_kernel<kDw>    dW of the piece
//
// The four products are one kernel: CTAs that stay, one per SM, in pairs (256 x 256 of the result, 64 of the contraction at a time) or, where
// there is less to do, alone (128 x 256, 128 or 64), each with a warp that loads tiles by TMA, a warp that issues the tensor cores'
// products, and eight or sixteen warps that work on a finished tile in one half of tensor memory while the next one is summed in the other.
// Alone, an SM's shared memory brings in and reads 24 KB in the 128 cycles of a product of 16, more than it can (78 % of the tensor cores' cycles
// at a contraction of 50021); a pair shares B's tile (92 %).  All sums, the logits and the statistics are fp32.
//
// What bounds it: at 8192 x 4096 against 131072 forward and backward take 26.1 to 28.5 ms by the box for 35.2 TFLOP, 1240 to 1350 TFLOP/s: the
// power limit (the library's product, back to back, 1406 of measured), at clocks of 1.3 to 1.5 GHz.  8.8 of the 35.2 are the logits formed again.  Few
// rows: the weight is read three times and dW written, 8 x 4096 against 131072 798 us of kernels for 4.3 GB.
//
// dx and dW can have few tiles and long contractions.  As many tiles as go evenly to the workers are theirs whole; of the others the
// contraction is cut into slices, whose sums go to scratch and are added, in order, by castle_ce_sum_kernel.
//
// fp32 tensors: every value is the sum of three bf16 ones (8 bits each: 24), and a product is the six largest of the nine products
// of such parts (what is left out is 2^-24 of it), the smallest first.  So the same kernels serve, with six times the steps.
//
// What the tensor cores add to an accumulator loses more than rounding to nearest would, and the losses of a long sum add up (197 rows of 512,
// fp32: losses 3.3e-6 off, gradients of longer sums 1.7e-5, where fp32 arithmetic has 2e-7).  Where the result has 32 bits
// (the logits, and everything of fp32 tensors), accumulators are therefore emptied every `flush` steps into sums that
// the working warps keep in registers.  The logits formed again are the same sums, bit for bit, as those behind the log-sum-exp: summed in one go,
// they made a row's probabilities add up to 1 + 1e-3 (logits of some 60 over 4096 to 8192, fp16), more than what a learnt row has to move by.
//
// G in 16 bits is taken in units of a power of two (the largest c_i's), in fp16 with 2^14 on top, so that it keeps probabilities down to 2^-28 in full
// precision; the unit is multiplied back in fp32 at the end.  Where all rows have one coefficient (mean, sum) that is the unit and none
// of it is in G: -1 for a target that has no probability is exact, where c would be off by the same half step in every row (1789 rows
// against 132536, bf16: gradients 3.2e-3 off in their norm, 1.7e-3 by rounding the result).  A row's largest entry by far is
// mostly its target's.  What rounding took from it is kept in fp32, and dx gets its product with the target's row of W.  With a coefficient per row
// fp16 has half steps of 2^-39 of the largest for all rows: one whose own is 2^20 times smaller has its probabilities to 2^-19 only.
#include <type_traits>

#include "common.cuh"
#include "vec.cuh"

namespace castle {

enum CeMode { kLse, kGrad, kDx, kDw };

constexpr int kCeM = 128, kCeN = 256, kCeK = 64;
// The warps that work on tiles.  Sixteen hide what each waits for better where results are written (dW of 131072 x 4096 over 8 rows: 257 us,
// with eight 319); with eight a row's statistics have fewer parts.
// (Their 576 threads leave 96 registers.  The forms that keep sums spill some: G of fp32 140 to 164 bytes a thread, of 16 bits 56 to 68, dx and dW of fp32 16 to 52.)
template <CeMode MODE> constexpr int kCeWarps = MODE == kLse ? 8 : 16;
template <CeMode MODE> constexpr int kCeShares = kCeWarps<MODE> / 4;      // of a tile's columns
template <CeMode MODE> constexpr int kCeThreads = (kCeWarps<MODE> + 2) * 32;
constexpr uint32_t kCeA = kCeM * kCeK * 2;
constexpr uint32_t kCeRing = 4 * (kCeA + kCeN * kCeK * 2);   // stages: 4 of a CTA alone with a tile of 256 columns, 6 of 128 or of a pair, 8 of 64
constexpr int kCeStages = 8;
constexpr uint32_t kCeStaging = 16 * 2048;   // results on their way out: 32 rows x 64 bytes of each working warp
__device__ __forceinline__ uint32_t staging_off(int row, int chunk16) { return row * 64 + ((chunk16 ^ ((row >> 1) & 3)) << 4); }   // without bank conflicts
constexpr size_t kCeSmem = kCeRing + kCeStaging + 1024;
// The stages in turn: which, and in which of its barriers' two phases.
struct CeTurn {
  int stages, s = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ explicit CeTurn(int n) : stages(n) {}
  __device__ __forceinline__ void next() {
    if (++s == stages) { s = 0; phase ^= 1u; }
  }
};
constexpr int64_t kCeScratch = (int64_t)1 << 30;   // bytes that a piece of the vocabulary may take
// Steps between emptyings: of a 16-bit operand's logits (32 additions in the tensor cores), of fp32's parts (24).  With these the losses of
// 197 x 512 in fp32 are 6.7e-8 of their norm off (emptied every second step 3.0e-7, and 8 % faster); not emptied 3.3e-6 and, of logits over 1024 in 16 bits, 8 % faster (166 us, 152).
// (G's logits, too: 8192 x 4096 against 131072, forward and gradients, 28.2 ms for 27.5 without; 4096 x 1024 against 50021 1.49 ms for 1.45.)
constexpr int kCeFlush = 8, kCeFlushF32 = 1, kCeNoFlush = 1 << 30;
// What G's largest entries (below 2 units) are raised by.  The exponents of the other types reach, and products with rows near their largest number
// must not be 2^14 times as large.
template <typename OUT> constexpr float kCeUnit = std::is_same<OUT, __half>::value ? 16384.f : 1.f;

struct CeHead {          // at the start of the workspace, written by castle_ce_rows_kernel
  int rows;              // that take part
  int gathered;          // whether they lie in the copy
  int bad;               // targets outside the vocabulary
  unsigned done;         // CTAs of the join that have ended
  float unit;            // of G, multiplied back into dx and dW
};
struct CeRow { int target; float lse, coef; int row; };   // of the rows that take part, in order; coef: G's, row: in the caller's tensors

__device__ __forceinline__ int term_a(int term) { return 0x001102 >> 4 * term & 3; }
__device__ __forceinline__ int term_b(int term) { return 0x010120 >> 4 * term & 3; }   // one term: the last

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

// One value as one 16-bit number, or as three whose sum it is.
template <typename T> struct CePlanes {
  static constexpr int count = 1;
  using Op = T;
  static __device__ __forceinline__ void split(float v, float* p) { p[0] = v; }
};
constexpr float kCeMostBf16 = 3.38953139e38f;   // (2 - 2^-7) 2^127
template <> struct CePlanes<float> {
  static constexpr int count = 3;
  using Op = __nv_bfloat16;
  static __device__ __forceinline__ void split(float v, float* p) {
    p[0] = __bfloat162float(__float2bfloat16_rn(v));
    if (isinf(p[0]) && !isinf(v)) p[0] = copysignf(kCeMostBf16, v);   // a number beyond the largest bf16 one is that and a rest
    const float r = v - p[0];
    p[1] = isfinite(p[0]) ? __bfloat162float(__float2bfloat16_rn(r)) : 0.f;   // an infinity is its first part alone (times a part of zero it gives NaN)
    p[2] = isfinite(p[0]) ? r - p[1] : 0.f;
  }
};
// A row into its planes, by a warp; columns from dim to pitch are zero.
template <typename T>
__device__ __forceinline__ void copy_row(const T* src, uint16_t* dst, int64_t plane, int dim, int pitch, int lane) {
  using Op = typename CePlanes<T>::Op;
  constexpr int P = CePlanes<T>::count;
  if (dim % 8 == 0 && reinterpret_cast<uintptr_t>(src) % 16 == 0) {
    if constexpr (P == 1) {
#pragma unroll 4
      for (int c = lane * 8; c < dim; c += 256) *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(src + c);
      return;
    }
    for (int c0 = lane * 8; c0 < dim; c0 += 1024) {   // four loads on their way at a time
      Raw8<T> raw[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c0 + u * 256 < dim) raw[u] = *reinterpret_cast<const Raw8<T>*>(src + c0 + u * 256);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int c = c0 + u * 256;
        if (c >= dim) break;
        float v[8], w[P][8];
        load8<T>(reinterpret_cast<const T*>(&raw[u]), v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float a[P];
          CePlanes<T>::split(v[j], a);
#pragma unroll
          for (int q = 0; q < P; ++q) w[q][j] = a[q];
        }
#pragma unroll
        for (int q = 0; q < P; ++q) store8<Op>(reinterpret_cast<Op*>(dst + q * plane + c), w[q]);
      }
    }
    return;
  }
  if constexpr (sizeof(T) == 2) {
    // A row at an odd place: 16-byte blocks of memory, of which each eight columns have parts of two (24989 rows of 5859
    // 101 us, 5.8 TB/s read and written; by single elements 186).
    const int lead = (int)(reinterpret_cast<uintptr_t>(src) % 16 / 2);   // columns of the first block that are not the row's
    auto block = [&](int c) {                                            // columns [c, c + 8), a block of memory; those that are not there are zero
      uint32_t w[4];
      if (c >= 0 && c + 8 <= dim) {
        const uint4 q = *reinterpret_cast<const uint4*>(src + c);
        w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
      } else {
        const uint16_t* from = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = c + 2 * j;
          w[j] = (k >= 0 && k < dim ? from[k] : 0u) | (uint32_t)(k + 1 >= 0 && k + 1 < dim ? from[k + 1] : 0u) << 16;
        }
      }
      return make_uint4(w[0], w[1], w[2], w[3]);
    };
    auto shifted = [&](int c, const uint4& a, const uint4& b) {
      uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 6; ++j) w[j] = lead & 4 ? w[j + 2] : w[j];
#pragma unroll
      for (int j = 0; j < 5; ++j) w[j] = lead & 2 ? w[j + 1] : w[j];
      const int bits = lead % 2 * 16;
      *reinterpret_cast<uint4*>(dst + c) = make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                                                      __funnelshift_r(w[3], w[4], bits));
    };
    const int whole = dim + lead - 16;   // the last column whose two blocks are all the row's
#pragma unroll 4
    for (int c = 8 + lane * 8; c <= whole; c += 256)
      shifted(c, *reinterpret_cast<const uint4*>(src + c - lead), *reinterpret_cast<const uint4*>(src + c - lead + 8));
    const int end = lane == 0 ? 0 : max(8, whole / 8 * 8 + 8) + (lane - 1) * 8;   // the first, and three at most behind those
    if (lane < 4 && end < pitch) shifted(end, block(end - lead), block(end - lead + 8));
    return;
  }
#pragma unroll 4
  for (int c = lane * 2; c < pitch; c += 64) {
    float a[P], b[P];
    CePlanes<T>::split(c < dim ? load1<T>(src + c) : 0.f, a);
    CePlanes<T>::split(c + 1 < dim ? load1<T>(src + c + 1) : 0.f, b);
#pragma unroll
    for (int q = 0; q < P; ++q) *reinterpret_cast<uint32_t*>(dst + q * plane + c) = Elem<Op>::pack2(a[q], b[q]);
  }
}

// Every CTA reads all targets (and, in a backward with a gradient per row, these), so it needs nothing of the others.
template <typename T>
__global__ void __launch_bounds__(1024, 1) castle_ce_rows_kernel(const CeRowsParams p) {
  __shared__ int s[3][32];
  __shared__ float sf[32];
  __shared__ int place[1024];   // of a row in the gathered order, -1: it takes no part
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r0 = (int64_t)blockIdx.x * p.rows_per_cta, r1 = min(p.n, r0 + p.rows_per_cta);
  overlap_wait();
  int sums[3] = {0, 0, 0};   // rows that take part before the CTA's own, all of them, ignored ones
  float most = 0.f;
  for (int64_t i0 = tid; i0 < p.n; i0 += 1024 * 8) {
    int64_t t[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) t[u] = i0 + u * 1024 < p.n ? p.targets[i0 + u * 1024] : -1;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t i = i0 + u * 1024;
      const bool in = i < p.n, skip = t[u] == p.ignore, on = in && !skip && t[u] >= 0 && t[u] < p.vocab;
      sums[0] += on && i < r0;
      sums[1] += on;
      sums[2] += in && skip;
      if (p.each && on) {
        const float g = fabsf(p.dloss[i]);
        if (g < INFINITY) most = fmaxf(most, g);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
    for (int k = 0; k < 3; ++k) sums[k] += __shfl_xor_sync(0xffffffffu, sums[k], o);
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  }
  if (lane < 3) s[lane][warp] = lane == 0 ? sums[0] : lane == 1 ? sums[1] : sums[2];
  if (lane == 0) sf[warp] = most;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) sums[k] = s[k][lane];
  most = sf[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
    for (int k = 0; k < 3; ++k) sums[k] += __shfl_xor_sync(0xffffffffu, sums[k], o);
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  }
  int before = sums[0];
  const int all = sums[1], ignored = sums[2];
  float g_one = 0.f, unit = 1.f;
  if (p.dloss && !p.each) g_one = p.mean ? p.dloss[0] / (float)(p.n - ignored) : p.dloss[0];
  if (most > 0.f) unit = __uint_as_float(max(__float_as_uint(most) & 0x7f800000u, 0x00800000u));   // the largest coefficient's power of two
  const bool gather = all < p.n;
  if (blockIdx.x == 0 && tid == 0) {
    CeHead h;
    h.rows = all;
    h.gathered = gather || p.copy_always;
    h.bad = (int)(p.n - ignored) - all;
    h.done = 0;
    h.unit = all > 0 ? (p.each ? unit : g_one) * (1.f / kCeUnit<T>) : 0.f;   // (the mean over no rows is not a number, its gradients are zero)
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
    if (lane == 0) s[0][warp] = __popc(vote);
    __syncthreads();
    int at = before, total = 0;
    for (int k = 0; k < 32; ++k) {
      if (k < warp) at += s[0][k];
      total += s[0][k];
    }
    at += __popc(vote & ((1u << lane) - 1));
    before += total;
    place[tid] = on ? at : -1;
    if (on) {
      CeRow r;
      r.target = (int)t;
      r.row = (int)i;
      r.lse = p.lse ? p.lse[i] : 0.f;
      r.coef = p.each ? p.dloss[i] / unit * kCeUnit<T> : kCeUnit<T>;
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
#pragma unroll 4
          for (int c = lane; c < p.dim; c += 32) store1<T>(row + c, 0.f);
        }
      }
    }
  }
  // what dW's contraction over rows reads behind the last one
  if (!p.lse_out && (gather || p.copy_always) && blockIdx.x == gridDim.x - 1) {
    const int64_t plane = p.copy_rows * p.pitch;
    const int64_t end = min(p.copy_rows, ((int64_t)all + kCeK - 1) / kCeK * kCeK);
    for (int64_t k = all + warp; k < end; k += 32)
      for (int q = 0; q < p.planes; ++q)
        for (int c = lane * 8; c < p.pitch; c += 256) *reinterpret_cast<uint4*>(p.copy + q * plane + k * p.pitch + c) = make_uint4(0u, 0u, 0u, 0u);
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
constexpr int kCeWorkers = 148;   // CTAs of a launch
constexpr int kCeShare = 24;   // steps from which on it can pay to share tiles out
constexpr int kCeParts = 4 * kCeWorkers;   // tiles of one CTA that the slab holds at most
constexpr int kCeSlices = 37;     // most slices of a contraction
struct CeProduct {
  const CeHead* head;
  const CeRow* rows;
  int m, n, k;           // of the result and the contraction; m (kDw: k) is the number of rows that take part instead
  int bn;                // columns of a tile
  int a_rows, k_rows;    // rows that a load of A's tile brings (not kDw), and of the contraction that a step has (kDw): fewer where there are fewer
  int b_row0;            // where the piece begins in B's rows (kLse, kGrad: along n, kDx: along k)
  int vocab0;            // the piece's first column of z (kLse, kGrad)
  int terms, group;
  int flush;             // steps after which an accumulator is emptied
  bool share;            // tiles may be shared out among workers (kDx, kDw)
  bool vec, w_vec;       // out can be stored, the weight read 16 bytes at a time
  // kLse
  float2* parts;         // [kCeShares<kLse> per tile of n][parts_ld]
  float* target_logit;
  int64_t parts_ld;
  // kDx, kDw
  uint16_t* g;           // kGrad: [plane][row, up to the tiles' end][g_ld]
  int64_t g_ld, g_plane;
  float* lost;           // kGrad, kDx (16 bits): what rounding took from the target's entry of G, of each row that takes part
  const void* w;         // kDx: the weight, w_stride apart, of which the piece has rows [vocab0, vocab0 + k)
  int64_t w_stride;
  void* out;             // (rows, ld)
  int64_t ld, out_row0;
  float4* slab;          // parts of shared tiles: [part][column / 4][row of the tile]
  float* acc;            // kDx, several pieces of the vocabulary: sums so far, (rows that take part, acc_ld); else NULL
  int64_t acc_ld;
  bool acc_add, acc_out; // not the first piece; the last one
  int32_t* status;
};

// What a worker (a CTA, or a pair) does: tiles, and slices of the contraction (steps of 64) of those that do not go evenly to the workers.
// Slices are dealt out one after the other, each with all its tiles, so that workers that run together read the same part of the operands
// (one worker's equal share of all steps in a row instead read them from memory again and again: 243 us where this takes 160).
template <CeMode MODE, int PAIR> struct CeWork {
  int tiles_m, tiles_n, steps, whole, left, slices, per, workers, group;
  __device__ __forceinline__ CeWork(const CeProduct& p, int rows, int count) : workers(count) {
    tiles_m = ((MODE == kDw ? p.m : rows) + kCeM * PAIR - 1) / (kCeM * PAIR);
    tiles_n = (p.n + p.bn - 1) / p.bn;
    steps = ((MODE == kDw ? rows : p.k) + kCeK - 1) / kCeK;
    group = max(1, min(p.group, tiles_m));
    whole = tiles_m * tiles_n;
    left = 0;
    slices = 1;
    per = steps;
    if ((MODE == kDx || MODE == kDw) && p.share) {
      // The least time in steps (0.3 us): rounds times a slice's steps, and for several slices the launch that adds them (7 us) and its
      // 256 or 128 KB a part, written and read.
      const int rest = whole % workers;
      float best = (float)steps;
#pragma unroll
      for (int k = 0; k < 11; ++k) {
        const int s = k < 5 ? k + 2 : k == 5 ? 8 : k == 6 ? 12 : k == 7 ? 16 : k == 8 ? 24 : k == 9 ? 32 : kCeSlices;
        if (rest == 0 || s > steps || rest * s * PAIR > kCeParts) continue;
        const float time = (float)((rest * s + workers - 1) / workers) * (float)((steps + s - 1) / s) + 24.f + 0.18f * PAIR * (float)(rest * s);
        if (time < best) { best = time; slices = s; }
      }
      if (slices > 1) {
        per = (steps + slices - 1) / slices;
        slices = (steps + per - 1) / per;
        left = rest;
        whole -= rest;
      }
    }
  }
  // The i-th piece of a worker's work: tile, steps [k0, k1), its part's place in the slab (-1: the whole tile).  False: there is none.
  __device__ __forceinline__ bool at(int worker, int i, int& m, int& n, int& k0, int& k1, int& slot) const {
    int t = worker + i * workers;
    slot = -1;
    k0 = 0;
    k1 = steps;
    if (t >= whole) {
      const int part = t - whole;
      if (part >= left * slices) return false;
      const int slice = part / left;
      k0 = slice * per;
      k1 = min(steps, k0 + per);
      slot = part;
      t = whole + part - slice * left;
    }
    place(t, m, n);
    return true;
  }
  // Tiles in bands of `group` tiles of rows, down the rows first: workers that run together share rows of both operands.
  __device__ __forceinline__ void place(int t, int& m, int& n) const {
    const int band = t / (group * tiles_n), first = band * group, high = min(group, tiles_m - first);
    t -= band * group * tiles_n;
    n = t / high;
    m = first + t - n * high;
  }
};

// Where a row of the result goes, and for dx the row of W that its sums get a multiple of (NULL: none, or the target is of another piece).
template <typename OUT> struct CeOut { int64_t to; const OUT* w; float lost; };
template <CeMode MODE, typename OUT> __device__ __forceinline__ CeOut<OUT> ce_out(const CeProduct& p, int row, bool on) {
  CeOut<OUT> o{MODE == kDw ? p.out_row0 + row : 0, nullptr, 0.f};
  if (MODE == kDw || !on) return o;
  const CeRow r = p.rows[row];
  o.to = r.row;
  if constexpr (CePlanes<OUT>::count == 1) {
    const float lost = p.lost[row];
    if (r.target >= p.vocab0 && r.target < p.vocab0 + p.k) {
      o.w = static_cast<const OUT*>(p.w) + r.target * p.w_stride;
      o.lost = lost;
    }
  }
  return o;
}
template <typename OUT, int COUNT> __device__ __forceinline__ void ce_add_lost(const CeProduct& p, const CeOut<OUT>& o, int col, int have, float* v) {
  if (CePlanes<OUT>::count > 1 || !o.w || o.lost == 0.f) return;
  if (p.w_vec && COUNT % 8 == 0) {
#pragma unroll
    for (int j = 0; j < COUNT; j += 8)
      if (j < have) {
        float f[8];
        load8<OUT>(o.w + col + j, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j + i] = fmaf(o.lost, f[i], v[j + i]);
      }
  } else {
#pragma unroll
    for (int j = 0; j < COUNT; ++j)
      if (j < have) v[j] = fmaf(o.lost, load1<OUT>(o.w + col + j), v[j]);
  }
}

// Several pieces of the vocabulary: the sums of a row of dx so far are added, and kept unless this piece is the last.
template <int COUNT> __device__ __forceinline__ void ce_accumulate(const CeProduct& p, int64_t row, int col, int have, float* v) {
  float* acc = p.acc + row * p.acc_ld + col;
#pragma unroll
  for (int j = 0; j < COUNT; j += 4)
    if (j < have) {   // (acc_ld is a multiple of 8)
      if (p.acc_add) {
        const float4 old = *reinterpret_cast<const float4*>(acc + j);
        v[j] += old.x; v[j + 1] += old.y; v[j + 2] += old.z; v[j + 3] += old.w;
      }
      if (!p.acc_out) *reinterpret_cast<float4*>(acc + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    }
}

// T: the operands' type, OUT: the result's (kDx, kDw) or the caller's (kGrad: float means three planes of G).  REG: accumulators are emptied into
// registers on the way.
template <typename T, typename OUT, CeMode MODE, bool REG, int PAIR>
__global__ void __launch_bounds__(kCeThreads<MODE>, 1) castle_ce_kernel(const CeProduct p, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_copy,
                                                               const __grid_constant__ CUtensorMap map_b) {
  constexpr bool A_MN = MODE == kDw, B_MN = MODE == kDx || MODE == kDw;
  constexpr int SHARES = kCeShares<MODE>, WIDTH = kCeN / SHARES;
  constexpr int GRAIN = 16 * PAIR;   // columns come in multiples of it
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t bar_full[kCeStages], bar_free[kCeStages], bar_done[2], bar_read[2], bar_end;   // of a pair, full and read are the first CTA's
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = PAIR == 2 ? cluster_rank() : 0;
  if (tid == 0) {
    for (int s = 0; s < kCeStages; ++s) { mbar_init(&bar_full[s], 1); mbar_init(&bar_free[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&bar_done[s], 1); mbar_init(&bar_read[s], kCeWarps<MODE> * PAIR); }
    mbar_init(&bar_end, 1);
    mbar_fence_init();
    abort_flag = 0;
    tma_prefetch_desc(&map_a); tma_prefetch_desc(&map_b);
  }
  if (warp == 1) {
    if constexpr (PAIR == 2) tmem_alloc_pair(&tmem_base_s, 512);
    else { tmem_alloc(&tmem_base_s, 512); tmem_relinquish(); }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;
  volatile int* abortp = &abort_flag;
  overlap_wait();
  const CeHead head = *p.head;
  const CeWork<MODE, PAIR> work(p, head.rows, gridDim.x / PAIR);
  const int worker = blockIdx.x / PAIR;
  int m, n, k0, k1, slot;
  // fp32's parts: a stage has all of them where two such stages fit, and the six products of a step read them from there
  // (logits of 197 x 4096 against 256 74 us, a stage for each product 90; forward and gradients of 9472 x 4096 against 8192 9.4 ms / 10.6).
  const bool together = CePlanes<OUT>::count > 1 && 2 * 3 * (kCeA + p.bn / PAIR * kCeK * 2) <= kCeRing;
  const uint32_t parts = together ? 3 : 1, b_bytes = p.bn / PAIR * kCeK * 2, stage = parts * (kCeA + b_bytes);   // bytes
  CeTurn ring(min(kCeStages, (int)(kCeRing / stage)));
  // columns of a tile that are computed
  auto columns = [&](int n) { return min(p.bn, (p.n - n * p.bn + GRAIN - 1) / GRAIN * GRAIN); };

  if (warp == 0) {
    if (elect_one()) {
      const bool copy = head.gathered;
      const CUtensorMap* ma = MODE != kDx && MODE != kDw && copy ? &map_copy : &map_a;
      const CUtensorMap* mb = MODE == kDw && copy ? &map_copy : &map_b;
      // what a step brings, of the pair
      const uint32_t bytes = parts * PAIR * ((A_MN ? 2 * p.k_rows : p.a_rows) * 128 + (MODE == kDw ? kCeN / PAIR / 64 * p.k_rows * 128 : p.bn / PAIR * kCeK * 2));
      bool sent = false, ready = false;   // ready: the next stage was found free while this one's copies were sent (a wait takes 300 cycles even if it is over)
      for (int i = 0; work.at(worker, i, m, n, k0, k1, slot) && !*abortp; ++i) {
        const int m0 = (m * PAIR + rank) * kCeM, n0 = n * p.bn + (PAIR == 2 ? rank * (columns(n) / 2) : 0);
        for (int ks = k0; ks < k1; ++ks) {
          for (int term = together ? 5 : 6 - p.terms; term < 6; ++term) {
            const int s = ring.s, k = ks * kCeK;
            if (!ready && !mbar_wait_ok<true>(&bar_free[s], ring.phase ^ 1u, abortp)) { ks = k1; break; }
            ring.next();
            ready = mbar_test_wait(&bar_free[ring.s], ring.phase ^ 1u);
            if (rank == 0) mbar_expect_tx(&bar_full[s], bytes);
            sent = true;
            auto load = [&](void* dst, const CUtensorMap* map, int c0, int c1, int plane) {
              if constexpr (PAIR == 2) tma_load_4d_pair(dst, map, of_cta(&bar_full[s], 0), c0, c1, plane, 0);
              else tma_load_4d(dst, map, &bar_full[s], c0, c1, plane, 0);
            };
            for (uint32_t part = 0; part < parts; ++part) {
              uint8_t *a = smem + s * stage + part * kCeA, *b = smem + s * stage + parts * kCeA + part * b_bytes;
              const int pa = together ? (int)part : term_a(term), pb = together ? (int)part : term_b(term);
              if (A_MN) {
                load(a, ma, m0, k, pa);
                load(a + kCeA / 2, ma, m0 + 64, k, pa);
              } else {
                load(a, ma, k, m0, pa);
              }
              if (B_MN) {
#pragma unroll
                for (int j = 0; j < kCeN / PAIR / 64; ++j) load(b + j * 8192, mb, n0 + j * 64, k + (MODE == kDx ? p.b_row0 : 0), pb);
              } else {
                load(b, mb, k, p.b_row0 + n0, pb);
              }
            }
          }
        }
      }
      // a copy that nobody waited for (after an abort) must not arrive in another CTA's shared memory
      if (*abortp && rank == 0 && sent)
        for (int j = 0; j < ring.stages; ++j, ring.next()) mbar_drain(&bar_full[ring.s], ring.phase ^ 1u);   // the last round of each
      // nor must the other CTA's word that a stage is free: the second CTA of a pair waits for the last of each (stages never used are free)
      if (rank == 1)
        for (int j = 0; j < ring.stages && !*abortp; ++j, ring.next()) mbar_wait_ok<true>(&bar_free[ring.s], ring.phase ^ 1u, abortp);
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      auto commit = [&](uint64_t* bar) {
        if constexpr (PAIR == 2) mma_commit_pair(bar);
        else mma_commit(bar);
      };
      int turn = 0;
      bool read = false;    // the next accumulator was found free
      bool ready = false;   // the next stage was found filled (logits of 197 x 4096 against 256 in bf16 17.3 us, without looking ahead 20)
      for (int i = 0; work.at(worker, i, m, n, k0, k1, slot) && !*abortp; ++i) {
        const uint32_t idesc = make_idesc(kCeM * PAIR, 16, Elem<T>::fmt, A_MN, B_MN, false) + ((uint32_t)((columns(n) - 16) >> 3) << 17);
        for (; k0 < k1 && !*abortp; k0 += p.flush, ++turn) {
          const int acc = turn & 1, steps = min(p.flush, k1 - k0) * (together ? 1 : p.terms);
          const uint32_t d = tmem + acc * kCeN;
          const uint32_t phase = ((uint32_t)(turn >> 1) & 1u) ^ 1u;
          if ((PAIR == 2 || !read) && !(PAIR == 2 ? mbar_wait_ok_cluster(&bar_read[acc], phase, abortp) : mbar_wait_ok<true>(&bar_read[acc], phase, abortp))) break;
          tc_fence_after();
          for (int j = 0; j < steps; ++j) {
            const int s = ring.s;
            if (!ready && !mbar_wait_ok<true>(&bar_full[s], ring.phase, abortp)) break;
            tc_fence_after();
            ring.next();
            ready = mbar_test_wait(&bar_full[ring.s], ring.phase);
            for (int term = together ? 0 : 5; term < 6; ++term) {
              const uint32_t a = smem_u32(smem) + s * stage + (together ? term_a(term) * kCeA : 0),
                             b = smem_u32(smem) + s * stage + parts * kCeA + (together ? term_b(term) * b_bytes : 0);
              const uint64_t da = A_MN ? desc_mnmajor(a, 8192) : desc_kmajor(a), db = B_MN ? desc_mnmajor(b, 8192) : desc_kmajor(b);
#pragma unroll
              for (int q = 0; q < kCeK / 16; ++q) {
                if (MODE == kDw && q * 16 >= p.k_rows) break;
                const uint64_t ao = da + (uint64_t)(((A_MN ? 2048 : 32) * q) >> 4), bo = db + (uint64_t)(((B_MN ? 2048 : 32) * q) >> 4);
                const bool add = j > 0 || (together && term > 0) || q > 0;
                if constexpr (PAIR == 2) mma_ss_pair(d, ao, bo, idesc, add);
                else mma_ss(d, ao, bo, idesc, add);
              }
            }
            commit(&bar_free[s]);
          }
          commit(&bar_done[acc]);
          if (PAIR == 1) read = mbar_test_wait(&bar_read[acc ^ 1], ((uint32_t)((turn + 1) >> 1) & 1u) ^ 1u);
        }
      }
      commit(&bar_end);   // all products have read their operands
      mbar_drain(&bar_end, 0);
    }
  } else {
    const int quarter = warp & 3, share = (warp - 2) >> 2, width = p.bn / SHARES;   // a warp has 32 rows and a share of the columns
    const uint32_t src = tmem + share * width + ((uint32_t)(quarter * 32) << 16);
    uint8_t* staging = smem + kCeRing + (warp - 2) * 2048;
    const uint32_t read_at = PAIR == 2 ? of_cta(&bar_read[0], 0) : 0;
    int turn = 0;
    bool over = false;
    auto release = [&] {   // the accumulator has been read
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR == 2) mbar_arrive_at(read_at + (turn & 1) * 8);
        else mbar_arrive(&bar_read[turn & 1]);
      }
      ++turn;
    };
    for (int i = 0; !over && work.at(worker, i, m, n, k0, k1, slot); ++i) {
      const int local = rank * kCeM + quarter * 32 + lane, row = m * PAIR * kCeM + local, c_base = n * p.bn + share * width;
      const int cols = min(width, p.n - c_base);   // that there are; of the others up to the next grain are computed
      const bool empty = k1 <= k0;
      const bool on = row < (MODE == kDw ? p.m : head.rows), direct = slot < 0 && (!p.acc || p.acc_out);
      CeOut<OUT> dst{0, nullptr, 0.f};
      if constexpr (MODE == kDx || MODE == kDw) dst = ce_out<MODE, OUT>(p, row, on);
      float sums[REG ? WIDTH : 1];
      if constexpr (REG) {
#pragma unroll
        for (int j = 0; j < WIDTH; ++j) sums[j] = 0.f;
        for (; k0 < k1; k0 += p.flush) {
          if (mbar_wait_failed(&bar_done[turn & 1], (uint32_t)(turn >> 1) & 1u, abortp)) { over = true; break; }
          tc_fence_after();
#pragma unroll
          for (int c0 = 0; c0 < WIDTH; c0 += 16) {
            if (c0 >= cols) break;
            float v[16];
            tmem_ld16(src + (turn & 1) * kCeN + c0, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const float2 t = add2(make_float2(sums[c0 + j], sums[c0 + j + 1]), make_float2(v[j], v[j + 1]));
              sums[c0 + j] = t.x;
              sums[c0 + j + 1] = t.y;
            }
          }
          release();
        }
        if (over) break;
      } else if (!empty) {
        if (mbar_wait_failed(&bar_done[turn & 1], (uint32_t)(turn >> 1) & 1u, abortp)) break;
        tc_fence_after();
      }
      auto take = [&](int c0, float* v) {   // values [c0, c0 + 32) of the thread's part of a row
        if constexpr (REG) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = sums[c0 + j];
        } else if (MODE == kDw && empty) {   // no rows take part
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0.f;
        } else {
          tmem_ld32(src + (turn & 1) * kCeN + c0, v);
          tmem_ld_wait();
        }
      };
      bool held = !REG && !empty;
      auto last_taken = [&](bool last) {   // the next product into the accumulator runs under the rest
        if (held && last) {
          release();
          held = false;
        }
      };
      constexpr float kLog2e = 1.4426950408889634f;
      if constexpr (MODE == kLse) {
        const int target = on ? p.rows[row].target - p.vocab0 - c_base : -1;
        float best = -INFINITY, sum = 0.f;
#pragma unroll
        for (int c0 = 0; c0 < WIDTH; c0 += 32) {
          if (c0 >= cols) break;
          float v[32];
          take(c0, v);
          last_taken(c0 + 32 >= cols);
          if (c0 + 32 > cols) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = c0 + j < cols ? v[j] : -INFINITY;
          }
          float top = best;
#pragma unroll
          for (int j = 0; j < 32; ++j) top = fmaxf(top, v[j]);
          if (target >= c0 && target < min(c0 + 32, cols)) {
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
        if (on) p.parts[(int64_t)(n * SHARES + share) * p.parts_ld + row] = make_float2(best, sum);
      } else if constexpr (MODE == kGrad) {
        CeRow r;
        r.target = -1; r.lse = 0.f; r.coef = 0.f; r.row = 0;
        if (row < head.rows) r = p.rows[row];
        const int target = r.target - p.vocab0 - c_base;
        constexpr int PLANES = CePlanes<OUT>::count;
#pragma unroll
        for (int c0 = 0; c0 < WIDTH; c0 += 32) {
          if (c0 >= cols) break;
          float v[32];
          take(c0, v);
          last_taken(c0 + 32 >= cols);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 d = mul2(add2(make_float2(v[j], v[j + 1]), splat(-r.lse)), splat(kLog2e));
            v[j] = ex2_approx(d.x);
            v[j + 1] = ex2_approx(d.y);
          }
          if (target >= c0 && target < min(c0 + 32, cols)) {
            float g = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              v[j] = c0 + j == target ? v[j] - 1.f : v[j];
              g = c0 + j == target ? v[j] : g;
            }
            if (PLANES == 1) {
              g *= r.coef;
              const float lost = g - Elem<T>::to_f(Elem<T>::from_f(g));
              p.lost[row] = isfinite(lost) ? lost : 0.f;
            }
          }
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = r.coef == 0.f ? 0.f : v[j] * r.coef;
#pragma unroll
          for (int q = 0; q < PLANES; ++q) {
            __syncwarp();   // what was here before has been read
#pragma unroll
            for (int c = 0; c < 4; ++c) {   // a plane's part of each value, and what it leaves to the next
              uint4 o;
              uint32_t* u = &o.x;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                float* pair = v + c * 8 + 2 * j;
                u[j] = Elem<T>::pack2(pair[0], pair[1]);
                if (q + 1 < PLANES) {
                  const float2 f = Elem<T>::unpack2(u[j]);
                  pair[0] -= f.x;
                  pair[1] -= f.y;
                }
              }
              *reinterpret_cast<uint4*>(staging + staging_off(lane, c)) = o;
            }
            __syncwarp();
            // Four lanes store a row's 64 bytes; also the zeros of rows behind the last one.
            uint16_t* out = p.g + q * p.g_plane + (int64_t)(row - lane) * p.g_ld + c_base + c0;
            const int col = (lane & 3) * 8;
            if (c0 + col < cols) {   // (g_ld is a multiple of 8)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int at = j * 8 + (lane >> 2);
                *reinterpret_cast<uint4*>(out + at * p.g_ld + col) = *reinterpret_cast<const uint4*>(staging + staging_off(at, lane & 3));
              }
            }
          }
        }
      } else {
        const float unit = head.unit;
        const int64_t to = dst.to;
#pragma unroll
        for (int c0 = 0; c0 < WIDTH; c0 += 32) {
          if (c0 >= cols) break;
          float v[32];
          take(c0, v);
          last_taken(c0 + 32 >= cols);
          if (slot >= 0) {
            float4* out = p.slab + ((int64_t)slot * (kCeN / 4) + (share * width + c0) / 4) * (kCeM * PAIR) + local;
#pragma unroll
            for (int j = 0; j < 32; j += 4) out[(j / 4) * (kCeM * PAIR)] = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          } else {
            if constexpr (MODE == kDx) {
              ce_add_lost<OUT, 32>(p, dst, c_base + c0, min(32, cols - c0), v);
              if (p.acc && on) ce_accumulate<32>(p, row, c_base + c0, min(32, cols - c0), v);
            }
            if (!direct) continue;
            // Through shared memory, so that four lanes store 64 bytes of a row, or half a warp its words where rows are not
            // at 16-byte boundaries (dW of 24989 x 5859 over 23 rows 168 us; by single elements of 32 rows at a time 1416, and with rows of 5856 63).
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= unit;
            constexpr int PIECE = 16 / (int)sizeof(OUT), PANEL = 4 * PIECE;   // columns of 16 bytes, and of 64
            OUT* out = static_cast<OUT*>(p.out) + c_base;
#pragma unroll
            for (int h = 0; h < 32; h += PANEL) {
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const float* f = v + h + c * PIECE;
                if constexpr (sizeof(OUT) == 4) *reinterpret_cast<float4*>(staging + staging_off(lane, c)) = make_float4(f[0], f[1], f[2], f[3]);
                else store8<OUT>(reinterpret_cast<OUT*>(staging + staging_off(lane, c)), f);
              }
              __syncwarp();
              if (p.vec) {
                const int col = c0 + h + (lane & 3) * PIECE;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const int at = j * 8 + (lane >> 2);
                  int64_t row_to;
                  bool there;
                  if constexpr (MODE == kDw) {
                    there = row - lane + at < p.m;
                    row_to = to - lane + at;
                  } else {
                    const int target = __shfl_sync(0xffffffffu, on ? (int)to : -1, at);
                    there = target >= 0;
                    row_to = target;
                  }
                  if (there && col < cols)
                    *reinterpret_cast<uint4*>(out + row_to * p.ld + col) = *reinterpret_cast<const uint4*>(staging + staging_off(at, lane & 3));
                }
              } else {
                // Half a warp has a row, a lane a word of it; the single elements before and behind a row's words are stored by the row's own lane.
                constexpr bool HALVES = sizeof(OUT) == 2;
                const int k = lane % 16, side = lane / 16, have = min(PANEL, cols - c0 - h);
                OUT* const panel = out + c0 + h;
                auto lead = [](const OUT* row) { return HALVES ? (int)(reinterpret_cast<uintptr_t>(row) / 2 % 2) : 0; };
                const uint8_t* const from = staging + side * 64;
                auto word = [&](int j, int i) { return *reinterpret_cast<const uint32_t*>(from + j * 128 + (((i / 4) ^ (j & 3)) << 4) + i % 4 * 4); };   // (see staging_off)
                auto store = [&](OUT* row, int off, int j) {   // the (2 j + side)-th row of the warp's
                  *reinterpret_cast<uint32_t*>(row + (HALVES ? 2 * k + off : k)) = HALVES ? __funnelshift_r(word(j, k), word(j, (k + 1) % 16), off * 16) : word(j, k);
                };
                if constexpr (MODE == kDw) {
                  OUT* row_at = panel + (to - lane + side) * p.ld;
                  const int off = lead(row_at);   // (every second row begins alike)
                  const int rows = (HALVES ? 2 * k + off + 1 : k) < have ? p.m - (row - lane) - side : 0;
#pragma unroll 4
                  for (int j = 0; j < 16; ++j, row_at += 2 * p.ld)
                    if (2 * j < rows) store(row_at, off, j);
                } else {
#pragma unroll 4
                  for (int j = 0; j < 16; ++j) {
                    const int target = __shfl_sync(0xffffffffu, on ? (int)to : -1, 2 * j + side);
                    OUT* row_at = panel + (int64_t)target * p.ld;
                    const int off = lead(row_at);
                    if (target >= 0 && (HALVES ? 2 * k + off + 1 : k) < have) store(row_at, off, j);
                  }
                }
                if constexpr (HALVES) {
                  OUT* mine = panel + to * p.ld;
                  const int off = lead(mine);
                  auto element = [&](int i) { return *reinterpret_cast<const OUT*>(staging + staging_off(lane, i / 8) + i % 8 * 2); };
                  if (on && off) mine[0] = element(0);
                  if (on && (have - off) % 2 == 1) mine[have - 1] = element(have - 1);   // (nothing for a row of its first element alone)
                }
              }
              __syncwarp();
            }
          }
          __syncwarp();
        }
      }
      last_taken(true);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR == 2) {
    cluster_sync();   // the other's products read this CTA's tiles, its warps arrive at this CTA's barriers
    // The issuing thread has seen its last commit at its own CTA's barrier, which says nothing of the arrival here: a CTA that ended before would
    // have it in the shared memory of the next one on its SM.  (An issuer's commits arrive in order; this one comes after an abort, too.)
    if (rank == 1 && tid == 0) mbar_drain(&bar_end, 0);
  }
  if (warp == 1) {
    if constexpr (PAIR == 2) tmem_dealloc_pair(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
  if (tid == 0 && abort_flag) atomicOr(p.status, CASTLE_STATUS_WAIT_TIMEOUT);
}

// The parts of shared tiles, added in order: a thread per COLS values of a row, blockIdx.y the tile.
template <typename OUT, CeMode MODE, int PAIR, int COLS>
__global__ void __launch_bounds__(256) castle_ce_sum_kernel(const CeProduct p) {
  constexpr int ROWS = kCeM * PAIR;
  overlap_wait();
  const CeHead head = *p.head;
  const CeWork<MODE, PAIR> work(p, head.rows, kCeWorkers / PAIR);
  const int tile = blockIdx.y;
  if (tile >= work.left) return;
  int m, n;
  work.place(work.whole + tile, m, n);
  const int at = blockIdx.x * 256 + threadIdx.x, local = at % ROWS, first = at / ROWS * COLS;   // neighbouring threads: neighbouring rows
  const int row = m * ROWS + local, col = n * p.bn + first;
  const bool on = row < (MODE == kDw ? p.m : head.rows);
  if (col >= p.n) return;   // (a whole warp: its threads have neighbouring rows)
  float t[COLS];
#pragma unroll
  for (int j = 0; j < COLS; ++j) t[j] = 0.f;
  const int slices = on ? work.slices : 0;
#pragma unroll(COLS == 4 ? 8 : 2)
  for (int s = 0; s < slices; ++s) {
#pragma unroll
    for (int j = 0; j < COLS; j += 4) {
      const float4 v = p.slab[((int64_t)(s * work.left + tile) * (kCeN / 4) + (first + j) / 4) * ROWS + local];
      t[j] += v.x; t[j + 1] += v.y; t[j + 2] += v.z; t[j + 3] += v.w;
    }
  }
  const int have = min(COLS, p.n - col);
  const CeOut<OUT> dst = ce_out<MODE, OUT>(p, row, on);
  if constexpr (MODE == kDx) {
    ce_add_lost<OUT, COLS>(p, dst, col, have, t);
    if (p.acc && on) ce_accumulate<COLS>(p, row, col, have, t);
    if (p.acc && !p.acc_out) return;
  }
#pragma unroll
  for (int j = 0; j < COLS; ++j) t[j] *= head.unit;
  OUT* out = static_cast<OUT*>(p.out) + col;
  if constexpr (COLS == 16) {
    if (!p.vec) {   // rows at odd places: half a warp stores a row's 16 elements
      __shared__ float stage[8][32][17];
      const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, in = lane % 16;
#pragma unroll
      for (int j = 0; j < 16; ++j) stage[warp][lane][j] = t[j];
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        const int at = j + lane / 16, to = __shfl_sync(0xffffffffu, on ? (int)dst.to : -1, at);
        if (to >= 0 && in < have) store1<OUT>(out + to * p.ld + in, stage[warp][at][in]);
      }
      return;
    }
    if (!on) return;
#pragma unroll
    for (int j = 0; j < COLS; j += 8)
      if (j < have) store8<OUT>(out + dst.to * p.ld + j, t + j);
  } else {
    if (!on) return;
#pragma unroll
    for (int j = 0; j < COLS; ++j)
      if (j < have) store1<OUT>(out + dst.to * p.ld + j, t[j]);
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
  if constexpr (ROWS == 1) {   // trees: 256 parts one after the other would take as long as the rest
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) join(make_float2(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, sum, o)));
    if ((l & 31) == 0) s[l >> 5][0] = make_float2(best, sum);
  } else {
    s[l][r] = make_float2(best, sum);
  }
  __syncthreads();
  double loss = 0.0;
  if (l == 0 && row < rows) {
    for (int k = 1; k < (ROWS == 1 ? 8 : LANES); ++k) join(s[k][r]);
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
  __shared__ double ds[8];
  auto cta_sum = [&](double v) {   // of all threads; thread 0 has it
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) ds[threadIdx.x >> 5] = v;
    __syncthreads();
    return threadIdx.x == 0 ? ((ds[0] + ds[1]) + (ds[2] + ds[3])) + ((ds[4] + ds[5]) + (ds[6] + ds[7])) : 0.0;
  };
  const double mine = cta_sum(loss);
  if (threadIdx.x == 0) {
    p.sums[blockIdx.x] = mine;
    __threadfence();
    last = atomicAdd(&p.head->done, 1u) + 1 == gridDim.x;
    __threadfence();
  }
  __syncthreads();
  if (!last) return;
  double t = 0.0;
  for (int k = threadIdx.x; k < (int)gridDim.x; k += 256) t += __ldcg(p.sums + k);
  double total = cta_sum(t);
  if (threadIdx.x == 0) {
    if (p.mean) total /= (double)rows;
    p.loss[0] = p.head->bad ? __int_as_float(0x7fffffff) : (float)total;
  }
}

// ------------------------------------------------------------------------------------------------ host
// How a result of m x n over a contraction of k (all terms of it) is cut.  Pairs of CTAs are faster per row where the contraction is long and
// slower where it is short (the second CTA waits for the first's products at a tile's start and end), and pad the rows to 256 instead of
// 128.  us, pairs / single: logits and their gradient of 4096 x 1024 against 50021 281, 340 / 299, 369; 197 x 4096 against 131072 216, 231 / 231, 245;
// 300 x 1024 against 50021 48, 48 / 40, 42; 2000 x 512 against 8000 21, 26 / 19, 23.  dx of 4096 x 1024 312 / 340, of 600 x 1024 73 / 81, of 300 x 1024 56 / 51.
// dW, whose rows are the vocabulary: over 300 tokens 48 / 44, 600 61 / 66, 1000 33 / 36.  Narrower tiles (of single ones with one product's
// contraction each) as long as all of them run at once: logits of 130 x 512 against 256 6.0, with 256 columns 8.3; but two rounds of half
// tiles are slower than one of whole ones (50 x 768 against 32000 in fp32 55 / 43).  With one tile of rows, half as wide ones also where their
// rounds come out shorter (128 x 4096 against 131072, 7 of 128 columns for 4 of 256: logits 194 -> 188 us, their gradient 195 -> 192).
struct CeCut { int pair, bn; };
static CeCut ce_cut(CeMode mode, int64_t m, int64_t n, int64_t k) {
  const int64_t single = (m + 127) / 128 * 128, pairs = (m + 255) / 256 * 256;
  const bool logits = mode == kLse || mode == kGrad;
  const int64_t cost = mode == kDx ? 80 : k >= 1024 ? 85 : 108;   // of a pair's row, in hundredths of a single CTA's
  if (mode == kDw ? m > kCeM && k > 512 : pairs * cost < single * 100) {
    if (!logits || pairs / 256 * ((n + 255) / 256) >= 37) return {2, 256};   // (half of the pairs have a tile)
  }
  const int least = mode == kLse ? 32 * kCeShares<kLse> : mode == kGrad ? 32 * kCeShares<kGrad> : 256;   // 32 columns of each share
  int bn = 256;
  while (bn > least && single / 128 * ((2 * n + bn - 1) / bn) <= kCeWorkers) bn /= 2;
  if (logits && m <= kCeM && bn == 256) {   // one tile of rows: the weight's bytes are the time
    auto rounds = [&](int64_t width) { return ((n + width - 1) / width + kCeWorkers - 1) / kCeWorkers; };
    if (rounds(128) * 133 < rounds(256) * 256) bn = 128;
  }
  return {1, bn};
}

struct CePlan {
  int a_rows, k_rows;         // of a load, see CeProduct
  int planes, terms, pitch, piece_fwd, piece_bwd, parts_per_piece, pieces;
  bool copy_x, copy_w;        // operands are laid out anew: fp32, or rows that TMA cannot read
  int64_t copy_rows, g_rows;
  size_t rows, copy, wcopy, parts, running, logit, sums, g, lost, slab, acc, bytes;   // offsets
};

static CePlan ce_plan(int dtype, int64_t n, int dim, int64_t vocab, bool x_ok, bool w_ok, bool backward) {
  CePlan q{};
  auto up = [](int64_t v, int64_t to) { return (v + to - 1) / to * to; };
  const bool f32 = dtype == CASTLE_F32;
  q.planes = f32 ? 3 : 1;
  q.terms = f32 ? 6 : 1;
  q.pitch = (int)up(dim, 8);
  q.copy_x = f32 || !x_ok;
  q.copy_w = f32 || !w_ok;
  // A tile's rows behind the last one need not be loaded (their results go nowhere); of the contraction they have to be zero, 16 at a time.  Rows that
  // TMA has to fill take it longer than rows that it reads (8 x 4096 against 131072: logits 241 -> 187 us, their gradient 243 -> 180 (188 since its sums are emptied on the way), dW 257 -> 239).
  q.a_rows = (int)(n < kCeM ? up(n, 8) : kCeM);
  q.k_rows = (int)(n < kCeK ? up(n, 16) : kCeK);
  q.copy_rows = up(n, kCeK);
  q.g_rows = up(n, 2 * kCeM);
  const int64_t w_row = q.copy_w ? (int64_t)q.planes * q.pitch * 2 : 0;
  auto piece = [&](int64_t per_column) {
    int64_t v = kCeScratch / (per_column > 0 ? per_column : 1) / kCeN * kCeN;
    if (v < kCeN) v = kCeN;
    return (int)(v < vocab ? v : vocab);
  };
  q.piece_fwd = piece(w_row + q.copy_rows * kCeShares<kLse> * (int64_t)sizeof(float2) / kCeN);
  q.piece_bwd = piece(w_row + q.planes * q.g_rows * 2);
  q.pieces = (int)((vocab + q.piece_bwd - 1) / q.piece_bwd);
  size_t at = 1024;   // behind the CeHead
  auto take = [&](size_t bytes) { const size_t o = at; at += up((int64_t)bytes, 1024); return o; };
  q.rows = take((size_t)n * sizeof(CeRow));
  q.copy = take((size_t)q.planes * q.copy_rows * q.pitch * 2);
  const int64_t most = backward ? q.piece_bwd : q.piece_fwd;
  q.wcopy = take(q.copy_w ? (size_t)most * w_row : 0);
  if (!backward) {
    // so many for each tile of a row: of 256 columns, or 128 if the rows are one tile, or fewer where all tiles run at once (ce_cut)
    const int64_t width = n <= kCeM ? 128 : kCeN, wide = (q.piece_fwd + width - 1) / width;
    const int64_t few = kCeWorkers / ((n + kCeM - 1) / kCeM);
    q.parts_per_piece = kCeShares<kLse> * (int)(wide > few ? wide : few);
    q.parts = take((size_t)q.parts_per_piece * q.copy_rows * sizeof(float2));
    q.running = take((size_t)n * sizeof(float2));
    q.logit = take((size_t)n * sizeof(float));
    q.sums = take((size_t)((n + 7) / 8 + 256) * sizeof(double));
  } else {
    q.g = take((size_t)q.planes * q.g_rows * up(q.piece_bwd, 8) * 2);
    q.lost = take((size_t)n * sizeof(float));
    // the slab: as many parts as CeWork can choose
    auto parts = [&](const CeCut& cut, int64_t m, int64_t k) {
      const int64_t tiles = (m + kCeM * cut.pair - 1) / (kCeM * cut.pair) * ((dim + kCeN - 1) / kCeN), most = tiles * kCeSlices * cut.pair;
      return k < kCeShare * kCeK - kCeK + 1 ? 0 : most < kCeParts ? most : kCeParts;
    };
    const int64_t for_dx = parts(ce_cut(kDx, n, dim, (int64_t)q.piece_bwd * q.terms), n, q.piece_bwd);
    const int64_t for_dw = parts(ce_cut(kDw, q.piece_bwd, dim, n * q.terms), q.piece_bwd, n);
    q.slab = take((size_t)(for_dx > for_dw ? for_dx : for_dw) * kCeM * kCeN * sizeof(float));
    q.acc = take(q.pieces > 1 ? (size_t)n * up(dim, 8) * sizeof(float) : 0);
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

template <typename T, typename OUT, CeMode MODE, bool REG, int PAIR>
static cudaError_t ce_launch_as(const CeProduct& p, int64_t tiles, const CUtensorMap& a, const CUtensorMap& copy, const CUtensorMap& b, cudaStream_t st) {
  auto kernel = castle_ce_kernel<T, OUT, MODE, REG, PAIR>;
  const cudaError_t e = allow_smem(kernel, (int)kCeSmem);
  if (e != cudaSuccess) return e;
  const int64_t most = p.share ? kCeWorkers : tiles * PAIR;
  cudaLaunchConfig_t c = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = PAIR;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  c.gridDim = dim3((unsigned)(most < kCeWorkers ? most : kCeWorkers));
  c.blockDim = dim3(kCeThreads<MODE>);
  c.dynamicSmemBytes = kCeSmem;
  c.stream = st;
  c.attrs = attr;
  c.numAttrs = PAIR == 2 ? 2 : 1;
  return cudaLaunchKernelEx(&c, kernel, p, a, copy, b);
}
template <typename T, typename OUT, CeMode MODE>
static cudaError_t ce_launch(const CeProduct& p, int pair, int64_t tiles, const CUtensorMap& a, const CUtensorMap& copy, const CUtensorMap& b, cudaStream_t st) {
  constexpr bool F32 = CePlanes<OUT>::count > 1;
  if constexpr ((MODE == kLse || MODE == kGrad) && !F32) {   // one emptying of an accumulator is none: it is read where it is
    if (p.k > p.flush * kCeK)
      return pair == 2 ? ce_launch_as<T, OUT, MODE, true, 2>(p, tiles, a, copy, b, st) : ce_launch_as<T, OUT, MODE, true, 1>(p, tiles, a, copy, b, st);
  }
  return pair == 2 ? ce_launch_as<T, OUT, MODE, F32, 2>(p, tiles, a, copy, b, st) : ce_launch_as<T, OUT, MODE, F32, 1>(p, tiles, a, copy, b, st);
}

static int ce_rows_per_cta(int64_t n) {   // a CTA per SM, at least eight rows each (197 x 4096 in fp32 9 us, with 32 rows 20)
  const int64_t r = (n + 147) / 148;
  return (int)(r < 8 ? 8 : r);
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
  CE_TRY(ce_x_maps(c, q, op, q.a_rows, &x, &copy));
  for (int64_t v0 = 0; v0 < c.vocab; v0 += q.piece_fwd) {
    const int64_t count = c.vocab - v0 < q.piece_fwd ? c.vocab - v0 : q.piece_fwd;
    const CeCut cut = ce_cut(kLse, c.n, count, (int64_t)q.pitch * q.terms);
    const int tiles_n = (int)((count + cut.bn - 1) / cut.bn);
    CE_CUDA(ce_weight<OUT>(c, q, v0, count), "castle_linear_ce_fwd launch");
    CE_TRY(ce_w_map(c, q, op, count, cut.bn / cut.pair, &w));
    CeProduct p{};
    p.head = (const CeHead*)c.work; p.rows = (const CeRow*)(c.work + q.rows); p.n = (int)count; p.k = q.pitch; p.bn = cut.bn; p.a_rows = q.a_rows; p.k_rows = kCeK; p.b_row0 = q.copy_w ? 0 : (int)v0;
    p.vocab0 = (int)v0; p.terms = q.terms; p.group = 32 / cut.pair;
    p.flush = q.terms > 1 ? kCeFlushF32 : kCeFlush;
    p.parts = (float2*)(c.work + q.parts); p.parts_ld = q.copy_rows; p.target_logit = (float*)(c.work + q.logit); p.status = c.status;
    const int64_t tiles_m = (c.n + kCeM * cut.pair - 1) / (kCeM * cut.pair);
    CE_CUDA((ce_launch<T, OUT, kLse>(p, cut.pair, tiles_m * tiles_n, x, copy, w, c.st)), "castle_linear_ce_fwd launch");
    CeJoin j{};
    j.head = (CeHead*)c.work; j.rows = p.rows; j.parts = p.parts; j.running = (float2*)(c.work + q.running); j.target_logit = p.target_logit;
    j.sums = (double*)(c.work + q.sums); j.lse = lse; j.loss = loss; j.parts_ld = q.copy_rows; j.parts_n = kCeShares<kLse> * tiles_n;
    j.begin = v0 == 0; j.end = v0 + count == c.vocab; j.each = each; j.mean = c.reduction == CASTLE_REDUCE_MEAN;
    // few rows: a CTA or a warp each; many: neighbouring threads on neighbouring rows
    if (c.n < 256) CE_CUDA(launch_kernel(castle_ce_join_kernel<1>, dim3((unsigned)c.n), 256, 0, c.st, true, j), "castle_linear_ce_fwd launch");
    else if (c.n >= 4096) CE_CUDA(launch_kernel(castle_ce_join_kernel<32>, dim3((unsigned)((c.n + 31) / 32)), 256, 0, c.st, true, j), "castle_linear_ce_fwd launch");
    else CE_CUDA(launch_kernel(castle_ce_join_kernel<8>, dim3((unsigned)((c.n + 7) / 8)), 256, 0, c.st, true, j), "castle_linear_ce_fwd launch");
  }
  return 0;
}

template <typename OUT>
static int ce_backward(const CeCall& c, const CePlan& q, const float* lse, const float* dloss, void* dx, void* dw) {
  using T = typename CePlanes<OUT>::Op;
  const char* what = "castle_linear_ce_bwd launch";
  const int op = c.dtype == CASTLE_F16 ? CASTLE_F16 : CASTLE_BF16;
  CE_CUDA(ce_rows<OUT>(c, q, lse, dloss, dx, nullptr, nullptr), what);
  CUtensorMap x, copy, xk, copyk, w, wk, ga, gt;
  CE_TRY(ce_x_maps(c, q, op, q.a_rows, &x, &copy));
  CE_TRY(ce_x_maps(c, q, op, q.k_rows, &xk, &copyk));
  CeProduct base{};
  base.head = (const CeHead*)c.work; base.rows = (const CeRow*)(c.work + q.rows); base.terms = q.terms; base.flush = q.terms > 1 ? kCeFlushF32 : kCeNoFlush;
  base.status = c.status; base.ld = c.dim; base.bn = kCeN; base.a_rows = q.a_rows; base.k_rows = q.k_rows; base.slab = (float4*)(c.work + q.slab);
  base.lost = (float*)(c.work + q.lost);
  // What the workers share out: launched with the product whenever there could be something.
  auto product = [&](auto mode, const CeProduct& p, const CeCut& cut, int64_t m, const CUtensorMap& a, const CUtensorMap& acopy, const CUtensorMap& b) -> cudaError_t {
    constexpr CeMode MODE = decltype(mode)::value;
    const int64_t tiles = (m + kCeM * cut.pair - 1) / (kCeM * cut.pair) * ((p.n + kCeN - 1) / kCeN);
    const cudaError_t e = ce_launch<T, OUT, MODE>(p, cut.pair, tiles, a, acopy, b, c.st);
    if (e != cudaSuccess || !p.share) return e;
    const int64_t shared = tiles < kCeWorkers / cut.pair ? tiles : kCeWorkers / cut.pair;
    auto sum = [&](auto pair, auto cols) {
      constexpr int PAIR = decltype(pair)::value, COLS = decltype(cols)::value;
      return launch_kernel(castle_ce_sum_kernel<OUT, MODE, PAIR, COLS>, dim3(kCeM * PAIR * kCeN / COLS / 256, (unsigned)shared), 256, 0, c.st, true, p);
    };
    using std::integral_constant;
    // few tiles: many parts of each, added by many threads; else whole sectors of the result by each thread
    if (cut.pair == 1) return shared < 32 ? sum(integral_constant<int, 1>(), integral_constant<int, 4>()) : sum(integral_constant<int, 1>(), integral_constant<int, 16>());
    return shared < 16 ? sum(integral_constant<int, 2>(), integral_constant<int, 4>()) : sum(integral_constant<int, 2>(), integral_constant<int, 16>());
  };
  for (int64_t v0 = 0; v0 < c.vocab; v0 += q.piece_bwd) {
    const int64_t count = c.vocab - v0 < q.piece_bwd ? c.vocab - v0 : q.piece_bwd, pitch = (count + 7) / 8 * 8;
    uint16_t* gp = (uint16_t*)(c.work + q.g);
    const CeCut cut = ce_cut(kGrad, c.n, count, (int64_t)q.pitch * q.terms), cut_dx = ce_cut(kDx, c.n, c.dim, count * q.terms),
                cut_dw = ce_cut(kDw, count, c.dim, c.n * q.terms);
    CE_CUDA(ce_weight<OUT>(c, q, v0, count), what);
    CE_TRY(ce_w_map(c, q, op, count, cut.bn / cut.pair, &w));
    CE_TRY(ce_w_map(c, q, op, count, kCeK, &wk));
    CE_TRY(ce_map(&ga, gp, op, q.g_rows, (int)count, pitch, q.g_rows * pitch, q.planes, q.a_rows, "castle_linear_ce: logits' gradient"));
    CE_TRY(ce_map(&gt, gp, op, q.g_rows, (int)count, pitch, q.g_rows * pitch, q.planes, q.k_rows, "castle_linear_ce: logits' gradient"));
    CeProduct p = base;
    p.n = (int)count; p.k = q.pitch; p.bn = cut.bn; p.b_row0 = q.copy_w ? 0 : (int)v0; p.vocab0 = (int)v0; p.group = 32 / cut.pair;
    p.g = gp; p.g_ld = pitch; p.g_plane = q.g_rows * pitch;
    p.flush = q.terms > 1 ? kCeFlushF32 : kCeFlush;   // as in the forward: these are the logits that the log-sum-exp was formed of
    const int64_t tiles_m = (c.n + kCeM * cut.pair - 1) / (kCeM * cut.pair);
    CE_CUDA((ce_launch<T, OUT, kGrad>(p, cut.pair, tiles_m * ((count + cut.bn - 1) / cut.bn), x, copy, w, c.st)), what);
    if (dx) {
      p = base;
      p.vocab0 = (int)v0; p.w = c.w; p.w_stride = c.ws; p.w_vec = c.dim % 8 == 0 && (uintptr_t)c.w % 16 == 0 && c.ws % 8 == 0;
      p.n = c.dim; p.k = (int)count; p.b_row0 = q.copy_w ? 0 : (int)v0; p.out = dx; p.group = 16 / cut_dx.pair;
      p.vec = c.dim % 8 == 0 && (uintptr_t)dx % 16 == 0;
      p.share = (p.k + kCeK - 1) / kCeK >= kCeShare;
      if (q.pieces > 1) { p.acc = (float*)(c.work + q.acc); p.acc_ld = (c.dim + 7) / 8 * 8; p.acc_add = v0 > 0; p.acc_out = v0 + count == c.vocab; }
      CE_CUDA(product(std::integral_constant<CeMode, kDx>(), p, cut_dx, c.n, ga, ga, wk), what);
    }
    if (dw) {
      p = base;
      p.m = (int)count; p.n = c.dim; p.out = dw; p.out_row0 = v0; p.group = 16 / cut_dw.pair;
      p.vec = c.dim % 8 == 0 && (uintptr_t)dw % 16 == 0;
      p.share = (c.n + kCeK - 1) / kCeK >= kCeShare;
      CE_CUDA(product(std::integral_constant<CeMode, kDw>(), p, cut_dw, count, gt, copyk, xk), what);
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
