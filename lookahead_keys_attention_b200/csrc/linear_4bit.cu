// y = x W^T with weights of 4 bits, for the rows of a few tokens:
//
//     W[n, k] = scale[n, k / group] * (code[n, k] - zero[n, k / group])       zero = 8 where there are no zero points
//
// The product is a stream over the codes (half a byte per weight), so it is bound by HBM, and for small weights by a launch's latencies.
// It is computed with mma.sync: 16 weight rows are the first operand, 8 columns of x the second.  The sums of a group are fp32, and scales and
// zero points are applied to them, so that nothing but x and y is rounded to 16 bits.  For 16-bit rows a code enters as 16 + code, four bits
// at the top of a number's mantissa that one shift and one operation put there, and the rest is taken off by the sum of the group's x:
//     y[n] = sum over groups of  scale * (sum of (16 + code) x  -  (16 + zero) * sum of x)
// (the fp32 sums are some six times larger that way than with code - 8, which costs them less than three of 24 bits where y has 8 or 11).
// fp32 rows enter as three columns each, the bf16 parts of their 24 bits (8 bits each, exact), and codes as code - 8 (exact).
// For the types with fp32's range the codes enter as 2^-16 of that, and y is 2^16 of the sums: a group's sum is some hundred times larger than what
// its scale leaves of it, and would be infinite for rows near the type's largest number.
// (tcgen05 products want 128 rows of x or of W a step in shared memory, written there by the threads that unpack them: at a
// few columns the unpacking is the work, and a warp has its operand in registers already.)
//
// Layout of the codes: 2 KB for 16 rows and 256 k, as a warp reads them: 16 bytes for each lane 4 g + t (g < 8, t < 4) with row g and the first 128 k, 16 for
// each with row g + 8, and both again for the other 128 k; the 32-bit word j (j < 4) of them has k = 32 j + 8 t + {0 .. 7} of the 128, its bits
// 4 i .. 4 i + 3 k = 2 i of these eight, bits 16 + 4 i .. 2 i + 1.
// So a lane has eight adjacent k of each 32, the same as a 16-byte load of x gives it, and a shift and a mask leave two adjacent k in the halves
// of a register.
#include <algorithm>
#include <type_traits>
#include "common.cuh"
#include "decode_row.cuh"
#include "vec.cuh"

namespace castle {

constexpr int kL4Threads = 512, kL4Warps = kL4Threads / 32;
constexpr int kL4Tiles = 8;                                                 // 16 x 8 tiles that a warp leaves before they are added up
constexpr int kL4Smem = 220 * 1024;

struct Linear4Params {
  const void *x, *scales, *zeros;
  const uint4* codes;
  void* y;
  int64_t ldx;
  int rows, K, N, blocks;   // blocks of 256 k
  int shift, groups;        // log2(group / 32); groups of a row
  int kc, ks;               // CTAs of a cluster, which share K out; warps that share out a CTA's part of it
  int clusters, tiles;      // clusters; tiles of 16 weight rows
  int ldk;                  // elements between columns of x in shared memory
  bool vec;                 // rows of x can be read by 16 bytes
  int32_t* status;
  uint32_t mask, bits;      // CodeBits
};

template <typename T> struct CodeType { using type = T; static constexpr int parts = 1; };
template <> struct CodeType<float> { using type = __nv_bfloat16; static constexpr int parts = 3; };

// Codes 2 i and 2 i + 1 of the eight in a word as a pair of 16-bit numbers: `unit` times 16 + code for rows of 16 bits, code - 8 for the parts of fp32 ones.
// `mask` and `bits` are the kernel's arguments: with constants in their place the and and the or became an operation each, and moves of the constants.
template <typename T> struct CodeBits;
template <> struct CodeBits<__nv_bfloat16> {   // at: the top four of the mantissa's bits
  static constexpr int at = 3;
  static constexpr uint32_t mask = 0x00780078u, bits = 0x39803980u;
  static constexpr float unit = 1.f / 65536.f;
};
template <> struct CodeBits<__half> {
  static constexpr int at = 6;
  static constexpr uint32_t mask = 0x03c003c0u, bits = 0x4c004c00u;
  static constexpr float unit = 1.f;
};
template <> struct CodeBits<float> {           // 128 + code in bf16
  static constexpr int at = 0;
  static constexpr uint32_t mask = 0x000f000fu, bits = 0x3b003b00u;
  static constexpr float unit = 1.f / 65536.f;
};
template <typename T> __device__ __forceinline__ uint32_t code_pair(uint32_t w, int i, uint32_t mask, uint32_t bits) {
  const int right = 4 * i - CodeBits<T>::at;
  uint32_t v = right >= 0 ? w >> right : w << -right;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(v), "r"(mask), "r"(bits));   // v & mask | bits
  if constexpr (sizeof(T) == 4) {
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), __float2bfloat162_rn(136.f * CodeBits<T>::unit));
    v = *reinterpret_cast<const uint32_t*>(&d);
  }
  return v;
}

// The scales or zero points of a block's groups, as they lie.
template <typename T, int SPB> struct GroupRaw { uint32_t w[SPB * sizeof(T) > 4 ? SPB * sizeof(T) / 4 : 1]; };
// (volatile: they are to be on their way where they stand, blocks ahead of their use)
__device__ __forceinline__ uint32_t load_u16(const void* p) {
  uint16_t v;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t load_u32(const void* p) {
  uint32_t v;
  asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
template <typename T, int SPB, bool VEC>
__device__ __forceinline__ GroupRaw<T, SPB> load_group(const T* base, uint32_t row, int stretch, int shift, int groups) {   // stretch: the block's first 32 k
  GroupRaw<T, SPB> r;
  constexpr int bytes = SPB * sizeof(T);
  const T* at = base + (row + (stretch >> shift));
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < SPB; ++i) {
      const T* e = base + (row + min((stretch + i) >> shift, groups - 1));
      if constexpr (sizeof(T) == 4) r.w[i] = load_u32(e);
      else r.w[i / 2] = i % 2 ? r.w[i / 2] | load_u16(e) << 16 : load_u16(e);
    }
  } else if constexpr (SPB == 1) {
    r.w[0] = sizeof(T) == 2 ? load_u16(at) : load_u32(at);
  } else {
    if constexpr (bytes == 4) r.w[0] = load_u32(at);
    if constexpr (bytes == 8) asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "l"(at));
    if constexpr (bytes == 16) asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]) : "l"(at));
  }
  return r;
}
template <typename T, int SPB> __device__ __forceinline__ float group_value(const GroupRaw<T, SPB>& r, int i) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[i]);
  else {
    const float2 v = Elem<T>::unpack2(r.w[i / 2]);
    return i % 2 ? v.y : v.x;
  }
}

__device__ __forceinline__ uint4 load_stream(const uint4* p) {   // read once: not kept in the first-level cache, which the scales and zero points are for
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// Eight k of a column of x: a row's own values, or one of the three parts of fp32 ones.
template <typename T> __device__ __forceinline__ void stage8(const Linear4Params& p, int col, int k, float* v) {
  constexpr int parts = CodeType<T>::parts;
  const T* src = reinterpret_cast<const T*>(p.x) + (int64_t)(col / parts) * p.ldx + k;
  if (p.vec && k + 8 <= p.K) {
    load8<T>(src, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < p.K ? load1<T>(src + i) : 0.f;
  }
  if constexpr (parts == 3) {
    const int part = col % 3;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float rest = v[i];
      const float top = __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
      if (!(fabsf(rest) <= 3.4028235e38f)) { v[i] = part == 0 ? rest : 0.f; continue; }   // NaN and infinities are their first part
      rest -= top;
      const float mid = __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
      v[i] = part == 0 ? top : part == 1 ? mid : rest - mid;
    }
  }
}

// NT tiles of 8 columns; SPB groups in a block of 256 k (1: a group is a block or more), which a lane loads at once; not VEC: eight groups
// one by one, whatever their size and wherever they lie.
template <typename T, int NT, int SPB, bool VEC, bool ZEROS>
__global__ void __launch_bounds__(kL4Threads, 1) castle_linear_4bit_kernel(const __grid_constant__ Linear4Params p) {
  using E = typename CodeType<T>::type;
  constexpr int parts = CodeType<T>::parts, GM = kL4Tiles / NT;                // row tiles of a warp and batch
  constexpr int AHEAD = 2;                                                     // blocks of 256 k on their way; a whole number of turns is a batch
  static_assert(GM % AHEAD == 0, "a batch ends with a turn");
  constexpr bool SUMS = ZEROS || sizeof(T) == 2;
  constexpr int SPS = SPB < 2 ? 2 : SPB, SPAN = 8 / SPS;                       // sums of x in a block; stretches of 32 k that have them together
  extern __shared__ __align__(128) uint8_t raw[];
  __shared__ uint64_t bar;
  __shared__ int abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rank = p.kc > 1 ? (int)cluster_rank() : 0, cluster = blockIdx.x / p.kc;
  const int first = p.blocks * rank / p.kc, blocks = p.blocks * (rank + 1) / p.kc - first;   // this CTA's blocks
  const int cols = p.rows * parts;
  float* red = reinterpret_cast<float*>(raw);                                  // [warp][tile][16][8]
  E* xs = reinterpret_cast<E*>(raw + (size_t)kL4Warps * kL4Tiles * 128 * sizeof(float));   // [column][ldk]
  float* sums = reinterpret_cast<float*>(xs + (size_t)cols * p.ldk);           // [stretch][pair of columns][4]
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    mbar_fence_init();
    abort_flag = 0;
  }
  overlap_next();
  overlap_wait();
  __syncthreads();

  // ---- x, ahead of the codes in the queues: rows that lie as they are needed by bulk copies, others through the threads
  const int have = min(blocks * 256, p.K - first * 256);                       // k of this CTA that there are
  const bool bulk = parts == 1 && p.vec && p.K % 8 == 0;
  if (bulk && warp == 0) {
    if (lane == 0) mbar_expect_tx(&bar, cols * have * (uint32_t)sizeof(E));
    __syncwarp();
    if (lane < cols) bulk_g2s(xs + (int64_t)lane * p.ldk, reinterpret_cast<const T*>(p.x) + lane * p.ldx + first * 256, have * (uint32_t)sizeof(E), &bar);
  }

  // ---- this warp's walk: row tiles tile_begin + at_side, + side, ... of the cluster's, blocks [b0, b1) of each
  const int side = kL4Warps / p.ks, slice = warp % p.ks, at_side = warp / p.ks;
  const int b0 = first + blocks * slice / p.ks, b1 = first + blocks * (slice + 1) / p.ks;
  const int tile_begin = (int)((int64_t)p.tiles * cluster / p.clusters), tile_end = (int)((int64_t)p.tiles * (cluster + 1) / p.clusters);
  uint4 code[AHEAD][4];
  GroupRaw<T, SPB> scale[AHEAD][2], zero[ZEROS ? AHEAD : 1][2];
  // (offsets of 32 bits from the cluster's first row: addresses of 64 bits cost the loop as much as the codes' unpacking)
  const int nb = b1 - b0, tiles = tile_begin + at_side < tile_end ? (tile_end - tile_begin - at_side + side - 1) / side : 0;
  const uint4* code_base = p.codes + (int64_t)tile_begin * p.blocks * 128;
  const T* scale_base = reinterpret_cast<const T*>(p.scales) + (int64_t)tile_begin * 16 * p.groups;
  const T* zero_base = reinterpret_cast<const T*>(p.zeros) + (int64_t)tile_begin * 16 * p.groups;
  int to_fetch = tiles, next_block = b0, next_row = at_side * 16 + g;          // to_fetch: tiles that are not fetched to their end
  uint32_t code_at = (uint32_t)(at_side * p.blocks + b0) * 128 + lane, group0, group1;   // the next block's codes, its rows' first groups
  const uint32_t to_next = (uint32_t)(side * p.blocks - nb) * 128;
  const int last_row = p.N - 1 - tile_begin * 16;
  auto enter = [&]() {
    group0 = min(next_row, last_row) * p.groups;
    group1 = min(next_row + 8, last_row) * p.groups;
  };
  enter();
  auto fetch = [&](int s) {
    if (to_fetch == 0) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) code[s][i] = load_stream(code_base + code_at + 32 * i);
    scale[s][0] = load_group<T, SPB, VEC>(scale_base, group0, next_block * 8, p.shift, p.groups);
    scale[s][1] = load_group<T, SPB, VEC>(scale_base, group1, next_block * 8, p.shift, p.groups);
    if constexpr (ZEROS) {
      zero[s][0] = load_group<T, SPB, VEC>(zero_base, group0, next_block * 8, p.shift, p.groups);
      zero[s][1] = load_group<T, SPB, VEC>(zero_base, group1, next_block * 8, p.shift, p.groups);
    }
    code_at += 128;
    if (++next_block == b1) {
      next_block = b0;
      next_row += side * 16;
      code_at += to_next;
      --to_fetch;
      enter();
    }
  };
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) fetch(s);

  if (bulk) {
    const int rest = blocks * 256 - have;                                      // the last block's k that there are not
    for (int e = threadIdx.x; e < cols * rest; e += kL4Threads) xs[(int64_t)(e / rest) * p.ldk + have + e % rest] = Elem<E>::from_f(0.f);
    if (!mbar_wait_ok(&bar, 0, &abort_flag)) mbar_drain(&bar, 0);
  } else {
    const int eights = blocks * 32;
    for (int e = threadIdx.x; e < cols * eights; e += kL4Threads) {
      const int col = e / eights, k = e % eights * 8;
      float v[8];
      stage8<T>(p, col, first * 256 + k, v);
      store8<E>(xs + (int64_t)col * p.ldk + k, v);
    }
  }
  __syncthreads();
  if constexpr (SUMS) {   // eight lanes a stretch, in turn for its 32 or more k
    const int stretches = blocks * SPS, lane8 = threadIdx.x & 7;
    for (int e0 = 0; e0 < cols * stretches; e0 += kL4Threads / 8) {
      const int e = e0 + threadIdx.x / 8, col = e / stretches, k = e % stretches;
      float sum = 0.f;
      if (e < cols * stretches) {
#pragma unroll
        for (int i = 0; i < SPAN; i += 2) {                                    // 8 lanes x 8 k: 64 at a time
          if (SPAN > 1 || lane8 < 4) {
            float v[8];
            load8<E>(xs + (int64_t)col * p.ldk + (k * SPAN + i) * 32 + lane8 * 8, v);
#pragma unroll
            for (int q = 0; q < 8; ++q) sum = fmaf(v[q], CodeBits<T>::unit, sum);
          }
        }
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      // twice, as the sums of a lane's two rows begin with them; without zero points times -24, the codes' offset
      if (e < cols * stretches && lane8 == 0) {
        float* dst = sums + (k * NT * 4 + (col >> 1)) * 4 + (col & 1);
        dst[0] = dst[2] = ZEROS ? sum : -24.f * sum;
      }
    }
    __syncthreads();
  }

  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[i][q] = 0.f;
  const E* column[NT];   // (columns that there are not repeat the last one; nobody reads their results)
#pragma unroll
  for (int i = 0; i < NT; ++i) column[i] = xs + (int64_t)min(i * 8 + g, cols - 1) * p.ldk + 8 * t;
  const int x0 = (b0 - first) * 256, sum0 = (b0 - first) * SPS * NT * 16 + 4 * t;
  int left = nb, x_at = x0, sum_at = sum0;
  for (int batch = tile_begin; batch < tile_end; batch += side * GM) {
    const int batch_end = min(batch + side * GM, tile_end);
    const int mine = batch + at_side < batch_end ? (batch_end - batch - at_side + side - 1) / side : 0;   // row tiles of this warp
    float* dst = red + (size_t)warp * GM * NT * 128 + g * 8 + 2 * t;
    for (int u = mine * nb; u > 0; u -= AHEAD) {
#pragma unroll
      for (int s = 0; s < AHEAD; ++s) {
        if (s >= u) break;
        // The block's halves of 128 k have sums of their own, which are formed side by side where there is one tile of columns: a product waits
        // for the one before into the same sums.
        float c[2][NT][4];
        auto begin = [&](int h, int span) {   // the sums of half h for the group with stretch `span` of the sums of x
          constexpr int per = SPS / (SPB < SPS ? SPB : SPS);
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            if constexpr (SUMS) {
              const float4 sum = *reinterpret_cast<const float4*>(sums + sum_at + span * NT * 16 + i * 16);
              if constexpr (ZEROS) {
                constexpr float offset = sizeof(T) == 2 ? -16.f : 8.f;
                const float z0 = offset - group_value<T, SPB>(zero[s][0], span / per), z1 = offset - group_value<T, SPB>(zero[s][1], span / per);
                c[h][i][0] = z0 * sum.x; c[h][i][1] = z0 * sum.y; c[h][i][2] = z1 * sum.z; c[h][i][3] = z1 * sum.w;
              } else {
                c[h][i][0] = sum.x; c[h][i][1] = sum.y; c[h][i][2] = sum.z; c[h][i][3] = sum.w;
              }
            } else {
#pragma unroll
              for (int q = 0; q < 4; ++q) c[h][i][q] = 0.f;
            }
          }
        };
        auto end = [&](int h, int span) {
          constexpr int per = SPS / (SPB < SPS ? SPB : SPS);
          const float f0 = group_value<T, SPB>(scale[s][0], span / per), f1 = group_value<T, SPB>(scale[s][1], span / per);
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            acc[i][0] = fmaf(f0, c[h][i][0], acc[i][0]); acc[i][1] = fmaf(f0, c[h][i][1], acc[i][1]);
            acc[i][2] = fmaf(f1, c[h][i][2], acc[i][2]); acc[i][3] = fmaf(f1, c[h][i][3], acc[i][3]);
          }
        };
        auto unpack = [&](int h, int j, uint32_t (*a)[4]) {
          const uint4 lo = code[s][2 * h], hi = code[s][2 * h + 1];
          const uint32_t wl = j == 0 ? lo.x : j == 1 ? lo.y : j == 2 ? lo.z : lo.w, wh = j == 0 ? hi.x : j == 1 ? hi.y : j == 2 ? hi.z : hi.w;
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            a[m][0] = code_pair<T>(wl, 2 * m, p.mask, p.bits);
            a[m][1] = code_pair<T>(wh, 2 * m, p.mask, p.bits);
            a[m][2] = code_pair<T>(wl, 2 * m + 1, p.mask, p.bits);
            a[m][3] = code_pair<T>(wh, 2 * m + 1, p.mask, p.bits);
          }
        };
        if constexpr (NT == 1) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j % SPAN == 0) { begin(0, j / SPAN); begin(1, (4 + j) / SPAN); }
            uint32_t a[2][2][4];
            unpack(0, j, a[0]);
            unpack(1, j, a[1]);
            const uint4 x0 = *reinterpret_cast<const uint4*>(column[0] + x_at + 32 * j), x1 = *reinterpret_cast<const uint4*>(column[0] + x_at + 128 + 32 * j);
            mma_16x8x16<E>(c[0][0], a[0][0], x0.x, x0.y);
            mma_16x8x16<E>(c[1][0], a[1][0], x1.x, x1.y);
            mma_16x8x16<E>(c[0][0], a[0][1], x0.z, x0.w);
            mma_16x8x16<E>(c[1][0], a[1][1], x1.z, x1.w);
            if (j % SPAN == SPAN - 1) { end(0, j / SPAN); end(1, (4 + j) / SPAN); }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (j % SPAN == 0) begin(0, j / SPAN);
            uint32_t a[2][4];
            unpack(j / 4, j % 4, a);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              const uint4 b = *reinterpret_cast<const uint4*>(column[i] + x_at + 32 * j);
              mma_16x8x16<E>(c[0][i], a[0], b.x, b.y);
              mma_16x8x16<E>(c[0][i], a[1], b.z, b.w);
            }
            if (j % SPAN == SPAN - 1) end(0, j / SPAN);
          }
        }
        fetch(s);
        x_at += 256;
        sum_at += SPS * NT * 16;
        if (--left == 0) {
          left = nb; x_at = x0; sum_at = sum0;
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            *reinterpret_cast<float2*>(dst + i * 128) = make_float2(acc[i][0], acc[i][1]);
            *reinterpret_cast<float2*>(dst + i * 128 + 64) = make_float2(acc[i][2], acc[i][3]);
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[i][q] = 0.f;
          }
          dst += NT * 128;
        }
      }
    }
    if (p.kc > 1) cluster_sync(); else __syncthreads();
    // ---- the warps' and CTAs' shares of K, in order
    const int count = (batch_end - batch) * 16 * p.rows;
    for (int e = threadIdx.x * p.kc + rank; e < count; e += kL4Threads * p.kc) {
      const int row = e & 15, rest = e >> 4, tile = rest / p.rows, token = rest - tile * p.rows;
      const int n = (batch + tile) * 16 + row;
      float sum = 0.f;
#pragma unroll
      for (int q = 0; q < parts; ++q) {
        const int col = token * parts + q;
        const float* src = red + ((size_t)(tile % side * p.ks * GM + tile / side) * NT + col / 8) * 128 + row * 8 + col % 8;
        for (int r = 0; r < p.kc; ++r) {
#pragma unroll 4
          for (int w = 0; w < p.ks; ++w) sum += p.kc > 1 ? cluster_load(src + w * GM * NT * 128, r) : src[w * GM * NT * 128];
        }
      }
      if (n < p.N) store1<T>(reinterpret_cast<T*>(p.y) + (int64_t)token * p.N + n, sum * (1.f / CodeBits<T>::unit));
    }
    if (p.kc > 1) cluster_sync(); else __syncthreads();
  }
  if (threadIdx.x == 0 && abort_flag) atomicOr(p.status, CASTLE_STATUS_WAIT_TIMEOUT);
}

// The weights at full width, in the rows' type (rounded once): for the products of many fp32 rows and for the gradient of x.  A warp has 4 rows and 128 k, two words a
// thread, so that a store is 128 (fp32: 256) adjacent bytes of each row.  4096 x 4096 in us, bf16 and fp32: 15.2, 23.5 (the bytes take 6.4 and 11.6); a word a
// thread along a row 15.8, 27.2; 16 bytes of codes a thread, 64 bytes of a row at once, 15.7, 27.0, more of them a thread 17.2, 26.5.  What bounds it now: the
// first-level cache, at 87 % (4096 x 16384 bf16; the stores, and a scale for each row of a warp), with HBM at 34 % of the copy's rate.
template <typename T, bool ZEROS> __global__ void __launch_bounds__(256) castle_expand_4bit_kernel(const Linear4Params p, int64_t ldw) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = (warp & 1) * 4 + (lane >> 3), h = lane >> 2 & 1, t = lane & 3;
  const int part = blockIdx.y * 4 + (warp >> 1);   // of 128 k
  const int64_t n = (int64_t)blockIdx.x * 8 + g;
  if (n >= p.N || part * 128 >= p.K) return;
  const uint32_t* src = reinterpret_cast<const uint32_t*>(p.codes + (((n >> 4) * p.blocks * 2 + part) * 2 + (n >> 3 & 1)) * 32 + g * 4 + t);
  uint32_t w[2];
  float s[2], z[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = 2 * u + h;
    w[u] = __ldg(src + j);
    const int64_t at = n * p.groups + min((part * 4 + j) >> p.shift, p.groups - 1);
    s[u] = load1<T>(reinterpret_cast<const T*>(p.scales) + at);
    z[u] = ZEROS ? load1<T>(reinterpret_cast<const T*>(p.zeros) + at) : 8.f;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int k0 = part * 128 + (2 * u + h) * 32 + t * 8;
    if (k0 >= p.K) break;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {   // 2^23 + code, less 2^23
      const float code = __uint_as_float((w[u] >> (4 * (i >> 1) + 16 * (i & 1)) & 15u) | 0x4b000000u) - 8388608.f;
      v[i] = s[u] * (code - z[u]);
    }
    T* dst = reinterpret_cast<T*>(p.y) + n * ldw + k0;
    if (k0 + 8 <= p.K) {
      store8<T>(dst, v);
    } else {
      for (int i = 0; k0 + i < p.K; ++i) store1<T>(dst + i, v[i]);
    }
  }
}

// How K is shared out: the longest walk of a warp decides, its blocks and a fifth of one for each row tile that it begins and leaves (us with 16 / 8 /
// 4 warps to a tile, bf16: 1 x 4096 -> 4096 5.5 / 5.3 / 6.1, 8 x 4096 -> 16384 13.6 / 14.7 / 13.1, 1 x 8192 -> 32768 34.4 / 33.2 / 34.7, 1 x 16384 -> 1024 6.6 / 12.5 /
// 12.3).  Two CTAs of eight warps on an SM instead of one of sixteen: the same within 5 %.
static bool linear_4bit_plan(Linear4Params& p, int cols, size_t& smem) {
  int64_t best = -1;
  for (int kc = 1; kc <= 8 && kc <= p.blocks; kc *= 2) {
    const int most = (p.blocks + kc - 1) / kc, least = p.blocks / kc, ldk = most * 256 + 32;   // (columns 64 bytes apart in the banks)
    const size_t bytes = (size_t)kL4Warps * kL4Tiles * 128 * sizeof(float) + (size_t)cols * ldk * 2 + (size_t)most * 8 * (cols <= 8 ? 16 : cols <= 16 ? 32 : 64) * sizeof(float);
    if (bytes > kL4Smem) continue;
    const int clusters = std::min(p.tiles, kc == 8 ? 15 : kc == 4 ? 36 : 148 / kc), per = (p.tiles + clusters - 1) / clusters;
    for (int ks = 16; ks >= 1; ks /= 2) {
      if (ks > least) continue;   // (every warp has a block)
      const int side = kL4Warps / ks;
      const int64_t walk = (int64_t)((per + side - 1) / side) * (10 * ((most + ks - 1) / ks) + 2);
      // larger clusters end with a barrier of theirs and loads from each other: for a tenth and more
      if (best < 0 || walk * 10 < best * (kc > p.kc ? 9 : 10)) {
        best = walk;
        p.kc = kc; p.ks = ks; p.clusters = clusters; p.ldk = ldk;
        smem = bytes;
      }
    }
  }
  return best >= 0;
}

template <typename T, int NT, int SPB, bool VEC, bool ZEROS> static int launch_linear_4bit(const Linear4Params& p, size_t smem, cudaStream_t st) {
  auto kernel = castle_linear_4bit_kernel<T, NT, SPB, VEC, ZEROS>;
  Linear4Params q = p;
  q.mask = CodeBits<T>::mask;
  q.bits = CodeBits<T>::bits;
  cudaError_t e = allow_smem(kernel, kL4Smem);
  if (e != cudaSuccess) return cuda_fail(e, "castle_linear_4bit attribute");
  cudaLaunchConfig_t c = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)p.kc, 1, 1};
  c.gridDim = dim3(p.clusters * p.kc); c.blockDim = dim3(kL4Threads); c.dynamicSmemBytes = smem; c.stream = st;
  c.attrs = attr; c.numAttrs = p.kc > 1 ? 2 : 1;
  e = cudaLaunchKernelEx(&c, kernel, q);
  return e == cudaSuccess ? 0 : cuda_fail(e, "castle_linear_4bit launch");
}
template <typename T, int NT> static int launch_linear_4bit_nt(const Linear4Params& p, size_t smem, cudaStream_t st) {
  const int per_block = p.shift >= 3 ? 1 : 8 >> p.shift;
  // the groups of a block at once: a multiple of their number in a row, at their alignment (16 bytes is a load's most)
  const bool vec = p.groups % per_block == 0 && ((uintptr_t)p.scales | (uintptr_t)p.zeros) % (per_block * sizeof(T)) == 0;
  auto by_group = [&](auto zeros) {
    constexpr bool Z = decltype(zeros)::value;
    if (sizeof(T) == 4 && per_block == 8 && vec) return launch_linear_4bit<T, NT, 8, false, Z>(p, smem, st);
    return !vec ? launch_linear_4bit<T, NT, 8, false, Z>(p, smem, st) : per_block == 8 ? launch_linear_4bit<T, NT, 8, sizeof(T) == 2, Z>(p, smem, st)
           : per_block == 4 ? launch_linear_4bit<T, NT, 4, true, Z>(p, smem, st) : per_block == 2 ? launch_linear_4bit<T, NT, 2, true, Z>(p, smem, st) : launch_linear_4bit<T, NT, 1, true, Z>(p, smem, st);
  };
  return p.zeros ? by_group(std::true_type()) : by_group(std::false_type());
}
template <typename T> static int launch_linear_4bit_t(const Linear4Params& p, int cols, size_t smem, cudaStream_t st) {
  return cols <= 8 ? launch_linear_4bit_nt<T, 1>(p, smem, st) : cols <= 16 ? launch_linear_4bit_nt<T, 2>(p, smem, st) : launch_linear_4bit_nt<T, 4>(p, smem, st);
}

static int linear_4bit_check(const char* who, int32_t dtype, int32_t in_features, int64_t out_features, int32_t group, const void* codes, const void* scales, const void* zeros,
                             Linear4Params& p) {
  if (dtype < CASTLE_BF16 || dtype > CASTLE_F32) return reject("%s: unknown dtype %d", who, dtype);
  if (in_features <= 0 || in_features > (1 << 24) || out_features <= 0 || out_features > INT32_MAX / 2) return reject("%s: %d -> %lld not supported", who, in_features, (long long)out_features);
  if (group < 32 || group > (1 << 24) || (group & (group - 1))) return reject("%s: group size %d is not a power of two from 32 up", who, group);
  if (!codes || !scales) return reject("%s: null codes or scales", who);
  if ((uintptr_t)codes % 16 || ((uintptr_t)scales | (uintptr_t)zeros) % elem_size(dtype)) return reject("%s: the codes must be 16-byte aligned, scales and zero points aligned to their type", who);
  p.K = in_features; p.N = (int)out_features; p.blocks = (in_features + 255) / 256;
  p.groups = (in_features + group - 1) / group;
  p.shift = 0;
  while ((32 << p.shift) < group) ++p.shift;
  p.tiles = (p.N + 15) / 16;
  p.codes = static_cast<const uint4*>(codes); p.scales = scales; p.zeros = zeros;
  return 0;
}

}  // namespace castle

using namespace castle;

extern "C" int castle_linear_4bit_fits(int32_t dtype, int32_t rows, int32_t in_features) {
  const int parts = dtype == CASTLE_F32 ? 3 : 1;
  if (dtype < CASTLE_BF16 || dtype > CASTLE_F32 || rows < 1 || rows > 32 / parts || in_features <= 0 || in_features > (1 << 24)) return 0;
  Linear4Params p = {};
  p.blocks = (in_features + 255) / 256; p.tiles = 148;
  size_t smem = 0;
  return linear_4bit_plan(p, rows * parts, smem) ? 1 : 0;
}

extern "C" int castle_linear_4bit(int32_t dtype, int32_t rows, int32_t in_features, int64_t out_features, int32_t group, const void* x, int64_t row_stride,
                                  const void* codes, const void* scales, const void* zeros, void* y, int32_t* status, void* stream) {
  const char* who = "castle_linear_4bit";
  Linear4Params p = {};
  if (const int rc = linear_4bit_check(who, dtype, in_features, out_features, group, codes, scales, zeros, p)) return rc;
  if (!castle_linear_4bit_fits(dtype, rows, in_features)) return reject("%s: %d rows of %d not supported (see castle_linear_4bit_fits)", who, rows, in_features);
  if (!x || !y || ((uintptr_t)x | (uintptr_t)y) % elem_size(dtype)) return reject("%s: null rows or results, or not aligned to their type", who);
  if (row_stride < 0) return reject("%s: negative row stride", who);
  if (!status || (uintptr_t)status % 4) return reject("%s: null status, or not aligned", who);
  p.x = x; p.y = y; p.rows = rows; p.ldx = row_stride;
  p.vec = (uintptr_t)x % 16 == 0 && (rows == 1 || row_stride * elem_size(dtype) % 16 == 0);
  p.status = status;
  const int cols = rows * (dtype == CASTLE_F32 ? 3 : 1);
  size_t smem = 0;
  if (!linear_4bit_plan(p, cols, smem)) return reject("%s: %d rows of %d not supported", who, rows, in_features);
  const cudaStream_t st = (cudaStream_t)stream;
  if (dtype == CASTLE_BF16) return launch_linear_4bit_t<__nv_bfloat16>(p, cols, smem, st);
  if (dtype == CASTLE_F16) return launch_linear_4bit_t<__half>(p, cols, smem, st);
  return launch_linear_4bit_t<float>(p, cols, smem, st);
}

extern "C" int castle_expand_4bit(int32_t dtype, int32_t in_features, int64_t out_features, int32_t group, const void* codes, const void* scales, const void* zeros, void* w,
                                  int64_t row_stride, void* stream) {
  const char* who = "castle_expand_4bit";
  Linear4Params p = {};
  if (const int rc = linear_4bit_check(who, dtype, in_features, out_features, group, codes, scales, zeros, p)) return rc;
  if (!w || (uintptr_t)w % 16 || row_stride < in_features || row_stride * elem_size(dtype) % 16) return reject("%s: the weights must be 16-byte aligned, rows of a multiple of 16 bytes", who);
  p.y = w;
  const dim3 grid((unsigned)((p.N + 7) / 8), (unsigned)((p.K + 511) / 512));
  cudaError_t e = by_type(dtype, [&](auto v) {
    using T = decltype(v);
    return zeros ? launch_kernel(castle_expand_4bit_kernel<T, true>, grid, 256, 0, (cudaStream_t)stream, false, p, row_stride)
                 : launch_kernel(castle_expand_4bit_kernel<T, false>, grid, 256, 0, (cudaStream_t)stream, false, p, row_stride);
  });
  return e == cudaSuccess ? 0 : cuda_fail(e, "castle_expand_4bit launch");
}
