// y = x W^T with weights of 4 bits, for the rows of a few tokens:
//
//     W[n, k] = scale[n, k / group] * (code[n, k] - zero[n, k / group])       zero = 8 where there are no zero points
//
// The product is a stream over the codes (half a byte per weight), so it is bound by HBM, and for small weights by a launch's latencies.
// It is computed with mma.sync: 16 weight rows are the first operand, 8 columns of x the second.  The codes enter as code - 8, which
// both 16-bit types hold exactly, the sums of a group are fp32, and scales and zero points are applied to those sums:
//     y[n] = sum over groups of  scale * (sum of (code - 8) x  +  (8 - zero) * sum of x)
// so nothing but x and y is rounded to 16 bits.  fp32 rows enter as three columns each, the bf16 parts of their 24 bits (8 bits each, exact).
// (tcgen05 products want 128 rows of x or of W a step in shared memory, written there by the threads that unpack them: at a
// few columns the unpacking is the work, and a warp has its operand in registers already.)
//
// Layout of the codes: 64 bytes for 128 k of a row, word 4 t + j (t, j < 4) has k = 32 j + 8 t + {0 .. 7}; bits 4 i .. 4 i + 3 of it are
// k = 2 i of these eight, bits 16 + 4 i .. are 2 i + 1.  So a lane of a quad loads 16 bytes, has eight adjacent k of each 32, the same as a
// 16-byte load of x gives it, and a shift and a mask leave two adjacent k in the halves of a register.
#include <algorithm>
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
  int rows, K, N, blocks;   // blocks of 128 k
  int shift, groups;        // log2(group / 32); groups of a row
  int kc, ks;               // CTAs of a cluster, which share K out; warps that share out a CTA's part of it
  int clusters, tiles;      // clusters; tiles of 16 weight rows
  int ldk;                  // elements between columns of x in shared memory
  bool vec;                 // rows of x can be read by 16 bytes
};

template <typename T> struct CodeType { using type = T; static constexpr int parts = 1; };
template <> struct CodeType<float> { using type = __nv_bfloat16; static constexpr int parts = 3; };

// Two adjacent codes less eight: the low bits of 1024 (fp16) and 128 (bf16) are ones.
template <typename E> __device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  uint32_t r;
  if constexpr (Elem<E>::fmt == 1) {
    const uint32_t v = (w & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), __float2bfloat162_rn(136.f));
    r = *reinterpret_cast<const uint32_t*>(&d);
  } else {
    const uint32_t v = (w & 0x000f000fu) | 0x64006400u;
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&v), __float2half2_rn(1032.f));
    r = *reinterpret_cast<const uint32_t*>(&d);
  }
  return r;
}

__device__ __forceinline__ uint4 load_stream(const uint4* p) {   // read once: not kept in the first-level cache, which the scales and zero points are for
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ float cluster_load(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(of_cta(p, rank)) : "memory");
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

// NT tiles of 8 columns; SPB groups in a block of 128 k (1: a group is a block or more).
template <typename T, int NT, int SPB, bool ZEROS>
__global__ void __launch_bounds__(kL4Threads, 1) castle_linear_4bit_kernel(const Linear4Params p) {
  using E = typename CodeType<T>::type;
  constexpr int parts = CodeType<T>::parts, GM = kL4Tiles / NT;                // row tiles of a warp and batch
  constexpr int AHEAD = GM < 4 ? GM : 4;                                       // blocks of 128 k on their way; a whole number of turns is a batch
  extern __shared__ __align__(16) uint8_t raw[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rank = p.kc > 1 ? (int)cluster_rank() : 0, cluster = blockIdx.x / p.kc;
  const int first = p.blocks * rank / p.kc, blocks = p.blocks * (rank + 1) / p.kc - first;   // this CTA's blocks
  const int cols = p.rows * parts;
  float* red = reinterpret_cast<float*>(raw);                                  // [warp][tile][16][8]
  E* xs = reinterpret_cast<E*>(raw + (size_t)kL4Warps * kL4Tiles * 128 * sizeof(float));   // [column][ldk]
  float* sums = reinterpret_cast<float*>(xs + (size_t)cols * p.ldk);           // [32 k][column], with zero points
  overlap_next();
  overlap_wait();

  // ---- this warp's walk: row tiles tile0, tile0 + step, ... of the cluster's, blocks [b0, b1) of each
  const int side = kL4Warps / p.ks, slice = warp % p.ks, at_side = warp / p.ks;
  const int b0 = first + blocks * slice / p.ks, b1 = first + blocks * (slice + 1) / p.ks;
  const int tile_begin = (int)((int64_t)p.tiles * cluster / p.clusters), tile_end = (int)((int64_t)p.tiles * (cluster + 1) / p.clusters);
  uint4 code[AHEAD][2];
  T scale[AHEAD][SPB][2], zero[ZEROS ? AHEAD : 1][SPB][2];
  int next_tile = tile_begin + at_side, next_block = b0;
  auto fetch = [&](int s) {
    if (next_tile >= tile_end || b0 >= b1) return;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t n = min(next_tile * 16 + g + 8 * r, p.N - 1);
      code[s][r] = load_stream(p.codes + (n * p.blocks + next_block) * 4 + t);
#pragma unroll
      for (int i = 0; i < SPB; ++i) {
        const int64_t at = n * p.groups + min((next_block * 4 + i * (4 / SPB)) >> p.shift, p.groups - 1);
        scale[s][i][r] = reinterpret_cast<const T*>(p.scales)[at];
        if constexpr (ZEROS) zero[s][i][r] = reinterpret_cast<const T*>(p.zeros)[at];
      }
    }
    if (++next_block == b1) { next_block = b0; next_tile += side; }
  };
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) fetch(s);

  // ---- x into shared memory
  const int eights = blocks * 16;
  for (int e = threadIdx.x; e < cols * eights; e += kL4Threads) {
    const int col = e / eights, k = e % eights * 8;
    float v[8];
    stage8<T>(p, col, first * 128 + k, v);
    store8<E>(xs + (int64_t)col * p.ldk + k, v);
  }
  __syncthreads();
  if constexpr (ZEROS) {
    for (int e = threadIdx.x; e < cols * blocks * 4; e += kL4Threads) {
      const int col = e % cols, k = e / cols;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v[8];
        load8<E>(xs + (int64_t)col * p.ldk + k * 32 + i * 8, v);
#pragma unroll
        for (int q = 0; q < 8; ++q) sum += v[q];
      }
      sums[k * NT * 8 + col] = sum;
    }
    __syncthreads();
  }

  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[i][q] = 0.f;
  for (int batch = tile_begin; batch < tile_end; batch += side * GM) {
    const int batch_end = min(batch + side * GM, tile_end);
    const int mine = b0 < b1 && batch + at_side < batch_end ? (batch_end - batch - at_side + side - 1) / side : 0;   // row tiles of this warp
    int block = b0, nth = 0;
    for (int u = mine * (b1 - b0); u > 0; u -= AHEAD) {
#pragma unroll
      for (int s = 0; s < AHEAD; ++s) {
        if (s >= u) break;
        const uint4 lo = code[s][0], hi = code[s][1];
        float sc[SPB][2], ze[SPB][2];
#pragma unroll
        for (int i = 0; i < SPB; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            sc[i][r] = load1<T>(&scale[s][i][r]);
            if constexpr (ZEROS) ze[i][r] = 8.f - load1<T>(&zero[s][i][r]);
          }
        fetch(s);
        const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
        const int kb = (block - first) * 128;
        float c[NT][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j % (4 / SPB) == 0) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
              for (int q = 0; q < 4; ++q) c[i][q] = 0.f;
          }
          uint32_t a[2][4];
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            a[m][0] = code_pair<E>(wl[j] >> (8 * m));
            a[m][1] = code_pair<E>(wh[j] >> (8 * m));
            a[m][2] = code_pair<E>(wl[j] >> (8 * m + 4));
            a[m][3] = code_pair<E>(wh[j] >> (8 * m + 4));
          }
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            uint4 b = make_uint4(0, 0, 0, 0);
            if (i * 8 + g < cols) b = *reinterpret_cast<const uint4*>(xs + (int64_t)(i * 8 + g) * p.ldk + kb + 32 * j + 8 * t);
            mma_16x8x16<E>(c[i], a[0], b.x, b.y);
            mma_16x8x16<E>(c[i], a[1], b.z, b.w);
          }
          if constexpr (ZEROS) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              const float2 sum = *reinterpret_cast<const float2*>(sums + ((kb >> 5) + j) * NT * 8 + i * 8 + 2 * t);
              const float* z = ze[j / (4 / SPB)];
              c[i][0] = fmaf(z[0], sum.x, c[i][0]); c[i][1] = fmaf(z[0], sum.y, c[i][1]);
              c[i][2] = fmaf(z[1], sum.x, c[i][2]); c[i][3] = fmaf(z[1], sum.y, c[i][3]);
            }
          }
          if (j % (4 / SPB) == 4 / SPB - 1) {
            const float* f = sc[j / (4 / SPB)];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              acc[i][0] = fmaf(f[0], c[i][0], acc[i][0]); acc[i][1] = fmaf(f[0], c[i][1], acc[i][1]);
              acc[i][2] = fmaf(f[1], c[i][2], acc[i][2]); acc[i][3] = fmaf(f[1], c[i][3], acc[i][3]);
            }
          }
        }
        if (++block == b1) {
          block = b0;
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            float* dst = red + ((size_t)(warp * GM + nth) * NT + i) * 128;
            *reinterpret_cast<float2*>(dst + g * 8 + 2 * t) = make_float2(acc[i][0], acc[i][1]);
            *reinterpret_cast<float2*>(dst + (g + 8) * 8 + 2 * t) = make_float2(acc[i][2], acc[i][3]);
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[i][q] = 0.f;
          }
          ++nth;
        }
      }
    }
    if (p.kc > 1) cluster_sync(); else __syncthreads();
    // ---- the warps' and CTAs' shares of K, in order
    const int count = (batch_end - batch) * 16 * p.rows;
    for (int e = threadIdx.x * p.kc + rank; e < count; e += kL4Threads * p.kc) {
      const int row = e % 16, token = e / 16 % p.rows, tile = e / (16 * p.rows);
      const int n = (batch + tile) * 16 + row;
      float sum = 0.f;
      for (int r = 0; r < p.kc; ++r) {
        const int have = p.blocks * (r + 1) / p.kc - p.blocks * r / p.kc;
        for (int w = 0; w < p.ks; ++w) {
          if (have * w / p.ks == have * (w + 1) / p.ks) continue;   // a warp without blocks
#pragma unroll
          for (int q = 0; q < parts; ++q) {
            const int col = token * parts + q;
            const float* src = red + ((size_t)((tile % side * p.ks + w) * GM + tile / side) * NT + col / 8) * 128 + row * 8 + col % 8;
            sum += p.kc > 1 ? cluster_load(src, r) : *src;
          }
        }
      }
      if (n < p.N) store1<T>(reinterpret_cast<T*>(p.y) + (int64_t)token * p.N + n, sum);
    }
    if (p.kc > 1) cluster_sync(); else __syncthreads();
  }
}

// The weights at full width, in the rows' type (rounded once): for the products of many rows and for the gradient of x.
template <typename T, bool ZEROS> __global__ void __launch_bounds__(256) castle_expand_4bit_kernel(const Linear4Params p, int64_t ldw) {
  const int words = p.blocks * 16;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < (int64_t)p.N * words; e += (int64_t)gridDim.x * 256) {
    const int64_t n = e / words;
    const int word = (int)(e % words), k0 = word / 16 * 128 + (word % 4) * 32 + word % 16 / 4 * 8;
    if (k0 >= p.K) continue;
    const uint32_t w = reinterpret_cast<const uint32_t*>(p.codes)[e];
    const int64_t at = n * p.groups + (k0 / 32 >> p.shift);
    const float s = load1<T>(reinterpret_cast<const T*>(p.scales) + at), z = ZEROS ? load1<T>(reinterpret_cast<const T*>(p.zeros) + at) : 8.f;
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = s * ((float)(w >> (4 * i) & 15u) - z);
      v[2 * i + 1] = s * ((float)(w >> (4 * i + 16) & 15u) - z);
    }
    T* dst = reinterpret_cast<T*>(p.y) + n * ldw + k0;
    if (k0 + 8 <= p.K) {
      store8<T>(dst, v);
    } else {
      for (int i = 0; k0 + i < p.K; ++i) store1<T>(dst + i, v[i]);
    }
  }
}

// How K is shared out: the largest number of blocks that a warp walks through decides.
static bool linear_4bit_plan(Linear4Params& p, int cols, size_t& smem) {
  int64_t best = -1;
  for (int kc = 1; kc <= 8 && kc <= p.blocks; kc *= 2) {
    const int most = (p.blocks + kc - 1) / kc, ldk = most * 128 + 32;   // (columns 64 bytes apart in the banks)
    const size_t bytes = (size_t)kL4Warps * kL4Tiles * 128 * sizeof(float) + (size_t)cols * ldk * 2 + (p.zeros ? (size_t)most * 4 * (cols <= 8 ? 8 : cols <= 16 ? 16 : 32) * sizeof(float) : 0);
    if (bytes > kL4Smem) continue;
    const int clusters = std::min(p.tiles, kc == 8 ? 15 : kc == 4 ? 36 : 148 / kc), per = (p.tiles + clusters - 1) / clusters;
    for (int ks = 16; ks >= 1; ks /= 2) {
      if (ks > most) continue;
      const int side = kL4Warps / ks;
      const int64_t walk = (int64_t)((per + side - 1) / side) * ((most + ks - 1) / ks);
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

template <typename T, int NT, int SPB, bool ZEROS> static int launch_linear_4bit(const Linear4Params& p, size_t smem, cudaStream_t st) {
  auto kernel = castle_linear_4bit_kernel<T, NT, SPB, ZEROS>;
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
  e = cudaLaunchKernelEx(&c, kernel, p);
  return e == cudaSuccess ? 0 : cuda_fail(e, "castle_linear_4bit launch");
}
template <typename T, int NT> static int launch_linear_4bit_nt(const Linear4Params& p, size_t smem, cudaStream_t st) {
  if (p.zeros) return p.shift == 0 ? launch_linear_4bit<T, NT, 4, true>(p, smem, st) : p.shift == 1 ? launch_linear_4bit<T, NT, 2, true>(p, smem, st) : launch_linear_4bit<T, NT, 1, true>(p, smem, st);
  return p.shift == 0 ? launch_linear_4bit<T, NT, 4, false>(p, smem, st) : p.shift == 1 ? launch_linear_4bit<T, NT, 2, false>(p, smem, st) : launch_linear_4bit<T, NT, 1, false>(p, smem, st);
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
  p.K = in_features; p.N = (int)out_features; p.blocks = (in_features + 127) / 128;
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
  p.blocks = (in_features + 127) / 128; p.tiles = 148; p.zeros = &p;   // (with zero points it needs more)
  size_t smem = 0;
  return linear_4bit_plan(p, rows * parts, smem) ? 1 : 0;
}

extern "C" int castle_linear_4bit(int32_t dtype, int32_t rows, int32_t in_features, int64_t out_features, int32_t group, const void* x, int64_t row_stride,
                                  const void* codes, const void* scales, const void* zeros, void* y, void* stream) {
  const char* who = "castle_linear_4bit";
  Linear4Params p = {};
  if (const int rc = linear_4bit_check(who, dtype, in_features, out_features, group, codes, scales, zeros, p)) return rc;
  if (!castle_linear_4bit_fits(dtype, rows, in_features)) return reject("%s: %d rows of %d not supported (see castle_linear_4bit_fits)", who, rows, in_features);
  if (!x || !y || ((uintptr_t)x | (uintptr_t)y) % elem_size(dtype)) return reject("%s: null rows or results, or not aligned to their type", who);
  if (row_stride < 0) return reject("%s: negative row stride", who);
  p.x = x; p.y = y; p.rows = rows; p.ldx = row_stride;
  p.vec = (uintptr_t)x % 16 == 0 && (rows == 1 || row_stride * elem_size(dtype) % 16 == 0);
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
  const int64_t words = (int64_t)p.N * p.blocks * 16;
  const int ctas = (int)std::min<int64_t>((words + 255) / 256, 148 * 16);
  cudaError_t e = by_type(dtype, [&](auto v) {
    using T = decltype(v);
    return zeros ? launch_kernel(castle_expand_4bit_kernel<T, true>, dim3(ctas), 256, 0, (cudaStream_t)stream, false, p, row_stride)
                 : launch_kernel(castle_expand_4bit_kernel<T, false>, dim3(ctas), 256, 0, (cudaStream_t)stream, false, p, row_stride);
  });
  return e == cudaSuccess ? 0 : cuda_fail(e, "castle_expand_4bit launch");
}
