// Matrix-vector products with 4-bit weights and group scales (the client's
// head on the last decrypted token, and projections of a few rows).
//
//   y[b][n] = sum_g s[n][g] sum_{k in group g} (code[n][k] - z[n][g]) x[b][k],
// codes 0..15, z = 8 or stored per group.  Bytes bound: N K / 2 bytes of codes
// are read once for all rows.
//
// The products run on mma.sync m16n8k16 with 16 weight rows as M and up to 8
// rows of x as N: a difference code - z is a small integer, exact in bf16 and
// fp16, so the tensor cores form the integer-times-x sums of a group in
// binary32 and one multiply-add per group and output applies the scale.  A
// nibble becomes a number by placing it in the low mantissa bits of 128 (bf16)
// or 1024 (fp16) and subtracting 128 + z (1024 + z), exactly: one shift, one
// three-input logic operation and one packed subtraction for two weights.
//
// Layout (laid out once): tiles of 16 rows x 64 columns, 512 bytes, the tiles
// of a row block consecutive; lane l of a warp reads its 16 bytes of a tile as
// the A operands of four products.  Word m of lane (g = l / 4, t = l % 4) holds
// rows g and g + 8, columns 16 m + 4 t + 0..3: nibbles (0, 4) columns 0, 1 of row
// g, (1, 5) columns 0, 1 of row g + 8, (2, 6) and (3, 7) columns 2, 3.  Product m sums
// over its 16 columns in any order, so x is read as it lies: the lane's B
// operands of column block m are x[16 m + 4 t .. + 3].  The two rows of a lane
// share one word of scales.
//
// Rows in binary32 are split into three truncations to bf16 (8 + 8 + 8 bits:
// exact), each its own column of the product, and joined at the end.
//
// A cluster of 1, 2, 4 or 8 blocks shares a row block: the columns are split over
// the blocks (as many as it takes for x to fit shared memory), and over a
// block's warps in chunks of a few tiles.  x is laid out in shared memory once
// per block, in operand order, so a tile costs two 16-byte reads of it.  Every
// warp keeps the weights of its next chunk in flight in registers (a register
// is refilled as soon as its tile is done).  The warps' sums of a row block meet
// in shared memory, two buffers and one barrier per row block, and are added in
// a fixed order.
#include "b2f_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2f {
namespace {

constexpr int Q4_ROWS = 16;   // weight rows of a tile
constexpr int Q4_COLS = 64;   // columns of a tile
constexpr int Q4_MAX_WARPS = 16;

struct Q4Args {
  const uint4 *packed;
  const uint32_t *scales;   // [row block][group][8 pairs]
  const uint16_t *zeros;    // [row block][group][8 pairs] or null
  const void *x;
  void *y;
  long long ldx, ldy;
  int N, K, tiles_k, groups;
  int group_tiles;          // 64-column tiles of a group, 0 for groups of 32
  // ceil(2^32 / group_tiles), tile / group_tiles in one product (both below 2^14: exact);
  // 0 for groups of one tile
  uint32_t group_magic;
  int rows, cols, out_f32, x_vec, scale_bf16;
  int block_tiles;          // tiles of x of one block of a cluster
  int warps, cluster;
};

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1, __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1, __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// d = a b
template <class T>
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1, T t) {
#pragma unroll
  for (int i = 0; i < 4; ++i) d[i] = 0.0f;
  mma_16816(d, a, b0, b1, t);
}

// two nibbles (bits 0-3 and 16-19 of w) -> code - z in both halves; base is
// 128 (bf16) or 1024 (fp16) in both halves, bz = base + z
template <class T>
constexpr uint32_t kNibbleBase = 0x43004300u;
template <>
constexpr uint32_t kNibbleBase<__half> = 0x64006400u;

__device__ __forceinline__ uint32_t nibbles(uint32_t w, uint32_t bz, __nv_bfloat16) {
  const uint32_t v = (w & 0x000f000fu) | kNibbleBase<__nv_bfloat16>;
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v),
                                   *reinterpret_cast<const __nv_bfloat162 *>(&bz));
  return *reinterpret_cast<const uint32_t *>(&d);
}
__device__ __forceinline__ uint32_t nibbles(uint32_t w, uint32_t bz, __half) {
  const uint32_t v = (w & 0x000f000fu) | kNibbleBase<__half>;
  const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&v),
                            *reinterpret_cast<const __half2 *>(&bz));
  return *reinterpret_cast<const uint32_t *>(&d);
}

__device__ __forceinline__ float2 scale_pair(uint32_t v, int bf16) {
  if (bf16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}

// x[col][k .. k + 3] as two packed operands; columns past the rows and
// elements past K are zero.  SPLIT: column col is plane col % 3 of row col / 3.
template <class T, bool SPLIT>
__device__ __forceinline__ uint2 load_x(const Q4Args &a, int col, int k) {
  const int row = SPLIT ? col / 3 : col;
  if (row >= a.rows || k >= a.K) return make_uint2(0, 0);
  if (!SPLIT) {
    const T *p = static_cast<const T *>(a.x) + row * a.ldx + k;
    if (a.x_vec && k + 4 <= a.K) return __ldg(reinterpret_cast<const uint2 *>(p));
    unsigned short v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = k + i < a.K ? __ldg(reinterpret_cast<const unsigned short *>(p) + i) : 0;
    return make_uint2(v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16);
  } else {
    const float *p = static_cast<const float *>(a.x) + row * a.ldx + k;
    const int plane = col - 3 * row;
    float v[4];
    if (a.x_vec && k + 4 <= a.K) {
      const float4 f = __ldg(reinterpret_cast<const float4 *>(p));
      v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = k + i < a.K ? __ldg(p + i) : 0.0f;
    }
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // truncations: v = hi + mid + lo, each with 8 significant bits; an
      // infinity or NaN stays in the first plane
      const uint32_t hi = __float_as_uint(v[i]) & 0xffff0000u;
      const bool finite = (hi & 0x7f800000u) != 0x7f800000u;
      const float r1 = finite ? v[i] - __uint_as_float(hi) : 0.0f;
      const uint32_t mid = __float_as_uint(r1) & 0xffff0000u;
      const uint32_t lo = __float_as_uint(r1 - __uint_as_float(mid));
      const uint32_t first = finite ? hi : __float_as_uint(v[i]) | (v[i] != v[i] ? 0x400000u : 0u);
      u[i] = (plane == 0 ? first : plane == 1 ? mid : lo) >> 16;
    }
    return make_uint2(u[0] | u[1] << 16, u[2] | u[3] << 16);
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ float remote_f32(const float *p, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n"
               : "=r"(a)
               : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(a) : "memory");
  return v;
}
// a barrier of the block, or of its cluster of cs blocks
__device__ __forceinline__ void meet(int cs) {
  if (cs == 1) {
    __syncthreads();
  } else {
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
  }
}

// Cluster c of gridDim.x / cs takes row blocks c, c + clusters, ...; block r of a
// cluster takes tiles [r block_tiles, (r + 1) block_tiles), its warp w the chunks
// of TPW tiles w, w + warps, ... of those.  NT: 8-column tiles of x (planes
// counted).  Shared memory: x [block_tiles][2][cols][4 lanes] of 16 bytes, then
// two buffers of sums [warps][16][8 NT].
template <class T, bool SPLIT, int NT, int TPW, bool ZERO, bool G32>
__global__ void __launch_bounds__(32 * Q4_MAX_WARPS)
    q4_matvec_kernel(const Q4Args a) {
  extern __shared__ __align__(16) unsigned char q4_smem[];
  uint4 *xs = reinterpret_cast<uint4 *>(q4_smem);
  float *sums = reinterpret_cast<float *>(q4_smem + (size_t)a.block_tiles * a.cols * 128);
  constexpr int SUMS = Q4_ROWS * 8 * NT;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int cs = a.cluster, rank = cs == 1 ? 0 : (int)cluster_rank();
  const int row_blocks = (a.N + Q4_ROWS - 1) / Q4_ROWS;
  const int stride = gridDim.x / cs;
  const int tile0 = rank * a.block_tiles;
  const int tiles = max(0, min(a.block_tiles, a.tiles_k - tile0));
  const int chunks = (tiles + TPW - 1) / TPW;

  int rb = blockIdx.x / cs, chunk = warp;
  uint4 w[TPW];
  uint32_t sc[G32 ? 2 * TPW : TPW];
  uint16_t zr[ZERO ? (G32 ? 2 * TPW : TPW) : 1];
  // tile i of a chunk into its registers (zeros past the block's tiles)
  auto fetch = [&](int i, int r, int c) {
    const int kt = c * TPW + i;
    const bool in = r < row_blocks && kt < tiles;
    const int k = tile0 + kt;
    w[i] = in ? __ldcs(a.packed + ((long long)r * a.tiles_k + k) * 32 + lane)
              : make_uint4(0, 0, 0, 0);
    const int grp = G32 ? 2 * k : a.group_magic ? (int)__umulhi((uint32_t)k, a.group_magic) : k;
    const long long at = ((long long)r * a.groups + grp) * 8 + g;
    if (G32) {
      const bool two = in && grp + 1 < a.groups;
      sc[2 * i] = in ? __ldg(a.scales + at) : 0;
      sc[2 * i + 1] = two ? __ldg(a.scales + at + 8) : 0;
      if (ZERO) {
        zr[2 * i] = in ? __ldg(a.zeros + at) : 0;
        zr[2 * i + 1] = two ? __ldg(a.zeros + at + 8) : 0;
      }
    } else {
      sc[i] = in ? __ldg(a.scales + at) : 0;
      if (ZERO) zr[i] = in ? __ldg(a.zeros + at) : 0;
    }
  };
#pragma unroll
  for (int i = 0; i < TPW; ++i) fetch(i, rb, chunk);

  for (int i = threadIdx.x; i < tiles * a.cols * 4; i += blockDim.x) {
    const int q = i & 3, c = (i >> 2) % a.cols, kt = (i >> 2) / a.cols;
    const int k = (tile0 + kt) * Q4_COLS + 4 * q;
    uint4 *o = xs + ((size_t)kt * 2 * a.cols + c) * 4 + q;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint2 lo = load_x<T, SPLIT>(a, c, k + 32 * h);
      const uint2 hi = load_x<T, SPLIT>(a, c, k + 32 * h + 16);
      o[h * a.cols * 4] = make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
  }
  __syncthreads();

  float tot[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) tot[j][i] = 0.0f;

  for (int buf = 0; rb < row_blocks; buf ^= 1) {
    for (; chunk < chunks;) {
      int next = chunk + warps, next_rb = rb;
      if (next >= chunks) next = warp, next_rb = rb + stride;
#pragma unroll
      for (int i = 0; i < TPW; ++i) {
        const uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        const int kt = chunk * TPW + i;
        uint4 xv[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const bool on = 8 * j + g < a.cols && kt < tiles;
          const uint4 *xp = xs + ((size_t)kt * 2 * a.cols + 8 * j + g) * 4 + t;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            xv[j][h] = on ? xp[h * a.cols * 4] : make_uint4(0, 0, 0, 0);
        }
        float acc[NT][4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const int si = G32 ? 2 * i + m / 2 : i;
          uint32_t bz0 = kNibbleBase<T> + 0x00080008u, bz1 = bz0;
          if (ZERO) {
            bz0 = kNibbleBase<T> + (zr[ZERO ? si : 0] & 0xffu) * 0x00010001u;
            bz1 = kNibbleBase<T> + (uint32_t)(zr[ZERO ? si : 0] >> 8) * 0x00010001u;
          }
          uint32_t f[4];
          f[0] = nibbles(v[m], bz0, T());
          f[1] = nibbles(v[m] >> 4, bz1, T());
          f[2] = nibbles(v[m] >> 8, bz0, T());
          f[3] = nibbles(v[m] >> 12, bz1, T());
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint32_t b0 = m & 1 ? xv[j][m / 2].z : xv[j][m / 2].x;
            const uint32_t b1 = m & 1 ? xv[j][m / 2].w : xv[j][m / 2].y;
            if (m == 0 || (G32 && m == 2))
              mma_first(acc[j], f, b0, b1, T());
            else
              mma_16816(acc[j], f, b0, b1, T());
          }
          if (m == 3 || (G32 && m == 1)) {  // the group's (or the tile's part of its) sums
            const float2 s = scale_pair(sc[si], a.scale_bf16);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              tot[j][0] += s.x * acc[j][0];
              tot[j][1] += s.x * acc[j][1];
              tot[j][2] += s.y * acc[j][2];
              tot[j][3] += s.y * acc[j][3];
            }
          }
        }
        fetch(i, next_rb, next);
      }
      chunk += warps;
    }
    chunk = warp;
    // c0, c1: row g, columns 2t, 2t + 1; c2, c3: row g + 8
    float *out = sums + (buf * warps + warp) * SUMS;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float *o = out + g * 8 * NT + 8 * j + 2 * t;
      *reinterpret_cast<float2 *>(o) = make_float2(tot[j][0], tot[j][1]);
      *reinterpret_cast<float2 *>(o + 8 * 8 * NT) = make_float2(tot[j][2], tot[j][3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) tot[j][i] = 0.0f;
    }
    meet(cs);
    for (int i = threadIdx.x + rank * blockDim.x; i < Q4_ROWS * a.rows; i += cs * blockDim.x) {
      const int r = i & 15, b = i >> 4, n = rb * Q4_ROWS + r;
      if (n < a.N) {
        float v = 0.0f;
        for (int c = 0; c < cs; ++c)
          for (int u = 0; u < warps; ++u) {
            const float *s = sums + (buf * warps + u) * SUMS + r * 8 * NT;
            auto at = [&](int col) { return cs == 1 ? s[col] : remote_f32(s + col, c); };
            if (SPLIT)
              v += at(3 * b) + (at(3 * b + 2) + at(3 * b + 1));
            else
              v += at(b);
          }
        const long long at = b * a.ldy + n;
        if (SPLIT || a.out_f32)
          static_cast<float *>(a.y)[at] = v;
        else
          static_cast<T *>(a.y)[at] = (T)v;
      }
    }
    rb += stride;
  }
  if (cs > 1) meet(cs);  // no block leaves while its sums are read
}

// codes [N][K] (one byte each) -> tiles; pairs of scales and zero points
__global__ void q4_pack_kernel(const uint8_t *__restrict__ codes, int N, int K, int tiles_k,
                               uint32_t *__restrict__ packed) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int row_blocks = (N + Q4_ROWS - 1) / Q4_ROWS;
  if (i >= (long long)row_blocks * tiles_k * 128) return;
  const int m = (int)(i & 3), lane = (int)(i >> 2) & 31;
  const long long tile = i >> 7;
  const int kt = (int)(tile % tiles_k), rb = (int)(tile / tiles_k);
  const int g = lane >> 2, t = lane & 3;
  uint32_t v = 0;
#pragma unroll
  for (int nib = 0; nib < 8; ++nib) {
    const int row = rb * Q4_ROWS + g + 8 * (nib & 1);
    const int col = kt * Q4_COLS + 16 * m + 4 * t + (nib & 2) + (nib >> 2);
    const uint32_t c = row < N && col < K ? codes[(long long)row * K + col] & 15u : 8u;
    v |= c << (4 * nib);
  }
  packed[i] = v;
}

template <class E>
__global__ void q4_pairs_kernel(const E *__restrict__ in, int N, int groups,
                                E *__restrict__ out) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int row_blocks = (N + Q4_ROWS - 1) / Q4_ROWS;
  if (i >= (long long)row_blocks * groups * 16) return;
  const int second = (int)(i & 1), g = (int)(i >> 1) & 7;
  const long long q = i >> 4;
  const int grp = (int)(q % groups), row = (int)(q / groups) * Q4_ROWS + g + 8 * second;
  out[i] = row < N ? in[(long long)row * groups + grp] : (E)0;
}

template <class T>
__device__ __forceinline__ float as_float(T x) {
  return (float)x;
}

// One warp per (row, group): symmetric s = max|w| / 7, codes round(w / s) + 8;
// else the range [min(w, 0), max(w, 0)] on 16 steps with an integer zero point.
// s is rounded to its stored type first and the codes are taken against that.
template <class T, class S>
__global__ void q4_quantize_kernel(const T *__restrict__ w, long long ld, int N, int K,
                                   int group, int groups, int symmetric,
                                   uint8_t *__restrict__ codes, S *__restrict__ scales,
                                   uint8_t *__restrict__ zeros) {
  const long long item = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (item >= (long long)N * groups) return;
  const int row = (int)(item / groups), grp = (int)(item % groups);
  const int k0 = grp * group, k1 = min(k0 + group, K);
  float lo = 0.0f, hi = 0.0f;
  for (int k = k0 + lane; k < k1; k += 32) {
    const float v = as_float(w[row * ld + k]);
    lo = fminf(lo, v);
    hi = fmaxf(hi, v);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(~0u, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, o));
  }
  const S stored = (S)(symmetric ? __fdiv_rn(fmaxf(hi, -lo), 7.0f) : __fdiv_rn(hi - lo, 15.0f));
  const float s = (float)stored;
  float z = 8.0f;
  if (!symmetric) z = s > 0.0f ? fminf(fmaxf(rintf(__fdiv_rn(-lo, s)), 0.0f), 15.0f) : 0.0f;
  for (int k = k0 + lane; k < k1; k += 32) {
    const float v = as_float(w[row * ld + k]);
    const float c = s > 0.0f ? rintf(__fdiv_rn(v, s)) + z : z;
    codes[(long long)row * K + k] = (uint8_t)fminf(fmaxf(c, 0.0f), 15.0f);
  }
  if (lane == 0) {
    scales[item] = stored;
    if (zeros) zeros[item] = (uint8_t)z;
  }
}

constexpr size_t kQ4Smem = 227 * 1024;

size_t smem_bytes(const Q4Args &a, int nt) {
  return (size_t)a.block_tiles * a.cols * 128 + (size_t)2 * a.warps * Q4_ROWS * 8 * nt * 4;
}

template <class T, bool SPLIT, int NT, bool ZERO, bool G32>
int launch_matvec(Q4Args a, int sms, cudaStream_t s) {
  constexpr int TPW = NT > 1 || G32 ? 4 : 8;
  auto k = q4_matvec_kernel<T, SPLIT, NT, TPW, ZERO, G32>;
  // the fewest blocks whose shares of x fit shared memory
  size_t smem = 0;
  for (a.cluster = 1; a.cluster <= 8; a.cluster *= 2) {
    a.block_tiles = (a.tiles_k + a.cluster - 1) / a.cluster;
    const int chunks = (a.block_tiles + TPW - 1) / TPW;
    const int visits = (chunks + Q4_MAX_WARPS - 1) / Q4_MAX_WARPS;
    a.warps = (chunks + visits - 1) / visits;
    smem = (size_t)a.block_tiles * a.cols * 128 + (size_t)2 * a.warps * Q4_ROWS * 8 * NT * 4;
    if (smem <= kQ4Smem) break;
  }
  B2F_CHECK_ARG(a.cluster <= 8, "b2f_q4_matvec: %d columns of %d values do not fit", a.cols, a.K);
  B2F_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kQ4Smem));
  const int row_blocks = (a.N + Q4_ROWS - 1) / Q4_ROWS;
  // blocks of an SM: by shared memory and by 16 warps (128 registers a thread)
  const int per_sm = std::max(1, std::min<int>((int)(kQ4Smem / (smem + 1024)), 16 / a.warps));
  const int clusters = std::min(row_blocks, std::max(1, sms * per_sm / a.cluster));
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(clusters * a.cluster);
  c.blockDim = dim3(32 * a.warps);
  c.dynamicSmemBytes = smem;
  c.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = a.cluster > 1 ? 1 : 0;
  B2F_CUDA(cudaLaunchKernelEx(&c, k, a));
  B2F_LAUNCHED("q4_matvec_kernel");
  return B2F_OK;
}
template <class T, bool SPLIT, int NT>
int launch_cols(const Q4Args &a, int sms, cudaStream_t s) {
  if (a.zeros)
    return a.group_tiles ? launch_matvec<T, SPLIT, NT, true, false>(a, sms, s)
                         : launch_matvec<T, SPLIT, NT, true, true>(a, sms, s);
  return a.group_tiles ? launch_matvec<T, SPLIT, NT, false, false>(a, sms, s)
                       : launch_matvec<T, SPLIT, NT, false, true>(a, sms, s);
}
template <class T, bool SPLIT>
int launch_rows(const Q4Args &a, int sms, cudaStream_t s) {
  if (a.cols <= 8) return launch_cols<T, SPLIT, 1>(a, sms, s);
  if (a.cols <= 16) return launch_cols<T, SPLIT, 2>(a, sms, s);
  return launch_cols<T, SPLIT, 4>(a, sms, s);
}

int check_shape(const char *who, int64_t N, int64_t K, int group) {
  B2F_CHECK_ARG(N >= 1 && N <= (1ll << 30) && K >= 1 && K <= (1ll << 24),
                "%s: weight of %lld x %lld", who, (long long)N, (long long)K);
  B2F_CHECK_ARG(group == 32 || (group >= 64 && group % 64 == 0),
                "%s: group of %d (32 or a multiple of 64)", who, group);
  return B2F_OK;
}

}  // namespace
}  // namespace b2f

extern "C" {

size_t b2f_q4_packed_bytes(int64_t N, int64_t K) {
  if (N < 1 || K < 1) return 0;
  return (size_t)((N + 15) / 16) * (size_t)((K + 63) / 64) * 512;
}

int b2f_q4_pack(const uint8_t *codes, const void *scales, const uint8_t *zeros, int64_t N,
                int64_t K, int group, void *packed, void *packed_scales, void *packed_zeros,
                void *stream) {
  B2F_RANGE("b2f_q4_pack");
  using namespace b2f;
  if (int rc = check_shape("b2f_q4_pack", N, K, group)) return rc;
  B2F_CHECK_ARG(codes && scales && packed && packed_scales && !zeros == !packed_zeros,
                "b2f_q4_pack: null argument");
  B2F_CHECK_ARG((uintptr_t)packed % 16 == 0 && (uintptr_t)packed_scales % 16 == 0 &&
                    (uintptr_t)packed_zeros % 16 == 0 && (uintptr_t)scales % 2 == 0,
                "b2f_q4_pack: misaligned buffer (16 bytes)");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int tiles_k = (int)((K + 63) / 64), groups = (int)((K + group - 1) / group);
  const long long rb = (N + 15) / 16, words = rb * tiles_k * 128, pairs = rb * groups * 16;
  q4_pack_kernel<<<(unsigned)((words + 255) / 256), 256, 0, s>>>(
      codes, (int)N, (int)K, tiles_k, static_cast<uint32_t *>(packed));
  B2F_LAUNCHED("q4_pack_kernel");
  q4_pairs_kernel<uint16_t><<<(unsigned)((pairs + 255) / 256), 256, 0, s>>>(
      static_cast<const uint16_t *>(scales), (int)N, groups,
      static_cast<uint16_t *>(packed_scales));
  B2F_LAUNCHED("q4_pairs_kernel");
  if (zeros) {
    q4_pairs_kernel<uint8_t><<<(unsigned)((pairs + 255) / 256), 256, 0, s>>>(
        zeros, (int)N, groups, static_cast<uint8_t *>(packed_zeros));
    B2F_LAUNCHED("q4_pairs_kernel");
  }
  return B2F_OK;
}

int b2f_q4_quantize(const void *w, int dtype, int64_t ld, int64_t N, int64_t K, int group,
                    int symmetric, int scale_dtype, uint8_t *codes, void *scales,
                    uint8_t *zeros, void *stream) {
  B2F_RANGE("b2f_q4_quantize");
  using namespace b2f;
  if (int rc = check_shape("b2f_q4_quantize", N, K, group)) return rc;
  B2F_CHECK_ARG(w && codes && scales && !zeros == !!symmetric, "b2f_q4_quantize: null argument");
  B2F_CHECK_ARG(ld >= K, "b2f_q4_quantize: rows of %lld, %lld apart", (long long)K,
                (long long)ld);
  B2F_CHECK_ARG(dtype >= B2F_F32 && dtype <= B2F_BF16, "b2f_q4_quantize: dtype %d", dtype);
  B2F_CHECK_ARG(scale_dtype == B2F_F16 || scale_dtype == B2F_BF16,
                "b2f_q4_quantize: scale dtype %d", scale_dtype);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int groups = (int)((K + group - 1) / group);
  const long long warps = N * groups;
  const unsigned grid = (unsigned)((warps + 7) / 8);
  auto go = [&](auto *wt, auto *st) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(wt)>>;
    using S = std::remove_pointer_t<decltype(st)>;
    q4_quantize_kernel<T, S><<<grid, 256, 0, s>>>(wt, ld, (int)N, (int)K, group, groups,
                                                  symmetric, codes, st, zeros);
  };
  auto pick = [&](auto *wt) {
    if (scale_dtype == B2F_BF16)
      go(wt, static_cast<__nv_bfloat16 *>(scales));
    else
      go(wt, static_cast<__half *>(scales));
  };
  if (dtype == B2F_F32)
    pick(static_cast<const float *>(w));
  else if (dtype == B2F_F16)
    pick(static_cast<const __half *>(w));
  else
    pick(static_cast<const __nv_bfloat16 *>(w));
  B2F_LAUNCHED("q4_quantize_kernel");
  return B2F_OK;
}

int b2f_q4_matvec(const void *x, int dtype, int64_t ldx, int64_t rows, const void *packed,
                  const void *scales, int scale_dtype, const void *zeros, int64_t N, int64_t K,
                  int group, void *y, int out_f32, void *stream) {
  B2F_RANGE("b2f_q4_matvec");
  using namespace b2f;
  if (int rc = check_shape("b2f_q4_matvec", N, K, group)) return rc;
  B2F_CHECK_ARG(rows >= 0 && rows <= 1024, "b2f_q4_matvec: %lld rows (up to 1024)",
                (long long)rows);
  B2F_CHECK_ARG(dtype >= B2F_F32 && dtype <= B2F_BF16, "b2f_q4_matvec: dtype %d", dtype);
  B2F_CHECK_ARG(scale_dtype == B2F_F16 || scale_dtype == B2F_BF16,
                "b2f_q4_matvec: scale dtype %d", scale_dtype);
  if (rows == 0) return B2F_OK;
  B2F_CHECK_ARG(x && packed && scales && y, "b2f_q4_matvec: null argument");
  B2F_CHECK_ARG(ldx >= K || rows == 1, "b2f_q4_matvec: rows of %lld, %lld apart", (long long)K,
                (long long)ldx);
  const int esize = dtype == B2F_F32 ? 4 : 2;
  B2F_CHECK_ARG((uintptr_t)packed % 16 == 0 && (uintptr_t)scales % 16 == 0 &&
                    (uintptr_t)zeros % 16 == 0 && (uintptr_t)x % esize == 0 &&
                    (uintptr_t)y % (out_f32 ? 4 : esize) == 0,
                "b2f_q4_matvec: misaligned buffer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int dev = 0, sms = 0;
  B2F_CUDA(cudaGetDevice(&dev));
  B2F_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  Q4Args a{};
  a.packed = static_cast<const uint4 *>(packed);
  a.scales = static_cast<const uint32_t *>(scales);
  a.zeros = static_cast<const uint16_t *>(zeros);
  a.ldx = ldx;
  a.ldy = N;
  a.N = (int)N;
  a.K = (int)K;
  a.tiles_k = (int)((K + 63) / 64);
  a.groups = (int)((K + group - 1) / group);
  a.group_tiles = std::min(group / 64, a.tiles_k);  // 0 for groups of 32
  a.out_f32 = out_f32 != 0;
  a.group_magic = a.group_tiles > 1 ? (uint32_t)(((1ull << 32) + a.group_tiles - 1) / a.group_tiles)
                                    : 0;
  a.scale_bf16 = scale_dtype == B2F_BF16;
  a.x_vec = (uintptr_t)x % (4 * esize) == 0 && (rows == 1 || ldx % 4 == 0);
  // columns of the product in one pass: up to 32, and no more than 8 blocks'
  // shared memory holds of x (a part kept for the sums)
  const int planes = dtype == B2F_F32 ? 3 : 1;
  const long long fit = 8ll * (kQ4Smem - 72 * 1024) / (128ll * (a.tiles_k + 8));
  const int step = (int)std::min<long long>(32, fit) / planes;
  B2F_CHECK_ARG(step >= 1, "b2f_q4_matvec: %lld columns are more than shared memory holds",
                (long long)K);
  for (int64_t r0 = 0; r0 < rows; r0 += step) {
    a.rows = (int)std::min<int64_t>(step, rows - r0);
    a.cols = a.rows * planes;
    a.x = static_cast<const char *>(x) + r0 * ldx * esize;
    a.y = static_cast<char *>(y) + r0 * N * (out_f32 ? 4 : esize);
    const int rc = dtype == B2F_F32   ? launch_rows<__nv_bfloat16, true>(a, sms, s)
                   : dtype == B2F_F16 ? launch_rows<__half, false>(a, sms, s)
                                      : launch_rows<__nv_bfloat16, false>(a, sms, s);
    if (rc) return rc;
  }
  return B2F_OK;
}

}  // extern "C"
