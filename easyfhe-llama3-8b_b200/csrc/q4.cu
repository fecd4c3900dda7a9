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
  int N, K, tiles_k, groups, group_tiles;  // group_tiles: 64-column tiles of a group, 0 for 32
  int rows, out_f32, x_vec, per_warp;
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

template <bool SB>
__device__ __forceinline__ float2 scale_pair(uint32_t v) {
  if (SB) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
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

// One block: row blocks blockIdx.x, + gridDim.x, ...; warp w sums tiles
// [w per_warp, (w + 1) per_warp) of a row block, then the block adds the
// warps' sums in order.  NT: 8-column tiles of x (planes counted).
template <class T, bool SPLIT, int NT, bool ZERO, bool SB>
__global__ void __launch_bounds__(32 * Q4_MAX_WARPS)
    q4_matvec_kernel(const Q4Args a) {
  extern __shared__ float q4_sums[];  // [warps][16][8 NT]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int row_blocks = (a.N + Q4_ROWS - 1) / Q4_ROWS;
  const int k_begin = warp * a.per_warp, k_end = min(k_begin + a.per_warp, a.tiles_k);
  for (int rb = blockIdx.x; rb < row_blocks; rb += gridDim.x) {
    const uint4 *wp = a.packed + ((long long)rb * a.tiles_k) * 32 + lane;
    const uint32_t *sp = a.scales + (long long)rb * a.groups * 8 + g;
    const uint16_t *zp = ZERO ? a.zeros + (long long)rb * a.groups * 8 + g : nullptr;
    float tot[NT][4], acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) tot[j][i] = acc[j][i] = 0.0f;
    uint32_t bz0 = kNibbleBase<T> + 0x00080008u, bz1 = bz0;
    auto zero_of = [&](int grp) {
      if (!ZERO) return;
      const uint32_t z = __ldg(zp + grp * 8);
      bz0 = kNibbleBase<T> + (z & 0xff) * 0x00010001u;
      bz1 = kNibbleBase<T> + (z >> 8) * 0x00010001u;
    };
    // apply the group's scales to its sums and start the next group
    auto flush = [&](int grp) {
      const float2 s = scale_pair<SB>(__ldg(sp + grp * 8));
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        tot[j][0] += s.x * acc[j][0];
        tot[j][1] += s.x * acc[j][1];
        tot[j][2] += s.y * acc[j][2];
        tot[j][3] += s.y * acc[j][3];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
      }
    };
    for (int kt = k_begin; kt < k_end; ++kt) {
      const uint4 w4 = __ldg(wp + (long long)kt * 32);
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
      const int grp = a.group_tiles ? kt / a.group_tiles : 2 * kt;
      zero_of(grp);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        if (m == 2 && !a.group_tiles) {  // groups of 32: two per tile
          flush(grp);
          if (grp + 1 >= a.groups) break;  // columns past K
          zero_of(grp + 1);
        }
        uint32_t f[4];
        f[0] = nibbles(w[m], bz0, T());
        f[1] = nibbles(w[m] >> 4, bz1, T());
        f[2] = nibbles(w[m] >> 8, bz0, T());
        f[3] = nibbles(w[m] >> 12, bz1, T());
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint2 b = load_x<T, SPLIT>(a, 8 * j + g, kt * Q4_COLS + 16 * m + 4 * t);
          mma_16816(acc[j], f, b.x, b.y, T());
        }
      }
      if (!a.group_tiles) {
        if (grp + 1 < a.groups) flush(grp + 1);
      } else if (kt + 1 == k_end || (kt + 1) % a.group_tiles == 0) {
        flush(grp);
      }
    }
    // c0, c1: row g, columns 2t, 2t + 1; c2, c3: row g + 8
    float *out = q4_sums + warp * (Q4_ROWS * 8 * NT);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float *o = out + g * 8 * NT + 8 * j + 2 * t;
      o[0] = tot[j][0], o[1] = tot[j][1];
      o[8 * 8 * NT] = tot[j][2], o[8 * 8 * NT + 1] = tot[j][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < Q4_ROWS * a.rows; i += blockDim.x) {
      const int r = i & 15, b = i >> 4, n = rb * Q4_ROWS + r;
      if (n < a.N) {
        float v = 0.0f;
        for (int w = 0; w < warps; ++w) {
          const float *s = q4_sums + (w * Q4_ROWS + r) * 8 * NT;
          if (SPLIT) {
            // the small planes first
            const float lo = s[3 * b + 2] + s[3 * b + 1];
            v += s[3 * b] + lo;
          } else {
            v += s[b];
          }
        }
        const long long at = b * a.ldy + n;
        if (SPLIT || a.out_f32)
          static_cast<float *>(a.y)[at] = v;
        else
          static_cast<T *>(a.y)[at] = (T)v;
      }
    }
    __syncthreads();
  }
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

template <class T, bool SPLIT, int NT>
int launch_matvec(const Q4Args &a, bool zero, bool sb, int grid, int warps, cudaStream_t s) {
  const size_t smem = (size_t)warps * Q4_ROWS * 8 * NT * sizeof(float);
  auto go = [&](auto kernel) { kernel<<<grid, 32 * warps, smem, s>>>(a); };
  if (zero && sb)
    go(q4_matvec_kernel<T, SPLIT, NT, true, true>);
  else if (zero)
    go(q4_matvec_kernel<T, SPLIT, NT, true, false>);
  else if (sb)
    go(q4_matvec_kernel<T, SPLIT, NT, false, true>);
  else
    go(q4_matvec_kernel<T, SPLIT, NT, false, false>);
  B2F_LAUNCHED("q4_matvec_kernel");
  return B2F_OK;
}
template <class T, bool SPLIT>
int launch_matvec_cols(const Q4Args &a, int cols, bool zero, bool sb, int grid, int warps,
                       cudaStream_t s) {
  if (cols <= 8) return launch_matvec<T, SPLIT, 1>(a, zero, sb, grid, warps, s);
  if (cols <= 16) return launch_matvec<T, SPLIT, 2>(a, zero, sb, grid, warps, s);
  return launch_matvec<T, SPLIT, 4>(a, zero, sb, grid, warps, s);
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
  a.group_tiles = group / 64;
  a.out_f32 = out_f32 != 0;
  a.x_vec = (uintptr_t)x % (4 * esize) == 0 && (rows == 1 || ldx % 4 == 0);
  const int warps = std::min(a.tiles_k, 8);
  a.per_warp = (a.tiles_k + warps - 1) / warps;
  const int row_blocks = (a.N + Q4_ROWS - 1) / Q4_ROWS;
  const int grid = std::min(row_blocks, 4 * sms);
  const int planes = dtype == B2F_F32 ? 3 : 1, step = 32 / planes;
  for (int64_t r0 = 0; r0 < rows; r0 += step) {
    a.rows = (int)std::min<int64_t>(step, rows - r0);
    a.x = static_cast<const char *>(x) + r0 * ldx * esize;
    a.y = static_cast<char *>(y) + r0 * N * (out_f32 ? 4 : esize);
    const int cols = a.rows * planes;
    const bool z = zeros != nullptr, sb = scale_dtype == B2F_BF16;
    int rc;
    if (dtype == B2F_F32)
      rc = launch_matvec_cols<__nv_bfloat16, true>(a, cols, z, sb, grid, warps, s);
    else if (dtype == B2F_F16)
      rc = launch_matvec_cols<__half, false>(a, cols, z, sb, grid, warps, s);
    else
      rc = launch_matvec_cols<__nv_bfloat16, false>(a, cols, z, sb, grid, warps, s);
    if (rc) return rc;
  }
  return B2F_OK;
}

}  // extern "C"
