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
// Layout (laid out once): records of 16 rows x 64 columns, a row block's records
// consecutive: 512 bytes of codes, then the scales of the record's group (two
// groups of 32) and its zero points, so that one running pointer reaches all
// that a record needs.  A group of more than 64 columns repeats its scales in each
// of its records (544 bytes instead of 528 for groups of 128): addressing them by
// group cost 20 of 158 instructions a record, and it is instructions that bound one
// row.  Lane l of a warp reads its 16 bytes of a record as the A operands of four
// products.  Word 2 h + b of lane (g = l / 4, t = l % 4) holds rows g and g + 8, columns
// 32 h + 8 t + 4 b + 0..3: nibbles (0, 4) columns 0, 1 of row g, (1, 5) columns 0, 1 of
// row g + 8, (2, 6) and (3, 7) columns 2, 3.  A product sums over its columns in any
// order, so x is read as it lies: the lane's B operands of words 2 h and 2 h + 1 are the
// 8 values x[32 h + 8 t ..].  The two rows of a lane share one word of scales.
//
// Rows in binary32 are split into three truncations to bf16 (8 + 8 + 8 bits:
// exact), each its own column of the product, and joined at the end.
//
// Few rows leave most of those 8 columns idle, and the conversion of the nibbles is
// what bounds them (85 instructions a record, 58 us for one row against 128256 x 4096,
// where HBM alone takes 41; as digits 47 instructions and 48 us).  They run on mma.sync
// m16n8k32 u8 x s8 instead: codes are bytes as they lie, two instructions for eight of
// them, and x is a fixed-point number per row and 64 columns, X = round(x 2^sh) with
// the largest |X| in [2^29, 2^30], as four signed base-256 digits, each a column of the
// product.  The sums code X are exact integers; the zero point enters as the
// accumulator's first value, -z sum X, on top of 1.5 2^23, so that the sum's bits read as
// binary32 are the sum plus that constant and no conversion is needed.  X is off by at
// most 2^-30 of the largest of its 64 columns, which binary32 accumulation of the same
// products is not better than.
//
// A block takes row blocks in turn, its warps chunks of a few records along the
// columns (and, where those are few, several row blocks at once).  x is laid out in
// shared memory once per block, in operand order, so a record costs one or two 16-byte
// reads of it.  Every warp keeps its next chunk in flight in registers (a register is
// refilled as soon as its record is done).  The warps' sums meet in shared memory, two
// buffers and one barrier per q4_batch rounds, and are added in a fixed order.  Where x
// does not fit one block, a cluster of 2, 4 or 8 blocks splits the columns and adds its
// blocks' sums through distributed shared memory; splitting without need was no
// faster (8 rows of 4096 x 4096: 8.3 us on one, 9.0 on two, 11.4 on four blocks).
//
// Measured: one binary32 row against 128256 x 4096, groups of 128: 48 us (5.6 TB/s, 86 %
// of copy bandwidth); one bf16 row of 4096 x 4096: 6.0 us, where the launch, the set-up of
// x and one trip to memory bound; 8 fp16 rows of 4096 x 14336 with zero points: 17.5 us,
// bound by the set-up (every block stages all 8 rows) and by 1.7 row blocks an SM.
#include "plain.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2f {
namespace {

constexpr int Q4_ROWS = 16;   // weight rows of a tile
constexpr int Q4_COLS = 64;   // columns of a tile

// bytes of a record and where its zero points lie
constexpr int q4_record(bool g32, bool zero) {
  return 512 + (g32 ? 64 : 32) + (zero ? 32 : 0);
}
constexpr int q4_zeros_at(bool g32) { return 512 + (g32 ? 64 : 32); }

struct Q4Args {
  const unsigned char *packed;
  const void *x;
  void *y;
  long long ldx, ldy;
  int N, K, tiles_k;
  int rows, cols, dtype, out_f32, x_vec;
  int block_tiles;  // tiles of x of one block of a cluster
  int warps_k, warps_r;  // a block's warps: along the columns, over row blocks
  int cluster;
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
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1, __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1, __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// two nibbles (bits 0-3 and 16-19 of w) -> code - z in both halves; base is
// 128 (bf16) or 1024 (fp16) in both halves, bz = base + z
template <class T>
constexpr uint32_t kNibbleBase = 0x43004300u;
template <>
constexpr uint32_t kNibbleBase<__half> = 0x64006400u;

// (w & mask) | base as one instruction (written in C it became two)
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t base) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;\n" : "=r"(v) : "r"(w), "r"(mask), "r"(base));
  return v;
}
__device__ __forceinline__ uint32_t nibbles(uint32_t w, uint32_t bz, __nv_bfloat16) {
  const uint32_t v = and_or(w, 0x000f000fu, kNibbleBase<__nv_bfloat16>);
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v),
                                   *reinterpret_cast<const __nv_bfloat162 *>(&bz));
  return *reinterpret_cast<const uint32_t *>(&d);
}
__device__ __forceinline__ uint32_t nibbles(uint32_t w, uint32_t bz, __half) {
  const uint32_t v = and_or(w, 0x000f000fu, kNibbleBase<__half>);
  const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&v),
                            *reinterpret_cast<const __half2 *>(&bz));
  return *reinterpret_cast<const uint32_t *>(&d);
}

template <bool SB>
__device__ __forceinline__ float2 scale_pair(uint32_t v) {
  if (SB) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}

// d = c + a b, u8 x s8
__device__ __forceinline__ void mma_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1,
                                          const int (&c)[4]) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]),
        "r"(c[3]));
}

constexpr int kSumBase = 0x4B400000;  // bits of 1.5 2^23: + n reads as 1.5 2^23 + n, |n| < 2^22

// Four consecutive columns k.. of a row of x as they lie (binary32: a word each,
// 16-bit types: two in a word), zero past K.
__device__ __forceinline__ uint4 load_piece(const Q4Args &a, int row, int k) {
  const bool whole = a.x_vec && k + 4 <= a.K;
  const long long at = row * a.ldx + k;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (a.dtype == B2F_F32) {
    const uint32_t *p = static_cast<const uint32_t *>(a.x) + at;
    if (whole) return __ldg(reinterpret_cast<const uint4 *>(p));
    if (k < a.K) v.x = __ldg(p);
    if (k + 1 < a.K) v.y = __ldg(p + 1);
    if (k + 2 < a.K) v.z = __ldg(p + 2);
    if (k + 3 < a.K) v.w = __ldg(p + 3);
    return v;
  }
  const unsigned short *p = static_cast<const unsigned short *>(a.x) + at;
  if (whole) {
    const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p));
    v.x = u.x, v.y = u.y;
    return v;
  }
  if (k < a.K) v.x = __ldg(p);
  if (k + 1 < a.K) v.x |= (uint32_t)__ldg(p + 1) << 16;
  if (k + 2 < a.K) v.y = __ldg(p + 2);
  if (k + 3 < a.K) v.y |= (uint32_t)__ldg(p + 3) << 16;
  return v;
}

constexpr int Q4_AHEAD = 4;  // loads of x in flight per thread while a block lays it out

// Visits x of a block's tiles in pieces of 4 columns: put(tile, row, piece of the
// tile, values), 16 threads in a row on a tile's pieces.  Whole warps take part
// (`on` tells whether there is a piece), so put may exchange among its 16 lanes.
template <class Put>
__device__ __forceinline__ void q4_each_piece(const Q4Args &a, int tile0, int tiles, Put put) {
  const int total = tiles * a.rows * 16;
  for (int i0 = 0; i0 < total; i0 += Q4_AHEAD * blockDim.x) {
    uint4 v[Q4_AHEAD];
#pragma unroll
    for (int u = 0; u < Q4_AHEAD; ++u) {
      const int i = i0 + u * blockDim.x + threadIdx.x;
      const int row = (i >> 4) / tiles, kt = (i >> 4) - row * tiles;
      v[u] = i < total ? load_piece(a, row, (tile0 + kt) * Q4_COLS + 4 * (i & 15))
                       : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < Q4_AHEAD; ++u)
      if (i0 + u * blockDim.x < total) {
        const int i = i0 + u * blockDim.x + threadIdx.x;
        const int row = (i >> 4) / tiles, kt = (i >> 4) - row * tiles;
        put(i < total, kt, row, i & 15, v[u]);
      }
  }
}

// x as operands: [tile][2][cols][4 lanes] of 16 bytes (8 columns), a piece is half of
// them.  16-bit rows on 16-byte boundaries are copied as they lie, all in flight at once.
template <bool SPLIT>
__device__ __forceinline__ void q4_values(const Q4Args &a, int tile0, int tiles,
                                          unsigned char *xs) {
  if (!SPLIT && a.x_vec == 2) {
    for (int i = threadIdx.x; i < tiles * a.rows * 8; i += blockDim.x) {
      const int row = (i >> 3) / tiles, kt = (i >> 3) - row * tiles, q = i & 7;
      const int k = (tile0 + kt) * Q4_COLS + 8 * q;
      const int bytes = max(0, min(16, (a.K - k) * 2));  // the rest is filled with zeros
      const unsigned short *from =
          static_cast<const unsigned short *>(a.x) + (bytes ? row * a.ldx + k : 0);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(
                       (uint32_t)__cvta_generic_to_shared(
                           xs + ((size_t)(2 * kt + (q >> 2)) * a.cols + row) * 64 + (q & 3) * 16)),
                   "l"(from), "r"(bytes)
                   : "memory");
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
    return;
  }
  q4_each_piece(a, tile0, tiles, [&](bool on, int kt, int row, int q, const uint4 &v) {
    if (!on) return;
    unsigned char *o =
        xs + (size_t)(2 * kt + (q >> 3)) * a.cols * 64 + ((q >> 1) & 3) * 16 + (q & 1) * 8;
    if (!SPLIT) {
      *reinterpret_cast<uint2 *>(o + row * 64) = make_uint2(v.x, v.y);
    } else {
      // truncations: v = hi + mid + lo, each with 8 significant bits; an
      // infinity or NaN stays in the first plane
      const uint32_t x[4] = {v.x, v.y, v.z, v.w};
      uint32_t hi[4], mid[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        hi[e] = x[e] & 0xffff0000u;
        const bool finite = (hi[e] & 0x7f800000u) != 0x7f800000u;
        const float r1 = finite ? __uint_as_float(x[e]) - __uint_as_float(hi[e]) : 0.0f;
        mid[e] = __float_as_uint(r1) & 0xffff0000u;
        lo[e] = __float_as_uint(r1 - __uint_as_float(mid[e]));
        if (!finite && (x[e] & 0x7fffffu)) hi[e] |= 0x400000u;  // a NaN stays one
      }
      auto put = [&](int plane, const uint32_t (&y)[4]) {
        *reinterpret_cast<uint2 *>(o + (3 * row + plane) * 64) =
            make_uint2(__byte_perm(y[0], y[1], 0x7632), __byte_perm(y[2], y[3], 0x7632));
      };
      put(0, hi);
      put(1, mid);
      put(2, lo);
    }
  });
}

// x as digits: digits [tile][8 NT][4 lanes][4 words] of 4 bytes (a word's columns 0, 2,
// 1, 3: the order of its nibbles), factor [tile][8 NT] = 256^plane
// 2^-sh.  Columns past the last one are zero.  A NaN among x makes every sum of its row
// and tile NaN by plane 0's factor.  Infinities are no digits: their sum must not cancel
// before it is infinite.  They leave +-1 in plane 0 under a factor of -0, which marks them
// for q4_infinite.  Returns whether this thread met infinities.
template <int NT>
__device__ __forceinline__ bool q4_digits(const Q4Args &a, int tile0, int tiles,
                                          unsigned char *digits, float *factor) {
  bool infinite = false;
  const int idle = 2 * NT - a.rows;  // rows past the last one
  for (int i = threadIdx.x; i < tiles * idle * 16; i += blockDim.x) {
    const int kt = (i >> 4) / idle, c = 4 * a.rows + (((i >> 4) - kt * idle) << 2);
    reinterpret_cast<uint4 *>(digits)[(kt * 8 * NT + c) * 4 + (i & 15)] = make_uint4(0, 0, 0, 0);
    if ((i & 15) < 4) factor[kt * 8 * NT + c + (i & 3)] = 0.0f;
  }
  q4_each_piece(a, tile0, tiles, [&](bool on, int kt, int row, int q, const uint4 &raw) {
    float v[4] = {__uint_as_float(raw.x), __uint_as_float(raw.y), __uint_as_float(raw.z),
                  __uint_as_float(raw.w)};
    if (a.dtype == B2F_BF16) {
      v[0] = __uint_as_float(raw.x << 16), v[1] = __uint_as_float(raw.x & 0xffff0000u);
      v[2] = __uint_as_float(raw.y << 16), v[3] = __uint_as_float(raw.y & 0xffff0000u);
    } else if (a.dtype == B2F_F16) {
      const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&raw.x));
      const float2 hi = __half22float2(*reinterpret_cast<const __half2 *>(&raw.y));
      v[0] = lo.x, v[1] = lo.y, v[2] = hi.x, v[3] = hi.y;
    }
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
#pragma unroll
    for (int o = 8; o; o >>= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
    // top < 2^(e - 126): X = round(x 2^sh), sh = 156 - e, |X| <= 2^30 (sh at most
    // 126: what is lost lies below 2^-127).  Byte p of X + 0x80808080 is digit p + 128,
    // so that sum xor 0x80808080 holds the four signed digits.
    const int e = (int)(top >> 23);
    const int sh = min(156 - e, 126);
    const float up = __uint_as_float((uint32_t)(127 + sh) << 23);
    uint32_t D[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int X = __float2int_rn(v[j] * up);
      if (e == 255)
        X = (__float_as_uint(v[j]) & 0x7fffffffu) == 0x7f800000u ? (v[j] > 0 ? 1 : -1) : 0;
      D[j] = ((uint32_t)X + 0x80808080u) ^ 0x80808080u;
    }
    // bytes of plane p: columns 0, 2, 1, 3
    const uint32_t a01 = __byte_perm(D[0], D[2], 0x5140), a23 = __byte_perm(D[0], D[2], 0x7362);
    const uint32_t b01 = __byte_perm(D[1], D[3], 0x5140), b23 = __byte_perm(D[1], D[3], 0x7362);
    if (!on) return;
    uint32_t *o = reinterpret_cast<uint32_t *>(digits) +
                  ((kt * 8 * NT + row * 4) * 4 + ((q >> 1) & 3)) * 4 + 2 * (q >> 3) + (q & 1);
    o[0] = __byte_perm(a01, b01, 0x5410);
    o[16] = __byte_perm(a01, b01, 0x7632);
    o[32] = __byte_perm(a23, b23, 0x5410);
    o[48] = __byte_perm(a23, b23, 0x7632);
    if (q < 4) {
      float x = __uint_as_float((uint32_t)max(127 + 8 * q - sh, 1) << 23);
      if (e == 255) {
        x = q ? 0.0f : top == 0x7f800000u ? -0.0f : __uint_as_float(top);
        infinite |= top == 0x7f800000u;
      }
      factor[kt * 8 * NT + row * 4 + q] = x;
    }
  });
  return infinite;
}

// What the infinities of row b of x among a block's tiles make of the sums of weight rows g
// and g + 8 of row block rb: in each tile and group an infinity of the sign that all its
// products have, or NaN where they differ or one has a zero weight; 0 without infinities.
template <int NT, bool ZERO, bool G32, bool SB>
__device__ __noinline__ float2 q4_infinite(const Q4Args &a, int rb, int b, int tile0, int tiles,
                                           const unsigned char *digits, const float *factor) {
  constexpr int REC = q4_record(G32, ZERO), SUB = G32 ? 2 : 1;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float2 sum = make_float2(0.0f, 0.0f);
  for (int kt = 0; kt < tiles; ++kt) {
    const int col = kt * 8 * NT + 4 * b;
    if (__float_as_uint(factor[col]) != 0x80000000u) continue;
    const unsigned char *p = a.packed + ((long long)rb * a.tiles_k + tile0 + kt) * REC;
    const uint4 c = reinterpret_cast<const uint4 *>(p)[lane];
    const uint4 d = reinterpret_cast<const uint4 *>(digits)[col * 4 + t];
    const uint32_t code[4] = {c.x, c.y, c.z, c.w}, mark[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      int z0 = 8, z1 = 8;
      if (ZERO) {
        const uint16_t z = reinterpret_cast<const uint16_t *>(p + q4_zeros_at(G32))[8 * u + g];
        z0 = z & 255, z1 = z >> 8;
      }
      uint32_t seen = 0;  // 1: positive products, 2: negative, 4: of nothing; << 3 for row g + 8
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        if (G32 && u != m / 2) continue;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int sign = (int)(signed char)(mark[m] >> (8 * k));
          const int p0 = sign * ((int)((code[m] >> (8 * k)) & 15u) - z0);
          const int p1 = sign * ((int)((code[m] >> (8 * k + 4)) & 15u) - z1);
          if (sign)
            seen |= (p0 > 0 ? 1u : p0 < 0 ? 2u : 4u) | (p1 > 0 ? 8u : p1 < 0 ? 16u : 32u);
        }
      }
      seen |= __shfl_xor_sync(~0u, seen, 1);
      seen |= __shfl_xor_sync(~0u, seen, 2);
      if (!seen) continue;
      auto value = [](uint32_t v) { return v == 1 ? INFINITY : v == 2 ? -INFINITY : NAN; };
      const float2 s = scale_pair<SB>(reinterpret_cast<const uint32_t *>(p + 512)[8 * u + g]);
      sum.x += s.x * value(seen & 7u);
      sum.y += s.y * value(seen >> 3);
    }
  }
  return sum;
}

// first [tile][SUB][4 NT]: the accumulators' first values of two columns, twice (-8 sum
// X on kSumBase; with zero points sum X), from the digits.
template <int NT, bool ZERO, bool G32>
__device__ __forceinline__ void q4_first(int tiles, const unsigned char *digits, int *first) {
  constexpr int SUB = G32 ? 2 : 1;
  for (int i = threadIdx.x; i < tiles * 8 * NT; i += blockDim.x) {
    const int c = i % (8 * NT), kt = i / (8 * NT);
    int sum[2] = {0, 0};
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int4 d = *reinterpret_cast<const int4 *>(digits + (size_t)i * 64 + t * 16);
      sum[0] = __dp4a(d.x, 0x01010101, __dp4a(d.y, 0x01010101, sum[0]));
      sum[1] = __dp4a(d.z, 0x01010101, __dp4a(d.w, 0x01010101, sum[1]));
    }
    if (!G32) sum[0] += sum[1];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      int *f = first + ((kt * SUB + u) * 4 * NT + c / 2) * 4 + (c & 1);
      f[0] = f[2] = ZERO ? sum[u] : kSumBase - 8 * sum[u];
    }
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

constexpr int q4_batch(int nt) { return 4 / nt; }

// How x enters the products: in its own type, split into three of bf16, or as
// four digits of 8 bits.
enum Q4Rows { Q4_SAME, Q4_SPLIT, Q4_DIGITS };
constexpr int q4_max_warps(Q4Rows how) { return how == Q4_DIGITS ? 8 : 16; }
// shared memory of one tile of x, of the digits with first sums and factors
constexpr int q4_digit_bytes(int nt) { return 512 * nt; }
constexpr int q4_tile_bytes(bool digits, bool g32, int nt, int cols) {
  return digits ? q4_digit_bytes(nt) + ((g32 ? 2 : 1) * 64 + 32) * nt : cols * 128;
}

// Infinities join y when all else is there, a row block to a warp and a cluster's blocks one
// after the other.  Within the loop over the records, on its registers, they cost four rows
// of 128256 x 4096 14 us of 84 without one infinity among them.  A call, and ids read again,
// leave the loop its registers: one to four rows take as long as without (zero points: 1 %).
template <int NT, bool ZERO, bool G32, bool SB>
__device__ __forceinline__ void q4_join_infinite(const Q4Args &a) {
  extern __shared__ __align__(16) unsigned char q4_smem[];
  const unsigned char *xs = q4_smem + 16;
  const float *factor =
      reinterpret_cast<const float *>(xs + (size_t)a.block_tiles *
                                               (q4_digit_bytes(NT) + (G32 ? 2 : 1) * 64 * NT));
  const int cs = a.cluster;
  if (cs == 1) {
    __syncthreads();
    if (!*reinterpret_cast<volatile int *>(q4_smem)) return;
  }
  uint32_t tid, block_id;
  asm volatile("mov.u32 %0, %%tid.x;\n" : "=r"(tid));
  asm volatile("mov.u32 %0, %%ctaid.x;\n" : "=r"(block_id));
  const int warp = __shfl_sync(~0u, tid >> 5, 0), lane = tid & 31, warps = blockDim.x >> 5;
  const int rank = cs == 1 ? 0 : (int)cluster_rank();
  const int row_blocks = (a.N + Q4_ROWS - 1) / Q4_ROWS, wr = a.warps_r;
  const int stride = gridDim.x / cs * wr, tile0 = rank * a.block_tiles;
  const int tiles = max(0, min(a.block_tiles, a.tiles_k - tile0));
  auto add = [](auto *y, float v) { *y = (std::remove_pointer_t<decltype(y)>)((float)*y + v); };
#pragma unroll 1
  for (int turn = 0; turn < cs; ++turn) {
    if (turn == rank && *reinterpret_cast<volatile int *>(q4_smem)) {
#pragma unroll 1
      for (int i = warp, b0 = (int)block_id / cs * wr;; i += warps) {
        while (i >= wr && b0 < row_blocks) i -= wr, b0 += stride;
        if (b0 >= row_blocks) break;
        if (b0 + i >= row_blocks) continue;
#pragma unroll 1
        for (int b = 0; b < a.rows; ++b) {
          const float2 v = q4_infinite<NT, ZERO, G32, SB>(a, b0 + i, b, tile0, tiles, xs, factor);
          const long long n = (long long)(b0 + i) * Q4_ROWS + (lane >> 2), at = b * a.ldy + n;
#pragma unroll 1
          for (int r = 0; r < 2; ++r) {
            const float w = r ? v.y : v.x;
            if ((lane & 3) != 0 || w == 0.0f || n + 8 * r >= a.N) continue;
            if (a.out_f32 || a.dtype == B2F_F32)
              add(static_cast<float *>(a.y) + at + 8 * r, w);
            else if (a.dtype == B2F_F16)
              add(static_cast<__half *>(a.y) + at + 8 * r, w);
            else
              add(static_cast<__nv_bfloat16 *>(a.y) + at + 8 * r, w);
          }
        }
      }
    }
    if (cs > 1) meet(cs);
  }
}

// In round i cluster c takes the warps_r row blocks from (c + i clusters) warps_r on;
// block r of a cluster takes tiles [r block_tiles, (r + 1) block_tiles) of them, warp
// (r, k) of a block the chunks of TPW tiles k, k + warps_k, ... of row block r.  NT:
// 8-column tiles of x (planes counted).  Shared memory: 16 bytes of zeros, x
// [block_tiles][2][cols][4 lanes] of 16 bytes (digits: what q4_digits and q4_first
// write), then two buffers of sums [q4_batch(NT)][warps][16][8 NT] and, for clusters, of
// a block's totals [q4_batch(NT)][warps_r][rows][16]: the warps meet once per q4_batch
// rounds.
template <class T, Q4Rows HOW, int NT, int TPW, bool ZERO, bool G32, bool SB>
__global__ void __launch_bounds__(32 * q4_max_warps(HOW), HOW == Q4_DIGITS ? 2 : 1)
    q4_matvec_kernel(const Q4Args a) {
  constexpr bool SPLIT = HOW == Q4_SPLIT, INT = HOW == Q4_DIGITS;
  extern __shared__ __align__(16) unsigned char q4_smem[];
  unsigned char *xs = q4_smem + 16;
  int *first = reinterpret_cast<int *>(xs + (size_t)a.block_tiles * q4_digit_bytes(NT));
  float *factor = reinterpret_cast<float *>(first + a.block_tiles * (G32 ? 2 : 1) * 16 * NT);
  float *sums = reinterpret_cast<float *>(
      xs + (size_t)a.block_tiles * q4_tile_bytes(INT, G32, NT, a.cols));
  float *joined = sums + 2 * q4_batch(NT) * (blockDim.x >> 5) * Q4_ROWS * 8 * NT;
  constexpr int SUMS = Q4_ROWS * 8 * NT, REC = q4_record(G32, ZERO), SUB = G32 ? 2 : 1;
  constexpr int BATCH = q4_batch(NT);
  // the same in every lane, and known to be: its branches need no reconvergence
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int cs = a.cluster, rank = cs == 1 ? 0 : (int)cluster_rank();
  const int row_blocks = (a.N + Q4_ROWS - 1) / Q4_ROWS;
  const int wk = a.warps_k, wr = a.warps_r, warp_r = warp / wk, warp_k = warp - warp_r * wk;
  const int first_rb = blockIdx.x / cs * wr, stride = gridDim.x / cs * wr;
  const int tile0 = rank * a.block_tiles;
  const int tiles = max(0, min(a.block_tiles, a.tiles_k - tile0));
  const int chunks = (tiles + TPW - 1) / TPW;

  int rb = first_rb + warp_r, chunk = warp_k;
  uint4 w[TPW];
  uint32_t sc[TPW][SUB];
  uint16_t zr[TPW][SUB];
  const unsigned char *rec = nullptr;  // the next visit's first record
  int have = 0;                        // its tiles
  auto aim = [&](int r, int c) {
    have = r < row_blocks ? min(TPW, tiles - c * TPW) : 0;
    rec = a.packed + ((long long)r * a.tiles_k + tile0 + c * TPW) * REC;
  };
  auto fetch = [&](int i) {
    const unsigned char *p = rec + i * REC;
    w[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + lane);
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      sc[i][u] = __ldcs(reinterpret_cast<const uint32_t *>(p + 512) + 8 * u + g);
      if (ZERO)
        zr[i][u] = __ldcs(reinterpret_cast<const uint16_t *>(p + q4_zeros_at(G32)) + 8 * u + g);
    }
  };
  aim(rb, chunk);
#pragma unroll
  for (int i = 0; i < TPW; ++i)
    if (i < have) fetch(i);

  if (threadIdx.x == 0) *reinterpret_cast<uint4 *>(q4_smem) = make_uint4(0, 0, 0, 0);
  if constexpr (INT) {
    const int infinite = __syncthreads_or(q4_digits<NT>(a, tile0, tiles, xs, factor));
    if (threadIdx.x == 0) reinterpret_cast<uint4 *>(q4_smem)->x = infinite;
    q4_first<NT, ZERO, G32>(tiles, xs, first);
  } else {
    q4_values<SPLIT>(a, tile0, tiles, xs);
  }
  __syncthreads();

  // this lane's operands of a tile: two reads x_half apart, tiles x_tile apart;
  // a lane past the last column stays on the zeros
  int x_first[NT], x_half[NT], x_tile[NT];
  float tot[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const bool on = 8 * j + g < a.cols;
    x_first[j] = on ? 16 + ((8 * j + g) * 4 + t) * 16 : 0;
    x_half[j] = on ? a.cols * 64 : 0;
    x_tile[j] = on ? a.cols * 128 : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) tot[j][i] = 0.0f;
  }

  int xo[NT];
  // a chunk's digits, first sums and factors of this lane
  const unsigned char *dp = nullptr;
  const int4 *cp = nullptr;
  const float2 *fp = nullptr;
  auto consume_digits = [&](int i) {
    const uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const uint4 xv = *reinterpret_cast<const uint4 *>(dp + (i * NT + j) * 512);
      const float2 f = fp[(i * NT + j) * 4];
      int acc[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int u = G32 ? h : 0;
        if (G32 || h == 0) {
          const int4 c = cp[((i * SUB + u) * NT + j) * 4];
          acc[0] = c.x, acc[1] = c.y, acc[2] = c.z, acc[3] = c.w;
          if (ZERO) {
            const int z0 = zr[i][u] & 255, z1 = zr[i][u] >> 8;
            acc[0] = kSumBase - z0 * c.x, acc[1] = kSumBase - z0 * c.y;
            acc[2] = kSumBase - z1 * c.x, acc[3] = kSumBase - z1 * c.y;
          }
        }
        mma_16832(acc, v[2 * h] & 0x0f0f0f0fu, (v[2 * h] >> 4) & 0x0f0f0f0fu,
                  v[2 * h + 1] & 0x0f0f0f0fu, (v[2 * h + 1] >> 4) & 0x0f0f0f0fu,
                  h ? xv.z : xv.x, h ? xv.w : xv.y, acc);
        if (G32 || h == 1) {
          const float2 s = scale_pair<SB>(sc[i][u]);
          constexpr float base = 12582912.0f;  // kSumBase
          tot[j][0] += (s.x * f.x) * (__int_as_float(acc[0]) - base);
          tot[j][1] += (s.x * f.y) * (__int_as_float(acc[1]) - base);
          tot[j][2] += (s.y * f.x) * (__int_as_float(acc[2]) - base);
          tot[j][3] += (s.y * f.y) * (__int_as_float(acc[3]) - base);
        }
      }
    }
  };
  auto consume_values = [&](int i) {
    const uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
    uint4 xv[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      xv[j][0] = *reinterpret_cast<const uint4 *>(q4_smem + xo[j]);
      xv[j][1] = *reinterpret_cast<const uint4 *>(q4_smem + xo[j] + x_half[j]);
      xo[j] += x_tile[j];
    }
    float acc[NT][4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int u = G32 ? m / 2 : 0;
      uint32_t bz0 = kNibbleBase<T> + 0x00080008u, bz1 = bz0;
      if (ZERO) {
        bz0 = kNibbleBase<T> + (zr[i][u] & 0xffu) * 0x00010001u;
        bz1 = kNibbleBase<T> + (uint32_t)(zr[i][u] >> 8) * 0x00010001u;
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
      if (m == 3 || (G32 && m == 1)) {  // the sums of the record's (half's) group
        const float2 s = scale_pair<SB>(sc[i][u]);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          tot[j][0] += s.x * acc[j][0];
          tot[j][1] += s.x * acc[j][1];
          tot[j][2] += s.y * acc[j][2];
          tot[j][3] += s.y * acc[j][3];
        }
      }
    }
  };

  auto consume = [&](int i) {
    if constexpr (INT)
      consume_digits(i);
    else
      consume_values(i);
  };

  int buf = 0, met = 0;
  for (int lead = first_rb; lead < row_blocks; lead += stride, rb += stride) {
    while (rb < row_blocks && chunk < chunks) {
      const int now = have;
#pragma unroll
      for (int j = 0; j < NT; ++j) xo[j] = x_first[j] + chunk * TPW * x_tile[j];
      if (INT) {
        dp = xs + chunk * TPW * q4_digit_bytes(NT) + lane * 16;
        cp = reinterpret_cast<const int4 *>(first) + chunk * TPW * SUB * 4 * NT + t;
        fp = reinterpret_cast<const float2 *>(factor) + chunk * TPW * 4 * NT + t;
      }
      if (chunk + wk < chunks)
        aim(rb, chunk + wk);
      else
        aim(rb + stride, warp_k);
      if (now == TPW && have == TPW) {  // a full chunk, and another one follows
#pragma unroll
        for (int i = 0; i < TPW; ++i) {
          consume(i);
          fetch(i);
        }
      } else {
#pragma unroll
        for (int i = 0; i < TPW; ++i) {
          if (i < now) consume(i);
          if (i < have) fetch(i);
        }
      }
      chunk += wk;
    }
    chunk = warp_k;
    // c0, c1: row g, columns 2t, 2t + 1; c2, c3: row g + 8
    float *out = sums + ((buf * BATCH + met) * warps + warp) * SUMS;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float *o = out + g * 8 * NT + 8 * j + 2 * t;
      *reinterpret_cast<float2 *>(o) = make_float2(tot[j][0], tot[j][1]);
      *reinterpret_cast<float2 *>(o + 8 * 8 * NT) = make_float2(tot[j][2], tot[j][3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) tot[j][i] = 0.0f;
    }
    if (++met < BATCH && lead + stride < row_blocks) continue;
    __syncthreads();
    const int per = Q4_ROWS * a.rows, round = wr * per;
    // item i of the batch: round q, row block ir of it, row b of x, weight row r
    auto put = [&](int i, float v) {
      const int q = i / round, ir = (i - q * round) / per, r = i & 15;
      const int b = (i - q * round - ir * per) >> 4;
      const int n = (lead - (met - 1 - q) * stride + ir) * Q4_ROWS + r;
      if (n >= a.N) return;
      const long long at = b * a.ldy + n;
      if (SPLIT || a.out_f32 || (INT && a.dtype == B2F_F32))
        static_cast<float *>(a.y)[at] = v;
      else if (INT && a.dtype == B2F_F16)
        static_cast<__half *>(a.y)[at] = __float2half_rn(v);
      else
        static_cast<T *>(a.y)[at] = (T)v;
    };
    for (int i = threadIdx.x; i < met * round; i += blockDim.x) {
      const int q = i / round, ir = (i - q * round) / per, r = i & 15;
      const int b = (i - q * round - ir * per) >> 4;
      const float *s = sums + ((buf * BATCH + q) * warps + ir * wk) * SUMS + r * 8 * NT;
      float v = 0.0f;
#pragma unroll 4
      for (int u = 0; u < wk; ++u, s += SUMS) {
        if (INT)  // small digits first; what is not finite is in plane 0 alone
          v += s[4 * b + 3] + (s[4 * b + 2] + (s[4 * b + 1] + s[4 * b]));
        else if (SPLIT)
          v += s[3 * b] + (s[3 * b + 2] + s[3 * b + 1]);
        else
          v += s[b];
      }
      if (cs == 1)
        put(i, v);
      else
        joined[buf * BATCH * round + i] = v;
    }
    if (cs > 1) {
      meet(cs);
      for (int i = threadIdx.x + rank * blockDim.x; i < met * round; i += cs * blockDim.x) {
        float v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c)
          v[c] = c < cs ? remote_f32(joined + buf * BATCH * round + i, c) : 0.0f;
        put(i, ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])));
      }
    }
    met = 0;
    buf ^= 1;
  }
  if (cs > 1) meet(cs);  // no block leaves while its sums are read
  if constexpr (INT) q4_join_infinite<NT, ZERO, G32, SB>(a);
}

// codes [N][K] (one byte each), scales and zero points [N][groups] -> records.
// A warp writes one record: 4 words of codes a lane, then the scales and zeros.
__global__ void q4_pack_kernel(const uint8_t *__restrict__ codes,
                               const uint16_t *__restrict__ scales,
                               const uint8_t *__restrict__ zeros, int N, int K, int tiles_k,
                               int group, int groups, int record,
                               unsigned char *__restrict__ packed) {
  const long long tile = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const int row_blocks = (N + Q4_ROWS - 1) / Q4_ROWS;
  if (tile >= (long long)row_blocks * tiles_k) return;
  const int kt = (int)(tile % tiles_k), rb = (int)(tile / tiles_k);
  unsigned char *out = packed + tile * record;
  const int g = lane >> 2, t = lane & 3;
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int nib = 0; nib < 8; ++nib) {
      const int row = rb * Q4_ROWS + g + 8 * (nib & 1);
      const int col = kt * Q4_COLS + 32 * (m >> 1) + 8 * t + 4 * (m & 1) + (nib & 2) + (nib >> 2);
      const uint32_t c = row < N && col < K ? codes[(long long)row * K + col] & 15u : 8u;
      v[m] |= c << (4 * nib);
    }
  reinterpret_cast<uint4 *>(out)[lane] = make_uint4(v[0], v[1], v[2], v[3]);
  const int sub = group == 32 ? 2 : 1;
  if (lane < 16 * sub) {
    const int u = lane >> 4, r = rb * Q4_ROWS + ((lane & 15) >> 1) + 8 * (lane & 1);
    const int grp = group == 32 ? 2 * kt + u : kt / (group / 64);
    const bool in = r < N && grp < groups;  // zero scales past the weight
    reinterpret_cast<uint16_t *>(out + 512)[lane] = in ? scales[(long long)r * groups + grp] : 0;
    if (zeros)
      out[q4_zeros_at(sub == 2) + lane] = in ? zeros[(long long)r * groups + grp] & 15u : 8u;
  }
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

template <class T, Q4Rows HOW, int NT, bool ZERO, bool G32, bool SB>
int launch_matvec(Q4Args a, int dev, int sms, cudaStream_t s) {
  constexpr int TPW = NT > 1 || G32 ? 4 : 8;
  constexpr bool INT = HOW == Q4_DIGITS;
  B2F_CHECK_ARG(a.cols <= 8 * NT, "b2f_q4_matvec: %d columns of the product, %d fit", a.cols,
                8 * NT);
  auto k = q4_matvec_kernel<T, HOW, NT, TPW, ZERO, G32, SB>;
  constexpr int most = q4_max_warps(HOW);
  static std::atomic<uint64_t> allowed{0};
  if (int rc = allow_shared(k, (int)kQ4Smem, dev, allowed)) return rc;
  static const int regs = [&] {  // of a thread, as compiled
    cudaFuncAttributes f{};
    return cudaFuncGetAttributes(&f, k) == cudaSuccess ? (f.numRegs + 7) / 8 * 8 : 255;
  }();
  const int row_blocks = (a.N + Q4_ROWS - 1) / Q4_ROWS;
  auto smem_of = [&](int warps_k, int warps_r) {
    return 16 + (size_t)a.block_tiles * q4_tile_bytes(INT, G32, NT, a.cols) +
           (size_t)2 * q4_batch(NT) * warps_r * Q4_ROWS *
               (warps_k * 8 * NT + (a.cluster > 1 ? a.rows : 0)) * 4;
  };
  // the fewest blocks whose shares of x fit shared memory
  for (a.cluster = 1;; a.cluster *= 2) {
    a.block_tiles = (a.tiles_k + a.cluster - 1) / a.cluster;
    const int chunks = (a.block_tiles + TPW - 1) / TPW, visits = (chunks + most - 1) / most;
    a.warps_k = (chunks + visits - 1) / visits;
    if (smem_of(a.warps_k, 1) <= kQ4Smem) break;
    B2F_CHECK_ARG(a.cluster < 8, "b2f_q4_matvec: %d columns of %d values do not fit", a.cols, a.K);
  }
  auto blocks_of = [&](int warps_r) {  // blocks of an SM, 0: does not fit
    return std::min<int>((int)(kQ4Smem / smem_of(a.warps_k, warps_r)),
                         65536 / (regs * 32 * a.warps_k * warps_r));
  };
  // as many row blocks at once as the warps allow and the row blocks fill
  a.warps_r = most / a.warps_k;
  while (a.warps_r > 1 && blocks_of(a.warps_r) < 1) --a.warps_r;
  const int at_once = std::max(1, sms * std::max(1, blocks_of(a.warps_r)) / a.cluster);
  a.warps_r = std::min(a.warps_r, (row_blocks + at_once - 1) / at_once);
  const int warps = a.warps_k * a.warps_r;
  const int clusters = std::min((row_blocks + a.warps_r - 1) / a.warps_r,
                                std::max(1, sms * std::max(1, blocks_of(a.warps_r)) / a.cluster));
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(clusters * a.cluster);
  c.blockDim = dim3(32 * warps);
  c.dynamicSmemBytes = smem_of(a.warps_k, a.warps_r);
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
template <class T, Q4Rows HOW, int NT>
int launch_cols(const Q4Args &a, bool zero, bool g32, bool sb, int dev, int sms, cudaStream_t s) {
  if (zero && g32)
    return sb ? launch_matvec<T, HOW, NT, true, true, true>(a, dev, sms, s)
              : launch_matvec<T, HOW, NT, true, true, false>(a, dev, sms, s);
  if (zero)
    return sb ? launch_matvec<T, HOW, NT, true, false, true>(a, dev, sms, s)
              : launch_matvec<T, HOW, NT, true, false, false>(a, dev, sms, s);
  if (g32)
    return sb ? launch_matvec<T, HOW, NT, false, true, true>(a, dev, sms, s)
              : launch_matvec<T, HOW, NT, false, true, false>(a, dev, sms, s);
  return sb ? launch_matvec<T, HOW, NT, false, false, true>(a, dev, sms, s)
            : launch_matvec<T, HOW, NT, false, false, false>(a, dev, sms, s);
}
// Up to four binary32 rows, or one or two of a 16-bit type, as digits where every block
// has row blocks enough to spread their set-up over, else in their own type or split.
// Digits against the other, us: one binary32 row of 4096 columns for 8192 weight rows 10.1
// and 9.6, for 14336 12.1 and 13.1, for 128256 47.5 and 58.2; four 23.0 and 19.6 (14336),
// 32.6 and 32.9 (32768), 84 and 107 (128256); one bf16 row 18.1 and 19.7 (32768), 48.0 and
// 57.9 (128256), but three and four 79 and 60, 84 and 63.
int launch_rows(Q4Args a, bool zero, bool g32, bool sb, int dev, int sms, cudaStream_t s) {
  using B = __nv_bfloat16;
  const int nt = a.rows <= 2 ? 1 : 2;
  const size_t digits = (size_t)((a.tiles_k + 7) / 8) * q4_tile_bytes(true, g32, nt, 0) + 49168;
  const int spread = (a.N + Q4_ROWS - 1) / Q4_ROWS / sms;
  const bool wide = a.dtype == B2F_F32;
  if (a.rows <= (wide ? 4 : 2) && spread >= (wide && a.rows <= 2 ? 6 : 12) && digits <= kQ4Smem) {
    a.cols = 4 * a.rows;
    return a.rows <= 2 ? launch_cols<B, Q4_DIGITS, 1>(a, zero, g32, sb, dev, sms, s)
                       : launch_cols<B, Q4_DIGITS, 2>(a, zero, g32, sb, dev, sms, s);
  }
  if (a.dtype == B2F_F32) {
    a.cols = 3 * a.rows;
    return a.cols <= 8 ? launch_cols<B, Q4_SPLIT, 1>(a, zero, g32, sb, dev, sms, s)
                       : launch_cols<B, Q4_SPLIT, 2>(a, zero, g32, sb, dev, sms, s);
  }
  a.cols = a.rows;
  if (a.dtype == B2F_F16)
    return a.cols <= 8    ? launch_cols<__half, Q4_SAME, 1>(a, zero, g32, sb, dev, sms, s)
                          : launch_cols<__half, Q4_SAME, 2>(a, zero, g32, sb, dev, sms, s);
  return a.cols <= 8    ? launch_cols<B, Q4_SAME, 1>(a, zero, g32, sb, dev, sms, s)
                        : launch_cols<B, Q4_SAME, 2>(a, zero, g32, sb, dev, sms, s);
}

int check_shape(const char *who, int64_t N, int64_t K, int group) {
  // 131072 columns: 8 blocks' shared memory holds a binary32 row of them
  B2F_CHECK_ARG(N >= 1 && N <= (1ll << 30) && K >= 1 && K <= (1ll << 17),
                "%s: weight of %lld x %lld (up to 131072 columns)", who, (long long)N,
                (long long)K);
  B2F_CHECK_ARG(group == 32 || (group >= 64 && group % 64 == 0),
                "%s: group of %d (32 or a multiple of 64)", who, group);
  return B2F_OK;
}

}  // namespace
}  // namespace b2f

extern "C" {

size_t b2f_q4_packed_bytes(int64_t N, int64_t K, int group, int zeros) {
  if (N < 1 || K < 1) return 0;
  return (size_t)((N + 15) / 16) * (size_t)((K + 63) / 64) *
         (size_t)b2f::q4_record(group == 32, zeros != 0);
}

int b2f_q4_pack(const uint8_t *codes, const void *scales, const uint8_t *zeros, int64_t N,
                int64_t K, int group, void *packed, void *stream) {
  B2F_RANGE("b2f_q4_pack");
  using namespace b2f;
  if (int rc = check_shape("b2f_q4_pack", N, K, group)) return rc;
  B2F_CHECK_ARG(codes && scales && packed, "b2f_q4_pack: null argument");
  B2F_CHECK_ARG((uintptr_t)packed % 32 == 0 && (uintptr_t)scales % 2 == 0,
                "b2f_q4_pack: misaligned buffer (32 bytes)");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int tiles_k = (int)((K + 63) / 64), groups = (int)((K + group - 1) / group);
  const long long records = (N + 15) / 16 * tiles_k;
  q4_pack_kernel<<<(unsigned)((records + 7) / 8), 256, 0, s>>>(
      codes, static_cast<const uint16_t *>(scales), zeros, (int)N, (int)K, tiles_k, group, groups,
      q4_record(group == 32, zeros != nullptr), static_cast<unsigned char *>(packed));
  B2F_LAUNCHED("q4_pack_kernel");
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
                  int scale_dtype, int zeros, int64_t N, int64_t K, int group, void *y,
                  int out_f32, void *stream) {
  B2F_RANGE("b2f_q4_matvec");
  using namespace b2f;
  if (int rc = check_shape("b2f_q4_matvec", N, K, group)) return rc;
  B2F_CHECK_ARG(rows >= 0 && rows <= 1024, "b2f_q4_matvec: %lld rows (up to 1024)",
                (long long)rows);
  B2F_CHECK_ARG(dtype >= B2F_F32 && dtype <= B2F_BF16, "b2f_q4_matvec: dtype %d", dtype);
  B2F_CHECK_ARG(scale_dtype == B2F_F16 || scale_dtype == B2F_BF16,
                "b2f_q4_matvec: scale dtype %d", scale_dtype);
  if (rows == 0) return B2F_OK;
  B2F_CHECK_ARG(x && packed && y, "b2f_q4_matvec: null argument");
  B2F_CHECK_ARG(ldx >= K || rows == 1, "b2f_q4_matvec: rows of %lld, %lld apart", (long long)K,
                (long long)ldx);
  const int esize = dtype == B2F_F32 ? 4 : 2;
  B2F_CHECK_ARG((uintptr_t)packed % 32 == 0 && (uintptr_t)x % esize == 0 &&
                    (uintptr_t)y % (out_f32 ? 4 : esize) == 0,
                "b2f_q4_matvec: misaligned buffer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int dev = 0, sms = 0;
  if (int rc = current_device(&dev, &sms)) return rc;
  Q4Args a{};
  a.packed = static_cast<const unsigned char *>(packed);
  a.ldx = ldx;
  a.ldy = N;
  a.N = (int)N;
  a.K = (int)K;
  a.tiles_k = (int)((K + 63) / 64);
  a.out_f32 = out_f32 != 0;
  // 4 values at once, or (16-bit types) 8
  a.x_vec = (uintptr_t)x % (4 * esize) == 0 && (rows == 1 || ldx % 4 == 0);
  if (a.x_vec && esize == 2 && (uintptr_t)x % 16 == 0 && (rows == 1 || ldx % 8 == 0)) a.x_vec = 2;
  a.dtype = dtype;
  // rows in one pass: 4 of binary32 (8 of them as 24 columns took 217 us against 2 x 84
  // for 128256 weight rows), up to 16 of 16 bits (17 as 32 columns: 190 us, 16 of them:
  // 118), no more than 8 blocks' shared memory holds of x (72 KB of each kept for the
  // sums), and of 16 bits no more than two hold unless that is less than 8 rows (16 rows of
  // 14336 columns at once, on four blocks: 44 us, as 8 and 8: 2 x 17); the passes share the
  // rows out evenly
  auto fit = [&](int blocks) {
    return blocks * (long long)(kQ4Smem - 72 * 1024) / (128ll * (a.tiles_k + 8));
  };
  const long long most = dtype == B2F_F32 ? std::min(4ll, fit(8) / 3)
                                          : std::min(16ll, std::max(fit(2), std::min(8ll, fit(8))));
  const int64_t passes = (rows + most - 1) / most;
  const int step = (int)((rows + passes - 1) / passes);
  for (int64_t r0 = 0; r0 < rows; r0 += step) {
    a.rows = (int)std::min<int64_t>(step, rows - r0);
    a.x = static_cast<const char *>(x) + r0 * ldx * esize;
    a.y = static_cast<char *>(y) + r0 * N * (out_f32 ? 4 : esize);
    const int rc = launch_rows(a, zeros != 0, group == 32, scale_dtype == B2F_BF16, dev,
                               sms, s);
    if (rc) return rc;
  }
  return B2F_OK;
}

}  // extern "C"
