// Softmax cross entropy over a large vocabulary and its gradient, from hidden
// states h [T][D] and the head's weight W [V][D], without the logits z = h W^T
// [T][V] ever being kept.
//
//   lse_t  = log sum_v exp z_tv,     loss_t = lse_t - z_{t, label_t}
//   dz_tv  = g_t (exp(z_tv - lse_t) - [v = label_t])
//   dh     = dz W,                   dW = dz^T h
//
// Three matrix products on tcgen05 (bf16 or fp16 operands, binary32
// accumulators in tensor memory), one kernel template:
//   logits   A = h (K-major), B = W (K-major); the epilogue either reduces the
//            tile's columns to (max, sum of exp(z - max) - 1) per token, or turns them into
//            dz and stores that in the operand type;
//   dh       A = dz (K-major), B = W read along its rows (N-major);
//   dW       A = dz^T (M-major), B = h (N-major).
// The gradient walks the vocabulary in pieces whose dz fits a workspace: the
// logits of a piece are computed again, become dz at once, and both products
// consume it.  Ignored tokens are left out: the counted ones are gathered first,
// and the tiles are counted off from their number on the device.
//
// One block per SM: warp 0 loads tiles by TMA (128-byte swizzle) into a ring of
// stages, warp 1 issues the MMAs, 8 or 16 more read the accumulators; two
// accumulators in tensor memory let the epilogue of a tile run under the products
// of the next.  Either a block computes tiles of 128 x 256, or (dW, and the others
// with more than 128 tokens) two blocks of a cluster tiles of 256 x 256
// (cta_group::2), each loading half of both operands: 32 KB a K step instead of 48
// for as much of the product.  Outputs leave through shared memory as TMA
// stores.  Every wait is bounded: one that runs out is counted (b2f_vocab_loss_wait_errors),
// the block waits (bounded again) for its loads and products in flight, and all tiles that
// it still owes are NaN, which whatever is computed from them hands on.
//
// dz is rounded to the operand type before its two products (once from 65 tokens
// on: relative to each dz at most half a step of the type, the size of the rounding of
// the gradients themselves; what it leaves at the label joins dh and dW in binary32: it
// is shared by a token's whole row of dh, and a word that a token has as its label owes
// nearly all of its row of dW to that.  In two parts below, VL_LOW), and formed from
// p - 1 (expm1) at the label, where lse's own rounding is all that a confident token
// loses.  fp16 cannot hold g p of a rare word, so there dz is scaled by a power of two
// that brings the largest |g| to 2^14 and the products are scaled back in binary32.
//
// Measured on a 128256 x 4096 head in bf16: the score of 128 tokens 176-182 us (W read
// once at 88-91 % of copy bandwidth); a training step on them 855-905 us, its launches one by
// one 190 (logits) + 184 (dz: W again) + 156 (dh: W a third time) + 305 (dW; clearing as many
// bytes takes 350) + 23 (the small ones); a step on 4096 tokens 12.5-13.5 ms, 1.15-1.24 PFLOP/s
// over the four products of the counted tokens, under the power cap (cuBLAS sustains 1.385).
// dh, dW and the next piece's logits side by side on clusters of their own were no faster
// (672 against 660 us).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "plain.h"

namespace b2f {
namespace {

constexpr int VL_M = 128;       // rows of a block's part of a tile (TMEM lanes)
constexpr int VL_N = 256;       // columns of a tile
constexpr int VL_K = 64;        // K step: one 128-byte swizzle row
constexpr int VL_SLAB = 4096;   // 32 rows of 128 bytes that a warp stores at once
constexpr int VL_A_BYTES = VL_M * VL_K * 2;

// Shared memory of a block, CG blocks to a tile: stages of its rows of A and its share
// of B's columns, slabs of each epilogue warp, barriers.
template <int CG>
struct Block {
  static constexpr int n = VL_N / CG;  // columns of B
  static constexpr int stage = VL_A_BYTES + n * VL_K * 2;
  static constexpr int stages = CG == 1 ? 4 : 5;
  // epilogue warps, a quarter of them on each lane quarter, and the columns of each.
  // 16 of 64 columns halve the time of a tile's stores against 8 of 128 (dW of 128
  // tokens, whose products are short); beside one block's larger stages 8 fit.
  static constexpr int warps = CG == 1 ? 8 : 16;
  static constexpr int cols = VL_N * 4 / warps;
  static constexpr int threads = 32 * (2 + warps);
  static constexpr size_t smem = 1024 + (size_t)stages * stage + warps * VL_SLAB + 256;
};
static_assert(Block<1>::smem <= 227 * 1024 && Block<2>::smem <= 227 * 1024,
              "stages exceed shared memory");
// K steps of a logit that the tensor cores add up in one go: they truncate at every 16
// products, always towards zero, so the epilogue joins the sums of chunks of 512 products,
// rounded to nearest.  That takes the error of a loss of 0.2 to 0.9 over 3056 columns from
// 1.3e-5 - 2.1e-5 of it to 1.4e-6 - 2.8e-6 and costs 1.5 % of the score of 128 tokens; chunks
// of 256 halve the error again and cost 7 % (and 12 % of a step on 4096 tokens).
// Both passes over the logits cut them alike, for the errors of z and lse to cancel in dz.
constexpr int VL_CHUNK = 8;
// K steps of a gradient that they add up in one go, for the same reason: up to 1024 truncations,
// 1.2e-4 of a sum of one sign, a quarter of what rounding it to fp16 may cost.  dW of 2^20
// tokens with positive terms, in fp16, is off by 6e-5 to 9e-5 on average, in one go by 5.8e-3
// (in stretches of 1024 steps by up to 3.9e-4).
constexpr int VL_LONG = 256;
constexpr int VL_WAIT_LIMIT = 1 << 23;  // polls (each may suspend the thread for a while)
constexpr int VL_IDLE_LIMIT = 1 << 10;  // where nothing is to come (VocabArgs::idle)

__device__ int g_vocab_wait_errors;

enum Epilogue { EPI_STATS, EPI_DZ, EPI_PARTIAL, EPI_OUT };

// Up to this many tokens dz is carried as two numbers of the operand type, what the
// rounding of the first leaves in the second: rows 0 to 63 and 64 to 127 of a tile that
// would be half empty.  dh adds the two sums of a token, dW runs over both with the same
// rows of h.  The rounding of one dz, at the label, is shared by a whole row of dh and of
// dW, and over few tokens it does not average out: fp16 gradients of 8 to 64 tokens were
// off by 1.5 to 1.6 times what their own rounding costs, now by 1.0.  It takes 3 to 7 % of
// the time on a 128256 x 4096 head (508 to 523 us for dh of 64 tokens) and 5 to 8 us where
// all is latency; more tokens' dz would take a second tile and both products' time again.
constexpr int VL_LOW = 64;

// The counted tokens in the order of their labels (those of one label in their own), so
// that dW finds the tokens of its words: first[g] is the place of the first one whose label
// is 32 g or more, for g from 0 to the groups' number inclusive.  Labels outside the
// vocabulary count as its size, behind all words.
constexpr int VL_GROUP = 32;  // words that a warp of dW's epilogue holds
struct ByLabel {
  int *token, *label, *first;  // null: not wanted
  int groups;
};

// Tokens as the products see them: `rows` of the workspace, the counted ones first.
struct Counted {
  const int *count;          // how many; null: all of them
  const long long *labels;   // of the counted tokens
  const float *lse, *grad;
  const uint32_t *grad_max;  // bits of max |g| (fp16)
  const void *rows;          // [.][D]
  ByLabel by;
};

struct VocabArgs {
  int M, N, K;        // the product's sizes (M or K in tokens: at most that many)
  int splits;         // of K
  int n_first;        // logits: first word of the piece
  int k_first;        // dh: first word of the piece (row of W)
  int m_first;        // dW: first word of the piece (row of dW)
  int tokens_in_k;    // K counts tokens (dW), else M does
  int low;            // tokens, if rows VL_LOW.. of dz hold what rounding left of the others
  Counted tok;
  long long ignore;
  int vocab;
  float2 *part;       // [slots][M] (max, rest)
  float *label_logit; // [M]
  float *label_left;  // [M] what rounding left of dz at the label
  int accumulate;     // dh: add to the partial sums
  int idle;           // blocks (or pairs) from 1: this one loads nothing, its waits run out
};

// The tiles of a product, as every warp counts them off.
struct Tiles {
  int m_tiles, n_tiles, k_blocks, split_blocks, total;
};
struct Tile {
  int m, n, split;
};
// Tokens run fastest, so that the blocks at work share W's rows; dW's rows (8 KB of a
// 4096 wide head) are finished together: its columns run fastest.  dz starts from the
// last words, which the forward pass has left in L2.
template <int EPI>
__device__ __forceinline__ Tile tile_at(const Tiles &t, int i) {
  Tile r;
  if (EPI == EPI_OUT) {
    r.n = i % t.n_tiles, i /= t.n_tiles;
    r.m = i % t.m_tiles, r.split = i / t.m_tiles;
  } else {
    if (EPI == EPI_DZ) i = t.total - 1 - i;
    r.m = i % t.m_tiles, i /= t.m_tiles;
    r.n = i % t.n_tiles, r.split = i / t.n_tiles;
  }
  return r;
}
template <int CG>
__host__ __device__ inline Tiles tiles_of(const VocabArgs &a, int M, int K) {
  Tiles t;
  t.m_tiles = (M + CG * VL_M - 1) / (CG * VL_M);
  t.n_tiles = (a.N + VL_N - 1) / VL_N;
  t.k_blocks = (K + VL_K - 1) / VL_K;
  t.split_blocks = (t.k_blocks + a.splits - 1) / a.splits;
  t.total = t.m_tiles * t.n_tiles * a.splits;
  return t;
}

__device__ __forceinline__ uint32_t sptr(const void *p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void bar_init(uint64_t *bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(sptr(bar)), "r"(count));
}
__device__ __forceinline__ void bar_expect(uint64_t *bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(sptr(bar)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t *bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(sptr(bar)), "r"(parity)
      : "memory");
  return done;
}
// bounded; false when the wait ran out here or in another warp (*lost set)
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, volatile int *lost,
                                         int limit = VL_WAIT_LIMIT) {
  for (int it = 0; it < limit; ++it) {
    if (bar_try(bar, parity)) return true;
    if (*lost) return false;
  }
  *lost = 1;
  atomicAdd(&g_vocab_wait_errors, 1);
  return false;
}
// address of a shared-memory object in another block of the cluster
__device__ __forceinline__ uint32_t in_block(const void *p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(sptr(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void bar_arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar)
               : "memory");
}
__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// tile load; bar: shared::cluster address, of the pair's first block for CG 2
template <int CG>
__device__ __forceinline__ void tma_load(void *dst, const CUtensorMap *map, int x, int y,
                                         uint32_t bar) {
  if (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];\n" ::"r"(sptr(dst)),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        ".cta_group::2 [%0], [%1, {%2, %3}], [%4];\n" ::"r"(sptr(dst)),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap *map, int x, int y,
                                          const void *src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n"
               ::"l"((uint64_t)map), "r"(x), "r"(y), "r"(sptr(src))
               : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap *map, int x, int y, int z,
                                             const void *src, bool add) {
  if (add)
    asm volatile(
        "cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group "
        "[%0, {%1, %2, %3}], [%4];\n" ::"l"((uint64_t)map), "r"(x), "r"(y), "r"(z),
        "r"(sptr(src))
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];\n"
        ::"l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(sptr(src))
        : "memory");
}
__device__ __forceinline__ void store_commit() {
  asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
}
// this thread's stores have read their shared memory
__device__ __forceinline__ void store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");
}
__device__ __forceinline__ void store_wait() {
  asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
}
template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  if (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// the MMAs issued so far arrive on the barrier when done (CG 2: in both blocks)
template <int CG>
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
  if (CG == 1)
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(
            sptr(bar))
        : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;\n" ::"r"(sptr(bar)),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
      "%28, %29, %30, %31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_ld8(uint32_t addr, float (&v)[8]) {
  uint32_t r[8];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}

// Shared-memory operand with 128-byte swizzle.  K-major: rows of 64 K values,
// 8-row groups 1024 bytes apart.  M/N-major: 64 M/N values a row, one row per K;
// blocks of 64 M/N values lbo apart, groups of 8 K 1024 bytes apart.
__device__ __forceinline__ uint64_t swizzled_desc(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)((lbo >> 4) & 0x3FFF) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}

template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value)
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
  else
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// power of two S with S max|g| in [2^13, 2^14] (1 for a zero, infinite or NaN
// maximum): dz is formed times S for fp16
__device__ __forceinline__ float dz_scale(const uint32_t *grad_max) {
  const int e = (int)(*grad_max >> 23);  // sign bit clear
  if (e == 0 || e == 255) return 1.0f;
  const int k = min(max(127 + 13 - (e - 127), 1), 254);
  return __uint_as_float((uint32_t)k << 23);
}

constexpr float kLog2e = 1.4426950408889634f;

// 2^x, values below 2^-126 as zero
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// element h (-1: none) of v
__device__ __forceinline__ float pick(const float (&v)[32], int h) {
  float z = 0.0f;
#pragma unroll
  for (int j = 0; j < 32; ++j)
    if (j == h) z = v[j];
  return z;
}
// Running (max, rest) of logits, where sum exp(v - max) = 1 + rest: kept apart from the
// maximum's own 1, the rest of a confident token keeps its relative precision, and so does
// its loss.  An empty one is (-inf, -1) and must not make inf - inf of its own.
__device__ __forceinline__ void join(float &m, float &rest, float m1, float rest1) {
  const bool first = m >= m1;
  const float top = fmaxf(m, m1), base = top == -INFINITY ? 0.0f : top;
  const float less = first ? m1 : m, of_less = first ? rest1 : rest;
  rest = (first ? rest : rest1) + (1.0f + of_less) * ex2((less - base) * kLog2e);
  m = top;
}

// what v's rounding to T leaves (nothing of what T cannot hold)
template <class T>
__device__ __forceinline__ float left_over(float v) {
  float r;
  if constexpr (std::is_same<T, __half>::value)
    r = __half2float(__float2half_rn(v));
  else
    r = __bfloat162float(__float2bfloat16_rn(v));
  return isfinite(r) ? v - r : 0.0f;
}

// 32 columns of this warp's 32 rows into a slab (rows of 128 bytes, 16-byte chunks
// XORed with the row as TMA's 128-byte swizzle has them): as 64 bytes of 16-bit values
// (half 0 or 1 of the row) or 128 bytes of binary32.
template <class T>
__device__ __forceinline__ void put_half(unsigned char *slab, int lane, int half,
                                         const float (&v)[32]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint4 w;
    w.x = pack2<T>(v[8 * c], v[8 * c + 1]);
    w.y = pack2<T>(v[8 * c + 2], v[8 * c + 3]);
    w.z = pack2<T>(v[8 * c + 4], v[8 * c + 5]);
    w.w = pack2<T>(v[8 * c + 6], v[8 * c + 7]);
    *reinterpret_cast<uint4 *>(slab + lane * 128 + (((4 * half + c) ^ (lane & 7)) << 4)) = w;
  }
}
__device__ __forceinline__ void put_floats(unsigned char *slab, int lane, const float (&v)[32]) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<float4 *>(slab + lane * 128 + ((c ^ (lane & 7)) << 4)) =
        make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
}

// D[M][N] = sum_k A[m][k] B[n][k] per tile and split, handed to the epilogue.
// AMN / BMN: the operand lies in memory with M (N) contiguous, so a stage of it
// is blocks of 64 M (N) values x 64 K rows instead of rows of 64 K values.  CG: blocks
// that share a tile.
template <class T, int EPI, bool AMN, bool BMN, int CG>
__global__ void __launch_bounds__(Block<CG>::threads, 1)
    vocab_gemm_kernel(const __grid_constant__ CUtensorMap map_a,
                      const __grid_constant__ CUtensorMap map_b,
                      const __grid_constant__ CUtensorMap map_out, const VocabArgs a) {
  using B = Block<CG>;
  constexpr int TILE_M = CG * VL_M, STAGES = B::stages;
  constexpr bool LOGITS = EPI == EPI_STATS || EPI == EPI_DZ;
  extern __shared__ unsigned char vl_raw[];
  unsigned char *base = vl_raw + ((1024 - (sptr(vl_raw) & 1023)) & 1023);
  unsigned char *slabs = base + STAGES * B::stage;
  uint64_t *full = reinterpret_cast<uint64_t *>(slabs + B::warps * VL_SLAB);
  uint64_t *empty = full + STAGES, *acc_full = empty + STAGES, *acc_empty = acc_full + 2;
  uint64_t *drained = acc_empty + 2;
  uint32_t *tmem_ptr = reinterpret_cast<uint32_t *>(drained + 1);
  volatile int *lost = reinterpret_cast<volatile int *>(tmem_ptr + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  let_next_start();
  uint32_t rank = 0;
  if (CG > 1) asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(rank));
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) bar_init(full + s, 1), bar_init(empty + s, 1);
    for (int s = 0; s < 2; ++s) bar_init(acc_full + s, 1), bar_init(acc_empty + s, CG * B::warps);
    bar_init(drained, 1);
    *lost = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 1) {
    if (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(
                       sptr(tmem_ptr)),
                   "r"(2 * VL_N));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(
                       sptr(tmem_ptr)),
                   "r"(2 * VL_N));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::);
    }
  }
  fence_before();
  __syncthreads();
  if (CG > 1) cluster_meet();
  fence_after();
  const uint32_t tmem = *tmem_ptr;
  wait_for_previous();
  int M = a.M, K = a.K;
  if (a.tok.count) {
    const int count = *a.tok.count;
    (a.tokens_in_k ? K : M) = !a.low || EPI == EPI_DZ ? count : count ? 2 * VL_LOW : 0;
  }
  const Tiles ts = tiles_of<CG>(a, M, K);
  const int first = blockIdx.x / CG, step = gridDim.x / CG;
  const bool sums = ts.k_blocks > 0;  // no counted token: dW is zero without a product
  const bool idle = a.idle == first + 1;
  int it = 0;  // K steps loaded (warp 0) or multiplied (warp 1)

  if (warp == 0) {
    if (lane == 0 && sums && !idle) {
      bool ok = true;
      for (int tile = first; tile < ts.total && ok; tile += step) {
        const Tile at = tile_at<EPI>(ts, tile);
        const int mt = at.m, nt = at.n, split = at.split;
        const int kb0 = split * ts.split_blocks, kb1 = min(kb0 + ts.split_blocks, ts.k_blocks);
        const int m0 = mt * TILE_M + rank * VL_M, n0 = nt * VL_N + rank * B::n;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % STAGES;
          if (it >= STAGES &&
              !(ok = bar_wait(empty + s, ((it / STAGES) - 1) & 1, lost)))
            break;
          unsigned char *sa = base + s * B::stage, *sb = sa + VL_A_BYTES;
          if (rank == 0) bar_expect(full + s, CG * B::stage);
          const uint32_t bar = CG == 1 ? sptr(full + s) : in_block(full + s, 0);
          if (AMN) {
#pragma unroll
            for (int i = 0; i < VL_M / 64; ++i)
              tma_load<CG>(sa + i * 8192, &map_a, m0 + i * 64, kb * VL_K, bar);
          } else {
            tma_load<CG>(sa, &map_a, kb * VL_K, m0, bar);
          }
          if (BMN) {
#pragma unroll
            for (int i = 0; i < B::n / 64; ++i)
              tma_load<CG>(sb + i * 8192, &map_b, n0 + i * 64,
                           EPI == EPI_OUT && a.low ? 0 : a.k_first + kb * VL_K, bar);
          } else {
            tma_load<CG>(sb, &map_b, kb * VL_K, a.n_first + n0, bar);
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0 && sums && !idle) {
      constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)AMN << 15) |
                                 ((uint32_t)BMN << 16) | ((uint32_t)(VL_N >> 3) << 17) |
                                 ((uint32_t)(TILE_M >> 4) << 24);
      int n = 0;
      bool ok = true;
      for (int tile = first; tile < ts.total && ok; tile += step) {
        const int split = tile_at<EPI>(ts, tile).split;
        const int kb0 = split * ts.split_blocks, kb1 = min(kb0 + ts.split_blocks, ts.k_blocks);
        constexpr int chunk = LOGITS ? VL_CHUNK : VL_LONG;
        for (int kc = kb0; kc < kb1 && ok; kc += chunk, ++n) {
          const int buf = n & 1, end = min(kc + chunk, kb1);
          if (n >= 2 && !(ok = bar_wait(acc_empty + buf, ((n >> 1) - 1) & 1, lost))) break;
          fence_after();
          for (int kb = kc; kb < end; ++kb, ++it) {
            const int s = it % STAGES;
            if (!(ok = bar_wait(full + s, (it / STAGES) & 1, lost))) break;
            fence_after();
            const uint32_t sa = sptr(base + s * B::stage), sb = sa + VL_A_BYTES;
#pragma unroll
            for (int k = 0; k < VL_K / 16; ++k)
              mma_f16<CG>(tmem + buf * VL_N, swizzled_desc(sa + k * (AMN ? 2048 : 32), 8192),
                          swizzled_desc(sb + k * (BMN ? 2048 : 32), 8192), idesc,
                          kb > kc || k > 0);
            mma_commit<CG>(empty + s);
          }
          if (ok) mma_commit<CG>(acc_full + buf);
        }
      }
    }
  } else {
    // warps of lane quarter (warp & 3); those of a quarter share its columns
    const int quarter = warp & 3, part = (warp - 2) >> 2, row = quarter * 32 + lane;
    constexpr int COLS = B::cols;
    unsigned char *slab = slabs + (warp - 2) * VL_SLAB;
    int n = 0;
    float scale = 1.0f;
    if constexpr (std::is_same<T, __half>::value && EPI != EPI_STATS)
      scale = dz_scale(a.tok.grad_max);
    if (EPI != EPI_DZ) scale = 1.0f / scale;
    float run_max = -INFINITY, run_rest = -1.0f;  // stats of one row over a block's tiles
    bool ok = true;  // no wait of this warp ran out; none of its tiles is there after one did
    for (int tile = first; tile < ts.total; tile += step) {
      const Tile where = tile_at<EPI>(ts, tile);
      const int mt = where.m, nt = where.n, split = where.split;
      const int m0 = mt * TILE_M + rank * VL_M, n0 = nt * VL_N + part * COLS;
      const int t = m0 + row, cols = a.N - n0;  // columns of the product from n0 on
      auto accumulator = [&]() {
        return tmem + (n & 1) * VL_N + part * COLS + ((uint32_t)(quarter * 32) << 16);
      };
      auto ready = [&]() {
        ok = ok && __all_sync(~0u, bar_wait(acc_full + (n & 1), (n >> 1) & 1, lost,
                                            idle ? VL_IDLE_LIMIT : VL_WAIT_LIMIT));
        fence_after();
        return ok;
      };
      auto release = [&]() {
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive_at(in_block(acc_empty + (n & 1), 0));
        ++n;
      };
      // the slab, once its earlier store has read it
      auto next_slab = [&]() {
        if (lane == 0) store_wait_read();
        __syncwarp();
        return slab;
      };
      auto filled = [&]() {
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        __syncwarp();
      };
      // the tile's sums of this warp, its chunks joined; NaN where a wait ran out
      auto collect = [&](float(&z)[COLS / 32][32], int kb0, int kb1) {
        constexpr int chunk = LOGITS ? VL_CHUNK : VL_LONG;
        for (int kc = kb0; kc < kb1; kc += chunk) {
          if (!ready()) break;
          const uint32_t acc = accumulator();
#pragma unroll
          for (int i = 0; i < COLS / 32; ++i)
            if (EPI == EPI_OUT || 32 * i < cols) {
              if (kc == kb0) {
                tmem_ld32(acc + 32 * i, z[i]);
              } else {
#pragma unroll
                for (int q = 0; q < 32; q += 8) {
                  float more[8];
                  tmem_ld8(acc + 32 * i + q, more);
#pragma unroll
                  for (int j = 0; j < 8; ++j) z[i][q + j] += more[j];
                }
              }
            }
          release();
        }
        if (!ok) {
#pragma unroll
          for (int i = 0; i < COLS / 32; ++i)
#pragma unroll
            for (int j = 0; j < 32; ++j) z[i][j] = NAN;
        }
      };
      float z[COLS / 32][32];
      if constexpr (LOGITS) {
        collect(z, 0, ts.k_blocks);
        const bool live = t < M;
        const long long label = live ? a.tok.labels[t] : a.ignore;
        const long long at = label - a.n_first - n0;  // the label's column here
        // none past the last token: `ignore`, which stands in there, may be a word
        const int hit = live && at >= 0 && at < COLS && at < cols ? (int)at : -1;
        float g = 0.0f, lse = 0.0f;
        if (EPI == EPI_DZ && live && label != a.ignore) {
          g = a.tok.grad[t] * scale;
          lse = a.tok.lse[t];
          if (label < 0 || label >= a.vocab) g = NAN;
        }
        float mx = -INFINITY, rest = -1.0f;
#pragma unroll
        for (int c = 0; c < COLS; c += EPI == EPI_STATS ? 32 : 64) {
          if (c >= cols) break;
          if constexpr (EPI == EPI_STATS) {
            float(&v)[32] = z[c / 32];
            if (c + 32 > cols)
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (c + j >= cols) v[j] = -INFINITY;
            float m2 = v[0];
#pragma unroll
            for (int j = 1; j < 32; ++j) m2 = fmaxf(m2, v[j]);
            const float bs = m2 == -INFINITY ? 0.0f : m2;
            float all = 0.0f, below = 0.0f;  // below: without the largest
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float e = ex2((v[j] - bs) * kLog2e);
              all += e;
              if (!(e >= 1.0f)) below += e;
            }
            join(mx, rest, m2, below + (rintf(all - below) - 1.0f));
            if (hit >= c && hit < c + 32) a.label_logit[t] = pick(v, hit - c);
          } else {
            const bool two = CG == 1 && a.low;
            if (two && quarter >= 2) break;
            unsigned char *sl = next_slab();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              float(&v)[32] = z[c / 32 + q];
              const int h = hit - c - 32 * q;
              // with g = 0 all are 0, also where the logits are not finite
              const float own =
                  h >= 0 && h < 32 && g != 0.0f ? g * expm1f(pick(v, h) - lse) : 0.0f;
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const float p = ex2((v[j] - lse) * kLog2e);
                v[j] = g == 0.0f ? 0.0f : g * p;
                if (j == h) v[j] = own;
              }
              put_half<T>(sl, lane, q, v);
              if (!two && h >= 0 && h < 32) a.label_left[t] = left_over<T>(own);
            }
            filled();
            if (lane == 0 && m0 + quarter * 32 < (two ? VL_LOW : a.M)) {
              tma_store(&map_out, n0 + c, m0 + quarter * 32, sl);
              store_commit();
            }
            if (two) {
              sl = next_slab();
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                float(&v)[32] = z[c / 32 + q];
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = left_over<T>(v[j]);
                put_half<T>(sl, lane, q, v);
              }
              filled();
              if (lane == 0) {
                tma_store(&map_out, n0 + c, VL_LOW + quarter * 32, sl);
                store_commit();
              }
            }
          }
        }
        if constexpr (EPI == EPI_STATS) {
          // with one tile of tokens a block's tiles all hold the same rows: one entry
          // per block; else one per tile
          const bool one = a.M <= TILE_M;  // as the host counts the entries
          if (one) {
            join(run_max, run_rest, mx, rest);
            mx = run_max, rest = run_rest;
          }
          if (live && (!one || tile + step >= ts.total))
            a.part[(long long)((one ? first : nt) * (B::warps / 4) + part) * a.M + t] =
                make_float2(mx, rest);
        }
      } else if constexpr (EPI == EPI_PARTIAL) {
        const int kb0 = split * ts.split_blocks;
        collect(z, kb0, min(kb0 + ts.split_blocks, ts.k_blocks));
#pragma unroll
        for (int c = 0; c < COLS; c += 32) {
          if (c >= cols) break;
          unsigned char *sl = next_slab();
          put_floats(sl, lane, z[c / 32]);
          filled();
          const int r = m0 + quarter * 32;
          if (lane == 0 && r < a.M && (!a.low || r % VL_LOW < a.low)) {
            tma_store_3d(&map_out, n0 + c, m0 + quarter * 32, split, sl, a.accumulate);
            store_commit();
          }
        }
      } else {
        // the tokens whose label is one of this warp's words
        const int word0 = a.m_first + m0 + quarter * 32;
        int own = 0, own_end = 0;
        if (sums && a.tok.by.first)
          own = a.tok.by.first[word0 / VL_GROUP], own_end = a.tok.by.first[word0 / VL_GROUP + 1];
#pragma unroll
        for (int i = 0; i < COLS / 32; ++i)
#pragma unroll
          for (int j = 0; j < 32; ++j) z[i][j] = 0.0f;
        collect(z, 0, ts.k_blocks);
        // what rounding left of dz at the label, times the token's row of h: two columns a
        // lane, summed over the tokens of a word, then through the slab to the word's own
        // lane.  7 us of a step of 128 tokens (887) on a 128256 x 4096 head, below the noise
        // of one of 4096 (12.7 ms), 15 % where thousands of tokens all have one label
        static_assert(EPI != EPI_OUT || COLS == 64, "two columns a lane");
        if (own < own_end) {
          const T *h = static_cast<const T *>(a.tok.rows) + n0 + 2 * lane;
          float2 v = make_float2(0.0f, 0.0f);
#pragma unroll 1
          for (; own < own_end; ++own) {
            const int label = a.tok.by.label[own], token = a.tok.by.token[own];
            const float left = a.label_left[token];
            if (2 * lane < cols) {
              const float2 r =
                  unpack2<T>(*reinterpret_cast<const uint32_t *>(h + (long long)token * a.N));
              v.x = fmaf(left, r.x, v.x), v.y = fmaf(left, r.y, v.y);
            }
            if (own + 1 < own_end && a.tok.by.label[own + 1] == label) continue;
            float2 *through = reinterpret_cast<float2 *>(next_slab());
            through[lane] = v;
            __syncwarp();
            if (lane == label - word0) {
#pragma unroll
              for (int j = 0; j < 64; j += 4) {
                const float4 of = *reinterpret_cast<const float4 *>(through + j / 2);
                float *o = z[j / 32] + j % 32;
                o[0] += of.x, o[1] += of.y, o[2] += of.z, o[3] += of.w;
              }
            }
            v = make_float2(0.0f, 0.0f);
          }
        }
#pragma unroll
        for (int c = 0; c < COLS; c += 64) {
          if (c >= cols) break;
          unsigned char *sl = next_slab();
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float(&v)[32] = z[c / 32 + q];
            if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] *= scale;
            }
            put_half<T>(sl, lane, q, v);
          }
          filled();
          if (lane == 0 && m0 + quarter * 32 < a.M) {
            tma_store(&map_out, n0 + c, a.m_first + m0 + quarter * 32, sl);
            store_commit();
          }
        }
      }
    }
    if (EPI != EPI_STATS && lane == 0) store_wait();
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (*lost && rank == 0) {
    // loads in flight (all of a pair's arrive at its first block) and products end before
    // their memory is freed
    if (threadIdx.x == 0)
      for (int i = max(0, it - STAGES); i < it; ++i)
        for (int p = 0; p < VL_WAIT_LIMIT && !bar_try(full + i % STAGES, (i / STAGES) & 1); ++p) {
        }
    if (threadIdx.x == 32) {
      mma_commit<CG>(drained);
      for (int p = 0; p < VL_WAIT_LIMIT && !bar_try(drained, 0); ++p) {
      }
    }
    __syncwarp();
  }
  if (CG > 1) cluster_meet();
  fence_after();
  if (warp == 1) {
    if (CG == 1)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem),
                   "r"(2 * VL_N));
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem),
                   "r"(2 * VL_N));
  }
}

// Joins the tiles' (max, rest): block (8 tokens, 64 slices of the entries).  Ignored
// tokens get 0 and 0.  place: where a token's entries are (null: at its own number).
__global__ void __launch_bounds__(512)
    vocab_join_kernel(const float2 *__restrict__ part, const float *__restrict__ label_logit,
                      const long long *__restrict__ labels, long long ignore, int vocab,
                      const int *__restrict__ place, int T, int slots, float *__restrict__ loss,
                      float *__restrict__ lse) {
  __shared__ float2 sm[64][9];
  let_next_start();
  wait_for_previous();
  const int t = blockIdx.x * 8 + threadIdx.x;
  const bool live = t < T && labels[t] != ignore;
  const int at = live ? (place ? place[t] : t) : 0;
  float m = -INFINITY, s = -1.0f;
  if (live) {
#pragma unroll 8
    for (int n = threadIdx.y; n < slots; n += 64) {
      const float2 p = part[(long long)n * T + at];
      join(m, s, p.x, p.y);
    }
  }
  sm[threadIdx.y][threadIdx.x] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.y >= 8) return;
  for (int y = threadIdx.y + 8; y < 64; y += 8)
    join(m, s, sm[y][threadIdx.x].x, sm[y][threadIdx.x].y);
  sm[threadIdx.y][threadIdx.x] = make_float2(m, s);
  asm volatile("bar.sync 1, 64;\n" ::: "memory");
  if (threadIdx.y || t >= T) return;
  for (int y = 1; y < 8; ++y) join(m, s, sm[y][threadIdx.x].x, sm[y][threadIdx.x].y);
  const float ls = log1pf(s);
  lse[t] = live ? m + ls : 0.0f;
  float l = 0.0f;
  if (live) l = labels[t] >= 0 && labels[t] < vocab ? (m - label_logit[at]) + ls : NAN;
  loss[t] = l;
}

// What counting the tokens leaves in a workspace.
struct Count {
  int *place;          // where each counted token goes (-1: ignored)
  int *count;          // how many there are
  uint32_t *grad_max;  // bits of max |g|
  ByLabel by;
  int *other_token, *other_label;  // of the sort's alternate passes
  int vocab;
};
__device__ __forceinline__ int label_key(long long label, int vocab) {
  return label >= 0 && label < vocab ? (int)label : vocab;
}

// Counts the tokens, one block for all of them, and sorts the counted ones by label where
// that is wanted: digits of 8 bits from the lowest on, each pass stable, 4096 tokens at a
// time (a warp's 128 in four steps, ranked among the warp's by __match_any_sync).
__global__ void __launch_bounds__(1024)
    vocab_count_kernel(const long long *__restrict__ labels, long long ignore,
                       const float *__restrict__ grad, int T, const Count c) {
  __shared__ int sums[32];
  __shared__ uint32_t tops[32];
  __shared__ int digits[4][256];  // how often a digit occurs, then where its tokens go
  __shared__ int by_warp[32][256];
  let_next_start();
  wait_for_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool sort = c.by.first != nullptr;
  const int passes = sort ? (32 - __clz(c.vocab) + 7) / 8 : 0;
  int *label = passes & 1 ? c.other_label : c.by.label;  // of the next pass
  int *token = passes & 1 ? c.other_token : c.by.token;
  for (int i = threadIdx.x; i < 4 * 256; i += 1024) digits[i >> 8][i & 255] = 0;
  __syncthreads();
  int before = 0;
  uint32_t top = 0;
  for (int t0 = 0; t0 < T; t0 += 1024) {
    const int t = t0 + threadIdx.x;
    const bool in = t < T && labels[t] != ignore;
    const uint32_t mask = __ballot_sync(~0u, in);
    if (in && grad) top = max(top, __float_as_uint(fabsf(grad[t])));
    if (lane == 0) sums[warp] = __popc(mask);
    __syncthreads();
    int v = sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(~0u, v, o);
      if (lane >= o) v += u;
    }
    const int warps_before = __shfl_sync(~0u, v, warp) - __popc(mask);
    const int mine = before + warps_before + __popc(mask & ((1u << lane) - 1));
    before += __shfl_sync(~0u, v, 31);
    if (t < T) c.place[t] = in ? mine : -1;
    if (sort && in) {
      const int key = label_key(labels[t], c.vocab);
      label[mine] = key, token[mine] = mine;
      for (int p = 0; p < passes; ++p) atomicAdd(&digits[p][(key >> (8 * p)) & 255], 1);
    }
    __syncthreads();
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
  if (lane == 0) tops[warp] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) top = max(top, tops[w]);
    *c.count = before;
    if (c.grad_max) *c.grad_max = top;
  }
  for (int p = 0; p < passes; ++p) {
    int *to_label = label == c.by.label ? c.other_label : c.by.label;
    int *to_token = token == c.by.token ? c.other_token : c.by.token;
    if (warp == 0) {  // counts to places
      int v[8], sum = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = sum, sum += digits[p][8 * lane + k];
      int all = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(~0u, all, o);
        if (lane >= o) all += u;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) digits[p][8 * lane + k] = all - sum + v[k];
    }
    for (int i0 = 0; i0 < before; i0 += 4096) {
      for (int i = threadIdx.x; i < 32 * 256; i += 1024) by_warp[i >> 8][i & 255] = 0;
      __syncthreads();
      int key[4], tok[4], rank[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + warp * 128 + u * 32 + lane;
        const bool on = i < before;
        key[u] = on ? label[i] : 0, tok[u] = on ? token[i] : 0;
        const int d = (key[u] >> (8 * p)) & 255;
        const uint32_t same = __match_any_sync(~0u, on ? d : 256);
        const int seen = on ? by_warp[warp][d] : 0;
        rank[u] = seen + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (on && (same >> lane) == 1) by_warp[warp][d] = seen + __popc(same);
        __syncwarp();
      }
      __syncthreads();
      if (threadIdx.x < 256) {
        int at = digits[p][threadIdx.x];
        for (int w = 0; w < 32; ++w) {
          const int n = by_warp[w][threadIdx.x];
          by_warp[w][threadIdx.x] = at;
          at += n;
        }
        digits[p][threadIdx.x] = at;
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i0 + warp * 128 + u * 32 + lane < before) {
          const int at = by_warp[warp][(key[u] >> (8 * p)) & 255] + rank[u];
          to_label[at] = key[u], to_token[at] = tok[u];
        }
      __syncthreads();
    }
    label = to_label, token = to_token;
  }
}

// first[g] of the groups after the one of the label before (-1: none) up to this one's, and
// after the last label to the end: what the token of rank `rank` among the sorted sets.
__device__ __forceinline__ void set_first(const ByLabel &by, int rank, int total, int before,
                                          int label) {
  const int from = before < 0 ? 0 : before / VL_GROUP + 1;
  for (int g = from + threadIdx.x; g <= label / VL_GROUP; g += blockDim.x) by.first[g] = rank;
  if (rank == total - 1)
    for (int g = label / VL_GROUP + 1 + threadIdx.x; g <= by.groups; g += blockDim.x)
      by.first[g] = total;
}

// The counted tokens' rows, labels, lse and g, packed; up to 63 zero rows behind them
// fill the last K block of dW.  SELF: each block counts for itself (few tokens), and
// vocab_count_kernel's results are written here.
template <class T, bool SELF>
__global__ void __launch_bounds__(128)
    vocab_gather_kernel(const T *__restrict__ h, long long ldh, int D, int tokens, const Count c,
                        const long long *__restrict__ labels, long long ignore,
                        const float *__restrict__ lse, const float *__restrict__ grad,
                        T *__restrict__ out, long long *__restrict__ out_labels,
                        float *__restrict__ out_lse, float *__restrict__ out_grad) {
  __shared__ int sums[4][4];
  __shared__ uint32_t tops[4];
  let_next_start();
  const int t = blockIdx.x;
  const bool sort = c.by.first != nullptr;
  int p, total;
  if (SELF) {
    int before = 0, all = 0, rank = 0, last = -1;  // last: the label before in the order
    uint32_t top = 0;
    const int own = label_key(labels[t], c.vocab);
    for (int i = threadIdx.x; i < tokens; i += 128) {
      const long long label = labels[i];
      const bool in = label != ignore;
      all += in;
      before += in && i < t;
      const int key = label_key(label, c.vocab);
      if (in && (key < own || (key == own && i < t))) ++rank, last = max(last, key);
      if (in && grad) top = max(top, __float_as_uint(fabsf(grad[i])));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      all += __shfl_xor_sync(~0u, all, o);
      before += __shfl_xor_sync(~0u, before, o);
      rank += __shfl_xor_sync(~0u, rank, o);
      last = max(last, __shfl_xor_sync(~0u, last, o));
      top = max(top, __shfl_xor_sync(~0u, top, o));
    }
    const int w = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0)
      sums[w][0] = before, sums[w][1] = all, sums[w][2] = rank, sums[w][3] = last, tops[w] = top;
    __syncthreads();
    before = sums[0][0] + sums[1][0] + sums[2][0] + sums[3][0];
    total = sums[0][1] + sums[1][1] + sums[2][1] + sums[3][1];
    rank = sums[0][2] + sums[1][2] + sums[2][2] + sums[3][2];
    last = max(max(sums[0][3], sums[1][3]), max(sums[2][3], sums[3][3]));
    p = labels[t] != ignore ? before : -1;
    if (threadIdx.x == 0) {
      c.place[t] = p;
      if (t == 0)
        *c.count = total, *c.grad_max = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
      if (sort && p >= 0) c.by.token[rank] = p, c.by.label[rank] = own;
    }
    if (sort && p >= 0) set_first(c.by, rank, total, last, own);
  } else {
    wait_for_previous();
    p = c.place[t];
    total = *c.count;
    if (sort && t < total)
      set_first(c.by, t, total, t ? c.by.label[t - 1] : -1, c.by.label[t]);
  }
  if (p >= 0) {
    const uint4 *in = reinterpret_cast<const uint4 *>(h + t * ldh);
    uint4 *o = reinterpret_cast<uint4 *>(out + (long long)p * D);
    for (int i = threadIdx.x; i < D / 8; i += 128) o[i] = in[i];
    if (threadIdx.x == 0) {
      out_labels[p] = labels[t];
      if (lse) out_lse[p] = lse[t], out_grad[p] = grad[t];
    }
  }
  const int zero = total + t;
  if (t < 63 && zero < tokens) {
    uint4 *o = reinterpret_cast<uint4 *>(out + (long long)zero * D);
    for (int i = threadIdx.x; i < D / 8; i += 128) o[i] = make_uint4(0, 0, 0, 0);
  }
}

// Sum of the splits' dh and of what rounding left of dz at the label (one row of W a
// token), rounded once; zero rows for ignored tokens.  Four threads share
// the splits of four columns, and their sums are added in order.
template <class T>
__global__ void __launch_bounds__(256)
    vocab_sum_kernel(const float4 *__restrict__ partial, int splits, int tokens, int low, int d4,
                     const int *__restrict__ place, const uint32_t *__restrict__ grad_max,
                     const long long *__restrict__ labels, const float *__restrict__ label_left,
                     const T *__restrict__ w, long long ldw, int vocab,
                     uint2 *__restrict__ out) {
  __shared__ float4 sm[3][64];
  let_next_start();
  wait_for_previous();
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const long long i = (long long)blockIdx.x * 64 + x, n = (long long)tokens * d4;
  const int t = i < n ? (int)(i / d4) : 0, c = (int)(i - (long long)t * d4);
  const int p = i < n ? place[t] : -1;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](const float4 &w) { v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w; };
  if (p >= 0) {
    const float4 *from = partial + (long long)p * d4 + c;
    const long long split = low ? 2ll * VL_LOW * d4 : n;
#pragma unroll 4
    for (int s = y; s < splits; s += 4) {
      add(from[s * split]);
      if (low) add(from[s * split + (long long)VL_LOW * d4]);
    }
  }
  if (y) sm[y - 1][x] = v;
  __syncthreads();
  if (y || i >= n) return;
  for (int k = 0; k < 3; ++k) add(sm[k][x]);
  if (!low && p >= 0 && labels[p] >= 0 && labels[p] < vocab) {
    const uint2 row = *reinterpret_cast<const uint2 *>(w + labels[p] * ldw + 4 * c);
    const float left = label_left[p];
    const float2 a = unpack2<T>(row.x), b = unpack2<T>(row.y);
    v.x = fmaf(left, a.x, v.x), v.y = fmaf(left, a.y, v.y);
    v.z = fmaf(left, b.x, v.z), v.w = fmaf(left, b.y, v.w);
  }
  float scale = 1.0f;
  if constexpr (std::is_same<T, __half>::value) scale = 1.0f / dz_scale(grad_max);
  out[i] = make_uint2(pack2<T>(v.x * scale, v.y * scale), pack2<T>(v.z * scale, v.w * scale));
}

using TensorMapEncoder = PFN_cuTensorMapEncodeTiled_v12000;
TensorMapEncoder map_encoder() {
  static const TensorMapEncoder fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return (TensorMapEncoder) nullptr;
    return reinterpret_cast<TensorMapEncoder>(p);
  }();
  return fn;
}

int encode(CUtensorMap *m, CUtensorMapDataType type, int rank, const void *p,
           const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box) {
  const TensorMapEncoder enc = map_encoder();
  if (!enc) {
    set_error("the driver has no cuTensorMapEncodeTiled");
    return B2F_ERR_UNSUPPORTED;
  }
  const cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = enc(m, type, rank, const_cast<void *>(p), dims, strides, box, es,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("tensor map of %llu x %llu: error %d", (unsigned long long)dims[1],
              (unsigned long long)dims[0], (int)r);
    return B2F_ERR_CUDA;
  }
  return B2F_OK;
}
// matrix [rows][cols] of 16-bit values, rows ld apart, in boxes of 64 columns
template <class T>
int encode_map(CUtensorMap *m, const void *p, long long rows, long long cols, long long ld,
               int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  return encode(m, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                2, p, dims, strides, box);
}
// [splits][rows][cols] of binary32 in boxes of 32 x 32
int encode_partial(CUtensorMap *m, const float *p, long long splits, long long rows,
                   long long cols) {
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)splits};
  const cuuint64_t strides[2] = {(cuuint64_t)cols * 4, (cuuint64_t)(rows * cols) * 4};
  const cuuint32_t box[3] = {32, 32, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, p, dims, strides, box);
}

// Blocks that share a tile: two from 129 tokens on.  With up to 128 tokens W's bytes
// bound every product and half of a 256-row tile would be empty.
int blocks_per_tile(int64_t T) { return T > VL_M ? 2 : 1; }

// b2f_vocab_loss_idle_block's product (low byte) and block from 1 (the rest); 0: none
std::atomic<int64_t> g_idle{0};

template <class T, int EPI, bool AMN, bool BMN, int CG>
int launch_tiles(const CUtensorMap &ma, const CUtensorMap &mb, const CUtensorMap &mo, VocabArgs a,
                 bool chained, int dev, int sms, cudaStream_t s) {
  const int64_t idle = g_idle.load(std::memory_order_relaxed);
  a.idle = (idle & 255) == EPI ? (int)(idle >> 8) : 0;
  auto k = vocab_gemm_kernel<T, EPI, AMN, BMN, CG>;
  static std::atomic<uint64_t> allowed{0};
  if (int rc = allow_shared(k, (int)Block<CG>::smem, dev, allowed)) return rc;
  const int64_t m_tiles = (a.M + CG * VL_M - 1) / (CG * VL_M);
  const int64_t n_tiles = (a.N + VL_N - 1) / VL_N;
  B2F_CHECK_ARG(m_tiles * n_tiles * a.splits < (1ll << 31), "b2f_vocab_loss: too many tiles");
  const int tiles = (int)(m_tiles * n_tiles * a.splits);
  return launch_chained(k, dim3(CG * std::min(tiles, sms / CG)), dim3(Block<CG>::threads),
                        Block<CG>::smem, CG, chained, s, ma, mb, mo, a);
}
template <class T, int EPI, bool AMN, bool BMN>
int launch_gemm(const CUtensorMap &ma, const CUtensorMap &mb, const CUtensorMap &mo,
                const VocabArgs &a, int group, bool chained, int dev, int sms, cudaStream_t s) {
  return group == 2 ? launch_tiles<T, EPI, AMN, BMN, 2>(ma, mb, mo, a, chained, dev, sms, s)
                    : launch_tiles<T, EPI, AMN, BMN, 1>(ma, mb, mo, a, chained, dev, sms, s);
}

struct Shape {
  int T, D, V;
  long long ldh, ldw;
};

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// The counted tokens' place in a workspace.
struct CountedSpace {
  size_t place, count, gmax, labels, lse, grad, left, rows;
  size_t by_token, by_label, other_token, other_label, first;  // with `words`: sorted
  size_t end;
};
int groups_of(int64_t words) { return (int)((words + VL_N - 1) / VL_N * (VL_N / VL_GROUP)); }
CountedSpace counted_space(int64_t T, int64_t D, bool grad, int64_t words) {
  CountedSpace c{};
  size_t off = 0;
  auto take = [&](size_t n) {
    const size_t at = off;
    off += round256(n);
    return at;
  };
  c.place = take(T * 4), c.count = take(4), c.gmax = take(4), c.labels = take(T * 8);
  c.lse = take(grad ? T * 4 : 0), c.grad = take(grad ? T * 4 : 0);
  c.left = take(grad ? T * 4 : 0);
  c.rows = take((size_t)T * D * 2);
  c.by_token = take(words ? T * 4 : 0), c.by_label = take(words ? T * 4 : 0);
  c.other_token = take(words ? T * 4 : 0), c.other_label = take(words ? T * 4 : 0);
  c.first = take(words ? (groups_of(words) + 1) * 4ll : 0);
  c.end = off;
  return c;
}
template <class T>
int gather_counted(const void *h, const Shape &z, const long long *labels, long long ignore,
                   const float *lse, const float *grad, bool sorted, char *ws,
                   const CountedSpace &c, Counted *tok, cudaStream_t s) {
  auto ints = [&](size_t at) { return reinterpret_cast<int *>(ws + at); };
  Count n{ints(c.place), ints(c.count), reinterpret_cast<uint32_t *>(ws + c.gmax)};
  n.vocab = z.V;
  if (sorted) {
    n.by = {ints(c.by_token), ints(c.by_label), ints(c.first), groups_of(z.V)};
    n.other_token = ints(c.other_token), n.other_label = ints(c.other_label);
  }
  auto *lab = reinterpret_cast<long long *>(ws + c.labels);
  float *l = reinterpret_cast<float *>(ws + c.lse), *g = reinterpret_cast<float *>(ws + c.grad);
  // the first of its chain waits for all before it.  Up to 1024 tokens every block of
  // the gathering counts for itself, one launch less.
  T *rows = reinterpret_cast<T *>(ws + c.rows);
  const T *from = static_cast<const T *>(h);
  if (z.T <= 1024) {
    if (int rc = launch_chained(vocab_gather_kernel<T, true>, dim3(z.T), dim3(128), 0, 1, false, s,
                                from, z.ldh, z.D, z.T, n, labels, ignore, lse, grad, rows, lab, l,
                                g))
      return rc;
  } else {
    if (int rc = launch_chained(vocab_count_kernel, dim3(1), dim3(1024), 0, 1, false, s, labels,
                                ignore, grad, z.T, n))
      return rc;
    if (int rc = launch_chained(vocab_gather_kernel<T, false>, dim3(z.T), dim3(128), 0, 1, true, s,
                                from, z.ldh, z.D, z.T, n, labels, ignore, lse, grad, rows, lab, l,
                                g))
      return rc;
  }
  *tok = Counted{n.count, lab, l, g, n.grad_max, rows, n.by};
  return B2F_OK;
}

// The forward pass gathers the counted tokens too from 1024 tokens on, where a product
// over the ignored ones costs more than two more launches.
bool forward_gathers(int64_t T) { return T >= 1024; }
int64_t forward_slots(int64_t T, int64_t V, int sms) {
  const int64_t group = blocks_per_tile(T), tiles = (V + VL_N - 1) / VL_N;
  const int per = group == 1 ? Block<1>::warps / 4 : Block<2>::warps / 4;
  // entries of blocks where one tile holds all tokens, else of tiles
  return per * (T <= group * VL_M ? std::min<int64_t>(tiles, sms / group) : tiles);
}

// How the gradient is cut: words of a piece, splits of dh's sum over a piece.
struct Plan {
  int piece, pieces, splits;
  CountedSpace c;
  size_t dz, partial, total;
};
constexpr size_t kDzBytes = 256ull << 20;
// dz in two parts where the tile of 128 rows has room for both
bool dz_in_two(int64_t T) { return T <= VL_LOW; }
int64_t dz_rows(int64_t T) { return dz_in_two(T) ? 2 * VL_LOW : T; }

Plan grad_plan(int64_t T, int64_t V, int64_t D, bool need_h, int sms) {
  Plan p{};
  constexpr int unit = VL_N;
  int64_t words = (int64_t)(kDzBytes / 2 / (size_t)dz_rows(T)) / unit * unit;
  words = std::max<int64_t>(words, unit);
  p.pieces = (int)((V + words - 1) / words);
  p.piece = (int)(((V + p.pieces - 1) / p.pieces + unit - 1) / unit * unit);
  p.pieces = (int)((V + p.piece - 1) / p.piece);
  // splits of a piece's words in dh = dz W: the number (with at least 4 K blocks
  // each) whose rounds over the SMs leave the least idle, 6 K blocks counted for a
  // tile's store; at most 256 MB of partial sums beyond the first
  const int64_t group = blocks_per_tile(T), slots = sms / group;
  const int64_t rows = dz_rows(T);
  const int64_t tiles = ((T + group * VL_M - 1) / (group * VL_M)) *
                        ((D + VL_N - 1) / VL_N);
  const int64_t kb = (std::min<int64_t>(p.piece, V) + VL_K - 1) / VL_K;
  int64_t best = 0;
  p.splits = 1;
  for (int64_t n = 1; n <= slots && n <= std::max<int64_t>(1, kb / 4); ++n) {
    if (n > 1 && (size_t)(n - 1) * rows * D * 4 > (256ull << 20)) break;
    const int64_t per = (kb + n - 1) / n;
    if ((kb + per - 1) / per != n) continue;  // a split without work
    const int64_t cost = ((tiles * n + slots - 1) / slots) * (per + 6);
    if (!best || cost < best) best = cost, p.splits = (int)n;
  }
  p.c = counted_space(T, D, true, dz_in_two(T) ? 0 : V);
  size_t off = p.c.end;
  p.dz = off, off += round256((size_t)rows * p.piece * 2);
  p.partial = off;
  if (need_h) off += round256((size_t)p.splits * rows * D * 4);
  p.total = off;
  return p;
}

int check_shape(const char *who, int dtype, int64_t T, int64_t V, int64_t D, int64_t ldh,
                int64_t ldw) {
  B2F_CHECK_ARG(dtype == B2F_F16 || dtype == B2F_BF16, "%s: dtype %d (fp16 or bf16)", who, dtype);
  B2F_CHECK_ARG(T >= 0 && T <= (1 << 24) && V >= 1 && V <= (1 << 26) && D >= 8 &&
                    D <= (1 << 20) && D % 8 == 0,
                "%s: %lld tokens, %lld words, hidden size %lld (a multiple of 8)", who,
                (long long)T, (long long)V, (long long)D);
  B2F_CHECK_ARG(ldh >= D && ldw >= D && ldh % 8 == 0 && ldw % 8 == 0,
                "%s: rows %lld and %lld apart (multiples of 8, at least the hidden size)", who,
                (long long)ldh, (long long)ldw);
  return B2F_OK;
}

template <class T>
int forward(const void *h, const void *w, const Shape &z, const long long *labels,
            long long ignore, float *loss, float *lse, char *ws, int dev, int sms,
            cudaStream_t s) {
  VocabArgs a{};
  a.M = z.T, a.N = z.V, a.K = z.D, a.splits = 1;
  a.ignore = ignore, a.vocab = z.V;
  a.tok.labels = labels;
  const int group = blocks_per_tile(z.T);
  const int64_t slots = forward_slots(z.T, z.V, sms);
  a.label_logit = reinterpret_cast<float *>(ws);
  size_t off = round256((size_t)z.T * 4);
  a.part = reinterpret_cast<float2 *>(ws + off);
  off += round256((size_t)slots * z.T * 8);
  const int *place = nullptr;
  long long ldh = z.ldh;
  if (forward_gathers(z.T)) {
    const CountedSpace c = counted_space(z.T, z.D, false, 0);
    if (int rc = gather_counted<T>(h, z, labels, ignore, nullptr, nullptr, false, ws + off, c,
                                   &a.tok, s))
      return rc;
    h = ws + off + c.rows;
    ldh = z.D;
    place = reinterpret_cast<int *>(ws + off + c.place);
  }
  CUtensorMap ma, mb;
  if (int rc = encode_map<T>(&ma, h, z.T, z.D, ldh, VL_M)) return rc;
  if (int rc = encode_map<T>(&mb, w, z.V, z.D, z.ldw, VL_N / group)) return rc;
  if (int rc = launch_gemm<T, EPI_STATS, false, false>(ma, mb, ma, a, group, place != nullptr, dev,
                                                     sms, s))
    return rc;
  return launch_chained(vocab_join_kernel, dim3((z.T + 7) / 8), dim3(8, 64), 0, 1, true, s, a.part,
                        a.label_logit, labels, ignore, z.V, place, z.T, (int)slots, loss, lse);
}

template <class T>
int backward(const void *h, const void *w, const Shape &z, const long long *labels,
             long long ignore, const float *lse, const float *grad, void *dh, void *dw,
             const Plan &p, char *ws, int dev, int sms, cudaStream_t s) {
  T *hc = reinterpret_cast<T *>(ws + p.c.rows), *dz = reinterpret_cast<T *>(ws + p.dz);
  float *partial = reinterpret_cast<float *>(ws + p.partial);
  float *left = reinterpret_cast<float *>(ws + p.c.left);
  Counted tok;
  const int low = dz_in_two(z.T) ? z.T : 0, rows = (int)dz_rows(z.T);
  if (int rc = gather_counted<T>(h, z, labels, ignore, lse, grad, dw && !low, ws, p.c, &tok, s))
    return rc;
  const int group = blocks_per_tile(z.T);
  CUtensorMap h_k, h_n, w_k, w_n, dz_k, dz_m, dz_out, sums, dw_out;
  if (int rc = encode_map<T>(&h_k, hc, z.T, z.D, z.D, VL_M)) return rc;
  if (int rc = encode_map<T>(&w_k, w, z.V, z.D, z.ldw, VL_N / group)) return rc;
  if (int rc = encode_map<T>(&h_n, hc, z.T, z.D, z.D, VL_K)) return rc;
  if (int rc = encode_map<T>(&w_n, w, z.V, z.D, z.ldw, VL_K)) return rc;
  if (dh)
    if (int rc = encode_partial(&sums, partial, p.splits, rows, z.D)) return rc;
  if (dw)
    if (int rc = encode_map<T>(&dw_out, dw, z.V, z.D, z.D, 32)) return rc;
  for (int i = 0; i < p.pieces; ++i) {
    const int v0 = i * p.piece, words = std::min(p.piece, z.V - v0);
    VocabArgs a{};
    a.M = z.T, a.N = words, a.K = z.D, a.splits = 1;
    a.n_first = v0;
    a.tok = tok, a.ignore = ignore, a.vocab = z.V, a.low = low;
    a.label_left = left;
    if (int rc = encode_map<T>(&dz_out, dz, rows, words, p.piece, 32)) return rc;
    if (int rc = launch_gemm<T, EPI_DZ, false, false>(h_k, w_k, dz_out, a, group, true, dev, sms,
                                                      s))
      return rc;
    if (dh) {
      if (int rc = encode_map<T>(&dz_k, dz, rows, words, p.piece, VL_M)) return rc;
      VocabArgs b{};
      b.M = rows, b.N = z.D, b.K = words, b.low = low;
      // the last piece may have too few words for all the splits; one without a K block
      // would add what its accumulator held before
      const int kb = (words + VL_K - 1) / VL_K, per = (kb + p.splits - 1) / p.splits;
      b.splits = (kb + per - 1) / per;
      b.k_first = v0;
      b.tok = tok;
      b.accumulate = i > 0;
      if (int rc = launch_gemm<T, EPI_PARTIAL, false, true>(dz_k, w_n, sums, b, group, true, dev,
                                                            sms, s))
        return rc;
    }
    if (dw) {
      if (int rc = encode_map<T>(&dz_m, dz, rows, words, p.piece, VL_K)) return rc;
      VocabArgs b{};
      b.M = words, b.N = z.D, b.K = rows, b.splits = 1, b.low = low;
      b.m_first = v0;
      b.tok = tok, b.tokens_in_k = 1;
      b.label_left = left;
      if (int rc = launch_tiles<T, EPI_OUT, true, true, 2>(dz_m, h_n, dw_out, b, true, dev, sms, s))
        return rc;
    }
  }
  if (dh) {
    const long long n4 = (long long)z.T * z.D / 4;
    return launch_chained(vocab_sum_kernel<T>, dim3((unsigned)((n4 + 63) / 64)), dim3(256), 0, 1,
                          true, s, reinterpret_cast<const float4 *>(partial), p.splits, z.T,
                          low, z.D / 4, reinterpret_cast<const int *>(ws + p.c.place), tok.grad_max,
                          tok.labels, left, static_cast<const T *>(w), z.ldw, z.V,
                          static_cast<uint2 *>(dh));
  }
  return B2F_OK;
}

}  // namespace
}  // namespace b2f

extern "C" {

size_t b2f_vocab_loss_workspace(int64_t T, int64_t V, int64_t D) {
  using namespace b2f;
  int dev = 0, sms = 0;
  if (T < 1 || V < 1 || D < 1 || current_device(&dev, &sms)) return 0;
  return round256((size_t)T * 4) + round256((size_t)forward_slots(T, V, sms) * T * 8) +
         (forward_gathers(T) ? counted_space(T, D, false, 0).end : 0);
}

int b2f_vocab_loss(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, int dtype,
                   int64_t T, int64_t V, int64_t D, const int64_t *labels, int64_t ignore,
                   float *loss, float *lse, void *ws, size_t ws_bytes, void *stream) {
  B2F_RANGE("b2f_vocab_loss");
  using namespace b2f;
  if (int rc = check_shape("b2f_vocab_loss", dtype, T, V, D, ldh, ldw)) return rc;
  if (T == 0) return B2F_OK;
  B2F_CHECK_ARG(hidden && weight && labels && loss && lse && ws, "b2f_vocab_loss: null argument");
  B2F_CHECK_ARG(((uintptr_t)hidden | (uintptr_t)weight) % 16 == 0 && (uintptr_t)ws % 256 == 0,
                "b2f_vocab_loss: misaligned buffer (16 bytes, workspace 256)");
  int dev = 0, sms = 0;
  if (int rc = current_device(&dev, &sms)) return rc;
  B2F_CHECK_ARG(ws_bytes >= b2f_vocab_loss_workspace(T, V, D),
                "b2f_vocab_loss: workspace too small (%zu bytes)", ws_bytes);
  char *wsp = static_cast<char *>(ws);
  const Shape z{(int)T, (int)D, (int)V, ldh, ldw};
  auto *lab = reinterpret_cast<const long long *>(labels);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == B2F_F16
             ? forward<__half>(hidden, weight, z, lab, ignore, loss, lse, wsp, dev, sms, s)
             : forward<__nv_bfloat16>(hidden, weight, z, lab, ignore, loss, lse, wsp, dev, sms, s);
}

size_t b2f_vocab_loss_grad_workspace(int64_t T, int64_t V, int64_t D, int need_hidden) {
  using namespace b2f;
  int dev = 0, sms = 0;
  if (T < 1 || V < 1 || D < 1 || current_device(&dev, &sms)) return 0;
  return grad_plan(T, V, D, need_hidden != 0, sms).total;
}

int b2f_vocab_loss_grad(const void *hidden, int64_t ldh, const void *weight, int64_t ldw,
                        int dtype, int64_t T, int64_t V, int64_t D, const int64_t *labels,
                        int64_t ignore, const float *lse, const float *grad_loss,
                        void *grad_hidden, void *grad_weight, void *ws, size_t ws_bytes,
                        void *stream) {
  B2F_RANGE("b2f_vocab_loss_grad");
  using namespace b2f;
  if (int rc = check_shape("b2f_vocab_loss_grad", dtype, T, V, D, ldh, ldw)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (T == 0) {
    if (grad_weight) B2F_CUDA(cudaMemsetAsync(grad_weight, 0, (size_t)V * D * 2, s));
    return B2F_OK;
  }
  B2F_CHECK_ARG(hidden && weight && labels && lse && grad_loss && ws,
                "b2f_vocab_loss_grad: null argument");
  B2F_CHECK_ARG(grad_hidden || grad_weight, "b2f_vocab_loss_grad: no gradient asked for");
  B2F_CHECK_ARG(((uintptr_t)hidden | (uintptr_t)weight | (uintptr_t)grad_hidden |
                 (uintptr_t)grad_weight) % 16 == 0 && (uintptr_t)ws % 256 == 0,
                "b2f_vocab_loss_grad: misaligned buffer (16 bytes, workspace 256)");
  int dev = 0, sms = 0;
  if (int rc = current_device(&dev, &sms)) return rc;
  const Plan p = grad_plan(T, V, D, grad_hidden != nullptr, sms);
  B2F_CHECK_ARG(ws_bytes >= p.total, "b2f_vocab_loss_grad: workspace too small (%zu of %zu bytes)",
                ws_bytes, p.total);
  const Shape z{(int)T, (int)D, (int)V, ldh, ldw};
  auto *lab = reinterpret_cast<const long long *>(labels);
  char *w = static_cast<char *>(ws);
  return dtype == B2F_F16
             ? backward<__half>(hidden, weight, z, lab, ignore, lse, grad_loss, grad_hidden,
                                grad_weight, p, w, dev, sms, s)
             : backward<__nv_bfloat16>(hidden, weight, z, lab, ignore, lse, grad_loss,
                                       grad_hidden, grad_weight, p, w, dev, sms, s);
}

int b2f_vocab_loss_idle_block(int product, int block) {
  using namespace b2f;
  B2F_CHECK_ARG(product >= 0 && product <= 3 && block >= -1 && block < (1 << 20),
                "b2f_vocab_loss_idle_block: product %d, block %d", product, block);
  g_idle.store(((int64_t)(block + 1) << 8) | product, std::memory_order_relaxed);
  return B2F_OK;
}

int b2f_vocab_loss_wait_errors(void) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, b2f::g_vocab_wait_errors, sizeof(int)) != cudaSuccess) return -1;
  return v;
}

}  // extern "C"
