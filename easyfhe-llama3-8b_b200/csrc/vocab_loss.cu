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
//            tile's 256 columns to (max, sum of exp) per token, or turns
//            them into dz and stores that in the operand type;
//   dh       A = dz (K-major), B = W read along its rows (N-major);
//   dW       A = dz^T (M-major), B = h (N-major).
// The gradient walks the vocabulary in pieces whose dz fits a workspace: the
// logits of a piece are computed again, become dz at once, and both products
// consume it.
//
// One block per SM: warp 0 loads tiles by TMA (128-byte swizzle) into a ring of
// stages, warp 1 issues the MMAs (128 x 256 x 16), warps 2-5 read the
// accumulators; two accumulators in tensor memory let the epilogue of a tile
// run under the products of the next.  Every wait is bounded: a wait that
// runs out ends the block and is counted (b2f_vocab_loss_wait_errors).
//
// dz is rounded once to the operand type before its two products: relative to
// each dz at most half a step of the type, the size of the rounding of the
// gradients themselves, and formed from p - 1 (expm1) at the label, so a confident
// token keeps its relative precision.  fp16 cannot hold g p of a rare word, so
// there dz is scaled by a power of two that brings the largest |g| to 2^14 and
// the products are scaled back in binary32.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "plain.h"

namespace b2f {
namespace {

constexpr int VL_M = 128;       // rows of a tile (TMEM lanes)
constexpr int VL_N = 256;       // columns of a tile
constexpr int VL_K = 64;        // K step: one 128-byte swizzle row
constexpr int VL_STAGES = 4;
constexpr int VL_A_BYTES = VL_M * VL_K * 2;
constexpr int VL_B_BYTES = VL_N * VL_K * 2;
constexpr int VL_STAGE = VL_A_BYTES + VL_B_BYTES;
constexpr int VL_THREADS = 192;
constexpr int VL_BARRIERS = 256;  // bytes in front of the stages' alignment slack
constexpr size_t VL_SMEM = (size_t)VL_STAGES * VL_STAGE + VL_BARRIERS + 1024;
constexpr int VL_WAIT_LIMIT = 1 << 23;  // polls (each may suspend the thread for a while)
static_assert(VL_SMEM <= 227 * 1024, "stages exceed shared memory");

__device__ int g_vocab_wait_errors;

enum Epilogue { EPI_STATS, EPI_DZ, EPI_PARTIAL, EPI_OUT };

struct VocabArgs {
  int M, N, K;          // the product's sizes
  int m_tiles, n_tiles, splits, k_blocks, split_blocks;  // K blocks in all, of a split
  int n_first;          // first row of B's outer coordinate (logits: first word of the piece)
  int k_first;          // dh: first word of the piece (row of W)
  // logits
  const long long *labels;
  long long ignore;
  int vocab;
  float2 *part;         // [n_tiles][M] (max, sum)
  float *label_logit;   // [M]
  const float *lse, *grad;
  const uint32_t *grad_max;  // bits of max |g| (fp16 only)
  void *out;            // dz, dh or dW
  long long ld_out;
  // dh partial sums
  float *partial;       // [splits][M][N]
  int accumulate;
};

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
__device__ __forceinline__ void bar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(sptr(bar)) : "memory");
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
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, volatile int *lost) {
  for (int it = 0; it < VL_WAIT_LIMIT; ++it) {
    if (bar_try(bar, parity)) return true;
    if (*lost) return false;
  }
  *lost = 1;
  atomicAdd(&g_vocab_wait_errors, 1);
  return false;
}
__device__ __forceinline__ void tma_2d(void *dst, const CUtensorMap *map, int x, int y,
                                       uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];\n" ::"r"(sptr(dst)),
      "l"((uint64_t)map), "r"(x), "r"(y), "r"(sptr(bar))
      : "memory");
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(
          sptr(bar))
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

// power of two S with S max|g| in [2^13, 2^14] (1 for a zero, infinite or NaN
// maximum): dz is formed times S for fp16
__device__ __forceinline__ float dz_scale(const uint32_t *grad_max) {
  const int e = (int)(__ldg(grad_max) >> 23);  // sign bit clear
  if (e == 0 || e == 255) return 1.0f;
  const int k = min(max(127 + 13 - (e - 127), 1), 254);
  return __uint_as_float((uint32_t)k << 23);
}

constexpr float kLog2e = 1.4426950408889634f;

template <class T, int EPI>
__device__ __forceinline__ void epilogue_tile(const VocabArgs &a, uint32_t tmem, int m0, int n0,
                                              int split, int row) {
  const int t = m0 + row;
  const bool live = t < a.M;
  if constexpr (EPI == EPI_STATS || EPI == EPI_DZ) {
    const long long label = live ? a.labels[t] : a.ignore;
    // column of the label in this tile
    const long long at = label - a.n_first - n0;
    const int hit = at >= 0 && at < VL_N ? (int)at : -1;
    const int cols = min(VL_N, a.N - n0);
    if constexpr (EPI == EPI_STATS) {
      float mx = -INFINITY, sum = 0.0f;
      for (int c = 0; c < VL_N; c += 32) {
        if (c >= cols) break;
        __syncwarp();  // the tensor-memory load takes the whole warp
        float v[32];
        tmem_ld32(tmem + c, v);
        if (c + 32 > cols)
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c + j >= cols) v[j] = -INFINITY;
        float m2 = mx;
#pragma unroll
        for (int j = 0; j < 32; ++j) m2 = fmaxf(m2, v[j]);
        // an empty maximum must not make inf - inf of its own
        const float base = m2 == -INFINITY ? 0.0f : m2;
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 32; ++j) s += exp2f((v[j] - base) * kLog2e);
        sum = sum * exp2f((mx - base) * kLog2e) + s;
        mx = m2;
        if ((hit >> 5) == (c >> 5) && hit >= 0) {
          float z = 0.0f;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c + j == hit) z = v[j];
          if (live) a.label_logit[t] = z;
        }
      }
      if (live) a.part[(long long)(n0 / VL_N) * a.M + t] = make_float2(mx, sum);
    } else {
      const bool counted = live && label != a.ignore;
      const bool valid = label >= 0 && label < a.vocab;
      float g = counted ? a.grad[t] : 0.0f;
      if (counted && !valid) g = NAN;
      if constexpr (sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value)
        g *= dz_scale(a.grad_max);
      const float lse = live ? a.lse[t] : 0.0f;
      T *out = static_cast<T *>(a.out) + (long long)t * a.ld_out + n0;
      for (int c = 0; c < VL_N; c += 32) {
        if (c >= cols) break;
        __syncwarp();  // the tensor-memory load takes the whole warp
        float v[32];
        tmem_ld32(tmem + c, v);
        if (!live) continue;
        const int h = (hit >> 5) == (c >> 5) && hit >= 0 ? hit - c : -1;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float x = v[j] - lse;
          float p = exp2f(x * kLog2e);
          if (j == h) p = expm1f(x);
          v[j] = counted ? g * p : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 32; j += 8)
          if (c + j < cols) {
            uint4 w;
            w.x = pack2<T>(v[j], v[j + 1]);
            w.y = pack2<T>(v[j + 2], v[j + 3]);
            w.z = pack2<T>(v[j + 4], v[j + 5]);
            w.w = pack2<T>(v[j + 6], v[j + 7]);
            *reinterpret_cast<uint4 *>(out + c + j) = w;
          }
      }
    }
  } else {
    float scale = 1.0f;
    if constexpr (std::is_same<T, __half>::value) scale = 1.0f / dz_scale(a.grad_max);
    const int cols = min(VL_N, a.N - n0);
    for (int c = 0; c < VL_N; c += 32) {
      if (c >= cols) break;
      __syncwarp();
      float v[32];
      tmem_ld32(tmem + c, v);
      if (!live) continue;
      if constexpr (EPI == EPI_PARTIAL) {
        float *out = a.partial + ((long long)split * a.M + t) * a.N + n0 + c;
#pragma unroll
        for (int j = 0; j < 32; j += 4)
          if (c + j < cols) {
            float4 w = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            if (a.accumulate) {
              const float4 o = *reinterpret_cast<const float4 *>(out + j);
              w.x += o.x, w.y += o.y, w.z += o.z, w.w += o.w;
            }
            *reinterpret_cast<float4 *>(out + j) = w;
          }
      } else {
        T *out = static_cast<T *>(a.out) + (long long)t * a.ld_out + n0 + c;
#pragma unroll
        for (int j = 0; j < 32; j += 8)
          if (c + j < cols) {
            uint4 w;
            w.x = pack2<T>(v[j] * scale, v[j + 1] * scale);
            w.y = pack2<T>(v[j + 2] * scale, v[j + 3] * scale);
            w.z = pack2<T>(v[j + 4] * scale, v[j + 5] * scale);
            w.w = pack2<T>(v[j + 6] * scale, v[j + 7] * scale);
            *reinterpret_cast<uint4 *>(out + j) = w;
          }
      }
    }
  }
}

// D[M][N] = sum_k A[m][k] B[n][k] per tile and split, handed to the epilogue.
// AMN / BMN: the operand lies in memory with M (N) contiguous, so a stage of it
// is blocks of 64 M (N) values x 64 K rows instead of rows of 64 K values.
template <class T, int EPI, bool AMN, bool BMN>
__global__ void __launch_bounds__(VL_THREADS, 1)
    vocab_gemm_kernel(const __grid_constant__ CUtensorMap map_a,
                      const __grid_constant__ CUtensorMap map_b, const VocabArgs a) {
  extern __shared__ unsigned char vl_raw[];
  unsigned char *base = vl_raw + VL_BARRIERS;
  base += (1024 - (sptr(base) & 1023)) & 1023;
  uint64_t *full = reinterpret_cast<uint64_t *>(vl_raw + ((16 - (sptr(vl_raw) & 15)) & 15));
  uint64_t *empty = full + VL_STAGES, *acc_full = empty + VL_STAGES, *acc_empty = acc_full + 2;
  uint32_t *tmem_ptr = reinterpret_cast<uint32_t *>(acc_empty + 2);
  volatile int *lost = reinterpret_cast<volatile int *>(tmem_ptr + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < VL_STAGES; ++s) bar_init(full + s, 1), bar_init(empty + s, 1);
    for (int s = 0; s < 2; ++s) bar_init(acc_full + s, 1), bar_init(acc_empty + s, 128);
    *lost = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(
                     sptr(tmem_ptr)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_ptr;
  const int tiles = a.m_tiles * a.n_tiles * a.splits;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
        const int mt = tile % a.m_tiles, r = tile / a.m_tiles;
        const int nt = r % a.n_tiles, split = r / a.n_tiles;
        const int kb0 = split * a.split_blocks, kb1 = min(kb0 + a.split_blocks, a.k_blocks);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % VL_STAGES;
          if (it >= VL_STAGES &&
              !(ok = bar_wait(empty + s, ((it / VL_STAGES) - 1) & 1, lost)))
            break;
          unsigned char *sa = base + s * VL_STAGE, *sb = sa + VL_A_BYTES;
          bar_expect(full + s, VL_STAGE);
          if (AMN) {
#pragma unroll
            for (int i = 0; i < VL_M / 64; ++i)
              tma_2d(sa + i * 8192, &map_a, mt * VL_M + i * 64, kb * VL_K, full + s);
          } else {
            tma_2d(sa, &map_a, kb * VL_K, mt * VL_M, full + s);
          }
          if (BMN) {
#pragma unroll
            for (int i = 0; i < VL_N / 64; ++i)
              tma_2d(sb + i * 8192, &map_b, nt * VL_N + i * 64, a.k_first + kb * VL_K, full + s);
          } else {
            tma_2d(sb, &map_b, kb * VL_K, a.n_first + nt * VL_N, full + s);
          }
        }
      }
      if (!ok)  // let the loads in flight land before the block ends
        for (int i = max(0, it - VL_STAGES); i < it; ++i)
          for (int p = 0; p < VL_WAIT_LIMIT && !bar_try(full + i % VL_STAGES, (i / VL_STAGES) & 1);
               ++p) {
          }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)AMN << 15) |
                                 ((uint32_t)BMN << 16) | ((uint32_t)(VL_N >> 3) << 17) |
                                 ((uint32_t)(VL_M >> 4) << 24);
      int it = 0, n = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++n) {
        const int split = tile / (a.m_tiles * a.n_tiles);
        const int kb0 = split * a.split_blocks, kb1 = min(kb0 + a.split_blocks, a.k_blocks);
        const int buf = n & 1;
        if (n >= 2 && !(ok = bar_wait(acc_empty + buf, ((n >> 1) - 1) & 1, lost))) break;
        fence_after();
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % VL_STAGES;
          if (!(ok = bar_wait(full + s, (it / VL_STAGES) & 1, lost))) break;
          fence_after();
          const uint32_t sa = sptr(base + s * VL_STAGE), sb = sa + VL_A_BYTES;
#pragma unroll
          for (int k = 0; k < VL_K / 16; ++k)
            mma_f16(tmem + buf * VL_N, swizzled_desc(sa + k * (AMN ? 2048 : 32), 8192),
                    swizzled_desc(sb + k * (BMN ? 2048 : 32), 8192), idesc,
                    kb > kb0 || k > 0);
          mma_commit(empty + s);
        }
        if (ok) mma_commit(acc_full + buf);
      }
    }
  } else {
    const int row = (warp & 3) * 32 + lane;
    int n = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++n) {
      const int mt = tile % a.m_tiles, r = tile / a.m_tiles;
      const int nt = r % a.n_tiles, split = r / a.n_tiles;
      const int buf = n & 1;
      const bool ok = bar_wait(acc_full + buf, (n >> 1) & 1, lost);
      if (!__all_sync(~0u, ok)) break;
      fence_after();
      epilogue_tile<T, EPI>(a, tmem + buf * VL_N + ((uint32_t)((warp & 3) * 32) << 16),
                            mt * VL_M, nt * VL_N, split, row);
      fence_before();
      bar_arrive(acc_empty + buf);
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem),
                 "r"(512));
}

// Joins the tiles' (max, sum): block (32 tokens, 16 slices of the tiles).
__global__ void __launch_bounds__(512)
    vocab_join_kernel(const float2 *__restrict__ part, const float *__restrict__ label_logit,
                      const long long *__restrict__ labels, long long ignore, int vocab,
                      int T, int n_tiles, float *__restrict__ loss, float *__restrict__ lse) {
  __shared__ float2 sm[16][33];
  const int t = blockIdx.x * 32 + threadIdx.x;
  float m = -INFINITY, s = 0.0f;
  auto join = [&](float2 p) {
    const float m2 = fmaxf(m, p.x), base = m2 == -INFINITY ? 0.0f : m2;
    s = s * exp2f((m - base) * kLog2e) + p.y * exp2f((p.x - base) * kLog2e);
    m = m2;
  };
  if (t < T)
    for (int n = threadIdx.y; n < n_tiles; n += 16) join(part[(long long)n * T + t]);
  sm[threadIdx.y][threadIdx.x] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.y || t >= T) return;
  m = -INFINITY, s = 0.0f;
  for (int y = 0; y < 16; ++y) join(sm[y][threadIdx.x]);
  const long long label = labels[t];
  const float ls = logf(s);
  lse[t] = m + ls;
  float l = 0.0f;
  if (label != ignore) l = label >= 0 && label < vocab ? (m - label_logit[t]) + ls : NAN;
  loss[t] = l;
}

// Hidden states with the rows of ignored tokens set to zero (whatever lies
// there, infinities and NaN included, must not reach dW) and max |g|.
template <class T>
__global__ void __launch_bounds__(128)
    vocab_mask_kernel(const T *__restrict__ h, long long ldh, int D,
                      const long long *__restrict__ labels, long long ignore,
                      const float *__restrict__ grad, T *__restrict__ out,
                      uint32_t *__restrict__ grad_max) {
  const long long t = blockIdx.x;
  const bool counted = labels[t] != ignore;
  const uint4 *in = reinterpret_cast<const uint4 *>(h + t * ldh);
  uint4 *o = reinterpret_cast<uint4 *>(out + t * D);
  for (int i = threadIdx.x; i < D / 8; i += 128)
    o[i] = counted ? in[i] : make_uint4(0, 0, 0, 0);
  if (grad_max && threadIdx.x == 0 && counted)
    atomicMax(grad_max, __float_as_uint(fabsf(grad[t])));
}

// Sum of the splits' dh, in order, rounded once.
template <class T>
__global__ void vocab_sum_kernel(const float4 *__restrict__ partial, int splits, long long n4,
                                 const uint32_t *__restrict__ grad_max, uint2 *__restrict__ out) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n4) return;
  float4 v = partial[i];
  for (int s = 1; s < splits; ++s) {
    const float4 w = partial[(long long)s * n4 + i];
    v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
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

// matrix [rows][cols] of 16-bit values, rows ld apart, in boxes of 64 columns
template <class T>
int encode_map(CUtensorMap *m, const void *p, long long rows, long long cols, long long ld,
               int box_rows) {
  const TensorMapEncoder enc = map_encoder();
  if (!enc) {
    set_error("the driver has no cuTensorMapEncodeTiled");
    return B2F_ERR_UNSUPPORTED;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, es[2] = {1, 1};
  const CUresult r =
      enc(m,
          std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                         : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
          2, const_cast<void *>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("tensor map of %lld x %lld (rows %lld apart): error %d", rows, cols, ld, (int)r);
    return B2F_ERR_CUDA;
  }
  return B2F_OK;
}

int sm_count(int *sms) {
  int dev = 0;
  return current_device(&dev, sms);
}

template <class T, int EPI, bool AMN, bool BMN>
int launch_gemm(const CUtensorMap &ma, const CUtensorMap &mb, VocabArgs a, int sms,
                cudaStream_t s) {
  auto k = vocab_gemm_kernel<T, EPI, AMN, BMN>;
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  if (int rc = current_device(&dev, &sms)) return rc;
  if (int rc = allow_shared(k, (int)VL_SMEM, dev, allowed)) return rc;
  a.m_tiles = (a.M + VL_M - 1) / VL_M;
  a.n_tiles = (a.N + VL_N - 1) / VL_N;
  a.k_blocks = (a.K + VL_K - 1) / VL_K;
  a.split_blocks = (a.k_blocks + a.splits - 1) / a.splits;
  a.splits = (a.k_blocks + a.split_blocks - 1) / a.split_blocks;  // none empty
  const long long tiles = (long long)a.m_tiles * a.n_tiles * a.splits;
  B2F_CHECK_ARG(tiles < (1ll << 31), "b2f_vocab_loss: %lld tiles", tiles);
  k<<<(unsigned)std::min<long long>(tiles, sms), VL_THREADS, VL_SMEM, s>>>(ma, mb, a);
  B2F_LAUNCHED("vocab_gemm_kernel");
  return B2F_OK;
}

struct Shape {
  int T, D, V;
  long long ldh, ldw;
};

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// How the gradient is cut: words of a piece, splits of dh's sum over a piece.
struct Plan {
  int piece, pieces, splits;
  size_t hc, dz, partial, gmax, total;
};
constexpr size_t kDzBytes = 256ull << 20;

Plan grad_plan(int64_t T, int64_t V, int64_t D, bool need_h, int sms) {
  Plan p{};
  int64_t words = (int64_t)(kDzBytes / 2 / (size_t)T) / VL_N * VL_N;
  words = std::max<int64_t>(words, VL_N);
  p.pieces = (int)((V + words - 1) / words);
  p.piece = (int)(((V + p.pieces - 1) / p.pieces + VL_N - 1) / VL_N * VL_N);
  p.pieces = (int)((V + p.piece - 1) / p.piece);
  const int64_t tiles = ((T + VL_M - 1) / VL_M) * ((D + VL_N - 1) / VL_N);
  const int64_t kb = (std::min<int64_t>(p.piece, V) + VL_K - 1) / VL_K;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(sms / tiles, kb / 4));
  const int64_t per = (kb + p.splits - 1) / p.splits;
  p.splits = (int)((kb + per - 1) / per);  // every split of the first piece has work
  size_t off = 0;
  p.hc = off, off += round256((size_t)T * D * 2);
  p.dz = off, off += round256((size_t)T * p.piece * 2);
  p.partial = off;
  if (need_h) off += round256((size_t)p.splits * T * D * 4);
  p.gmax = off, off += 256;
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
            long long ignore, float *loss, float *lse, void *ws, int sms, cudaStream_t s) {
  CUtensorMap ma, mb;
  if (int rc = encode_map<T>(&ma, h, z.T, z.D, z.ldh, VL_M)) return rc;
  if (int rc = encode_map<T>(&mb, w, z.V, z.D, z.ldw, VL_N)) return rc;
  VocabArgs a{};
  a.M = z.T, a.N = z.V, a.K = z.D, a.splits = 1;
  a.labels = labels, a.ignore = ignore, a.vocab = z.V;
  a.label_logit = static_cast<float *>(ws);
  a.part = reinterpret_cast<float2 *>(static_cast<char *>(ws) + round256((size_t)z.T * 4));
  if (int rc = launch_gemm<T, EPI_STATS, false, false>(ma, mb, a, sms, s)) return rc;
  vocab_join_kernel<<<(z.T + 31) / 32, dim3(32, 16), 0, s>>>(
      a.part, a.label_logit, labels, ignore, z.V, z.T, (z.V + VL_N - 1) / VL_N, loss, lse);
  B2F_LAUNCHED("vocab_join_kernel");
  return B2F_OK;
}

template <class T>
int backward(const void *h, const void *w, const Shape &z, const long long *labels,
             long long ignore, const float *lse, const float *grad, void *dh, void *dw,
             const Plan &p, char *ws, int sms, cudaStream_t s) {
  T *hc = reinterpret_cast<T *>(ws + p.hc), *dz = reinterpret_cast<T *>(ws + p.dz);
  float *partial = reinterpret_cast<float *>(ws + p.partial);
  uint32_t *gmax = nullptr;
  if (std::is_same<T, __half>::value) {
    gmax = reinterpret_cast<uint32_t *>(ws + p.gmax);
    B2F_CUDA(cudaMemsetAsync(gmax, 0, 4, s));
  }
  vocab_mask_kernel<T><<<z.T, 128, 0, s>>>(static_cast<const T *>(h), z.ldh, z.D, labels, ignore,
                                           grad, hc, gmax);
  B2F_LAUNCHED("vocab_mask_kernel");
  CUtensorMap h_k, h_n, w_k, w_n, dz_k, dz_m;
  if (int rc = encode_map<T>(&h_k, hc, z.T, z.D, z.D, VL_M)) return rc;
  if (int rc = encode_map<T>(&w_k, w, z.V, z.D, z.ldw, VL_N)) return rc;
  if (int rc = encode_map<T>(&h_n, hc, z.T, z.D, z.D, VL_K)) return rc;
  if (int rc = encode_map<T>(&w_n, w, z.V, z.D, z.ldw, VL_K)) return rc;
  for (int i = 0; i < p.pieces; ++i) {
    const int v0 = i * p.piece, words = std::min(p.piece, z.V - v0);
    VocabArgs a{};
    a.M = z.T, a.N = words, a.K = z.D, a.splits = 1;
    a.n_first = v0;
    a.labels = labels, a.ignore = ignore, a.vocab = z.V;
    a.lse = lse, a.grad = grad, a.grad_max = gmax;
    a.out = dz, a.ld_out = p.piece;
    if (int rc = launch_gemm<T, EPI_DZ, false, false>(h_k, w_k, a, sms, s)) return rc;
    if (dh) {
      if (int rc = encode_map<T>(&dz_k, dz, z.T, words, p.piece, VL_M)) return rc;
      VocabArgs b{};
      b.M = z.T, b.N = z.D, b.K = words, b.splits = p.splits;
      b.k_first = v0;
      b.partial = partial, b.accumulate = i > 0;
      if (int rc = launch_gemm<T, EPI_PARTIAL, false, true>(dz_k, w_n, b, sms, s)) return rc;
    }
    if (dw) {
      if (int rc = encode_map<T>(&dz_m, dz, z.T, words, p.piece, VL_K)) return rc;
      VocabArgs b{};
      b.M = words, b.N = z.D, b.K = z.T, b.splits = 1;
      b.grad_max = gmax;
      b.out = static_cast<T *>(dw) + (long long)v0 * z.D, b.ld_out = z.D;
      if (int rc = launch_gemm<T, EPI_OUT, true, true>(dz_m, h_n, b, sms, s)) return rc;
    }
  }
  if (dh) {
    const long long n4 = (long long)z.T * z.D / 4;
    vocab_sum_kernel<T><<<(unsigned)((n4 + 255) / 256), 256, 0, s>>>(
        reinterpret_cast<const float4 *>(partial), p.splits, n4, gmax,
        static_cast<uint2 *>(dh));
    B2F_LAUNCHED("vocab_sum_kernel");
  }
  return B2F_OK;
}

}  // namespace
}  // namespace b2f

extern "C" {

size_t b2f_vocab_loss_workspace(int64_t T, int64_t V, int64_t D) {
  using namespace b2f;
  if (T < 1 || V < 1) return 0;
  return round256((size_t)T * 4) + round256((size_t)((V + VL_N - 1) / VL_N) * T * 8);
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
  B2F_CHECK_ARG(ws_bytes >= b2f_vocab_loss_workspace(T, V, D),
                "b2f_vocab_loss: workspace too small (%zu bytes)", ws_bytes);
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const Shape z{(int)T, (int)D, (int)V, ldh, ldw};
  auto *lab = reinterpret_cast<const long long *>(labels);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == B2F_F16
             ? forward<__half>(hidden, weight, z, lab, ignore, loss, lse, ws, sms, s)
             : forward<__nv_bfloat16>(hidden, weight, z, lab, ignore, loss, lse, ws, sms, s);
}

size_t b2f_vocab_loss_grad_workspace(int64_t T, int64_t V, int64_t D, int need_hidden) {
  using namespace b2f;
  int sms = 0;
  if (T < 1 || V < 1 || D < 1 || sm_count(&sms)) return 0;
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
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const Plan p = grad_plan(T, V, D, grad_hidden != nullptr, sms);
  B2F_CHECK_ARG(ws_bytes >= p.total, "b2f_vocab_loss_grad: workspace too small (%zu of %zu bytes)",
                ws_bytes, p.total);
  const Shape z{(int)T, (int)D, (int)V, ldh, ldw};
  auto *lab = reinterpret_cast<const long long *>(labels);
  char *w = static_cast<char *>(ws);
  return dtype == B2F_F16
             ? backward<__half>(hidden, weight, z, lab, ignore, lse, grad_loss, grad_hidden,
                                grad_weight, p, w, sms, s)
             : backward<__nv_bfloat16>(hidden, weight, z, lab, ignore, lse, grad_loss,
                                       grad_hidden, grad_weight, p, w, sms, s);
}

int b2f_vocab_loss_wait_errors(void) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, b2f::g_vocab_wait_errors, sizeof(int)) != cudaSuccess) return -1;
  return v;
}

}  // extern "C"
