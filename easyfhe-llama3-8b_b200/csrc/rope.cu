// Rotary positions of the plaintext decoder layer (the plain twin that an
// encrypted layer is checked against).
//
// A pair (x0, x1) of a head at position p with frequency f:
//   y0 = x0 c - x1 s,  y1 = x1 c + x0 s,  c = m cos(p f),  s = m sin(p f),
// pairs (i, i + r/2) ("half") or (2i, 2i + 1) ("interleaved") of the first r
// elements of the head; the rest is copied.  The gradient is the rotation by
// the negative angle.
//
// Bytes bound: every element is read and written once, 3 operations each.  A
// block takes up to ROPE_TOKENS tokens of a sequence (one where there are few): its
// threads first compute the r/2 (c, s) of each token into shared memory (once per
// token, for all of its heads), then each thread keeps the (c, s) of its 16 bytes
// of pairs in registers and runs over the heads.  What paid beside that: sequences
// on the grid's second dimension, because a 64-bit division by their length per
// token and thread took more instructions than the rotation (32768 tokens of 40
// heads of 128 in bf16: 159 us with it, 109 without, 94 % of copy bandwidth), both
// loads of a head before anything else of it (131 us with the second one after the
// output's address), and registers for five blocks of 256 threads on an SM (four
// with two heads in flight per thread: 129 us).
// The angle of a far position needs more than binary32: p f is formed in binary64
// and reduced there to a fraction of a turn in [-1/2, 1/2] (off by 2^-52 of the turns).
// Heads of 16 bits take its sine and cosine in binary32 (the rounding of the fraction is
// 2^-26 of a turn at most, far below their own step); binary32 heads, which would feel that,
// take them in binary64 and round once; binary64 heads take binary64 sines of p f.
#include "plain.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2f {
namespace {

constexpr int ROPE_TOKENS = 4;     // tokens of a block, at most
constexpr int ROPE_THREADS = 256;  // at most

struct RopePart {
  const void *in;
  void *out;
  long long ib, is, ih, ob, os, oh;  // strides in elements
};
struct RopeArgs {
  RopePart part[2];
  int heads0, heads;  // heads of part 0, of both
  int block_tokens;
  long long batch, seq;
  int dim, rotary, interleaved;
  const void *pos;
  int pos64;
  long long pos_b, pos_s;  // strides of the positions
  const double *freqs;
  double factor;  // m; the gradient's sign is in `sign`
  int sign;
};

template <class T>
struct Wide {
  using V = float;
  using V2 = float2;
};
template <>
struct Wide<double> {
  using V = double;
  using V2 = double2;
};

__device__ __forceinline__ float to_wide(float x) { return x; }
__device__ __forceinline__ float to_wide(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_wide(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ double to_wide(double x) { return x; }
template <class T>
__device__ __forceinline__ T from_wide(typename Wide<T>::V x);
template <>
__device__ __forceinline__ float from_wide<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ double from_wide<double>(double x) {
  return x;
}
template <>
__device__ __forceinline__ __half from_wide<__half>(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_wide<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// m (cos, sin) of p f for heads of type T
template <class T>
__device__ __forceinline__ void turn_of(double p, double f, double factor, int sign,
                                        typename Wide<T>::V2 &o) {
  constexpr double kInv2Pi = 0.15915494309189533577;
  if constexpr (std::is_same<T, double>::value) {
    double s, c;
    sincos(p * f, &s, &c);
    o = make_double2(c * factor, (double)sign * s * factor);
    return;
  } else {
    double t = p * f * kInv2Pi;
    t -= rint(t);
    if constexpr (std::is_same<T, float>::value) {
      double s, c;
      sincospi(2.0 * t, &s, &c);
      o = make_float2((float)(c * factor), (float)((double)sign * s * factor));
    } else {
      float s, c;
      sincospif(2.0f * (float)t, &s, &c);
      o = make_float2(c * (float)factor, (float)sign * s * (float)factor);
    }
  }
}

// two roundings at once
__device__ __forceinline__ void put2(__nv_bfloat16 *o, float a, float b) {
  *reinterpret_cast<__nv_bfloat162 *>(o) = __floats2bfloat162_rn(a, b);
}
__device__ __forceinline__ void put2(__half *o, float a, float b) {
  *reinterpret_cast<__half2 *>(o) = __floats2half2_rn(a, b);
}
__device__ __forceinline__ void put2(float *o, float a, float b) { o[0] = a, o[1] = b; }
__device__ __forceinline__ void put2(double *o, double a, double b) { o[0] = a, o[1] = b; }

template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// block (x: 16-byte units of a head, y: heads), grid: ROPE_TOKENS tokens each.
// VEC elements per access; units [0, rot_units) rotate, the rest copy.
template <class T, int VEC>
__global__ void __launch_bounds__(ROPE_THREADS, 5)
    rope_kernel(const RopeArgs a, int rot_units, int units) {
  using W = typename Wide<T>::V;
  using W2 = typename Wide<T>::V2;
  extern __shared__ __align__(16) unsigned char rope_smem[];
  const int half = a.rotary / 2;
  // (c, s) of the block's tokens, cosines and sines apart
  W *cosines = reinterpret_cast<W *>(rope_smem), *sines = cosines + a.block_tokens * half;
  using P = Pack<T, VEC>;
  // pairs of a unit: half layout VEC of them, interleaved VEC / 2 (1 for VEC 1)
  const int pairs = a.interleaved && VEC > 1 ? VEC / 2 : VEC;
  const bool two = !(VEC > 1 && a.interleaved);  // a rotated unit is two accesses
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
  const long long s0 = (long long)blockIdx.x * a.block_tokens;
  const int nt = (int)min((long long)a.block_tokens, a.seq - s0);
  for (long long b = blockIdx.y; b < a.batch; b += gridDim.y) {
    for (int i = tid; i < nt * half; i += blockDim.x * blockDim.y) {
      const int t = i / half, j = i - t * half;
      const long long at = b * a.pos_b + (s0 + t) * a.pos_s;
      const double p = a.pos64 ? (double)static_cast<const long long *>(a.pos)[at]
                               : (double)static_cast<const int *>(a.pos)[at];
      W2 cs;
      turn_of<T>(p, a.freqs[j], a.factor, a.sign, cs);
      cosines[i] = cs.x;
      sines[i] = cs.y;
    }
    __syncthreads();
    const T *in0 = static_cast<const T *>(a.part[0].in) + b * a.part[0].ib + s0 * a.part[0].is;
    const T *in1 = static_cast<const T *>(a.part[1].in) + b * a.part[1].ib + s0 * a.part[1].is;
    T *out0 = static_cast<T *>(a.part[0].out) + b * a.part[0].ob + s0 * a.part[0].os;
    T *out1 = static_cast<T *>(a.part[1].out) + b * a.part[1].ob + s0 * a.part[1].os;
    for (int t = 0; t < nt; ++t) {
      for (int u = threadIdx.x; u < units; u += blockDim.x) {
        const bool rot = u < rot_units;
        W c[VEC], n[VEC];
        int e0, e1 = 0;  // element offsets of the unit's accesses
        if (rot) {
          e0 = a.interleaved ? u * pairs * 2 : u * VEC;
          e1 = a.interleaved ? e0 + 1 : e0 + half;
#pragma unroll
          for (int k = 0; k < VEC; ++k)
            if (k < pairs) {
              c[k] = cosines[t * half + u * pairs + k];
              n[k] = sines[t * half + u * pairs + k];
            }
        } else {
          e0 = a.rotary + (u - rot_units) * VEC;
        }
#pragma unroll 1
        for (int h = threadIdx.y; h < a.heads; h += blockDim.y) {
          const bool first = h < a.heads0;
          const T *in = first ? in0 + h * a.part[0].ih : in1 + (h - a.heads0) * a.part[1].ih;
          P x0, x1;
          x0 = *reinterpret_cast<const P *>(in + e0);
          if (rot && two) x1 = *reinterpret_cast<const P *>(in + e1);
          T *out = first ? out0 + h * a.part[0].oh : out1 + (h - a.heads0) * a.part[1].oh;
          P y0 = x0;
          if (rot && two) {
            P y1;
            if constexpr (VEC == 1) {
              const W lo = to_wide(x0.v[0]), hi = to_wide(x1.v[0]);
              y0.v[0] = from_wide<T>(lo * c[0] - hi * n[0]);
              y1.v[0] = from_wide<T>(hi * c[0] + lo * n[0]);
            } else {
#pragma unroll
              for (int k = 0; k < VEC; k += 2) {
                const W lo = to_wide(x0.v[k]), hi = to_wide(x1.v[k]);
                const W lo1 = to_wide(x0.v[k + 1]), hi1 = to_wide(x1.v[k + 1]);
                put2(y0.v + k, lo * c[k] - hi * n[k], lo1 * c[k + 1] - hi1 * n[k + 1]);
                put2(y1.v + k, hi * c[k] + lo * n[k], hi1 * c[k + 1] + lo1 * n[k + 1]);
              }
            }
            *reinterpret_cast<P *>(out + e1) = y1;
          } else if (rot) {
#pragma unroll
            for (int k = 0; k < VEC / 2; ++k) {
              const W lo = to_wide(x0.v[2 * k]), hi = to_wide(x0.v[2 * k + 1]);
              put2(y0.v + 2 * k, lo * c[k] - hi * n[k], hi * c[k] + lo * n[k]);
            }
          }
          *reinterpret_cast<P *>(out + e0) = y0;
        }
      }
      in0 += a.part[0].is, in1 += a.part[1].is;
      out0 += a.part[0].os, out1 += a.part[1].os;
    }
    __syncthreads();  // before the next sequence's angles
  }
}

template <class T>
int launch_rope(RopeArgs a, int parts, int sms, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int half = a.rotary / 2;
  bool vec = a.dim % V == 0 && a.rotary % V == 0 && (a.interleaved || half % V == 0);
  for (int i = 0; i < parts; ++i) {
    const RopePart &p = a.part[i];
    vec = vec && ((uintptr_t)p.in | (uintptr_t)p.out) % 16 == 0;
    for (long long st : {p.ib, p.is, p.ih, p.ob, p.os, p.oh}) vec = vec && st % V == 0;
  }
  // units of a head: rotated (two accesses of VEC in the half layout, one
  // interleaved; a pair for VEC 1), then copied
  const int v = vec ? V : 1;
  const int rot_units = vec && a.interleaved ? a.rotary / v : half / v;
  const int units = rot_units + (a.dim - a.rotary) / v;
  const int bx = std::min(units, 64);
  // heads split evenly over the passes that a block of at most 256 threads needs
  const int passes = (a.heads * bx + ROPE_THREADS - 1) / ROPE_THREADS;
  const int by = std::min((a.heads + passes - 1) / passes, ROPE_THREADS / bx);
  const dim3 block(bx, by);
  // few tokens: one to a block; more share a block's pipeline
  a.block_tokens = (int)std::max<long long>(
      1, std::min<long long>(ROPE_TOKENS, a.batch * a.seq / (8 * sms)));
  const dim3 grid((unsigned)((a.seq + a.block_tokens - 1) / a.block_tokens),
                  (unsigned)std::min<long long>(a.batch, 65535));
  const size_t smem = (size_t)a.block_tokens * half * 2 * sizeof(typename Wide<T>::V);
  if (vec)
    rope_kernel<T, V><<<grid, block, smem, s>>>(a, rot_units, units);
  else
    rope_kernel<T, 1><<<grid, block, smem, s>>>(a, rot_units, units);
  B2F_LAUNCHED("rope_kernel");
  return B2F_OK;
}

}  // namespace
}  // namespace b2f

extern "C" int b2f_rope(const b2f_rope_heads *parts, int num_parts, int dtype, int64_t batch,
                        int64_t seq, int dim, int rotary, int interleaved,
                        const void *positions, int positions64, int64_t pos_batch_stride,
                        int64_t pos_seq_stride, const double *freqs, double factor,
                        int gradient, void *stream) {
  B2F_RANGE("b2f_rope");
  using namespace b2f;
  B2F_CHECK_ARG(parts && num_parts >= 1 && num_parts <= 2, "b2f_rope: one or two parts");
  B2F_CHECK_ARG(batch >= 0 && seq >= 0, "b2f_rope: batch %lld, seq %lld", (long long)batch,
                (long long)seq);
  B2F_CHECK_ARG(dim >= 2 && dim <= 1024 && rotary >= 2 && rotary <= dim && rotary % 2 == 0,
                "b2f_rope: head of %d elements, %d rotated (an even number of 2 to dim, dim up "
                "to 1024)",
                dim, rotary);
  RopeArgs a{};
  long long heads = 0;
  for (int i = 0; i < num_parts; ++i) {
    B2F_CHECK_ARG(parts[i].heads >= 1 && parts[i].heads <= 4096, "b2f_rope: %d heads",
                  parts[i].heads);
    heads += parts[i].heads;
    a.part[i] = {parts[i].in,       parts[i].out,       parts[i].in_batch,
                 parts[i].in_seq,   parts[i].in_head,   parts[i].out_batch,
                 parts[i].out_seq,  parts[i].out_head};
  }
  B2F_CHECK_ARG(dtype >= B2F_F64 && dtype <= B2F_BF16, "b2f_rope: dtype %d", dtype);
  if (batch == 0 || seq == 0) return B2F_OK;
  B2F_CHECK_ARG(seq < (1ll << 31) && batch < (1ll << 31), "b2f_rope: %lld x %lld tokens",
                (long long)batch, (long long)seq);
  B2F_CHECK_ARG(positions && freqs, "b2f_rope: null positions or frequencies");
  const uintptr_t size = dtype == B2F_F64 ? 8 : dtype == B2F_F32 ? 4 : 2;
  for (int i = 0; i < num_parts; ++i)
    B2F_CHECK_ARG(parts[i].in && parts[i].out &&
                      ((uintptr_t)parts[i].in | (uintptr_t)parts[i].out) % size == 0,
                  "b2f_rope: null or misaligned heads");
  a.heads0 = parts[0].heads;
  a.heads = (int)heads;
  a.batch = batch;
  a.seq = seq;
  a.dim = dim;
  a.rotary = rotary;
  a.interleaved = interleaved != 0;
  a.pos = positions;
  a.pos64 = positions64 != 0;
  a.pos_b = pos_batch_stride;
  a.pos_s = pos_seq_stride;
  a.freqs = freqs;
  a.factor = factor;
  a.sign = gradient ? -1 : 1;
  int dev = 0, sms = 0;
  if (int rc = current_device(&dev, &sms)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case B2F_F64:
      return launch_rope<double>(a, num_parts, sms, s);
    case B2F_F32:
      return launch_rope<float>(a, num_parts, sms, s);
    case B2F_F16:
      return launch_rope<__half>(a, num_parts, sms, s);
    default:
      return launch_rope<__nv_bfloat16>(a, num_parts, sms, s);
  }
}
