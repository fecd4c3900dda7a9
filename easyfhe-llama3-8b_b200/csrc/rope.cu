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
// block takes TB tokens: its threads first compute the r/2 (c, s) of each
// token into shared memory (once per token, for all of its heads), then each
// thread keeps the (c, s) of its 16 bytes of pairs in registers and runs over
// the heads.  The angle of a far position needs more than binary32: p f is
// formed in binary64 and reduced there to a fraction of a turn in [-1/2,
// 1/2], whose sine and cosine are then taken in binary32 (the reduction's
// error is 2^-52 of the turns, the rounding of the fraction 2^-25 of a turn);
// binary64 inputs take binary64 sines of p f.
#include "b2f_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2f {
namespace {

constexpr int ROPE_TOKENS = 4;     // tokens of a block
constexpr int ROPE_THREADS = 256;  // at most

struct RopePart {
  const void *in;
  void *out;
  long long ib, is, ih, ob, os, oh;  // strides in elements
};
struct RopeArgs {
  RopePart part[2];
  int heads0, heads;  // heads of part 0, of both
  long long tokens, seq;
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

// (cos, sin) of p f
__device__ __forceinline__ void turn_of(double p, double f, float factor, int sign, float2 &o) {
  constexpr double kInv2Pi = 0.15915494309189533577;
  double t = p * f * kInv2Pi;
  t -= rint(t);
  float s, c;
  sincospif(2.0f * (float)t, &s, &c);
  o = make_float2(c * factor, (float)sign * s * factor);
}
__device__ __forceinline__ void turn_of(double p, double f, double factor, int sign, double2 &o) {
  double s, c;
  sincos(p * f, &s, &c);
  o = make_double2(c * factor, (double)sign * s * factor);
}

template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// block (x: 16-byte units of a head, y: heads), grid: ROPE_TOKENS tokens each.
// VEC elements per access; units [0, rot_units) rotate, the rest copy.
template <class T, int VEC>
__global__ void __launch_bounds__(ROPE_THREADS)
    rope_kernel(const RopeArgs a, int rot_units, int units) {
  using W = typename Wide<T>::V;
  using W2 = typename Wide<T>::V2;
  extern __shared__ __align__(16) unsigned char rope_smem[];
  W2 *cs = reinterpret_cast<W2 *>(rope_smem);
  const int half = a.rotary / 2;
  const long long t0 = (long long)blockIdx.x * ROPE_TOKENS;
  const int nt = (int)min((long long)ROPE_TOKENS, a.tokens - t0);
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
  for (int i = tid; i < nt * half; i += blockDim.x * blockDim.y) {
    const int t = i / half, j = i - t * half;
    const long long tok = t0 + t, b = tok / a.seq, s = tok - b * a.seq;
    const long long at = b * a.pos_b + s * a.pos_s;
    const double p = a.pos64 ? (double)static_cast<const long long *>(a.pos)[at]
                             : (double)static_cast<const int *>(a.pos)[at];
    turn_of(p, a.freqs[j], (W)a.factor, a.sign, cs[i]);
  }
  __syncthreads();
  using P = Pack<T, VEC>;
  for (int t = 0; t < nt; ++t) {
    const long long tok = t0 + t, b = tok / a.seq, s = tok - b * a.seq;
    for (int u = threadIdx.x; u < units; u += blockDim.x) {
      const bool rot = u < rot_units;
      // pairs of this unit: half layout VEC of them, interleaved VEC / 2 (1 for VEC 1)
      constexpr int NP = VEC;
      W2 c[NP];
      int e0, e1 = 0;  // element offsets of the unit's accesses
      const int pairs = a.interleaved ? (VEC > 1 ? VEC / 2 : 1) : VEC;
      if (rot) {
        e0 = a.interleaved ? u * pairs * 2 : u * VEC;
        e1 = a.interleaved ? e0 + 1 : e0 + half;
#pragma unroll
        for (int k = 0; k < NP; ++k)
          if (k < pairs) c[k] = cs[t * half + u * pairs + k];
      } else {
        e0 = a.rotary + (u - rot_units) * VEC;
      }
      for (int h = threadIdx.y; h < a.heads; h += blockDim.y) {
        const bool second = h >= a.heads0;
        const RopePart &pt = second ? a.part[1] : a.part[0];
        const int hh = second ? h - a.heads0 : h;
        const T *in = static_cast<const T *>(pt.in) + b * pt.ib + s * pt.is + hh * pt.ih;
        T *out = static_cast<T *>(pt.out) + b * pt.ob + s * pt.os + hh * pt.oh;
        const P x0 = *reinterpret_cast<const P *>(in + e0);
        P y0 = x0;
        if (rot) {
          if (VEC > 1 && a.interleaved) {
#pragma unroll
            for (int k = 0; k < VEC / 2; ++k) {
              const W lo = to_wide(x0.v[2 * k]), hi = to_wide(x0.v[2 * k + 1]);
              y0.v[2 * k] = from_wide<T>(lo * c[k].x - hi * c[k].y);
              y0.v[2 * k + 1] = from_wide<T>(hi * c[k].x + lo * c[k].y);
            }
          } else {
            const P x1 = *reinterpret_cast<const P *>(in + e1);
            P y1;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
              const W lo = to_wide(x0.v[k]), hi = to_wide(x1.v[k]);
              y0.v[k] = from_wide<T>(lo * c[k].x - hi * c[k].y);
              y1.v[k] = from_wide<T>(hi * c[k].x + lo * c[k].y);
            }
            *reinterpret_cast<P *>(out + e1) = y1;
          }
        }
        *reinterpret_cast<P *>(out + e0) = y0;
      }
    }
  }
}

template <class T>
int launch_rope(const RopeArgs &a, int parts, cudaStream_t s) {
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
  const unsigned grid = (unsigned)((a.tokens + ROPE_TOKENS - 1) / ROPE_TOKENS);
  const size_t smem = (size_t)ROPE_TOKENS * half * 2 * sizeof(typename Wide<T>::V);
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
  B2F_CHECK_ARG(seq <= (1ll << 32) / batch, "b2f_rope: %lld x %lld tokens", (long long)batch,
                (long long)seq);
  B2F_CHECK_ARG(positions && freqs, "b2f_rope: null positions or frequencies");
  const uintptr_t size = dtype == B2F_F64 ? 8 : dtype == B2F_F32 ? 4 : 2;
  for (int i = 0; i < num_parts; ++i)
    B2F_CHECK_ARG(parts[i].in && parts[i].out &&
                      ((uintptr_t)parts[i].in | (uintptr_t)parts[i].out) % size == 0,
                  "b2f_rope: null or misaligned heads");
  a.heads0 = parts[0].heads;
  a.heads = (int)heads;
  a.tokens = batch * seq;
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case B2F_F64:
      return launch_rope<double>(a, num_parts, s);
    case B2F_F32:
      return launch_rope<float>(a, num_parts, s);
    case B2F_F16:
      return launch_rope<__half>(a, num_parts, s);
    default:
      return launch_rope<__nv_bfloat16>(a, num_parts, s);
  }
}
