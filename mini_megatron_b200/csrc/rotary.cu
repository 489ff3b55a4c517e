// Rotary positions on the first heads of a packed [B, S, heads * d] activation.
//
// Pair i of a head, (a, b), at position p becomes
//   a' = m (a cos t - b sin t),  b' = m (b cos t + a sin t),  t = 2 pi p f_i
// with f_i in turns per position (64 bits) and m the magnitude of scaled
// variants; the gradient is the same rotation by -t.  Pairs are neighbours
// (2i, 2i + 1) or halves (i, i + r/2) of the first r elements of a head; the
// rest of the head and the other heads are copied, or left alone in place.
//
// Memory bounds it: every value is read and written once.  The angles cost
// nothing next to that because they depend on the token only: a CTA takes up
// to 4 tokens, copies what is not rotated, computes their r/2 sines and cosines
// once into shared memory (the turn p f_i in 64 bits, reduced to [-1/2, 1/2]
// before it is rounded to 32, so a position of millions keeps its angle to 2^-24
// of a turn) and then streams the rotated heads in 16-byte units, neighbouring
// threads on neighbouring units.  Values are rotated in 32 bits and rounded once.
//
// At 32 registers a thread 16 CTAs of 128 threads keep an SM's loads in flight.
// 16 x 1024 tokens of 36 heads of 64 in bf16, 24 of them rotated (151 MB): 28.0 us,
// 5.4 TB/s; 28.5 with 2 tokens, 29.5 with 256 threads, 32.8 with 256 threads, the
// angles first and the token's row found anew for every unit.  40 registers: 35 us.
// The same in fp32 (302 MB): 50.2 us, 6.0 TB/s.
#include "common.cuh"
#include "ops.h"

#include <algorithm>

namespace mmb {
namespace rope {

constexpr int kThreads = 128;
constexpr int kMaxTokens = 4;

struct Args {
  const void* x;
  void* y;
  long x_sb, x_ss, y_sb, y_ss;  // batch and token strides (elements)
  const void* positions;        // int32 / int64 or nullptr (token index in the row)
  int pos64;
  long pos_sb;                  // 0: the same positions for every row
  const double* freqs;          // [r / 2] turns per position
  float magnitude, sign;
  int S, d, rot, heads_rot, heads;
  long tokens;
  int per_cta;
  int copy;                     // 1: y is another tensor, the values that are not rotated are copied
};

template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static void load(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y), c = unpack_bf16x2(u.z), d = unpack_bf16x2(u.w);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
  }
  __device__ static void store(__nv_bfloat16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                              pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  __device__ static void load(const float* p, float (&v)[4]) {
    const float4 u = *reinterpret_cast<const float4*>(p);
    v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
  }
  __device__ static void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};

template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, 2048 / kThreads) rotary_kernel(const Args a) {
  pdl_trigger();
  constexpr int N = Vec<T>::N;
  extern __shared__ __align__(16) float s_sc[];  // [tokens of this CTA][2][r / 2]: cosines, then sines
  __shared__ long s_x[kMaxTokens], s_y[kMaxTokens];  // where the tokens' rows begin
  __shared__ double s_pos[kMaxTokens];
  const int half = a.rot / 2;
  const long t0 = (long)blockIdx.x * a.per_cta;
  const int nt = (int)min((long)a.per_cta, a.tokens - t0);
  pdl_wait();
  if (threadIdx.x < nt) {
    const long tok = t0 + threadIdx.x, b = tok / a.S, s = tok - b * a.S;
    s_x[threadIdx.x] = b * a.x_sb + s * a.x_ss;
    s_y[threadIdx.x] = b * a.y_sb + s * a.y_ss;
    double p = (double)s;
    if (a.positions)
      p = a.pos64 ? (double)static_cast<const long*>(a.positions)[b * a.pos_sb + s]
                  : (double)static_cast<const int*>(a.positions)[b * a.pos_sb + s];
    s_pos[threadIdx.x] = p;
  }
  __syncthreads();

  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  if (a.copy) {  // needs no angles
    const int tail = (a.d - a.rot) / N, full = a.d / N;
    const int copies = a.heads_rot * tail + (a.heads - a.heads_rot) * full;
    for (int u = threadIdx.x; u < nt * copies; u += kThreads) {
      const int t = u / copies, r = u - t * copies;
      long off;
      if (r < a.heads_rot * tail) {
        const int h = r / tail;
        off = (long)h * a.d + a.rot + (r - h * tail) * N;
      } else {
        off = (long)a.heads_rot * a.d + (long)(r - a.heads_rot * tail) * N;
      }
      *reinterpret_cast<uint4*>(y + s_y[t] + off) = *reinterpret_cast<const uint4*>(x + s_x[t] + off);
    }
  }
  for (int u = threadIdx.x; u < nt * half; u += kThreads) {
    const int t = u / half, i = u - t * half;
    const double turns = s_pos[t] * a.freqs[i];
    float sn, cs;
    sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
    s_sc[t * a.rot + i] = cs * a.magnitude;
    s_sc[t * a.rot + half + i] = sn * a.magnitude * a.sign;
  }
  __syncthreads();

  // rotated units: two vectors of one head (halves: one from each; neighbours: two adjacent ones)
  const int per_head = a.rot / (2 * N);
  const int per_tok = per_head * a.heads_rot;
  for (int u = threadIdx.x; u < nt * per_tok; u += kThreads) {
    const int t = u / per_tok, r = u - t * per_tok;
    const int h = r / per_head, g = r - h * per_head;
    const T* xp = x + s_x[t] + (long)h * a.d;
    T* yp = y + s_y[t] + (long)h * a.d;
    const int o0 = INTERLEAVED ? 2 * g * N : g * N;
    const int o1 = INTERLEAVED ? o0 + N : o0 + half;
    float v0[N], v1[N], w0[N], w1[N];
    Vec<T>::load(xp + o0, v0);
    Vec<T>::load(xp + o1, v1);
    const float* cs = s_sc + t * a.rot + g * N;  // the N pairs of this unit
    const float* sn = cs + half;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float c = cs[e], z = sn[e];
      if constexpr (INTERLEAVED) {
        const float p = e < N / 2 ? v0[(2 * e) % N] : v1[(2 * e) % N];
        const float q = e < N / 2 ? v0[(2 * e + 1) % N] : v1[(2 * e + 1) % N];
        (e < N / 2 ? w0 : w1)[(2 * e) % N] = p * c - q * z;
        (e < N / 2 ? w0 : w1)[(2 * e + 1) % N] = q * c + p * z;
      } else {
        w0[e] = v0[e] * c - v1[e] * z;
        w1[e] = v1[e] * c + v0[e] * z;
      }
    }
    Vec<T>::store(yp + o0, w0);
    Vec<T>::store(yp + o1, w1);
  }
}

}  // namespace rope

int rotary(const void* x, long x_sb, long x_ss, void* y, long y_sb, long y_ss, int is_f32, const void* positions,
           int pos64, long pos_sb, const double* freqs, float magnitude, float sign, int interleaved, long B, int S,
           int d, int rot, int heads_rot, int heads, int num_sms, cudaStream_t stream) {
  using namespace rope;
  const int N = is_f32 ? 4 : 8;
  if (rot < 2 * N || rot % (2 * N) || rot > d || d % N || heads_rot < 1 || heads_rot > heads || S < 1 || B < 1)
    return -1;
  Args a;
  a.x = x;
  a.y = y;
  a.x_sb = x_sb;
  a.x_ss = x_ss;
  a.y_sb = y_sb;
  a.y_ss = y_ss;
  a.positions = positions;
  a.pos64 = pos64;
  a.pos_sb = pos_sb;
  a.freqs = freqs;
  a.magnitude = magnitude;
  a.sign = sign;
  a.S = S;
  a.d = d;
  a.rot = rot;
  a.heads_rot = heads_rot;
  a.heads = heads;
  a.tokens = B * S;
  a.copy = (x != y);
  // few tokens: one per CTA, so that a short call still spreads over the SMs
  constexpr long kAngles = 47 * 1024;
  const long fit = kAngles / ((long)rot * (long)sizeof(float));  // the angles of a CTA's tokens in shared memory
  a.per_cta = (int)std::max(1L, std::min({(long)kMaxTokens, fit, a.tokens / (8L * num_sms)}));
  const long grid = (a.tokens + a.per_cta - 1) / a.per_cta;
  if (grid > 0x7fffffffL) return -2;
  const size_t smem = (size_t)a.per_cta * rot * sizeof(float);
  if (smem > (size_t)kAngles) return -3;
  if (is_f32) {
    if (interleaved) launch_early(0, rotary_kernel<float, true>, (unsigned)grid, kThreads, smem, stream, a);
    else launch_early(0, rotary_kernel<float, false>, (unsigned)grid, kThreads, smem, stream, a);
  } else {
    if (interleaved) launch_early(0, rotary_kernel<__nv_bfloat16, true>, (unsigned)grid, kThreads, smem, stream, a);
    else launch_early(0, rotary_kernel<__nv_bfloat16, false>, (unsigned)grid, kThreads, smem, stream, a);
  }
  return (int)cudaGetLastError();
}

}  // namespace mmb
