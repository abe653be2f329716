// scan.cuh -- what the selective scan's forward, backward and step kernels share.
//
//   dt = softplus(delta + delta_bias)             (or delta + delta_bias)
//   h[t] = exp(dt A) h[t-1] + dt u B[t]           per channel d and state n
//   y[t] = sum_n C[t] h[t] + skip u
// A thread owns four neighbouring states n of a channel; LPC lanes hold a channel's states
// (N <= 4 LPC, padded with A = B = C = 0, which add nothing) and a warp 32 / LPC lanes across
// channels. Time is cut into superchunks: the warps of a block take consecutive pieces of one,
// run the recurrence from zero, exchange their end states and decay products through shared
// memory and run it again from the state that enters their piece, with the decays kept in
// registers. So the exponentials, which bound the forward, are computed once.
#pragma once

#include <type_traits>

#include "rowvec.cuh"

namespace dudy {
namespace scan {

constexpr int kNS = 4;        // states of a thread, neighbours in n
constexpr int kWarps = 8;     // warps of a block: consecutive pieces of a superchunk
constexpr int kThreads = 32 * kWarps;
constexpr int kCkpt = 32;     // positions between saved states
constexpr int kMaxN = DUDY_SCAN_MAX_STATE;

struct Shape {
  int64_t B, D, L;
  int N, G;
  int softplus;
  __host__ __device__ int64_t R() const { return D / G; }
  __host__ __device__ int64_t ckpts() const { return (L + kCkpt - 1) / kCkpt; }
};

__device__ __forceinline__ int64_t clamp_len(const int32_t *lengths, int64_t b, int64_t L) {
  if (!lengths) return L;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : (n > L ? L : n);
}

// exp(x) for the decays. 16-bit tensors: one multiply and the base-2 exponential of the
// special function unit (relative error about 2^-22, against 2^-9 or 2^-12 of the result's
// rounding); fp32 tensors: the accurate exponential.
template <typename T>
__device__ __forceinline__ float decay(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}
template <>
__device__ __forceinline__ float decay<float>(float x) {
  return expf(x);
}

// softplus and its derivative. 16-bit tensors: log(1 + e) = e - e^2/2 + e^3/3 - e^4/4 where
// e = exp(x) is small (the logarithm of a rounded 1 + e would lose its digits), else the fast
// logarithm; both are exact to a few 2^-20. Above 20, log(1 + e) = x to fp32's precision.
template <typename T>
__device__ __forceinline__ float softplus(float x, float &slope) {
  const float e = __expf(x);
  slope = x > 20.f ? 1.f : __fdividef(e, 1.f + e);
  const float small = e * fmaf(-e, fmaf(-e, fmaf(-e, 0.25f, 1.f / 3.f), 0.5f), 1.f);
  return x > 20.f ? x : (e < 0.03f ? small : __logf(1.f + e));
}
template <>
__device__ __forceinline__ float softplus<float>(float x, float &slope) {
  const float e = expf(x);
  slope = x > 20.f ? 1.f : e / (1.f + e);
  return x > 20.f ? x : log1pf(e);
}

// Copies a tile of `rows` rows x TS positions of a [.., L] tensor into shared memory as it is
// (pitch PITCH elements): positions [t0, t0 + TS), zero at and behind `end`, and zero rows at
// and behind `valid`. 16-byte asynchronous copies where rows start on 16 bytes (`vec`).
template <typename T, int TS, int PITCH>
__device__ __forceinline__ void stage_rows(T *dst, const T *src, int rows, int valid, int64_t L,
                                           int64_t t0, int64_t end, bool vec) {
  constexpr int V = 16 / sizeof(T), VPR = TS / V;
  for (int i = threadIdx.x; i < rows * VPR; i += kThreads) {
    const int r = i / VPR, c = (i % VPR) * V;
    T *to = dst + r * PITCH + c;
    const int64_t t = t0 + c;
    if (r < valid && vec && t + V <= end) {
      cp_async16(to, src + (int64_t)r * L + t);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k)
        to[k] = r < valid && t + k < end ? src[(int64_t)r * L + t + k] : Elem<T>::from_f(0.f);
    }
  }
}

inline int lanes_per_channel(int64_t N) {
  return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16;
}

inline int validate(int64_t B, int64_t D, int64_t L, int64_t N, int64_t G, int dtype) {
  if (B <= 0 || D <= 0 || L <= 0) return refuse("B, D and L must be positive.");
  if (N < 1 || N > kMaxN)
    return refuse("N must be between 1 and " + std::to_string(kMaxN) + ", got " +
                  std::to_string(N) + ".");
  if (G <= 0 || D % G != 0)
    return refuse("D must be a multiple of the number of groups, got D=" + std::to_string(D) +
                  ", G=" + std::to_string(G) + ".");
  if (!dtype_known(dtype)) return refuse("Unsupported dtype.");
  if (L >= ((int64_t)1 << 30) || B * D >= ((int64_t)1 << 31) || B * D * L >= ((int64_t)1 << 40) ||
      B * G * N * L >= ((int64_t)1 << 40))
    return refuse("tensor too large.");
  return DUDY_OK;
}

template <typename F>
int by_type_and_lanes(int dtype, int64_t N, F &&f) {
  auto lanes = [&](auto t) {
    switch (lanes_per_channel(N)) {
      case 1: return f(t, std::integral_constant<int, 1>());
      case 2: return f(t, std::integral_constant<int, 2>());
      case 4: return f(t, std::integral_constant<int, 4>());
      case 8: return f(t, std::integral_constant<int, 8>());
      default: return f(t, std::integral_constant<int, 16>());
    }
  };
  if (dtype == DUDY_DTYPE_F32) return lanes(float());
  if (dtype == DUDY_DTYPE_F16) return lanes(__half());
  return lanes(__nv_bfloat16());
}

}  // namespace scan
}  // namespace dudy
