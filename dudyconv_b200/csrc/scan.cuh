// scan.cuh -- what the selective scan's forward, backward and step kernels share.
//
//   dt = softplus(delta + delta_bias)             (or delta + delta_bias)
//   h[t] = exp(dt A) h[t-1] + dt u B[t]           per channel d and state n
//   y[t] = sum_n C[t] h[t] + skip u
// A thread owns four neighbouring states n of two or four channels; LPC lanes hold a channel's
// states (N <= 4 LPC, padded with A = B = C = 0, which add nothing). The warps of a block take
// consecutive pieces of its sequence in turn, each on its own: a warp copies its piece's
// inputs, forms the decays exp(dt A) of all its positions (in registers), runs the recurrence
// from zero, and only then waits for the state that enters the piece. One multiply-add a state
// (the piece's decay product times what enters, plus its own end state) gives what it hands on
// to the next warp; it runs the recurrence again from the true state, for its outputs or
// gradients, while that one goes on. So each exponential is computed once, the chain from warp
// to warp is a few dozen instructions a piece, and no barrier joins the whole block:
// consecutive warps meet in pairs (bar.arrive / bar.sync on a barrier per neighbours, never two
// arrivals ahead, since the chain goes round the block before a warp arrives there again).
// Waiting before the recurrence instead, and running it once, made the chain the bound: 222
// and 861 us at the sizes below.
// The special function unit (16 a clock and SM, 59 us for the 268 M exponentials of B=16,
// D=256, L=4096, N=16) is the forward's floor, not HBM (17 us).
//
// Where there are too few rows of channels to fill the GPU, the sequence is cut into `splits`
// chunks, a block to each: a first kernel finds each chunk's end state from zero and its decay
// product, and the main kernel's block folds those of the chunks before its own into the state
// that it starts from. That doubles the exponentials and divides the steps in a row by `splits`.
//
// All arithmetic is fp32, two at a time where pairs lie side by side (__ffma2_rn).
#pragma once

#include <type_traits>

#include "rowvec.cuh"
#include "sm100.cuh"

namespace dudy {
namespace scan {

constexpr int kNS = 4;        // states of a thread, neighbours in n
constexpr int kWarps = 8;     // warps of a block: consecutive pieces of a superchunk
constexpr int kThreads = 32 * kWarps;
constexpr int kCkpt = 4;      // positions between saved states: a piece of the backward
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

// exp(dt A) as the base-2 exponential of the special function unit on dt A log2(e). Its rounding
// error is 3e-8 to 6e-8 of the result (rms, that of an fp32 rounding), but it is low by 0.6e-8 to
// 2e-8 on average for exponents of -0.001 to -0.1 (measured against float64 on 2^20 arguments a
// range), and a bias, unlike the rounding around it, adds up over the hundreds of positions that a
// slow state remembers. kCentre in the exponent, a relative 1.7e-8 (a fourth of a half rounding), takes
// it out; without it the error of dA was three times as large. Outside that range: with the constant the
// mean is 1.1e-8 too high for exponents above -0.001; below -0.5 the instruction is low by 5e-8 to
// 7e-8, of which the constant takes 1.7e-8 back, but there a state halves every second position and
// little adds up. At dt = 0 the result is still 1. (The accurate expf cost the fp32 kernels five more
// instructions a state and gave the same errors.)
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kCentre = 2.4e-8f;
__device__ __forceinline__ float decay(float dt, float a_log2e) {
  return ex2(fmaf(dt, a_log2e, kCentre));
}
__device__ __forceinline__ float2 decays(float2 dt, float2 a_log2e) {
  const float2 x = __ffma2_rn(dt, a_log2e, both(kCentre));
  return make_float2(ex2(x.x), ex2(x.y));
}

// What leaves a chunk: its decays' product times what enters, and its end from zero. A chunk of decays
// above 1 may have a product beyond fp32; where nothing enters, nothing of it is passed on. (Written
// out as a selection: as a branch, each chunk's loads waited for the chunk before; 40 us instead of
// 36 at B=1, D=256, L=4096, N=16. A second, guarded pass where the first ends in NaN cost every
// kernel registers: 1 to 7%.)
__device__ __forceinline__ float pass_chunk(float prod, float in, float end) {
  float v = fmaf(prod, in, end);
  asm("{.reg .pred p; setp.eq.f32 p, %1, 0f00000000; selp.f32 %0, %2, %0, p;}" : "+f"(v) : "f"(in), "f"(end));
  return v;
}

// softplus(x) = max(x, 0) + log(1 + e), e = exp(-|x|), and its derivative. 16-bit tensors take
// log(1 + e) = 2 artanh(e / (2 + e)) by its power series: the argument is at most 1/3, so seven
// terms leave 2^-26, and small steps keep their relative precision (the logarithm of a rounded
// 1 + e would not). fp32 tensors: the accurate functions.
template <typename T>
__device__ __forceinline__ float softplus(float x, float &slope) {
  // exp(-|x|) with the exponent's rounding put back (at |x| = 5 it is 3e-7); beyond 100 it is
  // zero, also for infinities and the types' lowest values, and NaN stays NaN
  const float ax = fabsf(x) > 100.f ? 100.f : fabsf(x), t = -kLog2e * ax;
  float e = ex2(t);
  e = fmaf(e, kLn2 * fmaf(-kLog2e, ax, -t), e);
  const float s = e * rcp(2.f + e), q = s * s;
  float p = fmaf(q, 1.f / 13.f, 1.f / 11.f);
  p = fmaf(p, q, 1.f / 9.f);
  p = fmaf(p, q, 1.f / 7.f);
  p = fmaf(p, q, 1.f / 5.f);
  p = fmaf(p, q, 1.f / 3.f);
  p = fmaf(p, q, 1.f);
  slope = (x > 0.f ? 1.f : e) * rcp(1.f + e);
  return fmaf(s + s, p, fmaxf(x, 0.f));
}
template <>
__device__ __forceinline__ float softplus<float>(float x, float &slope) {
  const float e = expf(-fabsf(x));
  slope = (x > 0.f ? 1.f : e) / (1.f + e);
  return fmaxf(x, 0.f) + log1pf(e);
}

__device__ __forceinline__ float2 lo(const float4 &v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ float2 hi(const float4 &v) { return make_float2(v.z, v.w); }
__device__ __forceinline__ float4 quad(const float2 &a, const float2 &b) {
  return make_float4(a.x, a.y, b.x, b.y);
}

// Input rows come in by stretches of one piece for each warp, copied by all the block's threads
// into one of three buffers (rows of whole 16-byte pieces: a warp's own piece of a row is 8 to
// 16 bytes, and copying it alone cost the load pipe eight times as many accesses). A warp that
// begins a piece of stretch s issues its part of stretch s + 2, waits for its part of s + 1
// (issued a stretch ago), takes what it needs of s into its own shared memory, and arrives for
// s + 1: when all have arrived, s + 1 has landed and buffer (s + 3) % 3 is free.
constexpr int kStages = 3;
constexpr int kHeld = 2;        // 16-byte copies of a stretch whose places a thread keeps at hand
constexpr int kSiteStage = 970;  // wait site of a stretch that never came

// One thread's 16 bytes of a stretch: the same row and place in it for every stretch.
template <typename T>
struct RowCopy {
  const T *src;  // null: nothing to copy (a padding row, zeroed once)
  int dst, c;
};
template <typename T>
__device__ __forceinline__ void row_copy(T *raw, const RowCopy<T> &x, int64_t t0, int64_t end,
                                         bool vec) {
  constexpr int V = 16 / sizeof(T);
  if (!x.src) return;
  T *to = raw + x.dst;
  if (vec && t0 + x.c + V <= end) {
    cp_async16(to, x.src + t0);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      to[k] = t0 + x.c + k < end ? x.src[t0 + k] : Elem<T>::from_f(0.f);
  }
}

struct Ready {  // one barrier a buffer, an arrival a warp
  uint64_t bar[kStages];
  int abort;
};
__device__ __forceinline__ void ready_init(Ready &r) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) sm100::mbar_init(&r.bar[i], kWarps);
    r.abort = 0;
    sm100::fence_barrier_init();
  }
  __syncthreads();
}
__device__ __forceinline__ void ready_arrive(Ready &r, int stretch) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) sm100::mbar_arrive(&r.bar[stretch % kStages]);
}
// A stretch that does not come within the library's limit is recorded; the block goes on, so
// that every warp still meets its neighbours.
__device__ __forceinline__ void ready_wait(Ready &r, int stretch, int *err) {
  sm100::mbar_wait(&r.bar[stretch % kStages], (stretch / kStages) & 1, err, &r.abort, kSiteStage,
                   stretch);
}

// Two warps meet: one arrives and goes on, the other waits for it.
__device__ __forceinline__ void pair_wait(int id) {
  asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory");
}
__device__ __forceinline__ void pair_arrive(int id) {
  asm volatile("bar.arrive %0, 64;" ::"r"(id) : "memory");
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

// saved states go out and come back by 16 bytes where a channel's number of them allows it
inline int require_checkpoints(const void *p, int64_t N) {
  if (N % 4 != 0 || aligned_to_16(p)) return DUDY_OK;
  return refuse("checkpoints must be 16-byte aligned.");
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
