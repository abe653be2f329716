// short_conv.cu -- the short causal depthwise conv in front of a state space scan: whole
// sequences forward and backward, and one token per sequence.
//
//   v[b,d,t]   = bias[d] + sum_{j<S} w[d,j] xe[b,d,t-(S-1)+j]        (tap S-1 = current token)
//   out[b,d,t] = v * sigmoid(v)   (or v)
// xe is x with the S-1 inputs before position 0 in front of it (the carried state, or zeros);
// the state after a sequence is the last S-1 values of xe[.., :length]. Backward:
//   dv[t] = dout[t] (s + v s (1 - s)), s = sigmoid(v);  dxe[t] = sum_j w_j dv[t + S-1-j]
//   dw_j  = sum_{b,t} dv[t] xe[t-(S-1)+j];  dbias = sum_{b,t} dv[t]
// Positions at and behind a sequence's length are not read, give zeros and carry no gradient.
//
// The forward reads and writes each row once, the backward reads two rows and writes one: 67 and
// 101 MB at B=16, D=256, L=4096 in fp16, 10.3 and 15.4 us of HBM at 6540 GB/s. With rows from HBM they
// take 16.8 us (4.0 TB/s, 61%; the special function unit is 59% busy, the issue slots 61%) and 45 us
// with the parameter sums. The backward waits for latency: all of a segment's loads come first,
// then all its arithmetic, and 80 registers leave three blocks an SM (33% of the warps), so the issue
// slots are 55% busy (40 instructions an element with S = 4) and HBM 34% (2.2 TB/s). Multiply-adds two
// positions at a time (__ffma2_rn) took 91 registers and 13% more time, or spilled and won nothing;
// segments of 512 positions took 9% more. A warp takes up to 1024 positions of a row, 256 at a time,
// eight to a lane (16-byte accesses); the S-1 <= 7 inputs before a lane's own come from the lane before
// it by shuffles, so no row is read twice, and all of a segment's loads are in flight at once.
// The backward walks its positions from the right, because dx needs the S-1 values of dv behind
// it: those come from the next lane, and at the right end of a block from the block done just
// before. Parameter gradients are summed in registers over the segment, once across the warp, and
// by a second kernel over batch and segments in a fixed order.
#include "rowvec.cuh"

namespace dudy {
namespace {

constexpr int kWarps = 8;          // warps of a block
constexpr int kBlockT = 256;       // positions a warp holds at a time
constexpr int kSegBlocks = 4;      // blocks of a backward segment
constexpr int64_t kSegT = kBlockT * kSegBlocks;

struct ConvShape {
  int64_t rows, D, L;
  unsigned segs;
  int silu, vec;
};

__device__ __forceinline__ int clamp_len(const int32_t *lengths, int64_t b, int64_t L) {
  if (!lengths) return (int)L;
  const int64_t n = lengths[b];
  return (int)(n < 0 ? 0 : (n > L ? L : n));
}

// xe[t] for t < 0: the state's entry, or zero
template <typename T, int S>
__device__ __forceinline__ float before(const T *state_row, int t) {
  return state_row && t >= -(S - 1) ? ldf(state_row + (S - 1) + t) : 0.f;
}

// The S-1 inputs before position `t0`, in lane 31 (where the lane before lane 0 would be)
template <typename T, int S>
__device__ __forceinline__ void inputs_before(const T *row, const T *state_row, int t0, int len,
                                              int lane, float (&v)[S - 1]) {
#pragma unroll
  for (int i = 0; i < S - 1; ++i) {
    const int p = t0 - (S - 1) + i;
    v[i] = 0.f;
    if (lane == 31) v[i] = p < 0 ? before<T, S>(state_row, p) : (p < len ? ldf(row + p) : 0.f);
  }
}

// The lane's window xw[0 .. S-2] = xe[t-(S-1) .. t-1], xw[S-1 ..] = xe[t .. t+7] from its own eight
// and, by a shuffle, the lane before; lane 0's come from lane 31's `left`.
template <int S>
__device__ __forceinline__ void window(const float (&x)[8], const float (&left)[S - 1], int lane,
                                       float (&xw)[8 + S - 1]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) xw[S - 1 + i] = x[i];
#pragma unroll
  for (int i = 0; i < S - 1; ++i)
    xw[i] = __shfl_sync(0xffffffffu, lane == 31 ? left[i] : x[8 - (S - 1) + i], lane + 31);
}

// the row and segment of a warp; false: none
__device__ __forceinline__ bool place(const ConvShape &s, int64_t &row, int &lo, int &hi) {
  row = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  lo = (int)(blockIdx.y * (unsigned)kSegT);
  hi = lo + kSegT < s.L ? lo + (int)kSegT : (int)s.L;
  return row < s.rows;
}

template <typename T, int S>
__global__ void __launch_bounds__(kWarps * 32)
short_conv_fwd_kernel(const T *__restrict__ x, const T *__restrict__ w, const T *__restrict__ bias,
                      const T *__restrict__ state, const int32_t *__restrict__ lengths,
                      T *__restrict__ out, T *__restrict__ final_state, ConvShape s) {
  const int lane = threadIdx.x & 31;
  int64_t row;
  int lo, hi;
  if (!place(s, row, lo, hi)) return;
  const unsigned d = (unsigned)row % (unsigned)s.D;
  const int len = clamp_len(lengths, (unsigned)row / (unsigned)s.D, s.L);
  const T *xr = x + row * s.L;
  const T *sr = state ? state + row * (S - 1) : nullptr;
  T *outr = out + row * s.L;
  RowEight<T> xs[kSegBlocks];
#pragma unroll
  for (int k = 0; k < kSegBlocks; ++k)
    if (lo + k * kBlockT < hi) xs[k].load(xr, lo + k * kBlockT + lane * 8, len, s.vec);
  float wt[S];
#pragma unroll
  for (int j = 0; j < S; ++j) wt[j] = ldf(w + d * S + j);
  const float bv = bias ? ldf(bias + d) : 0.f;
  float left[S - 1];
  inputs_before<T, S>(xr, sr, lo, len, lane, left);
#pragma unroll
  for (int k = 0; k < kSegBlocks; ++k) {
    const int t0 = lo + k * kBlockT, t = t0 + lane * 8;
    if (t0 >= hi) break;
    float xv[8], xw[8 + S - 1], o[8];
    xs[k].get(xv);
    window<S>(xv, left, lane, xw);
#pragma unroll
    for (int i = 0; i < S - 1; ++i) left[i] = xv[8 - (S - 1) + i];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[i] = bv;
#pragma unroll
      for (int j = 0; j < S; ++j) o[i] = fmaf(wt[j], xw[i + j], o[i]);
    }
    if (s.silu) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float2 v = make_float2(o[i], o[i + 1]), p = mul2(v, sigmoid2<T>(v));
        o[i] = p.x;
        o[i + 1] = p.y;
      }
    }
    if (t + 8 > len) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = t + i < len ? o[i] : 0.f;
    }
    row_store8(outr, t, (int)s.L, o, s.vec);
  }
  if (final_state && lo == 0 && lane < S - 1) {
    const int p = len - (S - 1) + lane;
    stf(final_state + row * (S - 1) + lane, p < 0 ? before<T, S>(sr, p) : ldf(xr + p));
  }
}

// dv of two positions from their pre-activations and the output's gradients
template <typename T>
__device__ __forceinline__ float2 dv_of(float2 v, float2 go) {
  const float2 sg = sigmoid2<T>(v), rest = fma2(sg, both(-1.f), both(1.f));
  return mul2(go, mul2(sg, fma2(v, rest, both(1.f))));
}

template <typename T, int S>
__global__ void __launch_bounds__(kWarps * 32)
short_conv_bwd_kernel(const T *__restrict__ go, const T *__restrict__ gfinal,
                      const T *__restrict__ x, const T *__restrict__ w,
                      const T *__restrict__ bias, const T *__restrict__ state,
                      const int32_t *__restrict__ lengths, T *__restrict__ gx,
                      T *__restrict__ gstate, float *__restrict__ part, ConvShape s) {
  const int lane = threadIdx.x & 31;
  int64_t row;
  int lo, hi;
  if (!place(s, row, lo, hi)) return;
  const unsigned d = (unsigned)row % (unsigned)s.D, b = (unsigned)row / (unsigned)s.D;
  const int len = clamp_len(lengths, b, s.L);
  const T *xr = x + row * s.L;
  const T *gr = go + row * s.L;
  T *gxr = gx + row * s.L;
  const T *sr = state ? state + row * (S - 1) : nullptr;
  const T *fr = gfinal ? gfinal + row * (S - 1) : nullptr;
  RowEight<T> xs[kSegBlocks], gs[kSegBlocks];
#pragma unroll
  for (int k = kSegBlocks - 1; k >= 0; --k)
    if (lo + k * kBlockT < hi) {
      xs[k].load(xr, lo + k * kBlockT + lane * 8, len, s.vec);
      gs[k].load(gr, lo + k * kBlockT + lane * 8, len, s.vec);
    }
  float wt[S];
#pragma unroll
  for (int j = 0; j < S; ++j) wt[j] = ldf(w + d * S + j);
  const float bv = bias ? ldf(bias + d) : 0.f;
  float dw[S], db = 0.f;
#pragma unroll
  for (int j = 0; j < S; ++j) dw[j] = 0.f;

  float first[S - 1];
  inputs_before<T, S>(xr, sr, lo, len, lane, first);
  // dv at the S-1 positions behind the segment: lane i takes position hi + i
  float behind[S];
  {
    float mine = 0.f;
    const int p = hi + lane;
    if (lane < S - 1 && p < len) {
      float v = bv;
#pragma unroll
      for (int j = 0; j < S; ++j) {
        const int q = p - (S - 1) + j;
        v = fmaf(wt[j], q < 0 ? before<T, S>(sr, q) : ldf(xr + q), v);
      }
      mine = s.silu ? dv_of<T>(both(v), both(ldf(gr + p))).x : ldf(gr + p);
    }
#pragma unroll
    for (int i = 0; i < S - 1; ++i) behind[i] = __shfl_sync(0xffffffffu, mine, i);
  }
#pragma unroll
  for (int b4 = kSegBlocks - 1; b4 >= 0; --b4) {
    const int t0 = lo + b4 * kBlockT, t = t0 + lane * 8;
    if (t0 >= hi) continue;
    float xv[8], xw[8 + S - 1], left[S - 1], dv[8 + S - 1];
    xs[b4].get(xv);
    if (b4 > 0) {
      float next[8];
      xs[b4 > 0 ? b4 - 1 : 0].get(next);
#pragma unroll
      for (int i = 0; i < S - 1; ++i) left[i] = next[8 - (S - 1) + i];
    } else {
#pragma unroll
      for (int i = 0; i < S - 1; ++i) left[i] = first[i];
    }
    window<S>(xv, left, lane, xw);
    {
      float g[8];
      gs[b4].get(g);
      if (s.silu) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          float2 v = both(bv);
#pragma unroll
          for (int j = 0; j < S; ++j) {
            v.x = fmaf(wt[j], xw[i + j], v.x);
            v.y = fmaf(wt[j], xw[i + j + 1], v.y);
          }
          const float2 p = dv_of<T>(v, make_float2(g[i], g[i + 1]));
          dv[i] = p.x;
          dv[i + 1] = p.y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) dv[i] = g[i];
      }
    }
    if (t + 8 > len) {
#pragma unroll
      for (int i = 0; i < 8; ++i) dv[i] = t + i < len ? dv[i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      db += dv[i];
#pragma unroll
      for (int j = 0; j < S; ++j) dw[j] = fmaf(dv[i], xw[i + j], dw[j]);
    }
#pragma unroll
    for (int i = 0; i < S - 1; ++i) {
      const float right = __shfl_down_sync(0xffffffffu, dv[i], 1);
      dv[8 + i] = lane == 31 ? behind[i] : right;
      behind[i] = __shfl_sync(0xffffffffu, dv[i], 0);
    }
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[i] = 0.f;
#pragma unroll
      for (int j = 0; j < S; ++j) o[i] = fmaf(wt[j], dv[i + S - 1 - j], o[i]);
    }
    if (fr && t + 8 > len - (S - 1)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = t + i - (len - (S - 1));
        if (k >= 0 && k < S - 1) o[i] += ldf(fr + k);
      }
    }
    if (t + 8 > len) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = t + i < len ? o[i] : 0.f;
    }
    row_store8(gxr, t, (int)s.L, o, s.vec);
    if (gstate && t0 == 0 && lane == 0) {
#pragma unroll
      for (int i = 0; i < S - 1; ++i) {
        float v = 0.f;
#pragma unroll
        for (int j = 0; j <= i; ++j) v = fmaf(wt[j], dv[i - j], v);
        // the state's entries that are still in the final state
        if (fr && i >= len) v += ldf(fr + (i - len));
        stf(gstate + row * (S - 1) + i, v);
      }
    }
  }
  // part[(j * D + d) * per + b * segs + seg], j = S the bias
  const int64_t per = s.rows / s.D * s.segs, at = (int64_t)b * s.segs + blockIdx.y;
#pragma unroll
  for (int j = 0; j <= S; ++j) {
    float v = j < S ? dw[j] : db;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) part[(j * s.D + d) * per + at] = v;
  }
}

// One warp per parameter: the sum of its `per` parts, lane by lane and then across the lanes.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
short_conv_param_kernel(const float *__restrict__ part, T *__restrict__ gw, T *__restrict__ gb,
                        int64_t D, int S, int64_t per) {
  const int lane = threadIdx.x & 31;
  const int64_t i = blockIdx.x * (int64_t)kWarps + (threadIdx.x >> 5);
  if (i >= D * (S + 1)) return;
  float v = 0.f;
  for (int64_t k = lane; k < per; k += 32) v += part[i * per + k];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane) return;
  const int64_t j = i / D, d = i % D;
  if (j < S) stf(gw + d * S + j, v);
  else if (gb) stf(gb + d, v);
}

// One token per sequence: a thread per (b, d); the state moves one place to the left.
template <typename T>
__global__ void __launch_bounds__(128)
short_conv_step_kernel(const T *__restrict__ x, T *__restrict__ state, const T *__restrict__ w,
                       const T *__restrict__ bias, T *__restrict__ out, int64_t rows, int64_t D,
                       int S, int silu) {
  const int64_t row = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (row >= rows) return;
  const int64_t d = row % D;
  T *sr = state + row * (S - 1);
  const T xv = x[row];
  float v = bias ? ldf(bias + d) : 0.f;
#pragma unroll
  for (int j = 0; j < DUDY_SHORT_CONV_MAX_TAPS - 1; ++j) {
    if (j >= S - 1) break;
    const T e = sr[j];
    v = fmaf(ldf(w + d * S + j), Elem<T>::to_f(e), v);
    if (j > 0) sr[j - 1] = e;
  }
  sr[S - 2] = xv;
  v = fmaf(ldf(w + d * S + S - 1), Elem<T>::to_f(xv), v);
  if (silu) v *= sigmoid_for<T>(v);
  stf(out + row, v);
}

int validate(int64_t B, int64_t D, int64_t L, int64_t S, int dtype) {
  if (B <= 0 || D <= 0 || L <= 0) return refuse("B, D and L must be positive.");
  if (S < 2 || S > DUDY_SHORT_CONV_MAX_TAPS)
    return refuse("S must be between 2 and " + std::to_string(DUDY_SHORT_CONV_MAX_TAPS) +
                  ", got " + std::to_string(S) + ".");
  if (!dtype_known(dtype)) return refuse("Unsupported dtype.");
  if (cdiv(L, kSegT) > 65535 || D >= ((int64_t)1 << 31) || B >= ((int64_t)1 << 31) ||
      B * D >= ((int64_t)1 << 31))
    return refuse("tensor too large.");
  return DUDY_OK;
}

size_t workspace_bytes(int64_t B, int64_t D, int64_t L, int64_t S) {
  return (size_t)((S + 1) * D * B * cdiv(L, kSegT)) * sizeof(float);
}

struct FwdArgs {
  const void *x, *w, *bias, *state;
  const int32_t *lengths;
  void *out, *final_state;
};
struct BwdArgs {
  const void *go, *gfinal, *x, *w, *bias, *state;
  const int32_t *lengths;
  void *gx, *gw, *gb, *gstate;
  float *part;
};

template <typename T, int S>
int fwd_launch(const FwdArgs &a, ConvShape s, cudaStream_t st) {
  s.vec = s.L % 8 == 0 && aligned_to_16(a.x) && aligned_to_16(a.out);
  short_conv_fwd_kernel<T, S><<<dim3((unsigned)cdiv(s.rows, kWarps), s.segs), kWarps * 32, 0, st>>>(
      (const T *)a.x, (const T *)a.w, (const T *)a.bias, (const T *)a.state, a.lengths,
      (T *)a.out, (T *)a.final_state, s);
  return check_launch("short_conv_fwd_kernel");
}

template <typename T, int S>
int bwd_launch(const BwdArgs &a, ConvShape s, cudaStream_t st) {
  s.vec = s.L % 8 == 0 && aligned_to_16(a.x) && aligned_to_16(a.go) && aligned_to_16(a.gx);
  short_conv_bwd_kernel<T, S><<<dim3((unsigned)cdiv(s.rows, kWarps), s.segs), kWarps * 32, 0, st>>>(
      (const T *)a.go, (const T *)a.gfinal, (const T *)a.x, (const T *)a.w, (const T *)a.bias,
      (const T *)a.state, a.lengths, (T *)a.gx, (T *)a.gstate, a.part, s);
  if (int rc = check_launch("short_conv_bwd_kernel")) return rc;
  short_conv_param_kernel<T><<<(unsigned)cdiv(s.D * (S + 1), kWarps), kWarps * 32, 0, st>>>(
      a.part, (T *)a.gw, (T *)a.gb, s.D, S, s.rows / s.D * s.segs);
  return check_launch("short_conv_param_kernel");
}

template <typename T>
int fwd_by_taps(const FwdArgs &a, const ConvShape &s, int64_t S, cudaStream_t st) {
  switch (S) {
    case 2: return fwd_launch<T, 2>(a, s, st);
    case 3: return fwd_launch<T, 3>(a, s, st);
    case 4: return fwd_launch<T, 4>(a, s, st);
    case 5: return fwd_launch<T, 5>(a, s, st);
    case 6: return fwd_launch<T, 6>(a, s, st);
    case 7: return fwd_launch<T, 7>(a, s, st);
    default: return fwd_launch<T, 8>(a, s, st);
  }
}

template <typename T>
int bwd_by_taps(const BwdArgs &a, const ConvShape &s, int64_t S, cudaStream_t st) {
  switch (S) {
    case 2: return bwd_launch<T, 2>(a, s, st);
    case 3: return bwd_launch<T, 3>(a, s, st);
    case 4: return bwd_launch<T, 4>(a, s, st);
    case 5: return bwd_launch<T, 5>(a, s, st);
    case 6: return bwd_launch<T, 6>(a, s, st);
    case 7: return bwd_launch<T, 7>(a, s, st);
    default: return bwd_launch<T, 8>(a, s, st);
  }
}

template <typename T>
int step_launch(const void *x, void *state, const void *w, const void *bias, void *out,
                int64_t rows, int64_t D, int S, int silu, cudaStream_t st) {
  short_conv_step_kernel<T><<<(unsigned)cdiv(rows, 128), 128, 0, st>>>(
      (const T *)x, (T *)state, (const T *)w, (const T *)bias, (T *)out, rows, D, S, silu);
  return check_launch("short_conv_step_kernel");
}

}  // namespace
}  // namespace dudy

extern "C" {

int dudy_short_conv_forward(const void *x, const void *weight, const void *bias,
                            const void *state, const int32_t *lengths, void *out,
                            void *final_state, int64_t B, int64_t D, int64_t L, int64_t S,
                            int silu, int dtype, void *stream) {
  using namespace dudy;
  clear_error();
  if (int rc = validate(B, D, L, S, dtype)) return rc;
  if (!x || !weight || !out) return refuse("null tensor pointer");
  if (int rc = require_apart(state, final_state)) return rc;  // its lanes read entries that others write
  if (int rc = require_sm100()) return rc;
  const FwdArgs a{x, weight, bias, state, lengths, out, final_state};
  const ConvShape s{B * D, D, L, (unsigned)cdiv(L, kSegT), silu, 0};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case DUDY_DTYPE_F32: return fwd_by_taps<float>(a, s, S, st);
    case DUDY_DTYPE_F16: return fwd_by_taps<__half>(a, s, S, st);
    default: return fwd_by_taps<__nv_bfloat16>(a, s, S, st);
  }
}

size_t dudy_short_conv_backward_workspace_size(int64_t B, int64_t D, int64_t L, int64_t S,
                                               int dtype) {
  if (dudy::validate(B, D, L, S, dtype)) return 0;
  return (dudy::workspace_bytes(B, D, L, S) + 255) & ~size_t(255);
}

int dudy_short_conv_backward(const void *go, const void *grad_final, const void *x,
                             const void *weight, const void *bias, const void *state,
                             const int32_t *lengths, void *grad_x, void *grad_weight,
                             void *grad_bias, void *grad_state, void *workspace,
                             size_t workspace_bytes, int64_t B, int64_t D, int64_t L, int64_t S,
                             int silu, int dtype, void *stream) {
  using namespace dudy;
  clear_error();
  if (int rc = validate(B, D, L, S, dtype)) return rc;
  if (!go || !x || !weight || !grad_x || !grad_weight) return refuse("null tensor pointer");
  if (int rc = require_workspace(workspace, workspace_bytes,
                                 dudy_short_conv_backward_workspace_size(B, D, L, S, dtype)))
    return rc;
  if (int rc = require_sm100()) return rc;
  const BwdArgs a{go, grad_final, x, weight, bias, state, lengths, grad_x, grad_weight, grad_bias,
                  grad_state, (float *)workspace};
  const ConvShape s{B * D, D, L, (unsigned)cdiv(L, kSegT), silu, 0};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case DUDY_DTYPE_F32: return bwd_by_taps<float>(a, s, S, st);
    case DUDY_DTYPE_F16: return bwd_by_taps<__half>(a, s, S, st);
    default: return bwd_by_taps<__nv_bfloat16>(a, s, S, st);
  }
}

int dudy_short_conv_step(const void *x, void *state, const void *weight, const void *bias,
                         void *out, int64_t B, int64_t D, int64_t S, int silu, int dtype,
                         void *stream) {
  using namespace dudy;
  clear_error();
  if (int rc = validate(B, D, 1, S, dtype)) return rc;
  if (!x || !state || !weight || !out) return refuse("null tensor pointer");
  if (int rc = require_sm100()) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case DUDY_DTYPE_F32:
      return step_launch<float>(x, state, weight, bias, out, B * D, D, (int)S, silu, st);
    case DUDY_DTYPE_F16:
      return step_launch<__half>(x, state, weight, bias, out, B * D, D, (int)S, silu, st);
    default:
      return step_launch<__nv_bfloat16>(x, state, weight, bias, out, B * D, D, (int)S, silu, st);
  }
}

}  // extern "C"
