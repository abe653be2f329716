// block_norm.cu -- what stands between two blocks of a [B, D, L] model, in one pass each way:
// the gate and norm of a block's output, the scaled residual, and the next block's norm.
//
//   g  = x * z * sigmoid(z)                      (or g = x without a gate)
//   p  = norm(g) * post_weight + post_bias
//   r' = r + scale * p                           (the residual stream)
//   y  = norm(r') * pre_weight + pre_bias        (the next block's input)
// norm(v) = (v - m) / sqrt(mean((v - m)^2) + eps) over the D channels of a token, m = mean(v)
// (layer) or 0 (rms). y is formed from r' before its rounding. Backward, with hat = norm(v)
// and inv its factor, d = the gradient of hat:
//   back(d) = inv * (d - hat mean(d hat) - [layer] mean(d))
//   dr = dr' + back2(dy pre_weight);  dp = dr scale;  dg = back1(dp post_weight)
//   dx = dg z s, dz = dg x (s + z s (1 - s));  parameter gradients are sums over all tokens.
// The backward recomputes g and r' in fp32 from x, z, r and the saved statistics.
//
// A token's channels lie L elements apart, so a block takes a tile of neighbouring tokens
// (lanes along t, coalesced) and all channels, and sums over its rows of threads.
#include "rowvec.cuh"

namespace dudy {
namespace {

constexpr int kThreads = 256;

struct NormShape {
  int64_t B, D, L;
  float eps;
};

struct NormFwd {
  const void *x, *gate, *residual, *w1, *b1, *scale, *w2, *b2;
  void *y, *rout;
  float *stats;  // [4, B*L]: mean1, inv1, mean2, inv2; or null
};

struct NormBwd {
  const void *gy, *grout, *x, *gate, *residual, *w1, *b1, *scale, *w2;
  const float *stats;
  void *gx, *ggate, *gresidual;
  float *part;  // [5][tiles][D]: post_weight, pre_weight, scale, post_bias, pre_bias
};

// Sum over the block's threads that share threadIdx.x % TX, known to all of them.
template <int TX>
__device__ __forceinline__ float tile_sum(float v, float *red) {
  const int tid = threadIdx.x, tx = tid % TX;
#pragma unroll
  for (int o = 16; o >= TX; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  constexpr int kW = kThreads / 32;
  __syncthreads();
  if ((tid & 31) < TX) red[(tid >> 5) * TX + tx] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kW; ++i) s += red[i * TX + tx];
  return s;
}

template <typename T>
__device__ __forceinline__ float opt(const T *p, int64_t d, float other) {
  return p ? ldf(p + d) : other;
}

// Any D and L: the tile is read once per sum and once for the result (from L1 / L2 after the
// first time); one token per thread and TX neighbouring tokens per tile.
template <typename T, typename R, int TX, bool LAYER>
__global__ void __launch_bounds__(kThreads)
block_norm_fwd_any_kernel(NormFwd a, NormShape s) {
  constexpr int TY = kThreads / TX;
  __shared__ float red[kThreads / 32 * TX];
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  const int64_t tiles = (s.L + TX - 1) / TX;
  const int64_t b = blockIdx.x / tiles, t = blockIdx.x % tiles * TX + tx;
  const bool in = t < s.L;
  const T *x = (const T *)a.x, *z = (const T *)a.gate;
  const R *r = (const R *)a.residual;
  const T *w1 = (const T *)a.w1, *b1 = (const T *)a.b1, *sc = (const T *)a.scale;
  const T *w2 = (const T *)a.w2, *b2 = (const T *)a.b2;
  const int64_t base = b * s.D * s.L + t;
  const float rd = 1.f / (float)s.D;

  auto gated = [&](int64_t d) {
    const float xv = ldf(x + base + d * s.L);
    if (!z) return xv;
    const float zv = ldf(z + base + d * s.L);
    return xv * zv * sigmoid_for<T>(zv);
  };
  float m1 = 0.f, m2 = 0.f;
  if (LAYER) {
    float v = 0.f;
    if (in)
      for (int64_t d = ty; d < s.D; d += TY) v += gated(d);
    m1 = tile_sum<TX>(v, red) * rd;
  }
  float v = 0.f;
  if (in)
    for (int64_t d = ty; d < s.D; d += TY) {
      const float c = gated(d) - m1;
      v = fmaf(c, c, v);
    }
  const float inv1 = rsqrtf(fmaf(tile_sum<TX>(v, red), rd, s.eps));
  auto stream = [&](int64_t d) {
    const float p = fmaf((gated(d) - m1) * inv1, ldf(w1 + d), opt(b1, d, 0.f));
    return fmaf(opt(sc, d, 1.f), p, ldf(r + base + d * s.L));
  };
  if (LAYER) {
    v = 0.f;
    if (in)
      for (int64_t d = ty; d < s.D; d += TY) v += stream(d);
    m2 = tile_sum<TX>(v, red) * rd;
  }
  v = 0.f;
  if (in)
    for (int64_t d = ty; d < s.D; d += TY) {
      const float c = stream(d) - m2;
      v = fmaf(c, c, v);
    }
  const float inv2 = rsqrtf(fmaf(tile_sum<TX>(v, red), rd, s.eps));
  if (!in) return;
  for (int64_t d = ty; d < s.D; d += TY) {
    const float rv = stream(d);
    stf((R *)a.rout + base + d * s.L, rv);
    stf((T *)a.y + base + d * s.L, fmaf((rv - m2) * inv2, ldf(w2 + d), opt(b2, d, 0.f)));
  }
  if (a.stats && ty == 0) {
    const int64_t n = s.B * s.L, i = b * s.L + t;
    a.stats[i] = m1;
    a.stats[n + i] = inv1;
    a.stats[2 * n + i] = m2;
    a.stats[3 * n + i] = inv2;
  }
}

template <typename T, typename R, int TX, bool LAYER>
__global__ void __launch_bounds__(kThreads)
block_norm_bwd_any_kernel(NormBwd a, NormShape s) {
  constexpr int TY = kThreads / TX;
  __shared__ float red[kThreads / 32 * TX];
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  const int64_t tiles = (s.L + TX - 1) / TX;
  const int64_t b = blockIdx.x / tiles, t = blockIdx.x % tiles * TX + tx;
  const bool in = t < s.L;
  const T *x = (const T *)a.x, *z = (const T *)a.gate, *gy = (const T *)a.gy;
  const R *r = (const R *)a.residual, *gr = (const R *)a.grout;
  const T *w1 = (const T *)a.w1, *b1 = (const T *)a.b1, *sc = (const T *)a.scale;
  const T *w2 = (const T *)a.w2;
  const int64_t base = b * s.D * s.L + t;
  const float rd = 1.f / (float)s.D;
  float m1 = 0.f, inv1 = 0.f, m2 = 0.f, inv2 = 0.f;
  if (in) {
    const int64_t n = s.B * s.L, i = b * s.L + t;
    if (LAYER) m1 = a.stats[i], m2 = a.stats[2 * n + i];
    inv1 = a.stats[n + i];
    inv2 = a.stats[3 * n + i];
  }
  struct Tok {
    float hat1, p, hat2, xv, zv, sg;
  };
  auto token = [&](int64_t d) {
    Tok k;
    const int64_t o = base + d * s.L;
    k.xv = ldf(x + o);
    float g = k.xv;
    k.zv = k.sg = 0.f;
    if (z) {
      k.zv = ldf(z + o);
      k.sg = sigmoid_for<T>(k.zv);
      g *= k.zv * k.sg;
    }
    k.hat1 = (g - m1) * inv1;
    k.p = fmaf(k.hat1, ldf(w1 + d), opt(b1, d, 0.f));
    k.hat2 = (fmaf(opt(sc, d, 1.f), k.p, ldf(r + o)) - m2) * inv2;
    return k;
  };
  // mean(d2 hat2), mean(d2) with d2 = dy pre_weight
  float v = 0.f, u = 0.f;
  if (in)
    for (int64_t d = ty; d < s.D; d += TY) {
      const float d2 = ldf(gy + base + d * s.L) * ldf(w2 + d);
      v = fmaf(d2, token(d).hat2, v);
      u += d2;
    }
  const float c2 = tile_sum<TX>(v, red) * rd;
  const float e2 = LAYER ? tile_sum<TX>(u, red) * rd : 0.f;
  auto dres = [&](int64_t d, const Tok &k) {
    const float d2 = ldf(gy + base + d * s.L) * ldf(w2 + d);
    const float up = gr ? ldf(gr + base + d * s.L) : 0.f;
    return fmaf(inv2, fmaf(-k.hat2, c2, d2) - e2, up);
  };
  v = u = 0.f;
  if (in)
    for (int64_t d = ty; d < s.D; d += TY) {
      const Tok k = token(d);
      const float d1 = dres(d, k) * opt(sc, d, 1.f) * ldf(w1 + d);
      v = fmaf(d1, k.hat1, v);
      u += d1;
    }
  const float c1 = tile_sum<TX>(v, red) * rd;
  const float e1 = LAYER ? tile_sum<TX>(u, red) * rd : 0.f;
  // all threads of a warp go round together: the parameter sums run across its lanes
  const int64_t ntiles = gridDim.x, tile = blockIdx.x;
  for (int64_t d0 = 0; d0 < s.D; d0 += TY) {
    const int64_t d = d0 + ty;
    const bool here = in && d < s.D;
    float q[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
    if (here) {
      const Tok k = token(d);
      const float dr = dres(d, k), dp = dr * opt(sc, d, 1.f);
      const float dg = inv1 * (fmaf(-k.hat1, c1, dp * ldf(w1 + d)) - e1);
      const int64_t o = base + d * s.L;
      const float dy = ldf(gy + o);
      stf((R *)a.gresidual + o, dr);
      if (z) {
        stf((T *)a.gx + o, dg * k.zv * k.sg);
        stf((T *)a.ggate + o, dg * k.xv * k.sg * fmaf(k.zv, 1.f - k.sg, 1.f));
      } else {
        stf((T *)a.gx + o, dg);
      }
      q[0] = dp * k.hat1;
      q[1] = dy * k.hat2;
      q[2] = dr * k.p;
      q[3] = dp;
      q[4] = dy;
    }
#pragma unroll
    for (int i = 0; i < 5; ++i) {
#pragma unroll
      for (int o = TX / 2; o > 0; o >>= 1) q[i] += __shfl_xor_sync(0xffffffffu, q[i], o);
      if (tx == 0 && d < s.D) a.part[(i * ntiles + tile) * s.D + d] = q[i];
    }
  }
}

// One column of threads per 32 channels: eight rows of threads take every eighth tile, then
// the rows' sums are added in order.
template <typename T>
__global__ void __launch_bounds__(256)
block_norm_param_kernel(const float *__restrict__ part, T *g0, T *g1, T *g2, T *g3, T *g4,
                        int64_t tiles, int64_t D) {
  __shared__ float red[8][32];
  T *const outs[5] = {g0, g1, g2, g3, g4};
  T *out = outs[blockIdx.y];
  if (!out) return;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t d = blockIdx.x * 32ll + tx;
  const float *p = part + blockIdx.y * tiles * D;
  float v = 0.f;
  if (d < D)
    for (int64_t i = ty; i < tiles; i += 8) v += p[i * D + d];
  red[ty][tx] = v;
  __syncthreads();
  if (ty || d >= D) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) v += red[i][tx];
  stf(out + d, v);
}

int validate(int64_t B, int64_t D, int64_t L, int dtype, int rdtype) {
  if (B <= 0 || D <= 0 || L <= 0) return refuse("B, D and L must be positive.");
  if (!dtype_known(dtype)) return refuse("Unsupported dtype.");
  if (rdtype != dtype && rdtype != DUDY_DTYPE_F32)
    return refuse("residual dtype must equal x dtype or be float32.");
  if (B >= ((int64_t)1 << 31) || D >= ((int64_t)1 << 31) || L >= ((int64_t)1 << 31) ||
      B * L >= ((int64_t)1 << 31) || B * L * D >= ((int64_t)1 << 40))
    return refuse("tensor too large.");
  return DUDY_OK;
}

int tile_tokens(int64_t L) { return L >= 32 ? 32 : (L >= 8 ? 8 : 1); }
int64_t tile_count(int64_t B, int64_t L) { return B * cdiv(L, tile_tokens(L)); }

template <typename T, typename R, bool LAYER>
int fwd_launch(const NormFwd &a, const NormShape &s, cudaStream_t st) {
  const unsigned grid = (unsigned)tile_count(s.B, s.L);
  switch (tile_tokens(s.L)) {
    case 32: block_norm_fwd_any_kernel<T, R, 32, LAYER><<<grid, kThreads, 0, st>>>(a, s); break;
    case 8: block_norm_fwd_any_kernel<T, R, 8, LAYER><<<grid, kThreads, 0, st>>>(a, s); break;
    default: block_norm_fwd_any_kernel<T, R, 1, LAYER><<<grid, kThreads, 0, st>>>(a, s);
  }
  return check_launch("block_norm_fwd_any_kernel");
}

struct ParamGrads {
  void *w1, *w2, *scale, *b1, *b2;
};

template <typename T, typename R, bool LAYER>
int bwd_launch(const NormBwd &a, const ParamGrads &g, const NormShape &s, cudaStream_t st) {
  const int64_t tiles = tile_count(s.B, s.L);
  const unsigned grid = (unsigned)tiles;
  switch (tile_tokens(s.L)) {
    case 32: block_norm_bwd_any_kernel<T, R, 32, LAYER><<<grid, kThreads, 0, st>>>(a, s); break;
    case 8: block_norm_bwd_any_kernel<T, R, 8, LAYER><<<grid, kThreads, 0, st>>>(a, s); break;
    default: block_norm_bwd_any_kernel<T, R, 1, LAYER><<<grid, kThreads, 0, st>>>(a, s);
  }
  if (int rc = check_launch("block_norm_bwd_any_kernel")) return rc;
  const dim3 pg((unsigned)cdiv(s.D, 32), 5);
  block_norm_param_kernel<T><<<pg, 256, 0, st>>>(a.part, (T *)g.w1, (T *)g.w2, (T *)g.scale,
                                                  (T *)g.b1, (T *)g.b2, tiles, s.D);
  return check_launch("block_norm_param_kernel");
}

// calls f with the element types of (dtype, residual dtype)
template <typename F>
int by_types(int dtype, int rdtype, F &&f) {
  if (dtype == DUDY_DTYPE_F32) return f(float(), float());
  if (dtype == DUDY_DTYPE_F16)
    return rdtype == DUDY_DTYPE_F32 ? f(__half(), float()) : f(__half(), __half());
  return rdtype == DUDY_DTYPE_F32 ? f(__nv_bfloat16(), float())
                                  : f(__nv_bfloat16(), __nv_bfloat16());
}

}  // namespace
}  // namespace dudy

extern "C" {

int dudy_block_norm_forward(const void *x, const void *gate, const void *residual,
                            const void *post_weight, const void *post_bias, const void *scale,
                            const void *pre_weight, const void *pre_bias, void *y,
                            void *residual_out, float *stats, int64_t B, int64_t D, int64_t L,
                            int layer, float eps, int dtype, int residual_dtype, void *stream) {
  using namespace dudy;
  clear_error();
  if (int rc = validate(B, D, L, dtype, residual_dtype)) return rc;
  if (!x || !residual || !post_weight || !pre_weight || !y || !residual_out)
    return refuse("null tensor pointer");
  if (int rc = require_sm100()) return rc;
  const NormFwd a{x, gate, residual, post_weight, post_bias, scale, pre_weight, pre_bias, y,
                  residual_out, stats};
  const NormShape s{B, D, L, eps};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return by_types(dtype, residual_dtype, [&](auto t, auto r) {
    return layer ? fwd_launch<decltype(t), decltype(r), true>(a, s, st)
                 : fwd_launch<decltype(t), decltype(r), false>(a, s, st);
  });
}

size_t dudy_block_norm_backward_workspace_size(int64_t B, int64_t D, int64_t L, int dtype,
                                               int residual_dtype) {
  if (dudy::validate(B, D, L, dtype, residual_dtype)) return 0;
  const size_t n = 5 * (size_t)dudy::tile_count(B, L) * (size_t)D * sizeof(float);
  return (n + 255) & ~size_t(255);
}

int dudy_block_norm_backward(const void *grad_y, const void *grad_residual_out, const void *x,
                             const void *gate, const void *residual, const void *post_weight,
                             const void *post_bias, const void *scale, const void *pre_weight,
                             const float *stats, void *grad_x, void *grad_gate,
                             void *grad_residual, void *grad_post_weight, void *grad_post_bias,
                             void *grad_scale, void *grad_pre_weight, void *grad_pre_bias,
                             void *workspace, size_t workspace_bytes, int64_t B, int64_t D,
                             int64_t L, int layer, int dtype, int residual_dtype, void *stream) {
  using namespace dudy;
  clear_error();
  if (int rc = validate(B, D, L, dtype, residual_dtype)) return rc;
  if (!grad_y || !x || !residual || !post_weight || !pre_weight || !stats || !grad_x ||
      !grad_residual || (gate && !grad_gate))
    return refuse("null tensor pointer");
  if (int rc = require_workspace(workspace, workspace_bytes,
                                 dudy_block_norm_backward_workspace_size(B, D, L, dtype,
                                                                         residual_dtype)))
    return rc;
  if (int rc = require_sm100()) return rc;
  const NormBwd a{grad_y, grad_residual_out, x, gate, residual, post_weight, post_bias, scale,
                  pre_weight, stats, grad_x, grad_gate, grad_residual, (float *)workspace};
  const ParamGrads g{grad_post_weight, grad_pre_weight, grad_scale, grad_post_bias, grad_pre_bias};
  const NormShape s{B, D, L, 0.f};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return by_types(dtype, residual_dtype, [&](auto t, auto r) {
    return layer ? bwd_launch<decltype(t), decltype(r), true>(a, g, s, st)
                 : bwd_launch<decltype(t), decltype(r), false>(a, g, s, st);
  });
}

}  // extern "C"
