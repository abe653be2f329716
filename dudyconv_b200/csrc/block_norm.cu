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
#include <type_traits>

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

// ---- D <= 1024: the tile in registers ------------------------------------------------------
// 512 threads hold a tile of 4 TX tokens x all channels, four tokens and up to four channels to
// a thread, so each tensor moves once. TX = 8 (rows of 64 bytes in 16-bit types) up to D = 256,
// then 4 and 2.
constexpr int kTileThreads = 512;
constexpr int kV = 4;  // tokens of a thread

template <typename T>
using Four = RowFour<T>;

template <typename T>
__device__ __forceinline__ void get4(const Four<T> &f, float (&v)[kV]) {
#pragma unroll
  for (int i = 0; i < kV; ++i) v[i] = f.get(i);
}

struct TileRed {
  float part[2][kTileThreads / 32][32];
  float total[2][32];
};

// Sums of the four tokens' values over the block's rows of threads, known to all threads of the
// tokens: across the rows of a warp by shuffles, across the warps by sixteen lanes a token.
// `turn` alternates between two sets of buffers, so two barriers are enough.
template <int TX>
__device__ __forceinline__ void tile_sum4(float (&v)[kV], TileRed &m, int &turn) {
  constexpr int kW = kTileThreads / 32, TOK = TX * kV;
  const int tid = threadIdx.x, tx = tid % TX;
#pragma unroll
  for (int o = 16; o >= TX; o >>= 1)
#pragma unroll
    for (int i = 0; i < kV; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if ((tid & 31) < TX)
    *reinterpret_cast<float4 *>(&m.part[turn][tid >> 5][tx * kV]) =
        make_float4(v[0], v[1], v[2], v[3]);
  __syncthreads();
  if (tid < TOK * kW) {
    float s = m.part[turn][tid % kW][tid / kW];
#pragma unroll
    for (int o = kW / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (tid % kW == 0) m.total[turn][tid / kW] = s;
  }
  __syncthreads();
  const float4 t = *reinterpret_cast<const float4 *>(&m.total[turn][tx * kV]);
  v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  turn ^= 1;
}

template <typename T, typename R, int TX, int ROWS, bool LAYER>
__global__ void __launch_bounds__(kTileThreads, ROWS <= 4 && sizeof(T) == 2 ? 2 : 1)
block_norm_fwd_tile_kernel(NormFwd a, NormShape s, bool vec) {
  constexpr int TY = kTileThreads / TX;
  __shared__ __align__(16) TileRed red;
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  const int64_t tiles = (s.L + TX * kV - 1) / (TX * kV);
  const int64_t b = blockIdx.x / tiles, t = blockIdx.x % tiles * (TX * kV) + tx * kV;
  const int64_t left = s.L - t, base = b * s.D * s.L + t;
  const bool in = left > 0;
  const float rd = 1.f / (float)s.D;
  int turn = 0;
  const T *xp = (const T *)a.x + base, *zp = a.gate ? (const T *)a.gate + base : nullptr;
  const R *rp = (const R *)a.residual + base;
  Four<T> xr[ROWS], zr[ROWS];
  Four<R> rr[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t d = ty + i * TY;
    if (in && d < s.D) {
      row_load4(xr[i], xp + d * s.L, 0, left, vec);
      if (zp) row_load4(zr[i], zp + d * s.L, 0, left, vec);
      row_load4(rr[i], rp + d * s.L, 0, left, vec);
    }
  }
  float g[ROWS][kV], m1[kV], m2[kV], q[kV];
#pragma unroll
  for (int k = 0; k < kV; ++k) m1[k] = m2[k] = 0.f;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const bool ok = in && ty + i * TY < s.D;
    if (ok) {
      get4(xr[i], g[i]);
      if (zp) {
        float z[kV];
        get4(zr[i], z);
#pragma unroll
        for (int k = 0; k < kV; ++k) g[i][k] *= z[k] * sigmoid_for<T>(z[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < kV; ++k) {
      if (!ok) g[i][k] = 0.f;
      m1[k] += g[i][k];
    }
  }
  if (LAYER) {
    tile_sum4<TX>(m1, red, turn);
#pragma unroll
    for (int k = 0; k < kV; ++k) m1[k] *= rd;
  } else {
#pragma unroll
    for (int k = 0; k < kV; ++k) m1[k] = 0.f;
  }
  auto squares = [&](const float (&m)[kV]) {
#pragma unroll
    for (int k = 0; k < kV; ++k) q[k] = 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
      if (!LAYER || ty + i * TY < s.D)
#pragma unroll
        for (int k = 0; k < kV; ++k) q[k] = fmaf(g[i][k] - m[k], g[i][k] - m[k], q[k]);
    tile_sum4<TX>(q, red, turn);
#pragma unroll
    for (int k = 0; k < kV; ++k) q[k] = rsqrtf(fmaf(q[k], rd, s.eps));
  };
  squares(m1);
  float inv1[kV];
#pragma unroll
  for (int k = 0; k < kV; ++k) inv1[k] = q[k];
  // the residual stream takes g's place
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t d = ty + i * TY;
    if (in && d < s.D) {
      const float w = ldf((const T *)a.w1 + d), o = LAYER ? opt((const T *)a.b1, d, 0.f) : 0.f;
      const float c = opt((const T *)a.scale, d, 1.f);
      float r[kV];
      get4(rr[i], r);
#pragma unroll
      for (int k = 0; k < kV; ++k)
        g[i][k] = fmaf(c, fmaf((g[i][k] - m1[k]) * inv1[k], w, o), r[k]);
      row_store4((R *)a.rout + base + d * s.L, 0, left, g[i], vec);
    }
#pragma unroll
    for (int k = 0; k < kV; ++k) m2[k] += g[i][k];
  }
  if (LAYER) {
    tile_sum4<TX>(m2, red, turn);
#pragma unroll
    for (int k = 0; k < kV; ++k) m2[k] *= rd;
  } else {
#pragma unroll
    for (int k = 0; k < kV; ++k) m2[k] = 0.f;
  }
  squares(m2);
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t d = ty + i * TY;
    if (!in || d >= s.D) continue;
    const float w = ldf((const T *)a.w2 + d), o = LAYER ? opt((const T *)a.b2, d, 0.f) : 0.f;
    float y[kV];
#pragma unroll
    for (int k = 0; k < kV; ++k) y[k] = fmaf((g[i][k] - m2[k]) * q[k], w, o);
    row_store4((T *)a.y + base + d * s.L, 0, left, y, vec);
  }
  if (a.stats && ty == 0) {
    const int64_t n = s.B * s.L, at = b * s.L + t;
#pragma unroll
    for (int k = 0; k < kV; ++k)
      if (k < left) {
        a.stats[at + k] = m1[k];
        a.stats[n + at + k] = inv1[k];
        a.stats[2 * n + at + k] = m2[k];
        a.stats[3 * n + at + k] = q[k];
      }
  }
}

template <int BYTES>
__device__ __forceinline__ void cp_async(void *smem, const void *gmem) {
  const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(gmem), "n"(BYTES)
               : "memory");
}

// The tile's five tensors in shared memory, each thread's own four-token pieces side by side
// (no thread reads another's, so its own copies' completion is all it waits for).
template <typename T, typename R, int ROWS>
struct NormTile {
  Four<T> x[ROWS][kTileThreads], z[ROWS][kTileThreads], gy[ROWS][kTileThreads];
  Four<R> r[ROWS][kTileThreads], gr[ROWS][kTileThreads];
  // two tiles where they fit beside TileRed in the 227 KB of a block
  static constexpr int kBytes = ROWS * kTileThreads * (3 * sizeof(Four<T>) + 2 * sizeof(Four<R>));
  static constexpr int kStages = 2 * kBytes <= 220 * 1024 ? 2 : 1;
};

// Persistent blocks: a block's next tile is copied while it works on this one, and the
// parameter sums stay in registers until its last.
template <typename T, typename R, int TX, int ROWS, bool LAYER>
__global__ void __launch_bounds__(kTileThreads, 1)
block_norm_bwd_tile_kernel(NormBwd a, NormShape s, int64_t ntiles, bool vec) {
  using Tile = NormTile<T, R, ROWS>;
  constexpr int TY = kTileThreads / TX;
  extern __shared__ __align__(16) char smem_raw[];
  Tile *stage = reinterpret_cast<Tile *>(smem_raw);
  __shared__ __align__(16) TileRed red;
  const int tid = threadIdx.x, tx = tid % TX, ty = tid / TX;
  const int64_t tiles = (s.L + TX * kV - 1) / (TX * kV), n = s.B * s.L;
  const float rd = 1.f / (float)s.D;
  int turn = 0;

  float w1[ROWS], b1[ROWS], sc[ROWS], w2[ROWS];
  float acc[5][ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t d = ty + i * TY;
    const bool ok = d < s.D;
    w1[i] = ok ? ldf((const T *)a.w1 + d) : 0.f;
    w2[i] = ok ? ldf((const T *)a.w2 + d) : 0.f;
    b1[i] = LAYER && ok ? opt((const T *)a.b1, d, 0.f) : 0.f;
    sc[i] = ok ? opt((const T *)a.scale, d, 1.f) : 0.f;
#pragma unroll
    for (int j = 0; j < 5; ++j) acc[j][i] = 0.f;
  }
  auto fetch = [&](int64_t tile, Tile &m) {
    const int64_t b = tile / tiles, t = tile % tiles * (TX * kV) + tx * kV;
    const int64_t left = s.L - t, base = b * s.D * s.L + t;
    if (left > 0)
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int64_t d = ty + i * TY, o = base + d * s.L;
        if (d >= s.D) continue;
        if (vec) {
          cp_async<sizeof(Four<T>)>(&m.x[i][tid], (const T *)a.x + o);
          if (a.gate) cp_async<sizeof(Four<T>)>(&m.z[i][tid], (const T *)a.gate + o);
          cp_async<sizeof(Four<R>)>(&m.r[i][tid], (const R *)a.residual + o);
          cp_async<sizeof(Four<T>)>(&m.gy[i][tid], (const T *)a.gy + o);
          if (a.grout) cp_async<sizeof(Four<R>)>(&m.gr[i][tid], (const R *)a.grout + o);
        } else {
          row_load4(m.x[i][tid], (const T *)a.x + o, 0, left, false);
          if (a.gate) row_load4(m.z[i][tid], (const T *)a.gate + o, 0, left, false);
          row_load4(m.r[i][tid], (const R *)a.residual + o, 0, left, false);
          row_load4(m.gy[i][tid], (const T *)a.gy + o, 0, left, false);
          if (a.grout) row_load4(m.gr[i][tid], (const R *)a.grout + o, 0, left, false);
        }
      }
    copies_commit();
  };
  int at = 0;
  if (blockIdx.x < ntiles) fetch(blockIdx.x, stage[0]);
  for (int64_t tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
    const int64_t b = tile / tiles, t = tile % tiles * (TX * kV) + tx * kV;
    const int64_t left = s.L - t, base = b * s.D * s.L + t;
    const bool in = left > 0;
    float m1[kV], inv1[kV], m2[kV], inv2[kV];
#pragma unroll
    for (int k = 0; k < kV; ++k) {
      const int64_t i = b * s.L + t + k;
      const bool ok = k < left;
      m1[k] = LAYER && ok ? a.stats[i] : 0.f;
      inv1[k] = ok ? a.stats[n + i] : 0.f;
      m2[k] = LAYER && ok ? a.stats[2 * n + i] : 0.f;
      inv2[k] = ok ? a.stats[3 * n + i] : 0.f;
    }
    if (Tile::kStages == 2 && tile + gridDim.x < ntiles) {
      fetch(tile + gridDim.x, stage[at ^ 1]);
      copies_wait<1>();
    } else {
      copies_wait<0>();
    }
    const Tile &m = stage[at];
    float hat1[ROWS][kV], hat2[ROWS][kV], sg[ROWS][kV], v[kV], u[kV];
#pragma unroll
    for (int k = 0; k < kV; ++k) v[k] = u[k] = 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const bool ok = in && ty + i * TY < s.D;
      float x[kV], z[kV], r[kV], gy[kV];
      get4(m.x[i][tid], x);
      get4(m.r[i][tid], r);
      get4(m.gy[i][tid], gy);
      if (a.gate) get4(m.z[i][tid], z);
#pragma unroll
      for (int k = 0; k < kV; ++k) {
        float g = x[k];
        sg[i][k] = 0.f;
        if (a.gate) {
          sg[i][k] = sigmoid_for<T>(z[k]);
          g *= z[k] * sg[i][k];
        }
        hat1[i][k] = ok ? (g - m1[k]) * inv1[k] : 0.f;
        hat2[i][k] =
            ok ? (fmaf(sc[i], fmaf(hat1[i][k], w1[i], b1[i]), r[k]) - m2[k]) * inv2[k] : 0.f;
        const float dy = ok ? gy[k] : 0.f, d2 = dy * w2[i];
        v[k] = fmaf(d2, hat2[i][k], v[k]);
        u[k] += d2;
        acc[1][i] = fmaf(dy, hat2[i][k], acc[1][i]);
        if (LAYER) acc[4][i] += dy;
      }
    }
    tile_sum4<TX>(v, red, turn);
    if (LAYER) tile_sum4<TX>(u, red, turn);
    float c2[kV], e2[kV];
#pragma unroll
    for (int k = 0; k < kV; ++k) {
      c2[k] = v[k] * rd;
      e2[k] = LAYER ? u[k] * rd : 0.f;
      v[k] = u[k] = 0.f;
    }
    // the gradient of p takes hat2's place
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int64_t d = ty + i * TY;
      const bool ok = in && d < s.D;
      float gy[kV], gr[kV], dr[kV];
      get4(m.gy[i][tid], gy);
      if (a.grout) get4(m.gr[i][tid], gr);
#pragma unroll
      for (int k = 0; k < kV; ++k) {
        const float up = a.grout ? gr[k] : 0.f;
        dr[k] = ok ? fmaf(inv2[k], fmaf(-hat2[i][k], c2[k], gy[k] * w2[i]) - e2[k], up) : 0.f;
        const float dp = dr[k] * sc[i], d1 = dp * w1[i];
        hat2[i][k] = d1;
        v[k] = fmaf(d1, hat1[i][k], v[k]);
        u[k] += d1;
        acc[0][i] = fmaf(dp, hat1[i][k], acc[0][i]);
        acc[2][i] = fmaf(dr[k], fmaf(hat1[i][k], w1[i], b1[i]), acc[2][i]);
        if (LAYER) acc[3][i] += dp;
      }
      if (ok) row_store4((R *)a.gresidual + base + d * s.L, 0, left, dr, vec);
    }
    tile_sum4<TX>(v, red, turn);
    if (LAYER) tile_sum4<TX>(u, red, turn);
#pragma unroll
    for (int k = 0; k < kV; ++k) {
      v[k] *= rd;
      u[k] = LAYER ? u[k] * rd : 0.f;
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int64_t d = ty + i * TY;
      if (!in || d >= s.D) continue;
      float x[kV], z[kV], gx[kV], gz[kV];
      get4(m.x[i][tid], x);
      if (a.gate) get4(m.z[i][tid], z);
#pragma unroll
      for (int k = 0; k < kV; ++k) {
        const float dg = inv1[k] * (fmaf(-hat1[i][k], v[k], hat2[i][k]) - u[k]);
        gx[k] = dg;
        if (a.gate) {
          const float h = dg * sg[i][k];
          gx[k] = h * z[k];
          gz[k] = h * x[k] * fmaf(z[k], 1.f - sg[i][k], 1.f);
        }
      }
      row_store4((T *)a.gx + base + d * s.L, 0, left, gx, vec);
      if (a.gate) row_store4((T *)a.ggate + base + d * s.L, 0, left, gz, vec);
    }
    if (Tile::kStages == 2) at ^= 1;
    else if (tile + gridDim.x < ntiles) fetch(tile + gridDim.x, stage[0]);
  }
#pragma unroll
  for (int j = 0; j < (LAYER ? 5 : 3); ++j)
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      float q = acc[j][i];
#pragma unroll
      for (int o = TX / 2; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
      const int64_t d = ty + i * TY;
      if (tx == 0 && d < s.D) a.part[(j * (int64_t)gridDim.x + blockIdx.x) * s.D + d] = q;
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

// ---- which kernel: tiles in registers where a sequence has tokens enough for one row of it and
// D fits, else the any-size kernel (few tokens: all threads go along D)
int any_tokens(int64_t L) { return L >= 32 ? 32 : (L >= 8 ? 8 : 1); }

int tile_tx(int64_t D, int64_t L) {
  if (D > 1024 || L < 8) return 0;
  return D <= 256 ? 8 : (D <= 512 ? 4 : 2);
}

// tiles of the kernel that runs, and the number of parts of its parameter sums
int64_t tile_count(int64_t B, int64_t D, int64_t L) {
  const int tx = tile_tx(D, L);
  return B * cdiv(L, tx ? tx * kV : any_tokens(L));
}
int64_t part_count(int64_t B, int64_t D, int64_t L) {
  const int64_t n = tile_count(B, D, L), sms = sm_count();
  return tile_tx(D, L) && n > sms ? sms : n;
}

bool aligned_to(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }

// calls f with the tile's lanes along tokens and the channels of a thread
template <typename F>
int by_tile(int64_t D, F &&f) {
  using std::integral_constant;
  if (D <= 64) return f(integral_constant<int, 8>(), integral_constant<int, 1>());
  if (D <= 128) return f(integral_constant<int, 8>(), integral_constant<int, 2>());
  if (D <= 256) return f(integral_constant<int, 8>(), integral_constant<int, 4>());
  if (D <= 512) return f(integral_constant<int, 4>(), integral_constant<int, 4>());
  return f(integral_constant<int, 2>(), integral_constant<int, 4>());
}

template <typename T, typename R, bool LAYER>
int fwd_launch(const NormFwd &a, const NormShape &s, cudaStream_t st) {
  const unsigned grid = (unsigned)tile_count(s.B, s.D, s.L);
  if (tile_tx(s.D, s.L)) {
    const bool vec = s.L % kV == 0 && aligned_to(a.x, sizeof(Four<T>)) &&
                     aligned_to(a.gate, sizeof(Four<T>)) && aligned_to(a.y, sizeof(Four<T>)) &&
                     aligned_to(a.residual, sizeof(Four<R>)) && aligned_to(a.rout, sizeof(Four<R>));
    return by_tile(s.D, [&](auto tx, auto rows) {
      block_norm_fwd_tile_kernel<T, R, decltype(tx)::value, decltype(rows)::value, LAYER>
          <<<grid, kTileThreads, 0, st>>>(a, s, vec);
      return check_launch("block_norm_fwd_tile_kernel");
    });
  }
  switch (any_tokens(s.L)) {
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
int bwd_main(const NormBwd &a, const NormShape &s, cudaStream_t st) {
  if (tile_tx(s.D, s.L)) {
    const bool vec = s.L % kV == 0 && aligned_to(a.x, sizeof(Four<T>)) &&
                     aligned_to(a.gate, sizeof(Four<T>)) && aligned_to(a.ggate, sizeof(Four<T>)) &&
                     aligned_to(a.gy, sizeof(Four<T>)) && aligned_to(a.gx, sizeof(Four<T>)) &&
                     aligned_to(a.residual, sizeof(Four<R>)) &&
                     aligned_to(a.grout, sizeof(Four<R>)) &&
                     aligned_to(a.gresidual, sizeof(Four<R>));
    const unsigned grid = (unsigned)part_count(s.B, s.D, s.L);
    const int64_t tiles = tile_count(s.B, s.D, s.L);
    return by_tile(s.D, [&](auto tx, auto rows) {
      constexpr int ROWS = decltype(rows)::value;
      using Tile = NormTile<T, R, ROWS>;
      const int smem = Tile::kStages * (int)sizeof(Tile);
      auto kern = block_norm_bwd_tile_kernel<T, R, decltype(tx)::value, ROWS, LAYER>;
      if (set_smem_once((const void *)kern, smem) != cudaSuccess)
        return check_launch("block_norm_bwd_tile_kernel shared memory");
      kern<<<grid, kTileThreads, smem, st>>>(a, s, tiles, vec);
      return check_launch("block_norm_bwd_tile_kernel");
    });
  }
  const unsigned grid = (unsigned)tile_count(s.B, s.D, s.L);
  switch (any_tokens(s.L)) {
    case 32: block_norm_bwd_any_kernel<T, R, 32, LAYER><<<grid, kThreads, 0, st>>>(a, s); break;
    case 8: block_norm_bwd_any_kernel<T, R, 8, LAYER><<<grid, kThreads, 0, st>>>(a, s); break;
    default: block_norm_bwd_any_kernel<T, R, 1, LAYER><<<grid, kThreads, 0, st>>>(a, s);
  }
  return check_launch("block_norm_bwd_any_kernel");
}

template <typename T, typename R, bool LAYER>
int bwd_launch(const NormBwd &a, const ParamGrads &g, const NormShape &s, cudaStream_t st) {
  if (int rc = bwd_main<T, R, LAYER>(a, s, st)) return rc;
  const dim3 pg((unsigned)cdiv(s.D, 32), 5);
  block_norm_param_kernel<T><<<pg, 256, 0, st>>>(a.part, (T *)g.w1, (T *)g.w2, (T *)g.scale,
                                                  (T *)g.b1, (T *)g.b2,
                                                  part_count(s.B, s.D, s.L), s.D);
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
  if (!layer && (post_bias || pre_bias)) return refuse("an rms norm has no bias.");
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
  const size_t n = 5 * (size_t)dudy::part_count(B, D, L) * (size_t)D * sizeof(float);
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
  if (!layer && (post_bias || grad_post_bias || grad_pre_bias))
    return refuse("an rms norm has no bias.");
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
