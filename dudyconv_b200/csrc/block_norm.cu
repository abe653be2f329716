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
// A block holds a tile of 8 TX tokens x all channels, eight tokens (16 bytes of a 16-bit row) and
// up to four (backward: two) channels to a thread, so each tensor moves once. TX = 4 (rows of 64
// bytes) up to D = 256, then 2 and 1. Persistent blocks copy their next tile into shared memory
// while they work on one, each thread's own pieces side by side (no thread reads another's, so its
// own copies' completion is all it waits for). Arithmetic goes two tokens at a time (__ffma2_rn).
// At B=16, D=256, L=4096 in fp16 with a gate, rms: 35 us forward (168 MB, 4.8 TB/s, 73% of a copy's
// 6540 GB/s) and 78 us backward with the parameter sums (268 MB, 3.4 TB/s). The backward's one block of
// 512 threads an SM waits as a whole at each of a tile's barriers: the issue slots are 45% busy (two
// norms' sums, the gate's sigmoid twice and three parameter sums an element), shared memory 54%, HBM
// 52%. Four tokens to a thread, with twice the addresses and sums a token, took 62 and 107 us;
// re-reading the tile for each sum, 462 in all.
constexpr int kFwdThreads = 256, kBwdThreads = 512;
constexpr int kV = 8;  // tokens of a thread

template <typename T>
using Piece = RowEight<T>;
using Two = float2[kV / 2];

template <int NT>
struct TileRed {
  float part[2][NT / 32][32];
  float total[2][32];
};

// Sums of the eight tokens' values over the block's rows of threads, known to all threads of the
// tokens: across the rows of a warp by shuffles, each lane ending with one token's, and across
// the warps by as many lanes a token. `turn` alternates between two sets of buffers, so two
// barriers are enough.
template <int TX, int NT>
__device__ __forceinline__ void tile_sum(Two &p, TileRed<NT> &m, int &turn) {
  constexpr int kW = NT / 32, TOK = TX * kV, LY = 32 / TX, SAME = LY / kV;
  const int tid = threadIdx.x, tx = tid % TX, ly = (tid & 31) / TX;
  float v[kV];
#pragma unroll
  for (int i = 0; i < kV / 2; ++i) v[2 * i] = p[i].x, v[2 * i + 1] = p[i].y;
  Scatter<TX, LY, kV>::sum(v, tid & 31);
  if (ly % SAME == 0) m.part[turn][tid >> 5][tx * kV + ly / SAME] = v[0];
  __syncthreads();
  if (tid < TOK * kW) {
    float s = m.part[turn][tid % kW][tid / kW];
#pragma unroll
    for (int o = kW / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (tid % kW == 0) m.total[turn][tid / kW] = s;
  }
  __syncthreads();
  const float4 t = *reinterpret_cast<const float4 *>(&m.total[turn][tx * kV]);
  const float4 u = *reinterpret_cast<const float4 *>(&m.total[turn][tx * kV + 4]);
  p[0] = make_float2(t.x, t.y);
  p[1] = make_float2(t.z, t.w);
  p[2] = make_float2(u.x, u.y);
  p[3] = make_float2(u.z, u.w);
  turn ^= 1;
}

template <typename T>
__device__ __forceinline__ void store_pairs(T *row, int left, const Two &p, bool vec) {
  float v[kV];
#pragma unroll
  for (int i = 0; i < kV / 2; ++i) v[2 * i] = p[i].x, v[2 * i + 1] = p[i].y;
  row_store8(row, 0, left, v, vec);
}

template <typename T>
__device__ __forceinline__ void fetch8(Piece<T> &to, const T *from, int left, bool vec) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(Piece<T>) / 16; ++i)
      cp_async16(reinterpret_cast<char *>(&to) + 16 * i, reinterpret_cast<const char *>(from) + 16 * i);
  } else {
    to.load(from, 0, left, false);
  }
}

// where a thread's tokens of a tile are
struct Place {
  int64_t first, base;  // of the tokens alone, and of channel 0's row
  int left;
};
template <int TX>
__device__ __forceinline__ Place place(unsigned tile, unsigned tiles, const NormShape &s) {
  const unsigned b = tile / tiles;
  const int t = (int)(tile - b * tiles) * (TX * kV) + threadIdx.x % TX * kV;
  return Place{b * s.L + t, b * s.D * s.L + t, (int)s.L - t};
}

template <typename T, typename R, int ROWS>
struct FwdTile {
  Piece<T> x[ROWS][kFwdThreads], z[ROWS][kFwdThreads];
  Piece<R> r[ROWS][kFwdThreads];
  static constexpr int kBytes = ROWS * kFwdThreads * (2 * sizeof(Piece<T>) + sizeof(Piece<R>));
  // two blocks an SM where two tiles of each fit, else one
  static constexpr int kBlocks = 2 * kBytes <= 104 * 1024 ? 2 : 1;
};

template <typename T, typename R, int TX, int ROWS, bool LAYER>
__global__ void __launch_bounds__(kFwdThreads, (FwdTile<T, R, ROWS>::kBlocks))
block_norm_fwd_tile_kernel(NormFwd a, NormShape s, unsigned ntiles, bool vec) {
  using Tile = FwdTile<T, R, ROWS>;
  constexpr int TY = kFwdThreads / TX;
  extern __shared__ __align__(16) char smem_raw[];
  Tile *stage = reinterpret_cast<Tile *>(smem_raw);
  __shared__ __align__(16) TileRed<kFwdThreads> red;
  const int tid = threadIdx.x, ty = tid / TX;
  const unsigned tiles = (unsigned)((s.L + TX * kV - 1) / (TX * kV));
  const float rd = 1.f / (float)s.D;
  const int D = (int)s.D;
  int turn = 0, at = 0;

  // residual + c1 hat1 + c0, y = c2 hat2 + c3
  float c1[ROWS], c0[ROWS], c2[ROWS], c3[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int d = ty + i * TY;
    const bool ok = d < D;
    const float sc = ok ? opt((const T *)a.scale, d, 1.f) : 0.f;
    c1[i] = ok ? sc * ldf((const T *)a.w1 + d) : 0.f;
    c0[i] = LAYER && ok ? sc * opt((const T *)a.b1, d, 0.f) : 0.f;
    c2[i] = ok ? ldf((const T *)a.w2 + d) : 0.f;
    c3[i] = LAYER && ok ? opt((const T *)a.b2, d, 0.f) : 0.f;
  }
  auto fetch = [&](unsigned tile, Tile &m) {
    const Place p = place<TX>(tile, tiles, s);
    if (p.left > 0)
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int d = ty + i * TY;
        if (d >= D) continue;
        const int64_t o = p.base + d * s.L;
        fetch8(m.x[i][tid], (const T *)a.x + o, p.left, vec);
        if (a.gate) fetch8(m.z[i][tid], (const T *)a.gate + o, p.left, vec);
        fetch8(m.r[i][tid], (const R *)a.residual + o, p.left, vec);
      }
    copies_commit();
  };
  if (blockIdx.x < ntiles) fetch(blockIdx.x, stage[0]);
  for (unsigned tile = blockIdx.x; tile < ntiles; tile += gridDim.x, at ^= 1) {
    const Place p = place<TX>(tile, tiles, s);
    if (tile + gridDim.x < ntiles) {
      fetch(tile + gridDim.x, stage[at ^ 1]);
      copies_wait<1>();
    } else {
      copies_wait<0>();
    }
    const Tile &m = stage[at];
    float2 g[ROWS][kV / 2];
    Two m1, m2, inv1, q;
#pragma unroll
    for (int k = 0; k < kV / 2; ++k) m1[k] = m2[k] = q[k] = both(0.f);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const bool ok = p.left > 0 && ty + i * TY < D;
#pragma unroll
      for (int k = 0; k < kV / 2; ++k) {
        float2 v = m.x[i][tid].pair(k);
        if (a.gate) {
          const float2 z = m.z[i][tid].pair(k);
          v = mul2(v, mul2(z, sigmoid2<T>(z)));
        }
        if (!ok) v = both(0.f);
        g[i][k] = v;
        if (LAYER) m1[k] = add2(m1[k], v);
        else q[k] = fma2(v, v, q[k]);
      }
    }
    // mean and 1 / sqrt(var + eps) of g; q holds the sum of squares of an rms norm
    auto statistics = [&](Two &mean, Two &inv) {
      if (LAYER) {
        tile_sum<TX>(mean, red, turn);
#pragma unroll
        for (int k = 0; k < kV / 2; ++k) mean[k] = mul2(mean[k], both(rd)), q[k] = both(0.f);
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
          if (ty + i * TY < D)
#pragma unroll
            for (int k = 0; k < kV / 2; ++k) {
              const float2 c = add2(g[i][k], neg2(mean[k]));
              q[k] = fma2(c, c, q[k]);
            }
      }
      tile_sum<TX>(q, red, turn);
#pragma unroll
      for (int k = 0; k < kV / 2; ++k) {
        inv[k] = make_float2(rsqrtf(fmaf(q[k].x, rd, s.eps)), rsqrtf(fmaf(q[k].y, rd, s.eps)));
        q[k] = both(0.f);
      }
    };
    statistics(m1, inv1);
    // the residual stream takes g's place
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int d = ty + i * TY;
      const bool ok = p.left > 0 && d < D;
#pragma unroll
      for (int k = 0; k < kV / 2; ++k) {
        const float2 hat = mul2(LAYER ? add2(g[i][k], neg2(m1[k])) : g[i][k], inv1[k]);
        float2 v = m.r[i][tid].pair(k);
        if (LAYER) v = add2(v, both(c0[i]));
        v = fma2(hat, both(c1[i]), v);
        if (!ok) v = both(0.f);
        g[i][k] = v;
        if (LAYER) m2[k] = add2(m2[k], v);
        else q[k] = fma2(v, v, q[k]);
      }
      if (ok) store_pairs((R *)a.rout + p.base + d * s.L, p.left, g[i], vec);
    }
    Two inv2;
    statistics(m2, inv2);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int d = ty + i * TY;
      if (p.left <= 0 || d >= D) continue;
      Two y;
#pragma unroll
      for (int k = 0; k < kV / 2; ++k) {
        const float2 hat = mul2(LAYER ? add2(g[i][k], neg2(m2[k])) : g[i][k], inv2[k]);
        y[k] = LAYER ? fma2(hat, both(c2[i]), both(c3[i])) : mul2(hat, both(c2[i]));
      }
      store_pairs((T *)a.y + p.base + d * s.L, p.left, y, vec);
    }
    if (a.stats && ty == 0 && p.left > 0) {
      const int64_t n = s.B * s.L;
      float *st = a.stats + p.first;
      if (LAYER) store_pairs(st, p.left, m1, vec), store_pairs(st + 2 * n, p.left, m2, vec);
      store_pairs(st + n, p.left, inv1, vec);
      store_pairs(st + 3 * n, p.left, inv2, vec);
    }
  }
}

template <typename T, typename R, int ROWS>
struct BwdTile {
  Piece<T> x[ROWS][kBwdThreads], z[ROWS][kBwdThreads], gy[ROWS][kBwdThreads];
  Piece<R> r[ROWS][kBwdThreads], gr[ROWS][kBwdThreads];
  static constexpr int kBytes = ROWS * kBwdThreads * (3 * sizeof(Piece<T>) + 2 * sizeof(Piece<R>));
  // two tiles where they fit beside the block's other shared memory
  static constexpr int kStages = 2 * kBytes <= 216 * 1024 ? 2 : 1;
};

// The parameter sums stay in registers until a block's last tile.
template <typename T, typename R, int TX, int ROWS, bool LAYER>
__global__ void __launch_bounds__(kBwdThreads, 1)
block_norm_bwd_tile_kernel(NormBwd a, NormShape s, unsigned ntiles, bool vec) {
  using Tile = BwdTile<T, R, ROWS>;
  constexpr int TY = kBwdThreads / TX;
  extern __shared__ __align__(16) char smem_raw[];
  Tile *stage = reinterpret_cast<Tile *>(smem_raw);
  __shared__ __align__(16) TileRed<kBwdThreads> red;
  const int tid = threadIdx.x, ty = tid / TX;
  const unsigned tiles = (unsigned)((s.L + TX * kV - 1) / (TX * kV));
  const int64_t n = s.B * s.L;
  const int D = (int)s.D;
  const float rd = 1.f / (float)s.D;
  int turn = 0;

  float w1[ROWS], b1[ROWS], sc[ROWS], w2[ROWS];
  // sums over tokens: dr hat1, dy hat2, dr, dy
  float2 acc[LAYER ? 4 : 2][ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int d = ty + i * TY;
    const bool ok = d < D;
    w1[i] = ok ? ldf((const T *)a.w1 + d) : 0.f;
    w2[i] = ok ? ldf((const T *)a.w2 + d) : 0.f;
    b1[i] = LAYER && ok ? opt((const T *)a.b1, d, 0.f) : 0.f;
    sc[i] = ok ? opt((const T *)a.scale, d, 1.f) : 0.f;
#pragma unroll
    for (int j = 0; j < (LAYER ? 4 : 2); ++j) acc[j][i] = both(0.f);
  }
  auto fetch = [&](unsigned tile, Tile &m) {
    const Place p = place<TX>(tile, tiles, s);
    if (p.left > 0)
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int d = ty + i * TY;
        if (d >= D) continue;
        const int64_t o = p.base + d * s.L;
        fetch8(m.x[i][tid], (const T *)a.x + o, p.left, vec);
        if (a.gate) fetch8(m.z[i][tid], (const T *)a.gate + o, p.left, vec);
        fetch8(m.r[i][tid], (const R *)a.residual + o, p.left, vec);
        fetch8(m.gy[i][tid], (const T *)a.gy + o, p.left, vec);
        if (a.grout) fetch8(m.gr[i][tid], (const R *)a.grout + o, p.left, vec);
      }
    copies_commit();
  };
  // the tile's statistics, by turns: mean1, inv1, mean2, inv2 of its tokens
  __shared__ __align__(16) Piece<float> stat[2][4][TX];
  auto fetch_stats = [&](unsigned tile, int buf) {
    const int tx = tid % TX, k = tid / TX;
    if (k >= 4 || (!LAYER && k % 2 == 0)) return;
    const Place p = place<TX>(tile, tiles, s);
    if (p.left > 0) fetch8(stat[buf][k][tx], a.stats + k * n + p.first, p.left, vec);
    else stat[buf][k][tx].load(a.stats, 0, 0, false);
  };
  int buf = 0;
  if (blockIdx.x < ntiles) {
    fetch_stats(blockIdx.x, 0);
    fetch(blockIdx.x, stage[0]);
  }
  for (unsigned tile = blockIdx.x; tile < ntiles; tile += gridDim.x, buf ^= 1) {
    const Place p = place<TX>(tile, tiles, s);
    const bool more = tile + gridDim.x < ntiles;
    const Tile &m = stage[Tile::kStages == 2 ? buf : 0];
    copies_wait<0>();
    __syncthreads();  // for the statistics: other threads copied them
    if (Tile::kStages == 2 && more) {
      fetch_stats(tile + gridDim.x, buf ^ 1);
      fetch(tile + gridDim.x, stage[buf ^ 1]);
    }
    const Piece<float> &m1 = stat[buf][0][tid % TX], &inv1 = stat[buf][1][tid % TX];
    const Piece<float> &m2 = stat[buf][2][tid % TX], &inv2 = stat[buf][3][tid % TX];
    const Two i1 = {inv1.pair(0), inv1.pair(1), inv1.pair(2), inv1.pair(3)};
    const Two i2 = {inv2.pair(0), inv2.pair(1), inv2.pair(2), inv2.pair(3)};
    Two v, u;
#pragma unroll
    for (int k = 0; k < kV / 2; ++k) v[k] = u[k] = both(0.f);
    float2 hat1[ROWS][kV / 2], hat2[ROWS][kV / 2];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const bool ok = p.left > 0 && ty + i * TY < D;
#pragma unroll
      for (int k = 0; k < kV / 2; ++k) {
        float2 g = m.x[i][tid].pair(k), r = m.r[i][tid].pair(k), dy = m.gy[i][tid].pair(k);
        if (a.gate) {
          const float2 z = m.z[i][tid].pair(k);
          g = mul2(g, mul2(z, sigmoid2<T>(z)));
        }
        if (!ok) g = r = dy = both(0.f);
        float2 h1 = mul2(LAYER ? add2(g, neg2(m1.pair(k))) : g, i1[k]);
        if (LAYER && !ok) h1 = both(0.f);
        float2 h2 = fma2(h1, both(sc[i] * w1[i]), r);
        if (LAYER) h2 = add2(h2, add2(both(sc[i] * b1[i]), neg2(m2.pair(k))));
        h2 = mul2(h2, i2[k]);
        if (LAYER && !ok) h2 = both(0.f);
        hat1[i][k] = h1;
        hat2[i][k] = h2;
        const float2 d2 = mul2(dy, both(w2[i]));
        v[k] = fma2(d2, h2, v[k]);
        acc[1][i] = fma2(dy, h2, acc[1][i]);
        if (LAYER) {
          u[k] = add2(u[k], d2);
          acc[3][i] = add2(acc[3][i], dy);
        }
      }
    }
    tile_sum<TX>(v, red, turn);
    if (LAYER) tile_sum<TX>(u, red, turn);
    Two c, e;
#pragma unroll
    for (int k = 0; k < kV / 2; ++k) {
      c[k] = mul2(v[k], both(-rd));
      e[k] = mul2(u[k], both(-rd));
      v[k] = u[k] = both(0.f);
    }
    // the gradient of hat1 takes hat2's place
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int d = ty + i * TY;
      const bool ok = p.left > 0 && d < D;
      Two dr;
#pragma unroll
      for (int k = 0; k < kV / 2; ++k) {
        float2 o = fma2(hat2[i][k], c[k], mul2(m.gy[i][tid].pair(k), both(w2[i])));
        if (LAYER) o = add2(o, e[k]);
        dr[k] = a.grout ? fma2(i2[k], o, m.gr[i][tid].pair(k)) : mul2(i2[k], o);
        if (!ok) dr[k] = both(0.f);
        const float2 d1 = mul2(dr[k], both(sc[i] * w1[i]));
        hat2[i][k] = d1;
        v[k] = fma2(d1, hat1[i][k], v[k]);
        acc[0][i] = fma2(dr[k], hat1[i][k], acc[0][i]);
        if (LAYER) {
          u[k] = add2(u[k], d1);
          acc[2][i] = add2(acc[2][i], dr[k]);
        }
      }
      if (ok) store_pairs((R *)a.gresidual + p.base + d * s.L, p.left, dr, vec);
    }
    tile_sum<TX>(v, red, turn);
    if (LAYER) tile_sum<TX>(u, red, turn);
#pragma unroll
    for (int k = 0; k < kV / 2; ++k) {
      c[k] = mul2(v[k], both(-rd));
      e[k] = mul2(u[k], both(-rd));
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int d = ty + i * TY;
      if (p.left <= 0 || d >= D) continue;
      Two gx, gz;
#pragma unroll
      for (int k = 0; k < kV / 2; ++k) {
        float2 o = fma2(hat1[i][k], c[k], hat2[i][k]);
        if (LAYER) o = add2(o, e[k]);
        gx[k] = mul2(i1[k], o);
        if (a.gate) {
          const float2 z = m.z[i][tid].pair(k), sg = sigmoid2<T>(z), h = mul2(gx[k], sg);
          gx[k] = mul2(h, z);
          gz[k] = mul2(mul2(h, m.x[i][tid].pair(k)),
                       fma2(z, fma2(sg, both(-1.f), both(1.f)), both(1.f)));
        }
      }
      store_pairs((T *)a.gx + p.base + d * s.L, p.left, gx, vec);
      if (a.gate) store_pairs((T *)a.ggate + p.base + d * s.L, p.left, gz, vec);
    }
    if (Tile::kStages == 1 && more) {
      fetch_stats(tile + gridDim.x, buf ^ 1);
      fetch(tile + gridDim.x, stage[0]);
    }
  }
  // post_weight: scale sum(dr hat1); pre_weight: sum(dy hat2); scale: sum(dr p) = w1 sum(dr hat1) +
  // b1 sum(dr); post_bias: scale sum(dr); pre_bias: sum(dy)
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    float q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      q[j] = j < (LAYER ? 4 : 2) ? acc[LAYER ? j : j & 1][i].x + acc[LAYER ? j : j & 1][i].y : 0.f;
#pragma unroll
      for (int o = TX / 2; o > 0; o >>= 1) q[j] += __shfl_xor_sync(0xffffffffu, q[j], o);
    }
    const int d = ty + i * TY;
    if (tid % TX || d >= D) continue;
    const float out[5] = {sc[i] * q[0], q[1], fmaf(w1[i], q[0], b1[i] * q[2]), sc[i] * q[2], q[3]};
#pragma unroll
    for (int j = 0; j < (LAYER ? 5 : 3); ++j)
      a.part[(j * (int64_t)gridDim.x + blockIdx.x) * s.D + d] = out[j];
  }
}

// The parameter gradients: the sum of the tiles' (or blocks') parts, 32 channels a block.
template <typename T>
__global__ void __launch_bounds__(1024)
block_norm_param_kernel(const float *__restrict__ part, T *g0, T *g1, T *g2, T *g3, T *g4,
                        int64_t tiles, int64_t D) {
  __shared__ float red[32][32];
  T *const outs[5] = {g0, g1, g2, g3, g4};
  T *out = outs[blockIdx.y];
  if (!out) return;
  const int64_t d = blockIdx.x * 32ll + (threadIdx.x & 31);
  const float v = column_sum<32>(part + blockIdx.y * tiles * D + d, tiles, D, d < D, red);
  if (threadIdx.x < 32 && d < D) stf(out + d, v);
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
  return D <= 256 ? 4 : (D <= 512 ? 2 : 1);
}

// tiles of the kernel that runs, and the number of parts of its parameter sums
int64_t tile_count(int64_t B, int64_t D, int64_t L) {
  const int tx = tile_tx(D, L);
  return B * cdiv(L, tx ? tx * kV : any_tokens(L));
}
int64_t part_count(int64_t B, int64_t D, int64_t L) {
  const int64_t n = tile_count(B, D, L), most = sm_count();
  return tile_tx(D, L) && n > most ? most : n;
}

// calls f with the tile's lanes along tokens and the channels of a thread
template <int NT, typename F>
int by_tile(int64_t D, F &&f) {
  using std::integral_constant;
  constexpr int kMost = 1024 / NT;  // channels of a thread at D = 256, 512, 1024
  if (D <= NT / 4) return f(integral_constant<int, 4>(), integral_constant<int, 1>());
  if (kMost == 4 && D <= 128) return f(integral_constant<int, 4>(), integral_constant<int, 2>());
  if (D <= 256) return f(integral_constant<int, 4>(), integral_constant<int, kMost>());
  if (D <= 512) return f(integral_constant<int, 2>(), integral_constant<int, kMost>());
  return f(integral_constant<int, 1>(), integral_constant<int, kMost>());
}

template <typename T, typename R, bool LAYER>
int fwd_launch(const NormFwd &a, const NormShape &s, cudaStream_t st) {
  const unsigned grid = (unsigned)tile_count(s.B, s.D, s.L);
  if (tile_tx(s.D, s.L)) {
    const bool vec = s.L % kV == 0 && aligned_to_16(a.x) &&
                     aligned_to_16(a.gate) && aligned_to_16(a.y) &&
                     aligned_to_16(a.residual) &&
                     aligned_to_16(a.rout) && aligned_to_16(a.stats);
    return by_tile<kFwdThreads>(s.D, [&](auto tx, auto rows) {
      using Tile = FwdTile<T, R, decltype(rows)::value>;
      const int smem = 2 * (int)sizeof(Tile), most = Tile::kBlocks * sm_count();
      auto kern = block_norm_fwd_tile_kernel<T, R, decltype(tx)::value, decltype(rows)::value, LAYER>;
      if (set_smem_once((const void *)kern, smem) != cudaSuccess)
        return check_launch("block_norm_fwd_tile_kernel shared memory");
      kern<<<grid < (unsigned)most ? grid : most, kFwdThreads, smem, st>>>(a, s, grid, vec);
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
    const bool vec = s.L % kV == 0 && aligned_to_16(a.x) &&
                     aligned_to_16(a.gate) && aligned_to_16(a.ggate) &&
                     aligned_to_16(a.gy) && aligned_to_16(a.gx) &&
                     aligned_to_16(a.residual) &&
                     aligned_to_16(a.grout) &&
                     aligned_to_16(a.gresidual) && aligned_to_16(a.stats);
    const unsigned grid = (unsigned)part_count(s.B, s.D, s.L);
    const int64_t tiles = tile_count(s.B, s.D, s.L);
    return by_tile<kBwdThreads>(s.D, [&](auto tx, auto rows) {
      constexpr int ROWS = decltype(rows)::value;
      using Tile = BwdTile<T, R, ROWS>;
      const int smem = Tile::kStages * (int)sizeof(Tile);
      auto kern = block_norm_bwd_tile_kernel<T, R, decltype(tx)::value, ROWS, LAYER>;
      if (set_smem_once((const void *)kern, smem) != cudaSuccess)
        return check_launch("block_norm_bwd_tile_kernel shared memory");
      kern<<<grid, kBwdThreads, smem, st>>>(a, s, (unsigned)tiles, vec);
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
  block_norm_param_kernel<T><<<pg, 1024, 0, st>>>(a.part, (T *)g.w1, (T *)g.w2, (T *)g.scale,
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
  if (!(eps > 0.f)) return refuse("eps must be positive.");
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
