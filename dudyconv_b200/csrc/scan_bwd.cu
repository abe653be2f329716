// scan_bwd.cu -- the selective scan's gradients.
//
// With a = exp(dt A) and g[t] = dL/dh[t]:  g[t] = C[t] dy[t] + a[t+1] g[t+1]   (from the right)
//   dC[n,t] = sum_d h dy                 dB[n,t] = sum_d g dt u        (channels of the group)
//   dA[d,n] = sum_{b,t} dt g a h[t-1]    ddt = u sum_n g B + sum_n A g a h[t-1]
//   du = dt sum_n g B + skip dy          ddelta = ddt softplus'        dskip = sum_{b,t} dy u
// Pieces of four positions go from the right end of a sequence to its left, from warp to warp
// of a block. The state that enters each was saved by the forward (16 bytes a state for every
// four positions: HBM has the time, and recovering them here would take a second chain in the
// other direction), so only g's recurrence runs from piece to piece.
//
// The sums over channels set the layout: a thread holds four channels x four states, so that
// most of a sum over channels or states happens in its registers and only the rest by
// shuffles. dB and dC of a block's channels are written as fp32 parts, one per block of
// channels, and added by a second kernel in a fixed order; so are dA and the two [D] sums over
// the batch and the chunks.
#include "scan.cuh"

namespace dudy {
namespace scan {
namespace {

constexpr int kND = 4;                 // channels of a thread
constexpr int kQ = 4;                  // positions of a piece
static_assert(kQ == kCkpt, "a state is saved at each piece's start");

struct Bwd {
  const void *go, *u, *delta, *Bm, *Cm;
  const float *gfinal, *A, *skip, *delta_bias, *ckpt;
  const int32_t *lengths;
  void *gu, *gdelta;
  float *ginit;
  float *part_b, *part_c;  // [tiles][B*G*N*L]
  float *part_a;           // [splits][B][D*N]
  float *part_d;           // [2][splits][B][D]: skip, delta_bias
  float *rend, *prod;      // [splits][B*D][N]: what a chunk passes to its left from zero, and its
                           // decays' product
  int64_t chunk;           // positions of a chunk, a multiple of kQ
  int splits, vec;
};

// a warp's own piece, positions outermost
template <int LPC>
struct BwdPiece {
  static constexpr int CT = 32 / LPC * kND;      // channels of a block
  static constexpr int NP = kNS * LPC;
  static constexpr int UI = (CT + 31) / 32;      // rows of u, delta and dy that a lane copies
  static constexpr int BI = (2 * NP + 31) / 32;  // rows of B and C
  float dt[kQ * CT], du[kQ * CT], go[kQ * CT];
  float u[kQ * CT], slope[kQ * CT];              // du's and ddelta's results take their places
  float bc[kQ * 2 * NP];                         // B and C of a position side by side
  float h0[2][CT * NP];                          // the states that enter this piece and the next
};
template <int LPC>
struct BwdSmem {
  BwdPiece<LPC> piece[kWarps];
  // handed on to the left, [warp][four of the thread's states][lane] (with the chunk's decay
  // product so far); the sums over warps at the end use the same room
  float4 pass[kWarps * kND * 32], total[kWarps * kND * 32];
};

// A thread's states lie in pairs of channels: e[p][n] holds channels 2p and 2p + 1 of state n,
// so that a position's dt, dt u and gradient of two channels are operands as they are read.
template <typename T, int LPC, bool PRE>
__global__ void __launch_bounds__(kThreads, 1)
scan_bwd_kernel(Bwd a, Shape s) {
  using Mine = BwdPiece<LPC>;
  constexpr int CT = Mine::CT, NP = Mine::NP;
  extern __shared__ __align__(16) char smem_raw[];
  BwdSmem<LPC> &all = *reinterpret_cast<BwdSmem<LPC> *>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ln = lane % LPC, ld = lane / LPC, n0 = ln * kNS, c0 = ld * kND;
  Mine &m = all.piece[warp];

  const int split = blockIdx.x % a.splits;
  if (PRE && split == 0) return;  // nothing lies to the left of the first chunk
  const int64_t bid = blockIdx.x / a.splits;
  const int R = (int)(s.D / s.G), tiles = (R + CT - 1) / CT;
  const int tile = (int)(bid % tiles);
  const int64_t bg = bid / tiles, b = bg / s.G, g = bg % s.G;
  const int chans = R - tile * CT < CT ? R - tile * CT : CT;
  const int64_t d0 = g * R + tile * CT, row0 = b * s.D + d0;
  const int64_t len = clamp_len(a.lengths, b, s.L);
  const int64_t from = split * a.chunk;
  const int64_t to = from + a.chunk < s.L ? from + a.chunk : s.L;
  const int64_t end = to < len ? to : len;
  const T *u = (const T *)a.u + row0 * s.L, *delta = (const T *)a.delta + row0 * s.L;
  const T *go = (const T *)a.go + row0 * s.L;
  const T *Bm = (const T *)a.Bm + bg * s.N * s.L, *Cm = (const T *)a.Cm + bg * s.N * s.L;
  T *gu = (T *)a.gu + row0 * s.L, *gdelta = (T *)a.gdelta + row0 * s.L;
  const int64_t nbc = s.B * s.G * s.N * s.L, nst = s.B * s.D * s.N;
  float *gB = a.part_b + tile * nbc + bg * s.N * s.L;
  float *gC = a.part_c + tile * nbc + bg * s.N * s.L;

  float2 A[2][kNS], dA[2][kNS], r[2][kNS], dskip[2], dbias[2], total[2][kNS];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    dskip[p] = dbias[p] = both(0.f);
#pragma unroll
    for (int i = 0; i < kNS; ++i) {
      float av[2], rv[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int c = c0 + 2 * p + x;
        const bool ok = c < chans && n0 + i < s.N;
        const int64_t at = (row0 + c) * s.N + n0 + i;
        av[x] = ok ? scaled<T>(a.A[(d0 + c) * s.N + n0 + i]) : 0.f;
        rv[x] = 0.f;
        if (!PRE && ok && warp == 0) {
          if (a.gfinal) rv[x] = a.gfinal[at];
          for (int k = a.splits - 1; k > split; --k)
            rv[x] = fmaf(a.prod[k * nst + at], rv[x], a.rend[k * nst + at]);
        }
      }
      A[p][i] = make_float2(av[0], av[1]);
      r[p][i] = make_float2(rv[0], rv[1]);
      dA[p][i] = both(0.f);
      total[p][i] = both(1.f);
    }
  }
  auto put = [&](float4 *dst, const float2 (&v)[2][kNS]) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      dst[(2 * p) * 32 + lane] = quad(v[p][0], v[p][1]);
      dst[(2 * p + 1) * 32 + lane] = quad(v[p][2], v[p][3]);
    }
  };
  auto take = [&](float2 (&v)[2][kNS], const float4 *src) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const float4 x = src[(2 * p) * 32 + lane], z = src[(2 * p + 1) * 32 + lane];
      v[p][0] = lo(x); v[p][1] = hi(x); v[p][2] = lo(z); v[p][3] = hi(z);
    }
  };

  // a lane's channels where it copies them
  float bias[Mine::UI], skip[Mine::UI];
#pragma unroll
  for (int k = 0; k < Mine::UI; ++k) {
    const int d = lane + k * 32;
    bias[k] = d < chans && a.delta_bias ? a.delta_bias[d0 + d] : 0.f;
    skip[k] = !PRE && d < chans && a.skip ? a.skip[d0 + d] : 0.f;
  }
  // the warp's next piece, in registers while this one is worked on
  RowFour<T> pu[Mine::UI], pd[Mine::UI], pg[Mine::UI], pb[Mine::BI];
  auto fetch = [&](int64_t t0) {
#pragma unroll
    for (int k = 0; k < Mine::UI; ++k) {
      const int d = lane + k * 32;
      if (d >= CT) break;
      const int64_t lim = d < chans ? end : 0;
      if (!PRE) row_load4(pu[k], u + d * s.L, t0, lim, a.vec);
      row_load4(pd[k], delta + d * s.L, t0, lim, a.vec);
      row_load4(pg[k], go + d * s.L, t0, lim, a.vec);
    }
#pragma unroll
    for (int k = 0; k < Mine::BI; ++k) {
      const int r = lane + k * 32, n = r % NP;
      if (r >= 2 * NP) break;
      row_load4(pb[k], (r < NP ? Bm : Cm) + n * s.L, t0, n < s.N ? end : 0, a.vec);
    }
  };
  using SumD = Scatter<LPC, 32 / LPC, 2 * kNS>;
  constexpr int kLeftD = SumD::kLeft, kGroups = 2 * kNS / kLeftD;
  constexpr int kSame = 32 / LPC / kGroups;  // lanes that end with the same values
  using SumN = Scatter<1, LPC, 2 * kND, 2>;
  constexpr int kLeftN = SumN::kLeft / 2, kOwners = kND / kLeftN, kEach = LPC / kOwners;
  // the states that enter the piece of positions from t0 on
  auto fetch_states = [&](int64_t t0, float *dst) {
    const float *src = a.ckpt + ((b * s.ckpts() + t0 / kCkpt) * s.D + d0) * s.N;
    const bool vec = s.N % 4 == 0;
#pragma unroll
    for (int i = lane; i < CT * (NP / 4); i += 32) {
      const int c = i / (NP / 4), n = i % (NP / 4) * 4;
      float *to = dst + c * NP + n;
      if (vec && c < chans && n < s.N) {
        cp_async16(to, src + c * s.N + n);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = c < chans && n + e < s.N ? src[c * s.N + n + e] : 0.f;
      }
    }
  };
  // piece k, counted from the right, is warp k % kWarps's
  const int pieces = end > from ? (int)((end - from + kQ - 1) / kQ) : 0;
  auto start = [&](int k) { return from + (int64_t)(pieces - 1 - k) * kQ; };
  int turn = 0;
  if (warp < pieces) {
    fetch(start(warp));
    if (!PRE) fetch_states(start(warp), m.h0[0]);
  }
  for (int k = warp; k < pieces; k += kWarps, turn ^= 1) {
    const int64_t t0 = start(k);
    if (!PRE) cp_async_wait_all();
    __syncwarp();
#pragma unroll
    for (int p = 0; p < Mine::UI; ++p) {
      const int d = lane + p * 32;
      if (d >= CT) break;
#pragma unroll
      for (int j = 0; j < kQ; ++j) {
        float dt = pd[p].get(j) + bias[p], slope = 1.f;
        if (s.softplus) dt = softplus<T>(dt, slope);
        if (t0 + j >= end) dt = slope = 0.f;
        m.dt[j * CT + d] = dt;
        m.go[j * CT + d] = pg[p].get(j);
        if (PRE) continue;
        const float uv = pu[p].get(j);
        m.du[j * CT + d] = dt * uv;
        m.u[j * CT + d] = uv;
        m.slope[j * CT + d] = slope;
      }
    }
#pragma unroll
    for (int p = 0; p < Mine::BI; ++p) {
      const int r = lane + p * 32;
      if (r >= 2 * NP) break;
#pragma unroll
      for (int j = 0; j < kQ; ++j) m.bc[j * 2 * NP + r] = pb[p].get(j);
    }
    __syncwarp();
    if (k + kWarps < pieces) {
      fetch(start(k + kWarps));
      if (!PRE) fetch_states(start(k + kWarps), m.h0[turn ^ 1]);
    }

    auto four = [](const float *p) { return *reinterpret_cast<const float4 *>(p); };
    auto twice = [&](int q, int which, float2 (&v)[kNS]) {
      const float4 x = four(m.bc + q * 2 * NP + which * NP + n0);
      v[0] = both(x.x); v[1] = both(x.y); v[2] = both(x.z); v[3] = both(x.w);
    };
    // dec[q]: position q's decay
    float2 dec[kQ][2][kNS], own[2][kNS], prod[2][kNS], bv[kNS], cv[kNS];
#pragma unroll
    for (int q = kQ - 1; q >= 0; --q) {
      const float4 dt = four(m.dt + q * CT + c0), gv = four(m.go + q * CT + c0);
      twice(q, 1, cv);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const float2 dtp = p ? hi(dt) : lo(dt), gy = p ? hi(gv) : lo(gv);
#pragma unroll
        for (int i = 0; i < kNS; ++i) {
          const float2 x = __fmul2_rn(dtp, A[p][i]);
          const float2 e = make_float2(decay<T>(x.x), decay<T>(x.y));
          dec[q][p][i] = e;
          own[p][i] = __fmul2_rn(e, q == kQ - 1 ? __fmul2_rn(cv[i], gy)
                                                 : __ffma2_rn(cv[i], gy, own[p][i]));
          prod[p][i] = q == kQ - 1 ? e : __fmul2_rn(prod[p][i], e);
        }
      }
    }
    // what enters the piece from the right, and what leaves it to the left
    if (k > 0) {
      const int before = (warp + kWarps - 1) % kWarps;
      pair_wait(1 + before);
      take(r, all.pass + before * kND * 32);
      if (PRE) take(total, all.total + before * kND * 32);
    }
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < kNS; ++i) {
        own[p][i] = __ffma2_rn(prod[p][i], r[p][i], own[p][i]);
        if (PRE) total[p][i] = __fmul2_rn(total[p][i], prod[p][i]);
      }
    if (k + 1 < pieces) {
      put(all.pass + warp * kND * 32, own);
      if (PRE) put(all.total + warp * kND * 32, total);
      pair_arrive(1 + warp);
    }
    if (PRE) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int i = 0; i < kNS; ++i) r[p][i] = own[p][i];
      continue;
    }
    // h[q]: the state before position q
    float2 h[kQ + 1][2][kNS];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const float4 x = four(m.h0[turn] + (c0 + 2 * p) * NP + n0);
      const float4 z = four(m.h0[turn] + (c0 + 2 * p + 1) * NP + n0);
      h[0][p][0] = make_float2(x.x, z.x);
      h[0][p][1] = make_float2(x.y, z.y);
      h[0][p][2] = make_float2(x.z, z.z);
      h[0][p][3] = make_float2(x.w, z.w);
    }
#pragma unroll
    for (int q = 0; q < kQ; ++q) {
      const float4 du = four(m.du + q * CT + c0);
      twice(q, 0, bv);
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int i = 0; i < kNS; ++i)
          h[q + 1][p][i] =
              __ffma2_rn(dec[q][p][i], h[q][p][i], __fmul2_rn(p ? hi(du) : lo(du), bv[i]));
    }
    // the gradients
    float dbc[SumD::kLeft][kQ];
#pragma unroll
    for (int q = kQ - 1; q >= 0; --q) {
      const float4 dt = four(m.dt + q * CT + c0), du = four(m.du + q * CT + c0);
      const float4 gv = four(m.go + q * CT + c0);
      twice(q, 0, bv);
      twice(q, 1, cv);
      float2 db[kNS], dc[kNS], sb[2], sa[2];
#pragma unroll
      for (int i = 0; i < kNS; ++i) db[i] = dc[i] = both(0.f);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const float2 dtp = p ? hi(dt) : lo(dt), dup = p ? hi(du) : lo(du);
        const float2 gy = p ? hi(gv) : lo(gv);
        sb[p] = sa[p] = both(0.f);
#pragma unroll
        for (int i = 0; i < kNS; ++i) {
          const float2 gg = __ffma2_rn(cv[i], gy, r[p][i]);
          r[p][i] = __fmul2_rn(dec[q][p][i], gg);
          const float2 w = __fmul2_rn(r[p][i], h[q][p][i]);
          dc[i] = __ffma2_rn(gy, h[q + 1][p][i], dc[i]);
          db[i] = __ffma2_rn(gg, dup, db[i]);
          sb[p] = __ffma2_rn(gg, bv[i], sb[p]);
          sa[p] = __ffma2_rn(w, A[p][i], sa[p]);
          dA[p][i] = __ffma2_rn(w, dtp, dA[p][i]);
        }
      }
      // dB, dC: over the lanes across channels; lane ld ends with values ld * left ..
      float v[2 * kNS];
#pragma unroll
      for (int i = 0; i < kNS; ++i) {
        v[i] = db[i].x + db[i].y;
        v[kNS + i] = dc[i].x + dc[i].y;
      }
      SumD::sum(v, lane);
#pragma unroll
      for (int i = 0; i < SumD::kLeft; ++i) dbc[i][q] = v[i];
      // the sums over states: a channel's two values stay together
      float z[2 * kND];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        z[4 * p] = sb[p].x; z[4 * p + 1] = sa[p].x;
        z[4 * p + 2] = sb[p].y; z[4 * p + 3] = sa[p].y;
      }
      SumN::sum(z, lane);
      if (ln % kEach == 0) {
#pragma unroll
        for (int i = 0; i < kLeftN; ++i) {
          const int at = q * CT + c0 + ln / kEach * kLeftN + i;
          const float gy = m.go[at], uj = m.u[at];
          const float sbv = z[2 * i];
          const float dd = fmaf(uj, sbv, z[2 * i + 1] * unscaled<T>()) * m.slope[at];
          m.u[at] = m.dt[at] * sbv;
          m.slope[at] = dd;
          (i & 1 ? dskip[i / 2].y : dskip[i / 2].x) += gy * uj;
          (i & 1 ? dbias[i / 2].y : dbias[i / 2].x) += dd;
        }
      }
    }
    if (ld % kSame == 0) {
#pragma unroll
      for (int i = 0; i < kLeftD; ++i) {
        const int at = ld / kSame * kLeftD + i, n = n0 + at % kNS;
        if (n >= s.N) continue;
        float o[4];
#pragma unroll
        for (int q = 0; q < kQ; ++q) o[q] = t0 + q < end ? dbc[i][q] : 0.f;
        row_store4((at < kNS ? gB : gC) + n * s.L, t0, to, o, s.L % 4 == 0);
      }
    }
    __syncwarp();
#pragma unroll
    for (int p = 0; p < Mine::UI; ++p) {
      const int d = lane + p * 32;
      if (d >= chans) break;
      float o[4], w[4];
#pragma unroll
      for (int j = 0; j < kQ; ++j) {
        const bool inside = t0 + j < end;
        o[j] = inside ? fmaf(skip[p], m.go[j * CT + d], m.u[j * CT + d]) : 0.f;
        w[j] = inside ? m.slope[j * CT + d] : 0.f;
      }
      row_store4(gu + d * s.L, t0, to, o, a.vec);
      row_store4(gdelta + d * s.L, t0, to, w, a.vec);
    }
  }
  if (PRE) {
    if (warp != (pieces ? (pieces - 1) % kWarps : 0)) return;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < kNS; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int c = c0 + 2 * p + x;
          if (c >= chans || n0 + i >= s.N) continue;
          const int64_t at = split * nst + (row0 + c) * s.N + n0 + i;
          a.rend[at] = x ? r[p][i].y : r[p][i].x;
          a.prod[at] = x ? total[p][i].y : total[p][i].x;
        }
    return;
  }
  // padded positions behind the last piece
  const int64_t rest = from + (int64_t)pieces * kQ;
  if (rest < to) {
    for (int d = warp; d < chans; d += kWarps)
      for (int64_t t = rest + lane; t < to; t += 32) {
        stf(gu + d * s.L + t, 0.f);
        stf(gdelta + d * s.L + t, 0.f);
      }
    for (int n = warp; n < s.N; n += kWarps)
      for (int64_t t = rest + lane; t < to; t += 32) gB[n * s.L + t] = gC[n * s.L + t] = 0.f;
  }
  if (a.ginit && split == 0 && warp == (pieces ? (pieces - 1) % kWarps : 0)) {
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < kNS; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int c = c0 + 2 * p + x;
          if (c < chans && n0 + i < s.N)
            a.ginit[(row0 + c) * s.N + n0 + i] = x ? r[p][i].y : r[p][i].x;
        }
  }
  // sums over the warps
  __syncthreads();
  put(all.pass + warp * kND * 32, dA);
  all.total[warp * 32 + lane] = quad(dskip[0], dskip[1]);
  all.total[(kWarps + warp) * 32 + lane] = quad(dbias[0], dbias[1]);
  __syncthreads();
  float *pa = a.part_a + (split * s.B + b) * s.D * s.N;
  for (int i = threadIdx.x; i < CT * NP; i += kThreads) {
    const int d = i / NP, n = i % NP;
    if (d >= chans || n >= s.N) continue;
    // put's place of pair p, state n % 4, channel d % 2
    const int p = d % kND / 2, j = n % kNS, l = d / kND * LPC + n / kNS;
    float v = 0.f;
    for (int w = 0; w < kWarps; ++w)
      v += reinterpret_cast<const float *>(all.pass + (w * kND + 2 * p + j / 2) * 32 + l)[j % 2 * 2 + d % 2];
    pa[(d0 + d) * s.N + n] = v;
  }
  for (int d = threadIdx.x; d < chans; d += kThreads) {
    const int l = d / kND * LPC + d % kND / kLeftN * kEach, j = d % kND % kLeftN;
    float v = 0.f, w = 0.f;
    for (int k = 0; k < kWarps; ++k) {
      v += reinterpret_cast<const float *>(all.total + k * 32 + l)[j];
      w += reinterpret_cast<const float *>(all.total + (kWarps + k) * 32 + l)[j];
    }
    a.part_d[(split * s.B + b) * s.D + d0 + d] = v;
    a.part_d[((a.splits + split) * s.B + b) * s.D + d0 + d] = w;
  }
}

// dB and dC: the sum of the channel blocks' parts, in order
template <typename T>
__global__ void __launch_bounds__(256)
scan_sum_parts_kernel(const float *__restrict__ pb, const float *__restrict__ pc,
                      T *__restrict__ gb, T *__restrict__ gc, int64_t n, int64_t tiles) {
  const float *p = blockIdx.y ? pc : pb;
  T *out = blockIdx.y ? gc : gb;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    float v = 0.f;
    for (int64_t k = 0; k < tiles; ++k) v += p[k * n + i];
    stf(out + i, v);
  }
}

// dA, dskip, ddelta_bias: the sum over batch and chunks, in order
__global__ void __launch_bounds__(256)
scan_param_kernel(const float *__restrict__ pa, const float *__restrict__ pd, float *ga,
                  float *gskip, float *gbias, int64_t parts, int64_t D, int64_t N) {
  const int64_t i = blockIdx.x * 256ll + threadIdx.x;
  if (i < D * N) {
    float v = 0.f;
    for (int64_t b = 0; b < parts; ++b) v += pa[b * D * N + i];
    ga[i] = v;
  }
  if (i < D) {
    float v = 0.f, w = 0.f;
    for (int64_t b = 0; b < parts; ++b) {
      v += pd[b * D + i];
      w += pd[(parts + b) * D + i];
    }
    if (gskip) gskip[i] = v;
    if (gbias) gbias[i] = w;
  }
}

int64_t channel_tiles(int64_t D, int64_t N, int64_t G) {
  return cdiv(D / G, 32 / lanes_per_channel(N) * kND);
}

// as the forward's chunks, with one block to an SM
int bwd_splits(int64_t B, int64_t D, int64_t L, int64_t N, int64_t G, int64_t *chunk) {
  const int64_t blocks = B * G * channel_tiles(D, N, G), places = sm_count();
  const int64_t most = cdiv(L, kWarps * kQ);
  int64_t n = blocks * 2 <= places ? places / blocks : 1;
  if (n > most) n = most;
  *chunk = cdiv(cdiv(L, n), kQ) * kQ;
  return (int)cdiv(L, *chunk);
}

struct Sizes {
  int64_t chunk, splits, bc, a, d, st;  // floats: each of part_b, part_c; part_a; part_d; rend, prod
  size_t bytes() const { return (size_t)(2 * bc + a + d + 2 * st) * sizeof(float); }
};
Sizes bwd_sizes(int64_t B, int64_t D, int64_t L, int64_t N, int64_t G) {
  Sizes z;
  z.splits = bwd_splits(B, D, L, N, G, &z.chunk);
  z.bc = cdiv(channel_tiles(D, N, G) * B * G * N * L, 4) * 4;
  z.a = z.splits * B * D * N;
  z.d = 2 * z.splits * B * D;
  z.st = z.splits > 1 ? z.splits * B * D * N : 0;
  return z;
}

struct Outs {
  void *gB, *gC;
  float *gA, *gskip, *gbias;
};

template <typename T, int LPC>
int bwd_launch(const Bwd &a, const Outs &o, const Shape &s, cudaStream_t st) {
  const int smem = (int)sizeof(BwdSmem<LPC>);
  auto main = scan_bwd_kernel<T, LPC, false>, pre = scan_bwd_kernel<T, LPC, true>;
  const int64_t tiles = channel_tiles(s.D, s.N, s.G);
  const unsigned blocks = (unsigned)(s.B * s.G * tiles * a.splits);
  if (a.splits > 1) {
    if (set_smem_once((const void *)pre, smem) != cudaSuccess)
      return check_launch("scan_bwd_kernel shared memory");
    pre<<<blocks, kThreads, smem, st>>>(a, s);
    if (int rc = check_launch("scan_bwd_kernel (chunk ends)")) return rc;
  }
  if (set_smem_once((const void *)main, smem) != cudaSuccess)
    return check_launch("scan_bwd_kernel shared memory");
  main<<<blocks, kThreads, smem, st>>>(a, s);
  if (int rc = check_launch("scan_bwd_kernel")) return rc;
  const int64_t n = s.B * s.G * s.N * s.L, cap = 8 * (int64_t)sm_count();
  const dim3 grid((unsigned)(cdiv(n, 256) < cap ? cdiv(n, 256) : cap), 2);
  scan_sum_parts_kernel<T><<<grid, 256, 0, st>>>(a.part_b, a.part_c, (T *)o.gB, (T *)o.gC, n,
                                                  tiles);
  if (int rc = check_launch("scan_sum_parts_kernel")) return rc;
  scan_param_kernel<<<(unsigned)cdiv(s.D * s.N, 256), 256, 0, st>>>(
      a.part_a, a.part_d, o.gA, o.gskip, o.gbias, s.B * a.splits, s.D, s.N);
  return check_launch("scan_param_kernel");
}

}  // namespace
}  // namespace scan
}  // namespace dudy

extern "C" {

size_t dudy_selective_scan_backward_workspace_size(int64_t B, int64_t D, int64_t L, int64_t N,
                                                   int64_t G, int dtype) {
  using namespace dudy;
  if (scan::validate(B, D, L, N, G, dtype)) return 0;
  return (scan::bwd_sizes(B, D, L, N, G).bytes() + 255) & ~size_t(255);
}

int dudy_selective_scan_backward(const void *go, const float *grad_final, const void *u,
                                 const void *delta, const float *A, const void *Bm,
                                 const void *Cm, const float *skip, const float *delta_bias,
                                 const float *checkpoints, const int32_t *lengths, void *grad_u,
                                 void *grad_delta, float *grad_A, void *grad_B, void *grad_C,
                                 float *grad_skip, float *grad_delta_bias, float *grad_state,
                                 void *workspace, size_t workspace_bytes, int64_t B, int64_t D,
                                 int64_t L, int64_t N, int64_t G, int softplus, int dtype,
                                 void *stream) {
  using namespace dudy;
  clear_error();
  if (int rc = scan::validate(B, D, L, N, G, dtype)) return rc;
  if (!go || !u || !delta || !A || !Bm || !Cm || !checkpoints || !grad_u || !grad_delta ||
      !grad_A || !grad_B || !grad_C)
    return refuse("null tensor pointer");
  if (int rc = require_workspace(workspace, workspace_bytes,
                                 dudy_selective_scan_backward_workspace_size(B, D, L, N, G, dtype)))
    return rc;
  if (int rc = require_sm100()) return rc;
  const scan::Sizes z = scan::bwd_sizes(B, D, L, N, G);
  float *pb = (float *)workspace, *pa = pb + 2 * z.bc, *pd = pa + z.a, *rend = pd + z.d;
  const int vec = L % 4 == 0 && aligned_to_16(u) && aligned_to_16(delta) && aligned_to_16(go) &&
                  aligned_to_16(Bm) && aligned_to_16(Cm) && aligned_to_16(grad_u) &&
                  aligned_to_16(grad_delta);
  const scan::Bwd a{go, u, delta, Bm, Cm, grad_final, A, skip, delta_bias, checkpoints, lengths,
                    grad_u, grad_delta, grad_state, pb, pb + z.bc, pa, pd, rend, rend + z.st,
                    z.chunk, (int)z.splits, vec};
  const scan::Outs o{grad_B, grad_C, grad_A, grad_skip, grad_delta_bias};
  const scan::Shape s{B, D, L, (int)N, (int)G, softplus};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return scan::by_type_and_lanes(dtype, N, [&](auto t, auto lanes) {
    return scan::bwd_launch<decltype(t), decltype(lanes)::value>(a, o, s, st);
  });
}

}  // extern "C"
