// scan_bwd.cu -- the selective scan's gradients.
//
// With a = exp(dt A) and g[t] = dL/dh[t]:  g[t] = C[t] dy[t] + a[t+1] g[t+1]   (from the right)
//   dC[n,t] = sum_d h dy                 dB[n,t] = sum_d g dt u        (channels of the group)
//   dA[d,n] = sum_{b,t} dt g a h[t-1]    ddt = u sum_n g B + sum_n A g a h[t-1]
//   du = dt sum_n g B + skip dy          ddelta = ddt softplus'        dskip = sum_{b,t} dy u
// Superchunks go from the right end of a sequence to its left. Within one, each warp runs its
// four positions forwards and backwards from zero, the end states of both directions are
// exchanged together, and it runs both again: forwards keeping the states, backwards forming
// the gradients. The state that enters a superchunk was saved by the forward.
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
constexpr int kQ = 4;                  // positions of a warp in a superchunk
constexpr int kTS = kWarps * kQ;       // positions of a superchunk
constexpr int kOP = kTS + 4;
static_assert(kTS == kCkpt, "a state is saved at each superchunk's start");

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
  int64_t chunk;           // positions of a chunk, a multiple of kTS
  int splits, vec;
};

template <typename T, int LPC>
struct BwdTile {
  static constexpr int CT = 32 / LPC * kND;      // channels of a block
  static constexpr int NP = kNS * LPC;
  static constexpr int PITCH = kTS + 16 / (int)sizeof(T);
  T raw_u[CT * PITCH], raw_d[CT * PITCH], raw_g[CT * PITCH];
  T raw_b[NP * PITCH], raw_c[NP * PITCH];
  float dt[kTS * CT], du[kTS * CT], go[kTS * CT];
  float u[kTS * CT], slope[kTS * CT];            // du's and ddelta's results take their places
  float2 b[kTS * NP], c[kTS * NP];               // each twice side by side
  float gb[NP * kOP], gc[NP * kOP];
  float h0[2][CT * NP];                          // the states saved at the superchunk's start
  // exchanged states, [warp][four of the thread's states][lane]: forward end, decay product and
  // backward end; the sums over warps at the end use the same room
  float4 end[kWarps * kND * 32], prod[kWarps * kND * 32], rend[kWarps * kND * 32];
  float4 rcarry[2 * kND * 32];
};

// A thread's states lie in pairs of channels: e[p][n] holds channels 2p and 2p + 1 of state n,
// so that a position's dt, dt u and gradient of two channels are operands as they are read.
template <typename T, int LPC, bool PRE>
__global__ void __launch_bounds__(kThreads, 1)
scan_bwd_kernel(Bwd a, Shape s) {
  using Tile = BwdTile<T, LPC>;
  constexpr int CT = Tile::CT, NP = Tile::NP, PITCH = Tile::PITCH;
  extern __shared__ __align__(16) char smem_raw[];
  Tile &m = *reinterpret_cast<Tile *>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ln = lane % LPC, ld = lane / LPC, n0 = ln * kNS, c0 = ld * kND;

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
  float *pb = a.part_b + tile * nbc + bg * s.N * s.L;
  float *pc = a.part_c + tile * nbc + bg * s.N * s.L;

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
        if (!PRE && ok) {
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
  // v = prod v + add over what a warp put
  auto fold = [&](float2 (&v)[2][kNS], const float4 *add, const float4 *prod) {
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 x = prod[(2 * p + i) * 32 + lane], e = add[(2 * p + i) * 32 + lane];
        v[p][2 * i] = __ffma2_rn(lo(x), v[p][2 * i], lo(e));
        v[p][2 * i + 1] = __ffma2_rn(hi(x), v[p][2 * i + 1], hi(e));
        if (PRE) {
          total[p][2 * i] = __fmul2_rn(total[p][2 * i], lo(x));
          total[p][2 * i + 1] = __fmul2_rn(total[p][2 * i + 1], hi(x));
        }
      }
  };
  if (warp == 0) put(m.rcarry, r);

  auto stage = [&](int64_t t0, int turn) {
    stage_rows<T, kTS, PITCH>(m.raw_d, delta, CT, chans, s.L, t0, end, a.vec);
    stage_rows<T, kTS, PITCH>(m.raw_g, go, CT, chans, s.L, t0, end, a.vec);
    stage_rows<T, kTS, PITCH>(m.raw_c, Cm, NP, s.N, s.L, t0, end, a.vec);
    if (PRE) return;
    stage_rows<T, kTS, PITCH>(m.raw_u, u, CT, chans, s.L, t0, end, a.vec);
    stage_rows<T, kTS, PITCH>(m.raw_b, Bm, NP, s.N, s.L, t0, end, a.vec);
    stage_states<NP>(m.h0[turn], a.ckpt + ((b * s.ckpts() + t0 / kCkpt) * s.D + d0) * s.N, CT,
                     chans, s.N);
  };
  const int supers = end > from ? (int)((end - from + kTS - 1) / kTS) : 0;
  if (supers) stage(from + (int64_t)(supers - 1) * kTS, 0);
  int turn = 0;
  for (int k = supers - 1; k >= 0; --k, turn ^= 1) {
    const int64_t t0 = from + (int64_t)k * kTS;
    cp_async_wait_all();
    __syncthreads();
    for (int i = threadIdx.x; i < CT * (kTS / 4); i += kThreads) {
      const int d = i % CT, c = i / CT * 4;
      const T *ru = m.raw_u + d * PITCH + c, *rd = m.raw_d + d * PITCH + c;
      const T *rg = m.raw_g + d * PITCH + c;
      const float bias = d < chans && a.delta_bias ? a.delta_bias[d0 + d] : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float dt = Elem<T>::to_f(rd[j]) + bias, slope = 1.f;
        if (s.softplus) dt = softplus<T>(dt, slope);
        if (t0 + c + j >= end) dt = slope = 0.f;
        const int at = (c + j) * CT + d;
        m.dt[at] = dt;
        m.go[at] = Elem<T>::to_f(rg[j]);
        if (PRE) continue;
        const float uv = Elem<T>::to_f(ru[j]);
        m.du[at] = dt * uv;
        m.u[at] = uv;
        m.slope[at] = slope;
      }
    }
    for (int i = threadIdx.x; i < NP * (kTS / 4); i += kThreads) {
      const int n = i % NP, c = i / NP * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m.c[(c + j) * NP + n] = both(Elem<T>::to_f(m.raw_c[n * PITCH + c + j]));
        if (!PRE) m.b[(c + j) * NP + n] = both(Elem<T>::to_f(m.raw_b[n * PITCH + c + j]));
      }
    }
    __syncthreads();
    if (k > 0) stage(t0 - kTS, turn ^ 1);

    // both directions from zero
    const float *sdt = m.dt + warp * kQ * CT + c0, *sdu = m.du + warp * kQ * CT + c0;
    const float *sgo = m.go + warp * kQ * CT + c0;
    const float2 *sb2 = m.b + warp * kQ * NP + n0, *sc2 = m.c + warp * kQ * NP + n0;
    auto four = [](const float *p) { return *reinterpret_cast<const float4 *>(p); };
    auto pairs = [](const float2 *p, float2 (&v)[kNS]) {
      const float4 x = reinterpret_cast<const float4 *>(p)[0];
      const float4 z = reinterpret_cast<const float4 *>(p)[1];
      v[0] = lo(x); v[1] = hi(x); v[2] = lo(z); v[3] = hi(z);
    };
    float2 dec[kQ][2][kNS], h[kQ][2][kNS], bv[kNS], cv[kNS];
    {
      float2 sum[2], loc[2][kNS];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        sum[p] = both(0.f);
#pragma unroll
        for (int i = 0; i < kNS; ++i) loc[p][i] = both(0.f);
      }
#pragma unroll
      for (int q = 0; q < kQ; ++q) {
        const float4 dt = four(sdt + q * CT);
        float4 du;
        if (!PRE) {
          du = four(sdu + q * CT);
          pairs(sb2 + q * NP, bv);
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const float2 dtp = p ? hi(dt) : lo(dt), dup = p ? hi(du) : lo(du);
          sum[p] = __fadd2_rn(sum[p], dtp);
#pragma unroll
          for (int i = 0; i < kNS; ++i) {
            const float2 x = __fmul2_rn(dtp, A[p][i]);
            dec[q][p][i] = make_float2(decay<T>(x.x), decay<T>(x.y));
            if (!PRE) loc[p][i] = __ffma2_rn(dec[q][p][i], loc[p][i], __fmul2_rn(dup, bv[i]));
          }
        }
      }
      if (!PRE) put(m.end + warp * kND * 32, loc);
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int i = 0; i < kNS; ++i) {
          const float2 x = __fmul2_rn(sum[p], A[p][i]);
          loc[p][i] = make_float2(decay<T>(x.x), decay<T>(x.y));
        }
      put(m.prod + warp * kND * 32, loc);
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int i = 0; i < kNS; ++i) loc[p][i] = both(0.f);
#pragma unroll
      for (int q = kQ - 1; q >= 0; --q) {
        const float4 gv = four(sgo + q * CT);
        pairs(sc2 + q * NP, cv);
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int i = 0; i < kNS; ++i)
            loc[p][i] = __fmul2_rn(dec[q][p][i], __ffma2_rn(cv[i], p ? hi(gv) : lo(gv), loc[p][i]));
      }
      put(m.rend + warp * kND * 32, loc);
    }
    __syncthreads();
    // what enters this warp's positions from the right, and from the left
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const float4 x = m.rcarry[(turn * kND + 2 * p) * 32 + lane];
      const float4 z = m.rcarry[(turn * kND + 2 * p + 1) * 32 + lane];
      r[p][0] = lo(x); r[p][1] = hi(x); r[p][2] = lo(z); r[p][3] = hi(z);
    }
    for (int w = kWarps - 1; w > (PRE ? (warp ? kWarps : -1) : warp); --w)
      fold(r, m.rend + w * kND * 32, m.prod + w * kND * 32);
    if (PRE) {
      if (warp == 0) put(m.rcarry + (turn ^ 1) * kND * 32, r);
      continue;
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const float4 x = *reinterpret_cast<const float4 *>(m.h0[turn] + (c0 + 2 * p) * NP + n0);
      const float4 z = *reinterpret_cast<const float4 *>(m.h0[turn] + (c0 + 2 * p + 1) * NP + n0);
      h[0][p][0] = make_float2(x.x, z.x);
      h[0][p][1] = make_float2(x.y, z.y);
      h[0][p][2] = make_float2(x.z, z.z);
      h[0][p][3] = make_float2(x.w, z.w);
    }
    for (int w = 0; w < warp; ++w) fold(h[0], m.end + w * kND * 32, m.prod + w * kND * 32);
    // forwards: h[q] is the state before position q
#pragma unroll
    for (int q = 0; q + 1 < kQ; ++q) {
      const float4 du = four(sdu + q * CT);
      pairs(sb2 + q * NP, bv);
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int i = 0; i < kNS; ++i)
          h[q + 1][p][i] =
              __ffma2_rn(dec[q][p][i], h[q][p][i], __fmul2_rn(p ? hi(du) : lo(du), bv[i]));
    }
    // backwards
#pragma unroll
    for (int q = kQ - 1; q >= 0; --q) {
      const int t = warp * kQ + q;
      const float4 dt = four(sdt + q * CT), du = four(sdu + q * CT), gv = four(sgo + q * CT);
      pairs(sb2 + q * NP, bv);
      pairs(sc2 + q * NP, cv);
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
          const float2 ah = __fmul2_rn(dec[q][p][i], h[q][p][i]);
          const float2 w = __fmul2_rn(gg, ah);
          dc[i] = __ffma2_rn(gy, __ffma2_rn(dup, bv[i], ah), dc[i]);
          db[i] = __ffma2_rn(gg, dup, db[i]);
          sb[p] = __ffma2_rn(gg, bv[i], sb[p]);
          sa[p] = __ffma2_rn(w, A[p][i], sa[p]);
          dA[p][i] = __ffma2_rn(w, dtp, dA[p][i]);
          r[p][i] = __fmul2_rn(dec[q][p][i], gg);
        }
      }
      // dB, dC: over the lanes across channels; lane ld ends with values ld * left ..
      float v[2 * kNS];
#pragma unroll
      for (int i = 0; i < kNS; ++i) {
        v[i] = db[i].x + db[i].y;
        v[kNS + i] = dc[i].x + dc[i].y;
      }
      using SumD = Scatter<LPC, 32 / LPC, 2 * kNS>;
      SumD::sum(v, lane);
      constexpr int kLeftD = SumD::kLeft, kGroups = 2 * kNS / kLeftD;
      constexpr int kSame = 32 / LPC / kGroups;  // lanes that hold the same values
      if (ld % kSame == 0) {
#pragma unroll
        for (int i = 0; i < kLeftD; ++i) {
          const int at = ld / kSame * kLeftD + i;
          (at < kNS ? m.gb : m.gc)[(n0 + at % kNS) * kOP + t] = v[i];
        }
      }
      // the sums over states: a channel's two values stay together
      float z[2 * kND];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        z[4 * p] = sb[p].x; z[4 * p + 1] = sa[p].x;
        z[4 * p + 2] = sb[p].y; z[4 * p + 3] = sa[p].y;
      }
      using SumN = Scatter<1, LPC, 2 * kND, 2>;
      SumN::sum(z, lane);
      constexpr int kLeftN = SumN::kLeft / 2, kOwners = kND / kLeftN, kEach = LPC / kOwners;
      if (ln % kEach == 0) {
#pragma unroll
        for (int i = 0; i < kLeftN; ++i) {
          const int c = c0 + ln / kEach * kLeftN + i, at = t * CT + c;
          const float gy = m.go[at], uj = m.u[at];
          const float sbv = z[2 * i], dd = fmaf(uj, sbv, z[2 * i + 1] * unscaled<T>()) * m.slope[at];
          m.u[at] = m.dt[at] * sbv;
          m.slope[at] = dd;
          (i & 1 ? dskip[i / 2].y : dskip[i / 2].x) += gy * uj;
          (i & 1 ? dbias[i / 2].y : dbias[i / 2].x) += dd;
        }
      }
    }
    if (warp == 0) put(m.rcarry + (turn ^ 1) * kND * 32, r);
    __syncthreads();
    // the superchunk's results
    for (int i = threadIdx.x; i < 2 * CT * (kTS / 8); i += kThreads) {
      const int x = i / CT, d = i % CT, c = x / 2 * 8;
      if (d >= chans) continue;
      const int64_t t = t0 + c;
      const float *src = (x & 1 ? m.slope : m.u) + c * CT + d;
      const float skip = !(x & 1) && a.skip ? a.skip[d0 + d] : 0.f;
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        o[j] = src[j * CT];
        if (!(x & 1)) o[j] = fmaf(skip, m.go[(c + j) * CT + d], o[j]);
        if (t + j >= end) o[j] = 0.f;
      }
      T *row = (x & 1 ? gdelta : gu) + d * s.L;
      if (a.vec) row_store8_until<T, true>(row, t, to, o);
      else row_store8_until<T, false>(row, t, to, o);
    }
    for (int i = threadIdx.x; i < 2 * s.N * (kTS / 8); i += kThreads) {
      const int x = i / (kTS / 8), n = x >> 1, c = i % (kTS / 8) * 8;
      const int64_t t = t0 + c;
      const float *src = (x & 1 ? m.gc : m.gb) + n * kOP + c;
      alignas(16) float o[8];
      *reinterpret_cast<float4 *>(o) = *reinterpret_cast<const float4 *>(src);
      *reinterpret_cast<float4 *>(o + 4) = *reinterpret_cast<const float4 *>(src + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (t + j >= end) o[j] = 0.f;
      float *row = (x & 1 ? pc : pb) + n * s.L;
      if (s.L % 8 == 0) row_store8_until<float, true>(row, t, to, o);
      else row_store8_until<float, false>(row, t, to, o);
    }
  }
  if (PRE) {
    if (warp) return;
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
  // padded positions behind the last superchunk
  const int64_t rest = from + (int64_t)supers * kTS;
  if (rest < to) {
    for (int d = warp; d < chans; d += kWarps)
      for (int64_t t = rest + lane; t < to; t += 32) {
        stf(gu + d * s.L + t, 0.f);
        stf(gdelta + d * s.L + t, 0.f);
      }
    for (int n = warp; n < s.N; n += kWarps)
      for (int64_t t = rest + lane; t < to; t += 32) pb[n * s.L + t] = pc[n * s.L + t] = 0.f;
  }
  if (a.ginit && split == 0 && warp == 0) {
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
  put(m.end + warp * kND * 32, dA);
  m.prod[warp * 32 + lane] = quad(dskip[0], dskip[1]);
  m.rend[warp * 32 + lane] = quad(dbias[0], dbias[1]);
  __syncthreads();
  float *pa = a.part_a + (split * s.B + b) * s.D * s.N;
  for (int i = threadIdx.x; i < CT * NP; i += kThreads) {
    const int d = i / NP, n = i % NP;
    if (d >= chans || n >= s.N) continue;
    // put's place of pair p, state n % 4, channel d % 2
    const int p = d % kND / 2, j = n % kNS, l = d / kND * LPC + n / kNS;
    float v = 0.f;
    for (int w = 0; w < kWarps; ++w)
      v += reinterpret_cast<const float *>(m.end + (w * kND + 2 * p + j / 2) * 32 + l)[j % 2 * 2 + d % 2];
    pa[(d0 + d) * s.N + n] = v;
  }
  using SumN = Scatter<1, LPC, 2 * kND, 2>;
  constexpr int kLeftN = SumN::kLeft / 2, kOwners = kND / kLeftN, kEach = LPC / kOwners;
  for (int d = threadIdx.x; d < chans; d += kThreads) {
    const int l = d / kND * LPC + d % kND / kLeftN * kEach, j = d % kND % kLeftN;
    float v = 0.f, w = 0.f;
    for (int k = 0; k < kWarps; ++k) {
      v += reinterpret_cast<const float *>(m.prod + k * 32 + l)[j];
      w += reinterpret_cast<const float *>(m.rend + k * 32 + l)[j];
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
  const int64_t supers = cdiv(L, kTS);
  int64_t n = blocks * 2 <= places ? places / blocks : 1;
  if (n > supers) n = supers;
  *chunk = cdiv(supers, n) * kTS;
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
  const int smem = (int)sizeof(BwdTile<T, LPC>);
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
  const int vec = L % 8 == 0 && aligned_to_16(u) && aligned_to_16(delta) && aligned_to_16(go) &&
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
