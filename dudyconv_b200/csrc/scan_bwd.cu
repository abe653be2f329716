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
// the batch.
#include "scan.cuh"

namespace dudy {
namespace scan {
namespace {

constexpr int kND = 4;                 // channels of a thread
constexpr int kQ = 4;                  // positions of a warp in a superchunk
constexpr int kTS = kWarps * kQ;       // positions of a superchunk
static_assert(kTS == kCkpt, "a state is saved at each superchunk's start");
constexpr int kST = kND * kNS;         // states of a thread

struct Bwd {
  const void *go, *u, *delta, *Bm, *Cm;
  const float *gfinal, *A, *skip, *delta_bias, *ckpt;
  const int32_t *lengths;
  void *gu, *gdelta;
  float *ginit;
  float *part_b, *part_c;  // [tiles][B*G*N*L]
  float *part_a;           // [B][D*N]
  float *part_d;           // [2][B][D]: skip, delta_bias
  int vec;
};

template <typename T, int LPC>
struct BwdSmem {
  static constexpr int CT = 32 / LPC * kND;      // channels of a block
  static constexpr int NP = kNS * LPC;
  static constexpr int PITCH = kTS + 16 / (int)sizeof(T);
  T raw_u[CT * PITCH], raw_d[CT * PITCH], raw_g[CT * PITCH];
  T raw_b[NP * PITCH], raw_c[NP * PITCH];
  float dt[kTS * CT], u[kTS * CT], go[kTS * CT], slope[kTS * CT];
  float b[kTS * NP], c[kTS * NP];
  float gu[CT * (kTS + 1)], gd[CT * (kTS + 1)];
  float gb[NP * (kTS + 1)], gc[NP * (kTS + 1)];
  // exchanged states, [warp][channel of the thread][lane]: forward end, decay product, and the
  // backward end; the sums over warps at the end use the same room
  float4 end[kWarps * kND * 32], prod[kWarps * kND * 32], rend[kWarps * kND * 32];
  float4 rcarry[2 * kND * 32];
};

template <typename T, int LPC>
__global__ void __launch_bounds__(kThreads, 1)
scan_bwd_kernel(Bwd a, Shape s) {
  using Smem = BwdSmem<T, LPC>;
  constexpr int CT = Smem::CT, NP = Smem::NP, PITCH = Smem::PITCH, OP = kTS + 1;
  extern __shared__ __align__(16) char smem_raw[];
  Smem &m = *reinterpret_cast<Smem *>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ln = lane % LPC, ld = lane / LPC, n0 = ln * kNS, c0 = ld * kND;

  const int64_t R = s.D / s.G, tiles = (R + CT - 1) / CT;
  const int64_t tile = blockIdx.x % tiles, bg = blockIdx.x / tiles;
  const int64_t b = bg / s.G, g = bg % s.G;
  const int chans = (int)(R - tile * CT < CT ? R - tile * CT : CT);
  const int64_t d0 = g * R + tile * CT, row0 = b * s.D + d0;
  const int64_t len = clamp_len(a.lengths, b, s.L);
  const T *u = (const T *)a.u + row0 * s.L, *delta = (const T *)a.delta + row0 * s.L;
  const T *go = (const T *)a.go + row0 * s.L;
  const T *Bm = (const T *)a.Bm + bg * s.N * s.L, *Cm = (const T *)a.Cm + bg * s.N * s.L;
  T *gu = (T *)a.gu + row0 * s.L, *gdelta = (T *)a.gdelta + row0 * s.L;
  const int64_t nbc = s.B * s.G * s.N * s.L;
  float *pb = a.part_b + tile * nbc + bg * s.N * s.L;
  float *pc = a.part_c + tile * nbc + bg * s.N * s.L;

  float A[kST], dA[kST], r[kST], skip[kND], dskip[kND], dbias[kND];
#pragma unroll
  for (int j = 0; j < kND; ++j) {
    const bool mine = c0 + j < chans;
    skip[j] = mine && a.skip ? a.skip[d0 + c0 + j] : 0.f;
    dskip[j] = dbias[j] = 0.f;
#pragma unroll
    for (int i = 0; i < kNS; ++i) {
      const bool ok = mine && n0 + i < s.N;
      A[j * kNS + i] = ok ? a.A[(d0 + c0 + j) * s.N + n0 + i] : 0.f;
      r[j * kNS + i] = ok && a.gfinal ? a.gfinal[(row0 + c0 + j) * s.N + n0 + i] : 0.f;
      dA[j * kNS + i] = 0.f;
    }
  }
  auto put = [&](float4 *to, const float *v) {
#pragma unroll
    for (int j = 0; j < kND; ++j)
      to[j * 32 + lane] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  };
  if (warp == 0) put(m.rcarry, r);

  auto stage = [&](int64_t t0) {
    stage_rows<T, kTS, PITCH>(m.raw_u, u, CT, chans, s.L, t0, len, a.vec);
    stage_rows<T, kTS, PITCH>(m.raw_d, delta, CT, chans, s.L, t0, len, a.vec);
    stage_rows<T, kTS, PITCH>(m.raw_g, go, CT, chans, s.L, t0, len, a.vec);
    stage_rows<T, kTS, PITCH>(m.raw_b, Bm, NP, s.N, s.L, t0, len, a.vec);
    stage_rows<T, kTS, PITCH>(m.raw_c, Cm, NP, s.N, s.L, t0, len, a.vec);
  };
  const int supers = (int)((len + kTS - 1) / kTS);
  if (supers) stage((int64_t)(supers - 1) * kTS);
  int parity = 0;
  for (int k = supers - 1; k >= 0; --k, parity ^= 1) {
    const int64_t t0 = (int64_t)k * kTS;
    float hin[kST];
#pragma unroll
    for (int i = 0; i < kST; ++i) {
      const int j = i / kNS, n = n0 + i % kNS;
      hin[i] = c0 + j < chans && n < s.N
                   ? a.ckpt[((row0 + c0 + j) * s.ckpts() + k) * s.N + n] : 0.f;
    }
    cp_async_wait_all();
    __syncthreads();
    for (int i = threadIdx.x; i < CT * (kTS / 8); i += kThreads) {
      const int d = i % CT, c = i / CT * 8;
      float uv[8], dv[8], gv[8];
      row_load8(m.raw_u + d * PITCH + c, uv);
      row_load8(m.raw_d + d * PITCH + c, dv);
      row_load8(m.raw_g + d * PITCH + c, gv);
      const float bias = d < chans && a.delta_bias ? a.delta_bias[d0 + d] : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float dt = dv[j] + bias, slope = 1.f;
        if (s.softplus) dt = softplus<T>(dt, slope);
        if (t0 + c + j >= len) dt = slope = 0.f;
        const int at = (c + j) * CT + d;
        m.dt[at] = dt;
        m.u[at] = uv[j];
        m.go[at] = gv[j];
        m.slope[at] = slope;
      }
    }
    for (int i = threadIdx.x; i < NP * (kTS / 8); i += kThreads) {
      const int n = i % NP, c = i / NP * 8;
      float bv[8], cv[8];
      row_load8(m.raw_b + n * PITCH + c, bv);
      row_load8(m.raw_c + n * PITCH + c, cv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        m.b[(c + j) * NP + n] = bv[j];
        m.c[(c + j) * NP + n] = cv[j];
      }
    }
    __syncthreads();
    if (k > 0) stage(t0 - kTS);

    // both directions from zero
    float dec[kQ][kST], h[kQ][kST], loc[kST];
    {
      float sum[kND];
#pragma unroll
      for (int i = 0; i < kST; ++i) loc[i] = 0.f;
#pragma unroll
      for (int j = 0; j < kND; ++j) sum[j] = 0.f;
#pragma unroll
      for (int q = 0; q < kQ; ++q) {
        const int t = warp * kQ + q;
        const float4 dt = *reinterpret_cast<const float4 *>(m.dt + t * CT + c0);
        const float4 uv = *reinterpret_cast<const float4 *>(m.u + t * CT + c0);
        const float4 bv = *reinterpret_cast<const float4 *>(m.b + t * NP + n0);
#pragma unroll
        for (int j = 0; j < kND; ++j) {
          const float dtj = (&dt.x)[j], du = dtj * (&uv.x)[j];
          sum[j] += dtj;
#pragma unroll
          for (int i = 0; i < kNS; ++i) {
            const int e = j * kNS + i;
            dec[q][e] = decay<T>(dtj * A[e]);
            loc[e] = fmaf(dec[q][e], loc[e], du * (&bv.x)[i]);
          }
        }
      }
      put(m.end + warp * kND * 32, loc);
#pragma unroll
      for (int e = 0; e < kST; ++e) loc[e] = decay<T>(sum[e / kNS] * A[e]);
      put(m.prod + warp * kND * 32, loc);
#pragma unroll
      for (int e = 0; e < kST; ++e) loc[e] = 0.f;
#pragma unroll
      for (int q = kQ - 1; q >= 0; --q) {
        const int t = warp * kQ + q;
        const float4 gv = *reinterpret_cast<const float4 *>(m.go + t * CT + c0);
        const float4 cv = *reinterpret_cast<const float4 *>(m.c + t * NP + n0);
#pragma unroll
        for (int e = 0; e < kST; ++e)
          loc[e] = dec[q][e] * fmaf((&cv.x)[e % kNS], (&gv.x)[e / kNS], loc[e]);
      }
      put(m.rend + warp * kND * 32, loc);
    }
    __syncthreads();
    // what enters this warp's positions from the left and from the right
    for (int w = 0; w < warp; ++w)
#pragma unroll
      for (int j = 0; j < kND; ++j) {
        const float4 p = m.prod[(w * kND + j) * 32 + lane], e = m.end[(w * kND + j) * 32 + lane];
#pragma unroll
        for (int i = 0; i < kNS; ++i)
          hin[j * kNS + i] = fmaf((&p.x)[i], hin[j * kNS + i], (&e.x)[i]);
      }
#pragma unroll
    for (int j = 0; j < kND; ++j) {
      const float4 c = m.rcarry[(parity * kND + j) * 32 + lane];
#pragma unroll
      for (int i = 0; i < kNS; ++i) r[j * kNS + i] = (&c.x)[i];
    }
    for (int w = kWarps - 1; w > warp; --w)
#pragma unroll
      for (int j = 0; j < kND; ++j) {
        const float4 p = m.prod[(w * kND + j) * 32 + lane], e = m.rend[(w * kND + j) * 32 + lane];
#pragma unroll
        for (int i = 0; i < kNS; ++i)
          r[j * kNS + i] = fmaf((&p.x)[i], r[j * kNS + i], (&e.x)[i]);
      }
    // forwards: h[q] is the state before position q
#pragma unroll
    for (int e = 0; e < kST; ++e) h[0][e] = hin[e];
#pragma unroll
    for (int q = 0; q + 1 < kQ; ++q) {
      const int t = warp * kQ + q;
      const float4 dt = *reinterpret_cast<const float4 *>(m.dt + t * CT + c0);
      const float4 uv = *reinterpret_cast<const float4 *>(m.u + t * CT + c0);
      const float4 bv = *reinterpret_cast<const float4 *>(m.b + t * NP + n0);
#pragma unroll
      for (int e = 0; e < kST; ++e) {
        const int j = e / kNS;
        h[q + 1][e] = fmaf(dec[q][e], h[q][e], (&dt.x)[j] * (&uv.x)[j] * (&bv.x)[e % kNS]);
      }
    }
    // backwards
#pragma unroll
    for (int q = kQ - 1; q >= 0; --q) {
      const int t = warp * kQ + q;
      const float4 dt = *reinterpret_cast<const float4 *>(m.dt + t * CT + c0);
      const float4 uv = *reinterpret_cast<const float4 *>(m.u + t * CT + c0);
      const float4 gv = *reinterpret_cast<const float4 *>(m.go + t * CT + c0);
      const float4 bv = *reinterpret_cast<const float4 *>(m.b + t * NP + n0);
      const float4 cv = *reinterpret_cast<const float4 *>(m.c + t * NP + n0);
      float db[kNS], dc[kNS], sb[kND], sa[kND];
#pragma unroll
      for (int i = 0; i < kNS; ++i) db[i] = dc[i] = 0.f;
#pragma unroll
      for (int j = 0; j < kND; ++j) {
        const float dtj = (&dt.x)[j], du = dtj * (&uv.x)[j], gy = (&gv.x)[j];
        sb[j] = sa[j] = 0.f;
#pragma unroll
        for (int i = 0; i < kNS; ++i) {
          const int e = j * kNS + i;
          const float gg = fmaf((&cv.x)[i], gy, r[e]);
          const float ah = dec[q][e] * h[q][e];
          const float ht = fmaf(du, (&bv.x)[i], ah);
          const float w = gg * ah;
          dc[i] = fmaf(gy, ht, dc[i]);
          db[i] = fmaf(gg, du, db[i]);
          sb[j] = fmaf(gg, (&bv.x)[i], sb[j]);
          sa[j] = fmaf(w, A[e], sa[j]);
          dA[e] = fmaf(w, dtj, dA[e]);
          r[e] = dec[q][e] * gg;
        }
      }
#pragma unroll
      for (int o = 16; o >= LPC; o >>= 1)
#pragma unroll
        for (int i = 0; i < kNS; ++i) {
          db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
          dc[i] += __shfl_xor_sync(0xffffffffu, dc[i], o);
        }
      if (ld == 0) {
#pragma unroll
        for (int i = 0; i < kNS; ++i) {
          m.gb[(n0 + i) * OP + t] = db[i];
          m.gc[(n0 + i) * OP + t] = dc[i];
        }
      }
#pragma unroll
      for (int o = LPC / 2; o > 0; o >>= 1)
#pragma unroll
        for (int j = 0; j < kND; ++j) {
          sb[j] += __shfl_xor_sync(0xffffffffu, sb[j], o);
          sa[j] += __shfl_xor_sync(0xffffffffu, sa[j], o);
        }
      if (ln == 0) {
        const float4 sl = *reinterpret_cast<const float4 *>(m.slope + t * CT + c0);
#pragma unroll
        for (int j = 0; j < kND; ++j) {
          const float gy = (&gv.x)[j], uj = (&uv.x)[j];
          const float dd = fmaf(uj, sb[j], sa[j]) * (&sl.x)[j];
          m.gu[(c0 + j) * OP + t] = fmaf((&dt.x)[j], sb[j], skip[j] * gy);
          m.gd[(c0 + j) * OP + t] = dd;
          dskip[j] = fmaf(gy, uj, dskip[j]);
          dbias[j] += dd;
        }
      }
    }
    if (warp == 0) put(m.rcarry + (parity ^ 1) * kND * 32, r);
    __syncthreads();
    // the superchunk's results
    for (int i = threadIdx.x; i < chans * kTS; i += kThreads) {
      const int d = i / kTS, t = i % kTS;
      if (t0 + t >= s.L) continue;
      const bool inside = t0 + t < len;
      stf(gu + d * s.L + t0 + t, inside ? m.gu[d * OP + t] : 0.f);
      stf(gdelta + d * s.L + t0 + t, inside ? m.gd[d * OP + t] : 0.f);
    }
    for (int i = threadIdx.x; i < s.N * kTS; i += kThreads) {
      const int n = i / kTS, t = i % kTS;
      if (t0 + t >= s.L) continue;
      const bool inside = t0 + t < len;
      pb[n * s.L + t0 + t] = inside ? m.gb[n * OP + t] : 0.f;
      pc[n * s.L + t0 + t] = inside ? m.gc[n * OP + t] : 0.f;
    }
  }
  // padded positions behind the last superchunk
  const int64_t from = (int64_t)supers * kTS;
  if (from < s.L) {
    for (int d = warp; d < chans; d += kWarps)
      for (int64_t t = from + lane; t < s.L; t += 32) {
        stf(gu + d * s.L + t, 0.f);
        stf(gdelta + d * s.L + t, 0.f);
      }
    for (int n = warp; n < s.N; n += kWarps)
      for (int64_t t = from + lane; t < s.L; t += 32) pb[n * s.L + t] = pc[n * s.L + t] = 0.f;
  }
  if (a.ginit && warp == 0) {
#pragma unroll
    for (int e = 0; e < kST; ++e) {
      const int j = e / kNS, n = n0 + e % kNS;
      if (c0 + j < chans && n < s.N) a.ginit[(row0 + c0 + j) * s.N + n] = r[e];
    }
  }
  // sums over the warps
  __syncthreads();
  put(m.end + warp * kND * 32, dA);
  m.prod[warp * 32 + lane] = make_float4(dskip[0], dskip[1], dskip[2], dskip[3]);
  m.rend[warp * 32 + lane] = make_float4(dbias[0], dbias[1], dbias[2], dbias[3]);
  __syncthreads();
  for (int i = threadIdx.x; i < CT * NP; i += kThreads) {
    const int d = i / NP, n = i % NP;
    if (d >= chans || n >= s.N) continue;
    const int j = d % kND, l = d / kND * LPC + n / kNS;
    float v = 0.f;
    for (int w = 0; w < kWarps; ++w)
      v += reinterpret_cast<const float *>(m.end + (w * kND + j) * 32 + l)[n % kNS];
    a.part_a[b * s.D * s.N + (d0 + d) * s.N + n] = v;
  }
  for (int d = threadIdx.x; d < chans; d += kThreads) {
    const int j = d % kND, l = d / kND * LPC;
    float v = 0.f, w = 0.f;
    for (int k = 0; k < kWarps; ++k) {
      v += reinterpret_cast<const float *>(m.prod + k * 32 + l)[j];
      w += reinterpret_cast<const float *>(m.rend + k * 32 + l)[j];
    }
    a.part_d[b * s.D + d0 + d] = v;
    a.part_d[(s.B + b) * s.D + d0 + d] = w;
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

// dA, dskip, ddelta_bias: the sum over the batch, in order
__global__ void __launch_bounds__(256)
scan_param_kernel(const float *__restrict__ pa, const float *__restrict__ pd, float *ga,
                  float *gskip, float *gbias, int64_t B, int64_t D, int64_t N) {
  const int64_t i = blockIdx.x * 256ll + threadIdx.x;
  if (i < D * N) {
    float v = 0.f;
    for (int64_t b = 0; b < B; ++b) v += pa[b * D * N + i];
    ga[i] = v;
  }
  if (i < D) {
    float v = 0.f, w = 0.f;
    for (int64_t b = 0; b < B; ++b) {
      v += pd[b * D + i];
      w += pd[(B + b) * D + i];
    }
    if (gskip) gskip[i] = v;
    if (gbias) gbias[i] = w;
  }
}

int64_t channel_tiles(int64_t D, int64_t N, int64_t G) {
  return cdiv(D / G, 32 / lanes_per_channel(N) * kND);
}

struct Outs {
  void *gB, *gC;
  float *gA, *gskip, *gbias;
};

template <typename T, int LPC>
int bwd_launch(const Bwd &a, const Outs &o, const Shape &s, cudaStream_t st) {
  const size_t smem = sizeof(BwdSmem<T, LPC>);
  auto kern = scan_bwd_kernel<T, LPC>;
  if (set_smem_once((const void *)kern, (int)smem) != cudaSuccess)
    return check_launch("scan_bwd_kernel shared memory");
  const int64_t tiles = channel_tiles(s.D, s.N, s.G);
  kern<<<(unsigned)(s.B * s.G * tiles), kThreads, smem, st>>>(a, s);
  if (int rc = check_launch("scan_bwd_kernel")) return rc;
  const int64_t n = s.B * s.G * s.N * s.L, cap = 8 * (int64_t)sm_count();
  const dim3 grid((unsigned)(cdiv(n, 256) < cap ? cdiv(n, 256) : cap), 2);
  scan_sum_parts_kernel<T><<<grid, 256, 0, st>>>(a.part_b, a.part_c, (T *)o.gB, (T *)o.gC, n,
                                                  tiles);
  if (int rc = check_launch("scan_sum_parts_kernel")) return rc;
  scan_param_kernel<<<(unsigned)cdiv(s.D * s.N, 256), 256, 0, st>>>(
      a.part_a, a.part_d, o.gA, o.gskip, o.gbias, s.B, s.D, s.N);
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
  const int64_t parts = 2 * scan::channel_tiles(D, N, G) * B * G * N * L;
  return ((size_t)(parts + B * D * N + 2 * B * D) * sizeof(float) + 255) & ~size_t(255);
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
  const int64_t tiles = scan::channel_tiles(D, N, G), n = B * G * N * L;
  float *ws = (float *)workspace;
  const int vec = L % 8 == 0 && aligned_to_16(u) && aligned_to_16(delta) && aligned_to_16(go) &&
                  aligned_to_16(Bm) && aligned_to_16(Cm);
  const scan::Bwd a{go, u, delta, Bm, Cm, grad_final, A, skip, delta_bias, checkpoints, lengths,
                    grad_u, grad_delta, grad_state, ws, ws + tiles * n, ws + 2 * tiles * n,
                    ws + 2 * tiles * n + B * D * N, vec};
  const scan::Outs o{grad_B, grad_C, grad_A, grad_skip, grad_delta_bias};
  const scan::Shape s{B, D, L, (int)N, (int)G, softplus};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return scan::by_type_and_lanes(dtype, N, [&](auto t, auto lanes) {
    return scan::bwd_launch<decltype(t), decltype(lanes)::value>(a, o, s, st);
  });
}

}  // extern "C"
