// scan_fwd.cu -- the selective scan forward over whole sequences, and over one token.
//
// Per state and position the forward needs one exponential and three multiply-adds: at N = 16
// the special function unit (16 a clock and SM) is the bound, not HBM (three 16-bit rows).
#include "scan.cuh"

namespace dudy {
namespace scan {
namespace {

constexpr int kQ = 16;                 // positions of a warp in a superchunk
constexpr int kTS = kWarps * kQ;       // positions of a superchunk

struct Fwd {
  const void *u, *delta, *Bm, *Cm;
  const float *A, *skip, *delta_bias, *init;
  const int32_t *lengths;
  void *y;
  float *final_state, *ckpt;
  int vec;
};

template <typename T, int LPC>
struct FwdSmem {
  static constexpr int CW = 32 / LPC;           // channels of a block (one per lane group)
  static constexpr int NP = kNS * LPC;          // padded states
  static constexpr int PITCH = kTS + 16 / (int)sizeof(T);
  T raw_u[CW * PITCH], raw_d[CW * PITCH], raw_b[NP * PITCH], raw_c[NP * PITCH];
  float2 du[kTS * CW];                          // (dt, dt u) of a position and channel
  float b[kTS * NP], c[kTS * NP];
  float y[CW * (kTS + 4)];
  float4 end[kWarps * 32], prod[kWarps * 32], carry[2 * 32];
};

template <typename T, int LPC>
__global__ void __launch_bounds__(kThreads)
scan_fwd_kernel(Fwd a, Shape s) {
  using Smem = FwdSmem<T, LPC>;
  constexpr int CW = Smem::CW, NP = Smem::NP, PITCH = Smem::PITCH, YP = kTS + 4;
  extern __shared__ __align__(16) char smem_raw[];
  Smem &m = *reinterpret_cast<Smem *>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ln = lane % LPC, ld = lane / LPC, n0 = ln * kNS;

  const int64_t R = s.D / s.G, tiles = (R + CW - 1) / CW;
  const int64_t tile = blockIdx.x % tiles, bg = blockIdx.x / tiles;
  const int64_t b = bg / s.G, g = bg % s.G;
  const int chans = (int)(R - tile * CW < CW ? R - tile * CW : CW);  // channels that exist
  const int64_t d0 = g * R + tile * CW, row0 = b * s.D + d0;
  const int64_t len = clamp_len(a.lengths, b, s.L);
  const T *u = (const T *)a.u + row0 * s.L, *delta = (const T *)a.delta + row0 * s.L;
  const T *Bm = (const T *)a.Bm + bg * s.N * s.L, *Cm = (const T *)a.Cm + bg * s.N * s.L;
  T *y = (T *)a.y + row0 * s.L;
  const bool mine = ld < chans;

  float A[kNS];
  float4 h0 = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kNS; ++i) {
    const bool ok = mine && n0 + i < s.N;
    A[i] = ok ? a.A[(d0 + ld) * s.N + n0 + i] : 0.f;
    if (ok && a.init) (&h0.x)[i] = a.init[(row0 + ld) * s.N + n0 + i];
  }
  if (warp == 0) m.carry[lane] = h0;

  auto stage = [&](int64_t t0) {
    stage_rows<T, kTS, PITCH>(m.raw_u, u, CW, chans, s.L, t0, len, a.vec);
    stage_rows<T, kTS, PITCH>(m.raw_d, delta, CW, chans, s.L, t0, len, a.vec);
    stage_rows<T, kTS, PITCH>(m.raw_b, Bm, NP, s.N, s.L, t0, len, a.vec);
    stage_rows<T, kTS, PITCH>(m.raw_c, Cm, NP, s.N, s.L, t0, len, a.vec);
  };
  const int supers = (int)((len + kTS - 1) / kTS);
  if (supers) stage(0);
  float h[kNS] = {h0.x, h0.y, h0.z, h0.w};
  for (int k = 0; k < supers; ++k) {
    const int64_t t0 = (int64_t)k * kTS;
    cp_async_wait_all();
    __syncthreads();
    // fp32 tiles, positions outermost, so that a thread reads its four states at once
    for (int i = threadIdx.x; i < CW * (kTS / 8); i += kThreads) {
      const int d = i % CW, c = i / CW * 8;
      float uv[8], dv[8];
      row_load8(m.raw_u + d * PITCH + c, uv);
      row_load8(m.raw_d + d * PITCH + c, dv);
      const bool ok = d < chans;
      const float bias = ok && a.delta_bias ? a.delta_bias[d0 + d] : 0.f;
      const float skip = ok && a.skip ? a.skip[d0 + d] : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float dt = dv[j] + bias, slope;
        if (s.softplus) dt = softplus<T>(dt, slope);
        if (t0 + c + j >= len) dt = 0.f;  // the state passes a padded position unchanged
        m.du[(c + j) * CW + d] = make_float2(dt, dt * uv[j]);
        m.y[d * YP + c + j] = skip * uv[j];
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
    if (k + 1 < supers) stage(t0 + kTS);

    // this warp's piece from a zero state
    float dec[kQ][kNS], sum = 0.f;
#pragma unroll
    for (int i = 0; i < kNS; ++i) h[i] = 0.f;
#pragma unroll
    for (int q = 0; q < kQ; ++q) {
      const int t = warp * kQ + q;
      const float2 du = m.du[t * CW + ld];
      const float4 bv = *reinterpret_cast<const float4 *>(m.b + t * NP + n0);
      sum += du.x;
#pragma unroll
      for (int i = 0; i < kNS; ++i) {
        dec[q][i] = decay<T>(du.x * A[i]);
        h[i] = fmaf(dec[q][i], h[i], du.y * (&bv.x)[i]);
      }
    }
    m.end[warp * 32 + lane] = make_float4(h[0], h[1], h[2], h[3]);
    m.prod[warp * 32 + lane] = make_float4(decay<T>(sum * A[0]), decay<T>(sum * A[1]),
                                           decay<T>(sum * A[2]), decay<T>(sum * A[3]));
    __syncthreads();
    // the state that enters it
    float4 in = m.carry[(k & 1) * 32 + lane];
    for (int w = 0; w < warp; ++w) {
      const float4 e = m.end[w * 32 + lane], p = m.prod[w * 32 + lane];
      in.x = fmaf(p.x, in.x, e.x);
      in.y = fmaf(p.y, in.y, e.y);
      in.z = fmaf(p.z, in.z, e.z);
      in.w = fmaf(p.w, in.w, e.w);
    }
    h[0] = in.x; h[1] = in.y; h[2] = in.z; h[3] = in.w;
    const int64_t tw = t0 + warp * kQ;
    if (a.ckpt && tw % kCkpt == 0 && tw < s.L && mine) {
      float *ck = a.ckpt + ((row0 + ld) * s.ckpts() + tw / kCkpt) * s.N + n0;
#pragma unroll
      for (int i = 0; i < kNS; ++i)
        if (n0 + i < s.N) ck[i] = h[i];
    }
    // and the piece again from there
#pragma unroll
    for (int q = 0; q < kQ; ++q) {
      const int t = warp * kQ + q;
      const float2 du = m.du[t * CW + ld];
      const float4 bv = *reinterpret_cast<const float4 *>(m.b + t * NP + n0);
      const float4 cv = *reinterpret_cast<const float4 *>(m.c + t * NP + n0);
      float acc = 0.f;
#pragma unroll
      for (int i = 0; i < kNS; ++i) {
        h[i] = fmaf(dec[q][i], h[i], du.y * (&bv.x)[i]);
        acc = fmaf((&cv.x)[i], h[i], acc);
      }
#pragma unroll
      for (int o = LPC / 2; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
      if (ln == 0) m.y[ld * YP + t] += acc;
    }
    if (warp == kWarps - 1) m.carry[((k + 1) & 1) * 32 + lane] = make_float4(h[0], h[1], h[2], h[3]);
    __syncwarp();
    // each warp stores its own positions
    for (int i = lane; i < CW * (kQ / 8); i += 32) {
      const int d = i / (kQ / 8), c = warp * kQ + i % (kQ / 8) * 8;
      if (d >= chans) continue;
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = t0 + c + j < len ? m.y[d * YP + c + j] : 0.f;
      if (a.vec) row_store8_until<T, true>(y + d * s.L, t0 + c, s.L, o);
      else row_store8_until<T, false>(y + d * s.L, t0 + c, s.L, o);
    }
  }
  // padded positions behind the last superchunk
  const int64_t from = (int64_t)supers * kTS;
  if (from < s.L)
    for (int d = warp; d < chans; d += kWarps)
      for (int64_t t = from + lane; t < s.L; t += 32) stf(y + d * s.L + t, 0.f);
  if (a.final_state && warp == kWarps - 1 && mine) {
#pragma unroll
    for (int i = 0; i < kNS; ++i)
      if (n0 + i < s.N) a.final_state[(row0 + ld) * s.N + n0 + i] = h[i];
  }
}

template <typename T, int LPC>
int fwd_launch(const Fwd &a, const Shape &s, cudaStream_t st) {
  const size_t smem = sizeof(FwdSmem<T, LPC>);
  auto kern = scan_fwd_kernel<T, LPC>;
  if (set_smem_once((const void *)kern, (int)smem) != cudaSuccess)
    return check_launch("scan_fwd_kernel shared memory");
  const int64_t grid = s.B * s.G * cdiv(s.R(), 32 / LPC);
  kern<<<(unsigned)grid, kThreads, smem, st>>>(a, s);
  return check_launch("scan_fwd_kernel");
}

// ---- one token per sequence -----------------------------------------------------------------
// LPC lanes per (b, d), four states each, the state updated in place.
template <typename T, int LPC>
__global__ void __launch_bounds__(128)
scan_step_kernel(const T *__restrict__ u, const T *__restrict__ delta, const float *__restrict__ A,
                 const T *__restrict__ Bm, const T *__restrict__ Cm,
                 const float *__restrict__ skip, const float *__restrict__ delta_bias,
                 float *__restrict__ state, T *__restrict__ y, int64_t rows, Shape s) {
  const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  const int64_t row = i / LPC;
  const int n0 = (int)(i % LPC) * kNS;
  const bool mine = row < rows;
  float acc = 0.f;
  float uv = 0.f;
  int64_t d = 0;
  if (mine) {
    const int64_t b = row / s.D;
    d = row % s.D;
    const int64_t bc = (b * s.G + d / (s.D / s.G)) * s.N;
    uv = ldf(u + row);
    float dt = ldf(delta + row) + (delta_bias ? delta_bias[d] : 0.f), slope;
    if (s.softplus) dt = softplus<T>(dt, slope);
    const float du = dt * uv;
#pragma unroll
    for (int k = 0; k < kNS; ++k) {
      const int n = n0 + k;
      if (n >= s.N) break;
      float *h = state + row * s.N + n;
      const float v = fmaf(decay<T>(dt * A[d * s.N + n]), *h, du * ldf(Bm + bc + n));
      *h = v;
      acc = fmaf(ldf(Cm + bc + n), v, acc);
    }
  }
#pragma unroll
  for (int o = LPC / 2; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (mine && n0 == 0) stf(y + row, fmaf(skip ? skip[d] : 0.f, uv, acc));
}

}  // namespace
}  // namespace scan
}  // namespace dudy

extern "C" {

size_t dudy_selective_scan_checkpoint_bytes(int64_t B, int64_t D, int64_t L, int64_t N,
                                            int64_t G, int dtype) {
  using namespace dudy;
  if (scan::validate(B, D, L, N, G, dtype)) return 0;
  return (size_t)(B * D * cdiv(L, scan::kCkpt) * N) * sizeof(float);
}

size_t dudy_selective_scan_forward_workspace_size(int64_t B, int64_t D, int64_t L, int64_t N,
                                                  int64_t G, int dtype) {
  using namespace dudy;
  if (scan::validate(B, D, L, N, G, dtype)) return 0;
  return 0;
}

int dudy_selective_scan_forward(const void *u, const void *delta, const float *A, const void *Bm,
                                const void *Cm, const float *skip, const float *delta_bias,
                                const float *state, const int32_t *lengths, void *y,
                                float *final_state, float *checkpoints, void *workspace,
                                size_t workspace_bytes, int64_t B, int64_t D, int64_t L,
                                int64_t N, int64_t G, int softplus, int dtype, void *stream) {
  using namespace dudy;
  clear_error();
  if (int rc = scan::validate(B, D, L, N, G, dtype)) return rc;
  if (!u || !delta || !A || !Bm || !Cm || !y) return refuse("null tensor pointer");
  if (int rc = require_workspace(workspace, workspace_bytes,
                                 dudy_selective_scan_forward_workspace_size(B, D, L, N, G, dtype)))
    return rc;
  if (int rc = require_sm100()) return rc;
  const int vec = L % 8 == 0 && aligned_to_16(u) && aligned_to_16(delta) && aligned_to_16(Bm) && aligned_to_16(Cm) &&
                  aligned_to_16(y);
  const scan::Fwd a{u, delta, Bm, Cm, A, skip, delta_bias, state, lengths, y, final_state,
                    checkpoints, vec};
  const scan::Shape s{B, D, L, (int)N, (int)G, softplus};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return scan::by_type_and_lanes(dtype, N, [&](auto t, auto lanes) {
    return scan::fwd_launch<decltype(t), decltype(lanes)::value>(a, s, st);
  });
}

int dudy_selective_scan_step(const void *u, const void *delta, const float *A, const void *Bm,
                             const void *Cm, const float *skip, const float *delta_bias,
                             float *state, void *y, int64_t B, int64_t D, int64_t N, int64_t G,
                             int softplus, int dtype, void *stream) {
  using namespace dudy;
  clear_error();
  if (int rc = scan::validate(B, D, 1, N, G, dtype)) return rc;
  if (!u || !delta || !A || !Bm || !Cm || !state || !y) return refuse("null tensor pointer");
  if (int rc = require_sm100()) return rc;
  const scan::Shape s{B, D, 1, (int)N, (int)G, softplus};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return scan::by_type_and_lanes(dtype, N, [&](auto t, auto lanes) {
    using T = decltype(t);
    constexpr int LPC = decltype(lanes)::value;
    const int64_t threads = B * D * LPC;
    scan::scan_step_kernel<T, LPC><<<(unsigned)cdiv(threads, 128), 128, 0, st>>>(
        (const T *)u, (const T *)delta, A, (const T *)Bm, (const T *)Cm, skip, delta_bias, state,
        (T *)y, B * D, s);
    return check_launch("scan_step_kernel");
  });
}

}  // extern "C"
