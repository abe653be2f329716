// scan_fwd.cu -- the selective scan forward over whole sequences, and over one token.
#include "scan.cuh"

namespace dudy {
namespace scan {
namespace {

constexpr int kND = 2;                 // channels of a thread
constexpr int kQ = 8;                  // positions of a warp in a superchunk
constexpr int kTS = kWarps * kQ;       // positions of a superchunk
constexpr int kYP = kTS + 4;
static_assert(kTS % kCkpt == 0 && kCkpt % kQ == 0, "states are saved where a warp's piece starts");

struct Fwd {
  const void *u, *delta, *Bm, *Cm;
  const float *A, *skip, *delta_bias, *init;
  const int32_t *lengths;
  void *y;
  float *final_state, *ckpt;
  float *end, *prod;   // [splits][B*D][N]: a chunk's end state from zero and its decays' product
  int64_t chunk;       // positions of a chunk, a multiple of kTS
  int splits, vec;
};

template <typename T, int LPC>
struct FwdTile {
  static constexpr int CT = 32 / LPC * kND;     // channels of a block
  static constexpr int NP = kNS * LPC;          // padded states
  static constexpr int UI = (CT * kTS / 4 + kThreads - 1) / kThreads;      // pieces of u a thread copies
  static constexpr int BI = (2 * NP * kTS / 8 + kThreads - 1) / kThreads;  // pieces of B and C
  float2 dt[kTS * CT], du[kTS * CT];            // dt and dt u, each twice side by side
  float bc[kTS * 2 * NP];                       // B and C of a position side by side
  float y[2][CT * kYP];
  float4 end[kWarps * kND * 32], prod[kWarps * kND * 32];
  float4 carry[2 * kND * 32];
};

// Four / eight neighbouring elements as they lie in memory; zero at and behind `end`.
template <typename T, int N>
struct Piece {
  T e[N];
  __device__ __forceinline__ void load(const T *row, int64_t t, int64_t end, bool vec) {
    if (vec && t + N <= end) {
      if constexpr (sizeof(e) == 8) {
        *reinterpret_cast<uint2 *>(e) = *reinterpret_cast<const uint2 *>(row + t);
      } else {
#pragma unroll
        for (int i = 0; i < (int)sizeof(e) / 16; ++i)
          reinterpret_cast<uint4 *>(e)[i] = reinterpret_cast<const uint4 *>(row + t)[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = t + i < end ? row[t + i] : Elem<T>::from_f(0.f);
    }
  }
};

// PRE: a chunk's end state from zero and its decay product only.
template <typename T, int LPC, bool PRE>
__global__ void __launch_bounds__(kThreads, 2)
scan_fwd_kernel(Fwd a, Shape s) {
  using Tile = FwdTile<T, LPC>;
  constexpr int CT = Tile::CT, NP = Tile::NP;
  extern __shared__ __align__(16) char smem_raw[];
  Tile &m = *reinterpret_cast<Tile *>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ln = lane % LPC, ld = lane / LPC, n0 = ln * kNS, c0 = ld * kND;

  const int R = (int)(s.D / s.G), tiles = (R + CT - 1) / CT;
  const int split = blockIdx.x % a.splits;
  if (PRE && split == a.splits - 1) return;  // nothing starts from the last chunk's end
  const int64_t bid = blockIdx.x / a.splits;
  const int tile = (int)(bid % tiles);
  const int64_t bg = bid / tiles, b = bg / s.G, g = bg % s.G;
  const int chans = R - tile * CT < CT ? R - tile * CT : CT;  // channels that exist
  const int64_t d0 = g * R + tile * CT, row0 = b * s.D + d0;
  const int64_t len = clamp_len(a.lengths, b, s.L);
  const int64_t from = split * a.chunk;                                  // this block's chunk
  const int64_t to = from + a.chunk < s.L ? from + a.chunk : s.L;
  const int64_t end = to < len ? to : len;                               // of it that is read
  const T *u = (const T *)a.u + row0 * s.L, *delta = (const T *)a.delta + row0 * s.L;
  const T *Bm = (const T *)a.Bm + bg * s.N * s.L, *Cm = (const T *)a.Cm + bg * s.N * s.L;
  T *y = (T *)a.y + row0 * s.L;

  float2 A[kND][2], h[kND][2], total[kND][2];
#pragma unroll
  for (int j = 0; j < kND; ++j) {
    float av[kNS], hv[kNS];
#pragma unroll
    for (int i = 0; i < kNS; ++i) {
      const bool ok = c0 + j < chans && n0 + i < s.N;
      const int64_t at = (row0 + c0 + j) * s.N + n0 + i, step = s.B * s.D * s.N;
      av[i] = ok ? scaled<T>(a.A[(d0 + c0 + j) * s.N + n0 + i]) : 0.f;
      hv[i] = 0.f;
      if (!PRE && ok) {
        if (a.init) hv[i] = a.init[at];
        for (int k = 0; k < split; ++k) hv[i] = fmaf(a.prod[k * step + at], hv[i], a.end[k * step + at]);
      }
    }
    A[j][0] = make_float2(av[0], av[1]);
    A[j][1] = make_float2(av[2], av[3]);
    h[j][0] = make_float2(hv[0], hv[1]);
    h[j][1] = make_float2(hv[2], hv[3]);
    total[j][0] = total[j][1] = both(1.f);
    if (warp == 0) m.carry[j * 32 + lane] = quad(h[j][0], h[j][1]);
  }

  // the next superchunk's elements, in registers while this one is worked on
  Piece<T, 4> pu[Tile::UI], pd[Tile::UI];
  Piece<T, 8> pb[Tile::BI];
  auto fetch = [&](int64_t t0) {
#pragma unroll
    for (int k = 0; k < Tile::UI; ++k) {
      const int i = threadIdx.x + k * kThreads, d = i % CT;
      if (i >= CT * kTS / 4) break;
      const int64_t lim = d < chans ? end : 0;
      pu[k].load(u + d * s.L, t0 + i / CT * 4, lim, a.vec);
      pd[k].load(delta + d * s.L, t0 + i / CT * 4, lim, a.vec);
    }
#pragma unroll
    for (int k = 0; k < Tile::BI; ++k) {
      const int i = threadIdx.x + k * kThreads, r = i % (2 * NP), n = r % NP;
      if (i >= 2 * NP * kTS / 8) break;
      pb[k].load((r < NP ? Bm : Cm) + n * s.L, t0 + i / (2 * NP) * 8, n < s.N ? end : 0, a.vec);
    }
  };
  auto store_y = [&](int64_t t0, const float *ys) {
    for (int i = threadIdx.x; i < chans * (kTS / 8); i += kThreads) {
      const int d = i / (kTS / 8), c = i % (kTS / 8) * 8;
      const int64_t t = t0 + c;
      alignas(16) float o[8];
      *reinterpret_cast<float4 *>(o) = *reinterpret_cast<const float4 *>(ys + d * kYP + c);
      *reinterpret_cast<float4 *>(o + 4) = *reinterpret_cast<const float4 *>(ys + d * kYP + c + 4);
      if (t + 8 > end)
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = t + j < end ? o[j] : 0.f;
      if (a.vec) row_store8_until<T, true>(y + d * s.L, t, to, o);
      else row_store8_until<T, false>(y + d * s.L, t, to, o);
    }
  };
  const int supers = end > from ? (int)((end - from + kTS - 1) / kTS) : 0;
  if (supers) fetch(from);
  for (int k = 0; k < supers; ++k) {
    const int64_t t0 = from + (int64_t)k * kTS;
    __syncthreads();
    // fp32 tiles, positions outermost, so that a thread reads its four states at once
#pragma unroll
    for (int p = 0; p < Tile::UI; ++p) {
      const int i = threadIdx.x + p * kThreads, d = i % CT, c = i / CT * 4;
      if (i >= CT * kTS / 4) break;
      const bool ok = d < chans;
      const float bias = ok && a.delta_bias ? a.delta_bias[d0 + d] : 0.f;
      const float skip = !PRE && ok && a.skip ? a.skip[d0 + d] : 0.f;
      alignas(16) float yv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float uv = Elem<T>::to_f(pu[p].e[j]);
        float dt = Elem<T>::to_f(pd[p].e[j]) + bias, slope;
        if (s.softplus) dt = softplus<T>(dt, slope);
        if (t0 + c + j >= end) dt = 0.f;  // the state passes a padded position unchanged
        m.dt[(c + j) * CT + d] = both(dt);
        m.du[(c + j) * CT + d] = both(dt * uv);
        yv[j] = skip * uv;
      }
      if (!PRE) *reinterpret_cast<float4 *>(m.y[k & 1] + d * kYP + c) = *reinterpret_cast<float4 *>(yv);
    }
#pragma unroll
    for (int p = 0; p < Tile::BI; ++p) {
      const int i = threadIdx.x + p * kThreads, r = i % (2 * NP), c = i / (2 * NP) * 8;
      if (i >= 2 * NP * kTS / 8) break;
#pragma unroll
      for (int j = 0; j < 8; ++j) m.bc[(c + j) * 2 * NP + r] = Elem<T>::to_f(pb[p].e[j]);
    }
    __syncthreads();
    if (k + 1 < supers) fetch(t0 + kTS);
    if (!PRE && k > 0) store_y(t0 - kTS, m.y[(k - 1) & 1]);

    // this warp's piece from a zero state
    const float2 *sdt = m.dt + warp * kQ * CT + c0, *sdu = m.du + warp * kQ * CT + c0;
    const float *sbc = m.bc + warp * kQ * 2 * NP + n0;
    float2 dec[kQ][kND][2];
    float sum[kND];
#pragma unroll
    for (int j = 0; j < kND; ++j) sum[j] = 0.f, h[j][0] = h[j][1] = both(0.f);
#pragma unroll
    for (int q = 0; q < kQ; ++q) {
      const float4 dt = *reinterpret_cast<const float4 *>(sdt + q * CT);
      const float4 du = *reinterpret_cast<const float4 *>(sdu + q * CT);
      const float4 bv = *reinterpret_cast<const float4 *>(sbc + q * 2 * NP);
#pragma unroll
      for (int j = 0; j < kND; ++j) {
        const float2 dtj = j ? hi(dt) : lo(dt), duj = j ? hi(du) : lo(du);
        sum[j] += dtj.x;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 x = __fmul2_rn(dtj, A[j][i]);
          dec[q][j][i] = make_float2(decay<T>(x.x), decay<T>(x.y));
          h[j][i] = __ffma2_rn(dec[q][j][i], h[j][i], __fmul2_rn(duj, i ? hi(bv) : lo(bv)));
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kND; ++j) {
      const float2 x = __fmul2_rn(both(sum[j]), A[j][0]), z = __fmul2_rn(both(sum[j]), A[j][1]);
      m.end[(warp * kND + j) * 32 + lane] = quad(h[j][0], h[j][1]);
      m.prod[(warp * kND + j) * 32 + lane] =
          make_float4(decay<T>(x.x), decay<T>(x.y), decay<T>(z.x), decay<T>(z.y));
    }
    __syncthreads();
    // the state that enters it
#pragma unroll
    for (int j = 0; j < kND; ++j) {
      const float4 c = m.carry[((k & 1) * kND + j) * 32 + lane];
      h[j][0] = lo(c);
      h[j][1] = hi(c);
    }
    const int before = PRE ? (warp == kWarps - 1 ? kWarps : 0) : warp;
    for (int w = 0; w < before; ++w)
#pragma unroll
      for (int j = 0; j < kND; ++j) {
        const float4 e = m.end[(w * kND + j) * 32 + lane], p = m.prod[(w * kND + j) * 32 + lane];
        h[j][0] = __ffma2_rn(lo(p), h[j][0], lo(e));
        h[j][1] = __ffma2_rn(hi(p), h[j][1], hi(e));
        if (PRE) {
          total[j][0] = __fmul2_rn(total[j][0], lo(p));
          total[j][1] = __fmul2_rn(total[j][1], hi(p));
        }
      }
    if (!PRE) {
      const int64_t tw = t0 + warp * kQ;
      if (a.ckpt && warp * kQ % kCkpt == 0 && tw < s.L) {
#pragma unroll
        for (int j = 0; j < kND; ++j) {
          float *ck = a.ckpt + ((b * s.ckpts() + tw / kCkpt) * s.D + d0 + c0 + j) * s.N + n0;
          const float v[kNS] = {h[j][0].x, h[j][0].y, h[j][1].x, h[j][1].y};
#pragma unroll
          for (int i = 0; i < kNS; ++i)
            if (c0 + j < chans && n0 + i < s.N) ck[i] = v[i];
        }
      }
      // and the piece again from there: v[j][q] is this thread's part of y
      float v[kND * kQ];
#pragma unroll
      for (int q = 0; q < kQ; ++q) {
        const float4 du = *reinterpret_cast<const float4 *>(sdu + q * CT);
        const float4 bv = *reinterpret_cast<const float4 *>(sbc + q * 2 * NP);
        const float4 cv = *reinterpret_cast<const float4 *>(sbc + q * 2 * NP + NP);
#pragma unroll
        for (int j = 0; j < kND; ++j) {
          const float2 duj = j ? hi(du) : lo(du);
          h[j][0] = __ffma2_rn(dec[q][j][0], h[j][0], __fmul2_rn(duj, lo(bv)));
          h[j][1] = __ffma2_rn(dec[q][j][1], h[j][1], __fmul2_rn(duj, hi(bv)));
          const float2 p = __ffma2_rn(hi(cv), h[j][1], __fmul2_rn(lo(cv), h[j][0]));
          v[j * kQ + q] = p.x + p.y;
        }
      }
      using Sum = Scatter<1, LPC, kND * kQ>;
      Sum::sum(v, lane);
      constexpr int kLeft = Sum::kLeft, kV = kLeft % 4 == 0 ? 4 : kLeft;
#pragma unroll
      for (int i = 0; i < kLeft; i += kV) {
        const int at = ln * kLeft + i;
        float *to = m.y[k & 1] + (c0 + at / kQ) * kYP + warp * kQ + at % kQ;
        if constexpr (kV == 4) {
          float4 o = *reinterpret_cast<float4 *>(to);
          o.x += v[i]; o.y += v[i + 1]; o.z += v[i + 2]; o.w += v[i + 3];
          *reinterpret_cast<float4 *>(to) = o;
        } else {
#pragma unroll
          for (int e = 0; e < kV; ++e) to[e] += v[i + e];
        }
      }
    }
    if (warp == kWarps - 1)
#pragma unroll
      for (int j = 0; j < kND; ++j)
        m.carry[(((k + 1) & 1) * kND + j) * 32 + lane] = quad(h[j][0], h[j][1]);
  }
  if (!PRE) {
    __syncthreads();
    if (supers) store_y(from + (int64_t)(supers - 1) * kTS, m.y[(supers - 1) & 1]);
    // padded positions behind the last superchunk
    const int64_t rest = from + (int64_t)supers * kTS;
    if (rest < to)
      for (int d = warp; d < chans; d += kWarps)
        for (int64_t t = rest + lane; t < to; t += 32) stf(y + d * s.L + t, 0.f);
  }
  const bool last = split == a.splits - 1;
  if (warp != kWarps - 1 || (!PRE && !(a.final_state && last))) return;
#pragma unroll
  for (int j = 0; j < kND; ++j) {
    const float v[kNS] = {h[j][0].x, h[j][0].y, h[j][1].x, h[j][1].y};
    const float p[kNS] = {total[j][0].x, total[j][0].y, total[j][1].x, total[j][1].y};
    const int64_t at = (row0 + c0 + j) * s.N + n0;
#pragma unroll
    for (int i = 0; i < kNS; ++i) {
      if (c0 + j >= chans || n0 + i >= s.N) continue;
      if (PRE) {
        a.end[split * s.B * s.D * s.N + at + i] = v[i];
        a.prod[split * s.B * s.D * s.N + at + i] = p[i];
      } else {
        a.final_state[at + i] = v[i];
      }
    }
  }
}

// Chunks of a sequence: as many as fill the GPU's places for blocks (two an SM), where the rows
// of channels alone leave at least half of them empty; whole superchunks each.
int64_t fwd_blocks(const Shape &s) {
  return s.B * s.G * cdiv(s.R(), 32 / lanes_per_channel(s.N) * kND);
}
int fwd_splits(const Shape &s, int64_t *chunk) {
  const int64_t blocks = fwd_blocks(s), places = 2 * (int64_t)sm_count();
  const int64_t supers = cdiv(s.L, kTS);
  int64_t n = blocks * 2 <= places ? places / blocks : 1;
  if (n > supers) n = supers;
  *chunk = cdiv(supers, n) * kTS;
  return (int)cdiv(s.L, *chunk);
}
size_t fwd_workspace(const Shape &s) {
  int64_t chunk;
  const int n = fwd_splits(s, &chunk);
  return n > 1 ? 2 * (size_t)n * s.B * s.D * s.N * sizeof(float) : 0;
}

template <typename T, int LPC>
int fwd_launch(const Fwd &a, const Shape &s, cudaStream_t st) {
  const int smem = (int)sizeof(FwdTile<T, LPC>);
  auto main = scan_fwd_kernel<T, LPC, false>, pre = scan_fwd_kernel<T, LPC, true>;
  const unsigned grid = (unsigned)(fwd_blocks(s) * a.splits);
  if (a.splits > 1) {
    if (set_smem_once((const void *)pre, smem) != cudaSuccess)
      return check_launch("scan_fwd_kernel shared memory");
    pre<<<grid, kThreads, smem, st>>>(a, s);
    if (int rc = check_launch("scan_fwd_kernel (chunk ends)")) return rc;
  }
  if (set_smem_once((const void *)main, smem) != cudaSuccess)
    return check_launch("scan_fwd_kernel shared memory");
  main<<<grid, kThreads, smem, st>>>(a, s);
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
      const float v = fmaf(decay<T>(dt * scaled<T>(A[d * s.N + n])), *h, du * ldf(Bm + bc + n));
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
  return (scan::fwd_workspace(scan::Shape{B, D, L, (int)N, (int)G, 1}) + 255) & ~size_t(255);
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
  const scan::Shape s{B, D, L, (int)N, (int)G, softplus};
  int64_t chunk;
  const int splits = scan::fwd_splits(s, &chunk);
  float *ws = (float *)workspace;
  const scan::Fwd a{u, delta, Bm, Cm, A, skip, delta_bias, state, lengths, y, final_state,
                    checkpoints, ws, splits > 1 ? ws + splits * B * D * N : nullptr, chunk, splits,
                    vec};
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
