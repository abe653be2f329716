// scan_fwd.cu -- the selective scan forward over whole sequences, and over one token.
//
// Measured with N = 16, D = 256, L = 4096: 179 us at B=16 in fp16 (197 when it saves the states
// for the backward, 268 MB more to write), against 59 us of exponentials and 17 us of HBM; 36 us
// at B=1 in bf16 (111 with one block for the sequence). Its 256 blocks of 16 channels at B=16 leave
// 40 SMs with one block where the others have two; there the pipe of shared memory and L1 (every lane
// reads its positions' dt, dt u, B and C; y goes out eight bytes a lane, along channels) is busiest,
// at 67%, before the issue slots' 56% and the special function unit's 39%. A
// recurrence costs two packed instructions a pair of states, so running it twice is cheap next to
// the exponentials. With the whole block on one piece, joined by barriers, it took 280 us.
#include "scan.cuh"

namespace dudy {
namespace scan {
namespace {

constexpr int kND = 2;                 // channels of a thread
constexpr int kQ = 8;                  // positions of a piece
constexpr int kTS = kWarps * kQ;       // positions of a stretch
constexpr int kYP = kQ + 4;
static_assert(kQ % kCkpt == 0, "states are saved within a piece");

struct Fwd {
  const void *u, *delta, *Bm, *Cm;
  const float *A, *skip, *delta_bias, *init;
  const int32_t *lengths;
  void *y;
  float *final_state, *ckpt;
  float *end, *prod;   // [splits][B*D][N]: a chunk's end state from zero and its decays' product
  int64_t chunk;       // positions of a chunk, a multiple of kQ
  int splits, vec;
  int *err;
};

// a warp's own piece
template <int LPC>
struct FwdPiece {
  static constexpr int CT = 32 / LPC * kND;     // channels of a block
  static constexpr int NP = kNS * LPC;          // padded states
  static constexpr int UI = (CT * kQ / 4 + 31) / 32;      // fours of u and delta that a lane takes
  static constexpr int BI = (2 * NP * kQ / 4 + 31) / 32;  // fours of B and C
  float4 dtu[kQ * CT / 2];                      // (dt, dt', dt u, dt' u') of two channels
  float bc[kQ * 2 * NP];                        // B and C of a position side by side
  float y[CT * kYP];
};
template <typename T, int LPC>
struct FwdSmem {
  static constexpr int CT = FwdPiece<LPC>::CT, NP = FwdPiece<LPC>::NP;
  static constexpr int PITCH = kTS + 16 / (int)sizeof(T);
  static constexpr int V = 16 / (int)sizeof(T), VPR = kTS / V;
  static constexpr int ROWS = 2 * CT + 2 * NP;  // u, delta, B, C as they lie in memory
  static constexpr int ITEMS = ROWS * VPR, EACH = (ITEMS + kThreads - 1) / kThreads;
  T raw[kStages][ROWS * PITCH];
  FwdPiece<LPC> piece[kWarps];
  float4 pass[kWarps * kND * 32];               // the state that a warp hands on
  float4 total[kWarps * kND * 32];              // and the chunk's decay product so far
  Ready ready;
};

// Where rows do not all start on 16 bytes (odd lengths), a stretch comes in by words, as it lies in
// memory: a 16-bit row that starts inside a word lies one element further on in its buffer
// (row_shift), where the 16 bytes between rows have room for it. The threads of a row take
// neighbouring words in turn. (fp32, B=5, D=256, L=1001: 47 us, 51 by elements, 43 at L=1000.)
template <typename T>
__device__ __forceinline__ int row_shift(const T *row) {
  return sizeof(T) == 2 ? (int)(reinterpret_cast<uintptr_t>(row) >> 1) & 1 : 0;
}
template <int TS, typename T>  // TS: positions of a stretch
__device__ __forceinline__ void row_words(T *raw, const RowCopy<T> &x, int64_t t0, int64_t end) {
  constexpr int V = 16 / sizeof(T), E = 4 / sizeof(T), kRow = TS / V;
  if (!x.src) return;
  const T *row = x.src - x.c + t0;
  T *to = raw + x.dst - x.c;
  const int64_t rest = end - t0;
  const int left = rest <= TS ? (int)rest : TS + 1;  // elements of the row that may be read
  const int sh = row_shift(row), own = x.c / V;
#pragma unroll
  for (int k = 0; k < (E > 1 ? 5 : 4); ++k) {
    if (k == 4 && (own || !sh)) break;
    const int word = k < 4 ? k * kRow + own : TS / E, e = word * E - sh;
    uint32_t *w = reinterpret_cast<uint32_t *>(to) + word;
    if (left <= e) {
      *w = 0u;
    } else if (e < 0 && t0 == 0) {  // nothing of this row lies before it
      *w = (uint32_t)*reinterpret_cast<const uint16_t *>(row) << 16;
    } else {
      cp_async4(w, row + e, left - e < E ? (left - e) * (int)sizeof(T) : 4);
    }
  }
}

// PRE: a chunk's end state from zero and its decay product only. VEC: all rows start on 16 bytes.
template <typename T, int LPC, bool PRE, bool VEC>
__global__ void __launch_bounds__(kThreads, 2)
scan_fwd_kernel(Fwd a, Shape s) {
  using Mine = FwdPiece<LPC>;
  constexpr int CT = Mine::CT, NP = Mine::NP;
  extern __shared__ __align__(16) char smem_raw[];
  using Smem = FwdSmem<T, LPC>;
  Smem &all = *reinterpret_cast<Smem *>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ln = lane % LPC, ld = lane / LPC, n0 = ln * kNS, c0 = ld * kND;
  Mine &m = all.piece[warp];

  const int split = blockIdx.x % a.splits;
  if (PRE && split == a.splits - 1) return;  // nothing starts from the last chunk's end
  const int R = (int)(s.D / s.G), tiles = (R + CT - 1) / CT;
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
  const int pieces = end > from ? (int)((end - from + kQ - 1) / kQ) : 0;

  float2 A[kND][2], h[kND][2], total[kND][2];
#pragma unroll
  for (int j = 0; j < kND; ++j) {
    float av[kNS], hv[kNS];
#pragma unroll
    for (int i = 0; i < kNS; ++i) {
      const bool ok = c0 + j < chans && n0 + i < s.N;
      const int64_t at = (row0 + c0 + j) * s.N + n0 + i, step = s.B * s.D * s.N;
      av[i] = ok ? kLog2e * a.A[(d0 + c0 + j) * s.N + n0 + i] : 0.f;
      hv[i] = 0.f;
      if (!PRE && ok && warp == 0) {
        if (a.init) hv[i] = a.init[at];
        for (int k = 0; k < split; ++k)
          hv[i] = pass_chunk(a.prod[k * step + at], hv[i], a.end[k * step + at]);
      }
    }
    A[j][0] = make_float2(av[0], av[1]);
    A[j][1] = make_float2(av[2], av[3]);
    h[j][0] = make_float2(hv[0], hv[1]);
    h[j][1] = make_float2(hv[2], hv[3]);
    total[j][0] = total[j][1] = both(1.f);
  }

  // a lane's channels where it takes u and delta
  float bias[Mine::UI], skip[Mine::UI];
#pragma unroll
  for (int k = 0; k < Mine::UI; ++k) {
    const int d = (lane + k * 32) % CT;
    bias[k] = d < chans && a.delta_bias ? a.delta_bias[d0 + d] : 0.f;
    skip[k] = !PRE && d < chans && a.skip ? a.skip[d0 + d] : 0.f;
  }
  const int stretches = (pieces + kWarps - 1) / kWarps;
  auto item = [&](int i) {
    const int row = i / Smem::VPR, c = i % Smem::VPR * Smem::V;
    const bool chan = row < 2 * CT;
    const int r = chan ? row % CT : (row - 2 * CT) % NP;
    const T *base = row < CT ? u : chan ? delta : row < 2 * CT + NP ? Bm : Cm;
    const bool ok = i < Smem::ITEMS && r < (chan ? chans : s.N);
    return RowCopy<T>{ok ? base + r * s.L + c : nullptr, row * Smem::PITCH + c, c};
  };
  // where row r of `rows` rows lies in its buffer
  auto shift = [&](const T *base, int r, int rows) {
    return r < rows ? row_shift(base) ^ (sizeof(T) == 2 ? r & (int)s.L & 1 : 0) : 0;
  };
  constexpr int kKeep = Smem::EACH < kHeld ? Smem::EACH : kHeld;
  RowCopy<T> held[kKeep];
#pragma unroll
  for (int k = 0; k < kKeep; ++k) held[k] = item(threadIdx.x + k * kThreads);
  auto stage = [&](int st) {
    if (st < stretches) {
      const int64_t t0 = from + (int64_t)st * kTS;
      T *raw = all.raw[st % kStages];
#pragma unroll
      for (int k = 0; k < Smem::EACH; ++k) {
        const RowCopy<T> x = k < kKeep ? held[k < kKeep ? k : 0] : item(threadIdx.x + k * kThreads);
        if (VEC) row_copy(raw, x, t0, end, true);
        else row_words<kTS>(raw, x, t0, end);
      }
    }
    copies_commit();
  };
  for (int i = threadIdx.x; i < Smem::ITEMS; i += kThreads) {
    const RowCopy<T> x = item(i);
    if (!x.src)
      for (int st = 0; st < kStages; ++st)
        *reinterpret_cast<uint4 *>(all.raw[st] + x.dst) = make_uint4(0, 0, 0, 0);
  }
  ready_init(all.ready);
  stage(0);
  stage(1);
  copies_wait<1>();
  ready_arrive(all.ready, 0);
  for (int st = 0; st < stretches; ++st) {
    const int k = st * kWarps + warp, buf = st % kStages, at = warp * kQ;
    const int64_t t0 = from + (int64_t)k * kQ;
    ready_wait(all.ready, st, a.err);
    __syncwarp();
    stage(st + 2);
    copies_wait<1>();
    // fp32, positions outermost, so that a thread reads its four states at once
    float *dtu = reinterpret_cast<float *>(m.dtu);
#pragma unroll
    for (int p = 0; p < Mine::UI; ++p) {
      const int i = lane + p * 32, d = i % CT, c = i / CT * 4;
      if (i >= CT * kQ / 4) break;
      RowFour<T> pu, pd;
      const T *src = all.raw[buf] + d * Smem::PITCH + at + c;
      if (VEC) {
        pu.load_all(src);
        pd.load_all(src + CT * Smem::PITCH);
      } else {
        pu.load_shifted(src, shift(u, d, chans));
        pd.load_shifted(src + CT * Smem::PITCH, shift(delta, d, chans));
      }
      alignas(16) float yv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float uv = pu.get(j);
        float dt = pd.get(j) + bias[p], slope;
        if (s.softplus) dt = softplus<T>(dt, slope);
        if (t0 + c + j >= end) dt = 0.f;  // the state passes a padded position unchanged
        float *dst = dtu + ((c + j) * (CT / 2) + d / 2) * 4 + d % 2;
        dst[0] = dt;
        dst[2] = dt * uv;
        yv[j] = skip[p] * uv;
      }
      if (!PRE) *reinterpret_cast<float4 *>(m.y + d * kYP + c) = *reinterpret_cast<float4 *>(yv);
    }
#pragma unroll
    for (int p = 0; p < Mine::BI; ++p) {
      const int i = lane + p * 32, r = i % (2 * NP), c = i / (2 * NP) * 4;
      if (i >= 2 * NP * kQ / 4) break;
      RowFour<T> pb;
      const T *src = all.raw[buf] + (2 * CT + r) * Smem::PITCH + at + c;
      if (VEC) pb.load_all(src);
      else pb.load_shifted(src, r < NP ? shift(Bm, r, (int)s.N) : shift(Cm, r - NP, (int)s.N));
#pragma unroll
      for (int j = 0; j < 4; ++j) m.bc[(c + j) * 2 * NP + r] = pb.get(j);
    }
    ready_arrive(all.ready, st + 1);
    if (k >= pieces) break;

    const float4 *sdt = m.dtu + ld;
    const float *sbc = m.bc + n0;
    float2 dec[kQ][kND][2], own[kND][2], prod[kND][2];
#pragma unroll
    for (int q = 0; q < kQ; ++q) {
      const float4 dt = sdt[q * (CT / 2)];
      const float4 bv = *reinterpret_cast<const float4 *>(sbc + q * 2 * NP);
#pragma unroll
      for (int j = 0; j < kND; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 e = decays(both(j ? dt.y : dt.x), A[j][i]);
          const float2 in = __fmul2_rn(both(j ? dt.w : dt.z), i ? hi(bv) : lo(bv));
          dec[q][j][i] = e;
          own[j][i] = q ? __ffma2_rn(e, own[j][i], in) : in;
          prod[j][i] = q ? __fmul2_rn(prod[j][i], e) : e;
        }
    }
    // the state that enters the piece, and the one that leaves it
    if (k > 0) {
      const int before = (warp + kWarps - 1) % kWarps;
      pair_wait(1 + before);
#pragma unroll
      for (int j = 0; j < kND; ++j) {
        const float4 v = all.pass[(before * kND + j) * 32 + lane];
        h[j][0] = lo(v);
        h[j][1] = hi(v);
        if (PRE) {
          const float4 p = all.total[(before * kND + j) * 32 + lane];
          total[j][0] = lo(p);
          total[j][1] = hi(p);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kND; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        own[j][i] = __ffma2_rn(prod[j][i], h[j][i], own[j][i]);
        if (PRE) total[j][i] = __fmul2_rn(total[j][i], prod[j][i]);
      }
    if (k + 1 < pieces) {
#pragma unroll
      for (int j = 0; j < kND; ++j) {
        all.pass[(warp * kND + j) * 32 + lane] = quad(own[j][0], own[j][1]);
        if (PRE) all.total[(warp * kND + j) * 32 + lane] = quad(total[j][0], total[j][1]);
      }
      pair_arrive(1 + warp);
    }
    if (PRE) {
#pragma unroll
      for (int j = 0; j < kND; ++j) h[j][0] = own[j][0], h[j][1] = own[j][1];
      continue;
    }
    auto save = [&](int64_t t, const float2 (&v)[kND][2]) {
      if (t >= end) return;
#pragma unroll
      for (int j = 0; j < kND; ++j) {
        if (c0 + j >= chans) break;
        float *ck = a.ckpt + ((b * s.ckpts() + t / kCkpt) * s.D + d0 + c0 + j) * s.N + n0;
        if (s.N % kNS == 0 && n0 < s.N) {
          *reinterpret_cast<float4 *>(ck) = quad(v[j][0], v[j][1]);
        } else {
          const float e[kNS] = {v[j][0].x, v[j][0].y, v[j][1].x, v[j][1].y};
#pragma unroll
          for (int i = 0; i < kNS; ++i)
            if (n0 + i < s.N) ck[i] = e[i];
        }
      }
    };
    if (a.ckpt) save(t0, h);
    // the recurrence from there; each state takes its decay's place
#pragma unroll
    for (int q = 0; q < kQ; ++q) {
      const float4 du = sdt[q * (CT / 2)];
      const float4 bv = *reinterpret_cast<const float4 *>(sbc + q * 2 * NP);
#pragma unroll
      for (int j = 0; j < kND; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 in = __fmul2_rn(both(j ? du.w : du.z), i ? hi(bv) : lo(bv));
          h[j][i] = __ffma2_rn(dec[q][j][i], h[j][i], in);
          dec[q][j][i] = h[j][i];
        }
      if ((q + 1) % kCkpt == 0 && q + 1 < kQ && a.ckpt) save(t0 + q + 1, h);
    }
    // v[j][q] is this thread's part of y
    float v[kND * kQ];
#pragma unroll
    for (int q = 0; q < kQ; ++q) {
      const float4 cv = *reinterpret_cast<const float4 *>(sbc + q * 2 * NP + NP);
#pragma unroll
      for (int j = 0; j < kND; ++j) {
        const float2 p = __ffma2_rn(hi(cv), dec[q][j][1], __fmul2_rn(lo(cv), dec[q][j][0]));
        v[j * kQ + q] = p.x + p.y;
      }
    }
    using Sum = Scatter<1, LPC, kND * kQ>;
    Sum::sum(v, lane);
    constexpr int kLeft = Sum::kLeft, kV = kLeft % 4 == 0 ? 4 : kLeft;
#pragma unroll
    for (int i = 0; i < kLeft; i += kV) {
      const int at = ln * kLeft + i;
      float *dst = m.y + (c0 + at / kQ) * kYP + at % kQ;
      if constexpr (kV == 4) {
        float4 o = *reinterpret_cast<float4 *>(dst);
        o.x += v[i]; o.y += v[i + 1]; o.z += v[i + 2]; o.w += v[i + 3];
        *reinterpret_cast<float4 *>(dst) = o;
      } else {
#pragma unroll
        for (int e = 0; e < kV; ++e) dst[e] += v[i + e];
      }
    }
    __syncwarp();
    if (!VEC) {  // neighbouring lanes to neighbouring positions
#pragma unroll 4
      for (int i = lane; i < CT * kQ; i += 32) {
        const int d = i / kQ, c = i % kQ;
        if (d < chans && t0 + c < to) stf(y + d * s.L + t0 + c, t0 + c < end ? m.y[d * kYP + c] : 0.f);
      }
      continue;
    }
#pragma unroll
    for (int p = 0; p < Mine::UI; ++p) {
      const int i = lane + p * 32, d = i % CT, c = i / CT * 4;
      if (i >= CT * kQ / 4) break;
      if (d >= chans) continue;
      float o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = t0 + c + j < end ? m.y[d * kYP + c + j] : 0.f;
      row_store4(y + d * s.L, t0 + c, to, o, true);
    }
  }
  if (!PRE) {  // padded positions behind the last piece
    const int64_t rest = from + (int64_t)pieces * kQ;
    if (rest < to)
      for (int d = warp; d < chans; d += kWarps)
        for (int64_t t = rest + lane; t < to; t += 32) stf(y + d * s.L + t, 0.f);
  }
  // the last piece's warp holds the end state
  if (warp != (pieces ? (pieces - 1) % kWarps : 0)) return;
  if (!PRE && !(a.final_state && split == a.splits - 1)) return;
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
// of channels alone leave at least half of them empty; whole pieces each.
int64_t fwd_blocks(const Shape &s) {
  return s.B * s.G * cdiv(s.R(), 32 / lanes_per_channel(s.N) * kND);
}
int fwd_splits(const Shape &s, int64_t *chunk) {
  const int64_t blocks = fwd_blocks(s), places = 2 * (int64_t)sm_count();
  // two stretches a chunk at least, and four without a cut: the first kernel costs about two
  const int64_t stretches = cdiv(s.L, kTS), most = stretches <= 4 ? 1 : cdiv(stretches, 2);
  int64_t n = blocks * 2 <= places ? places / blocks : 1;
  if (n > most) n = most;
  *chunk = cdiv(cdiv(s.L, n), kQ) * kQ;
  return (int)cdiv(s.L, *chunk);
}
size_t fwd_workspace(const Shape &s) {
  int64_t chunk;
  const int n = fwd_splits(s, &chunk);
  return n > 1 ? 2 * (size_t)n * s.B * s.D * s.N * sizeof(float) : 0;
}

template <typename T, int LPC>
int fwd_launch(const Fwd &a, const Shape &s, cudaStream_t st) {
  const int smem = (int)sizeof(FwdSmem<T, LPC>);
  auto main = a.vec ? scan_fwd_kernel<T, LPC, false, true> : scan_fwd_kernel<T, LPC, false, false>;
  auto pre = a.vec ? scan_fwd_kernel<T, LPC, true, true> : scan_fwd_kernel<T, LPC, true, false>;
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
      const float v = fmaf(decay(dt, kLog2e * A[d * s.N + n]), *h, du * ldf(Bm + bc + n));
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
  if (int rc = scan::require_checkpoints(checkpoints, N)) return rc;
  if (int rc = require_apart(state, final_state)) return rc;  // chunks' blocks read state when they start
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
                    vec, device_err_word()};
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
