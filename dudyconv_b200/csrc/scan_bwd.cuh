// scan_bwd.cuh -- the selective scan's gradients: the kernel (instantiated by element type in
// scan_bwd_f16.cu, scan_bwd_bf16.cu and scan_bwd_f32.cu; scan_bwd.cu has the rest).
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
// A thread holds two or four channels x four states, so that much of each sum over channels or
// states happens in its registers. dB and dC go
// across a warp's channels through shared memory, one word a lane and value, read back eight to
// a lane (by shuffles: 3% less with four channels, 7% more with two); the sums over states by
// shuffles. dB and dC of a block's channels are written as fp32
// parts, one per block of channels, and added by a second kernel in a fixed order; so are dA
// and the two [D] sums over the batch and the chunks.
//
// Measured with the sums kernel, N = 16, D = 256, L = 4096: 434 us at B=16 in fp16 (128 blocks of
// 32 channels, one an SM), 62 us at B=1 in bf16 (818 with one block for the sequence). The floors
// are 59 us of exponentials, 89 us of fp32 arithmetic (12 operations a state and position) and 60
// us of HBM with the saved states. It issues 23 instructions a lane's state and position, 168 us at
// full issue; eight warps an SM (255 registers a thread) do not hide their own latency and fill 45% of
// the slots. The busiest unit is the pipe of shared memory and L1, at 60%, to which the 4-byte stores of
// grad_u and grad_delta along channels add. With the whole block on one piece, joined by barriers, it
// took 722 us.
#pragma once

#include "scan.cuh"

namespace dudy {
namespace scan {

constexpr int kQ = 4;                  // positions of a piece
constexpr int kTS = kWarps * kQ;       // positions of a stretch
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
  int64_t chunk;           // positions of a chunk, a multiple of kTS
  int splits, vec;
  int *err;
};

// a warp's own piece, positions outermost
template <int LPC, int ND>
struct BwdPiece {
  static constexpr int CT = 32 / LPC * ND;       // channels of a block
  static constexpr int NP = kNS * LPC;
  static constexpr int UI = (CT * kQ / 2 + 31) / 32;      // pairs of u, delta, dy that a lane takes
  static constexpr int BI = (2 * NP * kQ / 4 + 31) / 32;  // fours of B and C
  float dt[kQ * CT], du[kQ * CT], go[kQ * CT];
  float u[kQ * CT], slope[kQ * CT];              // du's and ddelta's results take their places
  float bc[kQ * 2 * NP];                         // B and C of a position side by side
  float h0[2][CT * NP];                          // the states that enter this piece and the next
  float across[2][8 * 32];                       // dB's and dC's parts, by turns
};
template <typename T, int LPC, int ND>
struct BwdSmem {
  static constexpr int CT = BwdPiece<LPC, ND>::CT, NP = BwdPiece<LPC, ND>::NP;
  static constexpr int PITCH = kTS + 16 / (int)sizeof(T);
  static constexpr int V = 16 / (int)sizeof(T), VPR = kTS / V;
  static constexpr int ROWS = 3 * CT + 2 * NP;  // u, delta, dy, B, C as they lie in memory
  static constexpr int ITEMS = ROWS * VPR, EACH = (ITEMS + kThreads - 1) / kThreads;
  T raw[kStages][ROWS * PITCH];
  BwdPiece<LPC, ND> piece[kWarps];
  // handed on to the left, [warp][channel of the thread][lane] (with the chunk's decay product
  // so far); the sums over warps at the end use the same room
  float4 pass[kWarps * ND * 32], total[kWarps * ND * 32];
  Ready ready;
};

template <typename T, int LPC, int ND, bool PRE>
__global__ void __launch_bounds__(kThreads, ND == 2 ? 2 : 1)
scan_bwd_kernel(Bwd a, Shape s) {
  using Mine = BwdPiece<LPC, ND>;
  using Smem = BwdSmem<T, LPC, ND>;
  constexpr int CT = Mine::CT, NP = Mine::NP;
  extern __shared__ __align__(16) char smem_raw[];
  Smem &all = *reinterpret_cast<Smem *>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ln = lane % LPC, ld = lane / LPC, n0 = ln * kNS, c0 = ld * ND;
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

  // [channel][pair of states]
  float2 A[ND][2], dA[ND][2], r[ND][2], total[ND][2];
#pragma unroll
  for (int j = 0; j < ND; ++j) {
    float av[kNS], rv[kNS];
#pragma unroll
    for (int i = 0; i < kNS; ++i) {
      const bool ok = c0 + j < chans && n0 + i < s.N;
      const int64_t at = (row0 + c0 + j) * s.N + n0 + i;
      av[i] = ok ? kLog2e * a.A[(d0 + c0 + j) * s.N + n0 + i] : 0.f;
      rv[i] = 0.f;
      if (!PRE && ok && warp == 0) {
        if (a.gfinal) rv[i] = a.gfinal[at];
        for (int k = a.splits - 1; k > split; --k)
          rv[i] = pass_chunk(a.prod[k * nst + at], rv[i], a.rend[k * nst + at]);
      }
    }
    A[j][0] = make_float2(av[0], av[1]);
    A[j][1] = make_float2(av[2], av[3]);
    r[j][0] = make_float2(rv[0], rv[1]);
    r[j][1] = make_float2(rv[2], rv[3]);
    dA[j][0] = dA[j][1] = both(0.f);
    total[j][0] = total[j][1] = both(1.f);
  }
  // a lane's channels where it takes u, delta and dy
  float bias[Mine::UI], skip[Mine::UI];
#pragma unroll
  for (int k = 0; k < Mine::UI; ++k) {
    const int d = (lane + k * 32) % CT;
    bias[k] = d < chans && a.delta_bias ? a.delta_bias[d0 + d] : 0.f;
    skip[k] = !PRE && d < chans && a.skip ? a.skip[d0 + d] : 0.f;
  }

  // The chunk in whole stretches, so that copies start on 16 bytes; positions behind `end` count
  // as padding. Piece k, counted from the right, is warp k % kWarps's.
  const int stretches = end > from ? (int)((end - from + kTS - 1) / kTS) : 0;
  const int pieces = stretches * kWarps;
  auto item = [&](int i) {
    const int row = i / Smem::VPR, c = i % Smem::VPR * Smem::V;
    const bool chan = row < 3 * CT;
    const int r = chan ? row % CT : (row - 3 * CT) % NP;
    const T *base = row < CT ? u : row < 2 * CT ? delta : chan ? go : row < 3 * CT + NP ? Bm : Cm;
    bool ok = i < Smem::ITEMS && r < (chan ? chans : s.N);
    if (PRE) ok = ok && row >= CT && !(row >= 3 * CT && row < 3 * CT + NP);
    return RowCopy<T>{ok ? base + r * s.L + c : nullptr, row * Smem::PITCH + c, c};
  };
  constexpr int kKeep = Smem::EACH < kHeld ? Smem::EACH : kHeld;
  RowCopy<T> held[kKeep];
#pragma unroll
  for (int k = 0; k < kKeep; ++k) held[k] = item(threadIdx.x + k * kThreads);
  auto stage = [&](int st) {
    if (st >= stretches) return;
    const int64_t t0 = from + (int64_t)(stretches - 1 - st) * kTS;
    T *raw = all.raw[st % kStages];
#pragma unroll
    for (int k = 0; k < Smem::EACH; ++k)
      row_copy(raw, k < kKeep ? held[k < kKeep ? k : 0] : item(threadIdx.x + k * kThreads), t0,
               end, a.vec);
  };
  for (int i = threadIdx.x; i < Smem::ITEMS; i += kThreads) {
    const RowCopy<T> x = item(i);
    if (!x.src)
      for (int st = 0; st < kStages; ++st)
        *reinterpret_cast<uint4 *>(all.raw[st] + x.dst) = make_uint4(0, 0, 0, 0);
  }
  // the states that enter this warp's piece of a stretch
  auto stage_states = [&](int st) {
    if (PRE || st >= stretches) return;
    const int64_t t0 = from + (int64_t)(pieces - 1 - (st * kWarps + warp)) * kQ;
    const float *src = a.ckpt + ((b * s.ckpts() + t0 / kCkpt) * s.D + d0) * s.N;
    const bool in = t0 < end, vec = s.N % 4 == 0;
    float *dst = m.h0[st & 1];
#pragma unroll
    for (int i = lane; i < CT * (NP / 4); i += 32) {
      const int c = i / (NP / 4), n = i % (NP / 4) * 4;
      float *to = dst + c * NP + n;
      if (vec && in && c < chans && n < s.N) {
        cp_async16(to, src + c * s.N + n);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          to[e] = in && c < chans && n + e < s.N ? src[c * s.N + n + e] : 0.f;
      }
    }
  };
  using SumN = Scatter<1, LPC, 2 * ND, 2>;
  constexpr int kLeftN = SumN::kLeft / 2, kOwners = ND / kLeftN, kEach = LPC / kOwners;
  constexpr int DL = 32 / LPC;                   // lanes across channels
  constexpr int kOut = DL < 8 ? 8 / DL : 1;      // sums of dB and dC that a lane ends with
  constexpr int kShare = DL > 8 ? DL / 8 : 1;    // lanes that share one
  float dskip[kLeftN], dbias[kLeftN];
#pragma unroll
  for (int i = 0; i < kLeftN; ++i) dskip[i] = dbias[i] = 0.f;

  ready_init(all.ready);
  stage(0);
  stage_states(0);
  copies_commit();
  stage(1);
  copies_commit();
  copies_wait<1>();
  ready_arrive(all.ready, 0);
  for (int st = 0; st < stretches; ++st) {
    const int k = st * kWarps + warp, buf = st % kStages, at0 = (kWarps - 1 - warp) * kQ;
    const int64_t t0 = from + (int64_t)(pieces - 1 - k) * kQ;
    ready_wait(all.ready, st, a.err);
    __syncwarp();
    stage(st + 2);
    stage_states(st + 1);
    copies_commit();
    copies_wait<1>();
#pragma unroll
    for (int p = 0; p < Mine::UI; ++p) {
      const int i = lane + p * 32, d = i % CT, c = i / CT * 2;
      if (i >= CT * kQ / 2) break;
      const T *src = all.raw[buf] + d * Smem::PITCH + at0 + c;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float dt = ldf(src + CT * Smem::PITCH + j) + bias[p], slope = 1.f;
        if (s.softplus) dt = softplus<T>(dt, slope);
        if (t0 + c + j >= end) dt = slope = 0.f;
        const int to = (c + j) * CT + d;
        m.dt[to] = dt;
        m.go[to] = ldf(src + 2 * CT * Smem::PITCH + j);
        if (PRE) continue;
        const float uv = ldf(src + j);
        m.du[to] = dt * uv;
        m.u[to] = uv;
        m.slope[to] = slope;
      }
    }
#pragma unroll
    for (int p = 0; p < Mine::BI; ++p) {
      const int i = lane + p * 32, row = i % (2 * NP), c = i / (2 * NP) * 4;
      if (i >= 2 * NP * kQ / 4) break;
      RowFour<T> f;
      f.load_all(all.raw[buf] + (3 * CT + row) * Smem::PITCH + at0 + c);
#pragma unroll
      for (int j = 0; j < 4; ++j) m.bc[(c + j) * 2 * NP + row] = f.get(j);
    }
    ready_arrive(all.ready, st + 1);

    // a position's values of the thread's channels, each twice
    auto chan = [&](const float *p, int q, float2 (&v)[ND]) {
#pragma unroll
      for (int j = 0; j < ND; j += 2) {
        const float2 x = *reinterpret_cast<const float2 *>(p + q * CT + c0 + j);
        v[j] = both(x.x);
        v[j + 1] = both(x.y);
      }
    };
    float2 dt[ND], du[ND], gy[ND];
    auto four = [](const float *p) { return *reinterpret_cast<const float4 *>(p); };
    const float *sbc = m.bc + n0;
    // dec[q]: position q's decay
    float2 dec[kQ][ND][2], own[ND][2], prod[ND][2];
#pragma unroll
    for (int q = kQ - 1; q >= 0; --q) {
      chan(m.dt, q, dt);
      chan(m.go, q, gy);
      const float4 cv = four(sbc + q * 2 * NP + NP);
#pragma unroll
      for (int j = 0; j < ND; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 e = decays(dt[j], A[j][i]);
          const float2 ci = i ? hi(cv) : lo(cv);
          dec[q][j][i] = e;
          own[j][i] = __fmul2_rn(
              e, q == kQ - 1 ? __fmul2_rn(ci, gy[j]) : __ffma2_rn(ci, gy[j], own[j][i]));
          prod[j][i] = q == kQ - 1 ? e : __fmul2_rn(prod[j][i], e);
        }
    }
    // what enters the piece from the right, and what leaves it to the left
    if (k > 0) {
      const int before = (warp + kWarps - 1) % kWarps;
      pair_wait(1 + before);
#pragma unroll
      for (int j = 0; j < ND; ++j) {
        const float4 v = all.pass[(before * ND + j) * 32 + lane];
        r[j][0] = lo(v);
        r[j][1] = hi(v);
        if (PRE) {
          const float4 p = all.total[(before * ND + j) * 32 + lane];
          total[j][0] = lo(p);
          total[j][1] = hi(p);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        own[j][i] = __ffma2_rn(prod[j][i], r[j][i], own[j][i]);
        if (PRE) total[j][i] = __fmul2_rn(total[j][i], prod[j][i]);
      }
    if (k + 1 < pieces) {
#pragma unroll
      for (int j = 0; j < ND; ++j) {
        all.pass[(warp * ND + j) * 32 + lane] = quad(own[j][0], own[j][1]);
        if (PRE) all.total[(warp * ND + j) * 32 + lane] = quad(total[j][0], total[j][1]);
      }
      pair_arrive(1 + warp);
    }
    if (PRE) {
#pragma unroll
      for (int j = 0; j < ND; ++j) r[j][0] = own[j][0], r[j][1] = own[j][1];
      continue;
    }
    // h[q]: the state before position q
    float2 h[kQ + 1][ND][2];
#pragma unroll
    for (int j = 0; j < ND; ++j) {
      const float4 x = four(m.h0[st & 1] + (c0 + j) * NP + n0);
      h[0][j][0] = lo(x);
      h[0][j][1] = hi(x);
    }
#pragma unroll
    for (int q = 0; q < kQ; ++q) {
      chan(m.du, q, du);
      const float4 bv = four(sbc + q * 2 * NP);
#pragma unroll
      for (int j = 0; j < ND; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          h[q + 1][j][i] = __ffma2_rn(dec[q][j][i], h[q][j][i],
                                      __fmul2_rn(du[j], i ? hi(bv) : lo(bv)));
    }
    // the gradients
    float dbc[kOut][kQ];
#pragma unroll
    for (int q = kQ - 1; q >= 0; --q) {
      chan(m.dt, q, dt);
      chan(m.du, q, du);
      chan(m.go, q, gy);
      const float4 bv = four(sbc + q * 2 * NP), cv = four(sbc + q * 2 * NP + NP);
      float2 db[2], dc[2], sb[ND], sa[ND];
#pragma unroll
      for (int j = 0; j < ND; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 bi = i ? hi(bv) : lo(bv), ci = i ? hi(cv) : lo(cv);
          const float2 gg = __ffma2_rn(ci, gy[j], r[j][i]);
          r[j][i] = __fmul2_rn(dec[q][j][i], gg);
          const float2 w = __fmul2_rn(r[j][i], h[q][j][i]);
          dc[i] = j ? __ffma2_rn(gy[j], h[q + 1][j][i], dc[i]) : __fmul2_rn(gy[j], h[q + 1][j][i]);
          db[i] = j ? __ffma2_rn(gg, du[j], db[i]) : __fmul2_rn(gg, du[j]);
          sb[j] = i ? __ffma2_rn(gg, bi, sb[j]) : __fmul2_rn(gg, bi);
          sa[j] = i ? __ffma2_rn(w, A[j][i], sa[j]) : __fmul2_rn(w, A[j][i]);
          dA[j][i] = __ffma2_rn(w, dt[j], dA[j][i]);
        }
      }
      // dB, dC across the channels: value i of lane (ld, ln) to place i * 32 + ln * DL + ld, so
      // that the DL lanes' parts of a sum lie side by side; every second row has its fours
      // swapped in pairs, which spreads the reads of eight over all banks.
      float *across = m.across[q & 1];
      {
        const float v[8] = {db[0].x, db[0].y, db[1].x, db[1].y, dc[0].x, dc[0].y, dc[1].x, dc[1].y};
#pragma unroll
        for (int i = 0; i < 8; ++i) across[i * 32 + ((ln * DL + ld) ^ ((i & 1) << 2))] = v[i];
      }
      __syncwarp();
      {
        const int swap = (lane >> 2 & 1) << 2;
        const float4 x = four(across + ((lane * 8) ^ swap)), z = four(across + ((lane * 8 + 4) ^ swap));
        const float v[8] = {x.x, x.y, x.z, x.w, z.x, z.y, z.z, z.w};
        constexpr int kIn = DL < 8 ? DL : 8;
#pragma unroll
        for (int o = 0; o < kOut; ++o) {
          float t = 0.f;
#pragma unroll
          for (int i = 0; i < kIn; ++i) t = i ? t + v[o * kIn + i] : v[o * kIn];
#pragma unroll
          for (int x2 = 1; x2 < kShare; x2 <<= 1) t += __shfl_xor_sync(0xffffffffu, t, x2);
          dbc[o][q] = t;
        }
      }
      // the sums over states: a channel's two values stay together
      float z[2 * ND];
#pragma unroll
      for (int j = 0; j < ND; ++j) {
        z[2 * j] = sb[j].x + sb[j].y;
        z[2 * j + 1] = sa[j].x + sa[j].y;
      }
      SumN::sum(z, lane);
      if (ln % kEach == 0) {
#pragma unroll
        for (int i = 0; i < kLeftN; ++i) {
          const int at = q * CT + c0 + ln / kEach * kLeftN + i;
          const float gyj = m.go[at], uj = m.u[at];
          const float sbv = z[2 * i];
          const float dd = fmaf(uj, sbv, z[2 * i + 1] * kLn2) * m.slope[at];
          m.u[at] = m.dt[at] * sbv;
          m.slope[at] = dd;
          dskip[i] = fmaf(gyj, uj, dskip[i]);
          dbias[i] += dd;
        }
      }
    }
    // output o of dB and dC is state n0(o % LPC) + o / LPC % 4, dB where o / LPC < 4
    if (lane % kShare == 0) {
#pragma unroll
      for (int x = 0; x < kOut; ++x) {
        const int o = lane / kShare * kOut + x, i = o / LPC, n = o % LPC * kNS + i % kNS;
        if (n >= s.N) continue;
        float v[4];
#pragma unroll
        for (int q = 0; q < kQ; ++q) v[q] = t0 + q < end ? dbc[x][q] : 0.f;
        row_store4((i < kNS ? gB : gC) + n * s.L, t0, to, v, s.L % 4 == 0);
      }
    }
    __syncwarp();
#pragma unroll
    for (int p = 0; p < Mine::UI; ++p) {
      const int i = lane + p * 32, d = i % CT, c = i / CT * 2;
      if (i >= CT * kQ / 2) break;
      if (d >= chans) continue;
      float o[2], w[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int at = (c + j) * CT + d;
        const bool inside = t0 + c + j < end;
        o[j] = inside ? fmaf(skip[p], m.go[at], m.u[at]) : 0.f;
        w[j] = inside ? m.slope[at] : 0.f;
      }
      row_store2(gu + d * s.L, t0 + c, to, o, a.vec);
      row_store2(gdelta + d * s.L, t0 + c, to, w, a.vec);
    }
  }
  const int last = pieces ? kWarps - 1 : 0;  // the warp that holds what leaves the chunk
  if (PRE || (a.ginit && split == 0)) {
    if (warp == last) {
#pragma unroll
      for (int j = 0; j < ND; ++j) {
        const float v[kNS] = {r[j][0].x, r[j][0].y, r[j][1].x, r[j][1].y};
        const float p[kNS] = {total[j][0].x, total[j][0].y, total[j][1].x, total[j][1].y};
        const int64_t at = (row0 + c0 + j) * s.N + n0;
#pragma unroll
        for (int i = 0; i < kNS; ++i) {
          if (c0 + j >= chans || n0 + i >= s.N) continue;
          if (PRE) {
            a.rend[split * nst + at + i] = v[i];
            a.prod[split * nst + at + i] = p[i];
          } else {
            a.ginit[at + i] = v[i];
          }
        }
      }
    }
  }
  if (PRE) return;
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
  // sums over the warps
  __syncthreads();
  float *sums = reinterpret_cast<float *>(all.total);
#pragma unroll
  for (int j = 0; j < ND; ++j) all.pass[(warp * ND + j) * 32 + lane] = quad(dA[j][0], dA[j][1]);
#pragma unroll
  for (int i = 0; i < kLeftN; ++i) {
    sums[((warp * 2) * 32 + lane) * ND + i] = dskip[i];
    sums[((warp * 2 + 1) * 32 + lane) * ND + i] = dbias[i];
  }
  __syncthreads();
  float *pa = a.part_a + (split * s.B + b) * s.D * s.N;
  for (int i = threadIdx.x; i < CT * NP; i += kThreads) {
    const int d = i / NP, n = i % NP;
    if (d >= chans || n >= s.N) continue;
    const int l = d / ND * LPC + n / kNS;
    float v = 0.f;
    for (int w = 0; w < kWarps; ++w)
      v += reinterpret_cast<const float *>(all.pass + (w * ND + d % ND) * 32 + l)[n % kNS];
    pa[(d0 + d) * s.N + n] = v;
  }
  for (int d = threadIdx.x; d < chans; d += kThreads) {
    const int l = d / ND * LPC + d % ND / kLeftN * kEach, i = d % ND % kLeftN;
    float v = 0.f, w = 0.f;
    for (int k = 0; k < kWarps; ++k) {
      v += sums[((k * 2) * 32 + l) * ND + i];
      w += sums[((k * 2 + 1) * 32 + l) * ND + i];
    }
    a.part_d[(split * s.B + b) * s.D + d0 + d] = v;
    a.part_d[((a.splits + split) * s.B + b) * s.D + d0 + d] = w;
  }
}

template <typename T, int LPC, int ND>
int bwd_chain(const Bwd &a, const Shape &s, int64_t tiles, cudaStream_t st) {
  const int smem = (int)sizeof(BwdSmem<T, LPC, ND>);
  auto main = scan_bwd_kernel<T, LPC, ND, false>, pre = scan_bwd_kernel<T, LPC, ND, true>;
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
  return check_launch("scan_bwd_kernel");
}

// by lanes per channel, and four or two channels to a thread
template <typename T>
int bwd_chain_by(int lpc, bool four, const Bwd &a, const Shape &s, int64_t tiles,
                 cudaStream_t st) {
  switch (lpc) {
    case 1: return bwd_chain<T, 1, 2>(a, s, tiles, st);
    case 2: return bwd_chain<T, 2, 2>(a, s, tiles, st);
    case 4:
      return four ? bwd_chain<T, 4, 4>(a, s, tiles, st) : bwd_chain<T, 4, 2>(a, s, tiles, st);
    case 8: return bwd_chain<T, 8, 2>(a, s, tiles, st);
    default: return bwd_chain<T, 16, 2>(a, s, tiles, st);
  }
}
int bwd_chain_f16(int lpc, bool four, const Bwd &a, const Shape &s, int64_t tiles, cudaStream_t st);
int bwd_chain_bf16(int lpc, bool four, const Bwd &a, const Shape &s, int64_t tiles, cudaStream_t st);
int bwd_chain_f32(int lpc, bool four, const Bwd &a, const Shape &s, int64_t tiles, cudaStream_t st);

}  // namespace scan
}  // namespace dudy
