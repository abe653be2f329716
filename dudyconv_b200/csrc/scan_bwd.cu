// scan_bwd.cu -- the selective scan's gradients: the sums over blocks, the choice of the kernel
// and the C entry (the kernel is in scan_bwd.cuh).
#include <algorithm>

#include "scan_bwd.cuh"

namespace dudy {
namespace scan {
namespace {

// What the blocks left in parts, added in order: dB and dC over the channel blocks (blockIdx.y 0
// and 1), and dA, dskip and ddelta_bias over batch and chunks (blockIdx.y 2, 32 columns a block).
template <typename T>
__global__ void __launch_bounds__(256)
scan_sums_kernel(Bwd a, T *__restrict__ gB, T *__restrict__ gC, float *gA, float *gskip,
                 float *gbias, int64_t n, int64_t tiles, int64_t parts, int64_t D, int64_t N) {
  if (blockIdx.y < 2) {
    const float *p = blockIdx.y ? a.part_c : a.part_b;
    T *out = blockIdx.y ? gC : gB;
    const bool four = n % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
    const int64_t step = gridDim.x * 256ll;
    if (four) {
      for (int64_t i = (blockIdx.x * 256ll + threadIdx.x) * 4; i < n; i += step * 4) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int64_t k = 0; k < tiles; ++k) {
          const float4 x = *reinterpret_cast<const float4 *>(p + k * n + i);
          v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        }
        const float o[4] = {v.x, v.y, v.z, v.w};
        row_store4(out, i, n, o, true);
      }
    } else {
      for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += step) {
        float v = 0.f;
#pragma unroll 4
        for (int64_t k = 0; k < tiles; ++k) v += p[k * n + i];
        stf(out + i, v);
      }
    }
    return;
  }
  __shared__ float red[8][32];
  const int64_t states = D * N, cols = states + 2 * D;
  for (int64_t c0 = blockIdx.x * 32ll; c0 < cols; c0 += gridDim.x * 32ll) {
    const int64_t c = c0 + (threadIdx.x & 31), d = c - states;
    const float *p = c < states ? a.part_a + c : a.part_d + (d < D ? d : parts * D + d - D);
    const float v = column_sum<8>(p, parts, c < states ? states : D, c < cols, red);
    if (threadIdx.x >= 32 || c >= cols) continue;
    if (c < states) gA[c] = v;
    else if (d < D && gskip) gskip[d] = v;
    else if (d >= D && gbias) gbias[d - D] = v;
  }
}

// ---- which kernel ----
// Four channels to a thread where there are channels enough to give three quarters of the SMs a
// block of them and N is 9 to 16: fewer shuffles and shared loads a state, but 255 registers and
// one block an SM. B=16, D=256, L=4096, N=16, fp16: 434 us against 479; B=1: 70 against 62.
bool four_channels(int64_t B, int64_t D, int64_t N, int64_t G) {
  const int lpc = lanes_per_channel(N);
  return lpc == 4 && 4 * B * G * cdiv(D / G, 32 / lpc * 4) >= 3 * (int64_t)sm_count();
}
int64_t channel_tiles(int64_t D, int64_t N, int64_t G, bool four) {
  return cdiv(D / G, 32 / lanes_per_channel(N) * (four ? 4 : 2));
}

// as the forward's chunks, in whole stretches
constexpr int kLeast = 4;
int bwd_splits(int64_t B, int64_t D, int64_t L, int64_t N, int64_t G, bool four, int64_t *chunk) {
  const int64_t blocks = B * G * channel_tiles(D, N, G, four);
  const int64_t places = (four ? 1 : 2) * (int64_t)sm_count(), most = cdiv(L, kLeast * kTS);
  int64_t n = blocks * 2 <= places ? places / blocks : 1;
  if (n > most) n = most;
  *chunk = cdiv(cdiv(L, n), kTS) * kTS;
  return (int)cdiv(L, *chunk);
}

struct Sizes {
  bool four;
  int64_t tiles, chunk, splits;
  int64_t bc, a, d, st;  // floats: each of part_b, part_c; part_a; part_d; rend, prod
  size_t bytes() const { return (size_t)(2 * bc + a + d + 2 * st) * sizeof(float); }
};
Sizes bwd_sizes(int64_t B, int64_t D, int64_t L, int64_t N, int64_t G) {
  Sizes z;
  z.four = four_channels(B, D, N, G);
  z.tiles = channel_tiles(D, N, G, z.four);
  z.splits = bwd_splits(B, D, L, N, G, z.four, &z.chunk);
  z.bc = cdiv(z.tiles * B * G * N * L, 4) * 4;
  z.a = z.splits * B * D * N;
  z.d = 2 * z.splits * B * D;
  z.st = z.splits > 1 ? z.splits * B * D * N : 0;
  return z;
}

struct Outs {
  void *gB, *gC;
  float *gA, *gskip, *gbias;
};

template <typename T>
int bwd_sums(const Bwd &a, const Outs &o, const Shape &s, int64_t tiles, cudaStream_t st) {
  const int64_t n = s.B * s.G * s.N * s.L, cap = 8 * (int64_t)sm_count();
  const int64_t want = std::max(cdiv(n, 1024), cdiv(s.D * s.N + 2 * s.D, 32));
  scan_sums_kernel<T><<<dim3((unsigned)std::min(want, cap), 3), 256, 0, st>>>(
      a, (T *)o.gB, (T *)o.gC, o.gA, o.gskip, o.gbias, n, tiles, s.B * a.splits, s.D, s.N);
  return check_launch("scan_sums_kernel");
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
  if (int rc = scan::require_checkpoints(checkpoints, N)) return rc;
  // dB's and dC's parts go out and come back by 16 bytes where their number allows it
  if (B * G * N * L % 4 == 0 && !aligned_to_16(workspace))
    return refuse("workspace must be 16-byte aligned.");
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
                    z.chunk, (int)z.splits, vec, device_err_word()};
  const scan::Outs o{grad_B, grad_C, grad_A, grad_skip, grad_delta_bias};
  const scan::Shape s{B, D, L, (int)N, (int)G, softplus};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int lpc = scan::lanes_per_channel(N);
  int rc;
  switch (dtype) {
    case DUDY_DTYPE_F32:
      rc = scan::bwd_chain_f32(lpc, z.four, a, s, z.tiles, st);
      return rc ? rc : scan::bwd_sums<float>(a, o, s, z.tiles, st);
    case DUDY_DTYPE_F16:
      rc = scan::bwd_chain_f16(lpc, z.four, a, s, z.tiles, st);
      return rc ? rc : scan::bwd_sums<__half>(a, o, s, z.tiles, st);
    default:
      rc = scan::bwd_chain_bf16(lpc, z.four, a, s, z.tiles, st);
      return rc ? rc : scan::bwd_sums<__nv_bfloat16>(a, o, s, z.tiles, st);
  }
}

}  // extern "C"
