// torch_ext.cpp -- the torch-facing binding of libdudyconv_b200, built as the Python
// module `cuda_ops_ext`.
//
// It exposes the same surface the reference's Python layer binds to:
//   * pybind functions of `cuda_ops_ext` (reference cuda_ops/fused_dynamic_conv.cpp:58-101):
//     forward_chunk, forward_chunk_warmup, forward_chunk_cached_plan,
//     forward_chunk_clear_warmup_cache, forward_plan_name, backward_chunk,
//     backward_chunk_warmup, backward_chunk_cached_plan, backward_chunk_clear_warmup_cache,
//     backward_plan_name -- same argument names and defaults;
//   * TORCH_LIBRARY(fused_source_conv_mixed) with the 14 schemas of the reference
//     (cuda_ops/fused_source_conv_mixed_ops.cpp:354-505).
// Tensors are checked here (CUDA, dtype, shape; reference messages), outputs are
// allocated with the caching allocator, and all compute goes through the C ABI on the
// current stream. A nonzero C-ABI status becomes a RuntimeError (TORCH_CHECK).
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>
#include <torch/library.h>

#include <algorithm>
#include <cstdlib>
#include <map>
#include <mutex>
#include <string>
#include <tuple>
#include <vector>

#include "dudyconv_b200.h"

namespace {

int dtype_code(const torch::Tensor &t) {
  switch (t.scalar_type()) {
    case at::ScalarType::Float: return DUDY_DTYPE_F32;
    case at::ScalarType::Half: return DUDY_DTYPE_F16;
    case at::ScalarType::BFloat16: return DUDY_DTYPE_BF16;
    default: TORCH_CHECK(false, "Unsupported dtype: ", t.scalar_type(), ".");
  }
  return -1;
}

void check_status(int rc, const char *what) {
  TORCH_CHECK(rc == DUDY_OK, what, ": ", dudy_last_error(), " (status ", rc, ")");
}

bool debug_path() {
  static const bool on = std::getenv("DUDY_DEBUG_PATH") != nullptr ||
                         std::getenv("FDC_DEBUG_PATH") != nullptr;
  return on;
}

void *stream_ptr() { return reinterpret_cast<void *>(at::cuda::getCurrentCUDAStream().stream()); }

// ---------------------------------------------------------------------------------------
// dynamic conv
// ---------------------------------------------------------------------------------------
struct FdcDims {
  int64_t B, D, L, T, N, K;
};

// checks of the reference (cuda_ops/fused_dynamic_conv.py:108-186)
FdcDims check_fdc(const torch::Tensor &h, const torch::Tensor &kc, const torch::Tensor &mix,
                  int64_t off, int64_t dilation) {
  TORCH_CHECK(dilation > 0, "dilation must be positive.");
  TORCH_CHECK(h.is_cuda(), "h_full must be CUDA tensor.");
  TORCH_CHECK(kc.is_cuda(), "kernel_chunk must be CUDA tensor.");
  TORCH_CHECK(mix.is_cuda(), "kernel_mix must be CUDA tensor.");
  TORCH_CHECK(h.dim() == 3, "h_full must be [B,D,L], got ", h.sizes(), ".");
  TORCH_CHECK(kc.dim() == 4, "kernel_chunk must be [B,K,N,T], got ", kc.sizes(), ".");
  TORCH_CHECK(mix.dim() == 2, "kernel_mix must be [D,N], got ", mix.sizes(), ".");
  FdcDims d{h.size(0), h.size(1), h.size(2), kc.size(3), kc.size(2), kc.size(1)};
  TORCH_CHECK(kc.size(0) == d.B, "B mismatch: h_full=", d.B, ", kernel_chunk=", kc.size(0), ".");
  TORCH_CHECK(mix.size(0) == d.D, "D mismatch: h_full=", d.D, ", kernel_mix=", mix.size(0), ".");
  TORCH_CHECK(mix.size(1) == d.N, "N mismatch: kernel_chunk=", d.N, ", kernel_mix=", mix.size(1), ".");
  TORCH_CHECK(d.T > 0, "T must be positive.");
  TORCH_CHECK(d.K > 0, "K must be positive.");
  TORCH_CHECK(off >= 0, "t_offset must be non-negative.");
  TORCH_CHECK(off + d.T <= d.L, "t_offset + T must be <= L, got t_offset=", off, ", T=", d.T,
              ", L=", d.L, ".");
  dtype_code(h);
  TORCH_CHECK(kc.scalar_type() == h.scalar_type(), "kernel_chunk dtype must equal h_full dtype.");
  TORCH_CHECK(mix.scalar_type() == h.scalar_type(), "kernel_mix dtype must equal h_full dtype.");
  TORCH_CHECK(kc.device() == h.device() && mix.device() == h.device(),
              "all tensors must be on the same device.");
  TORCH_CHECK(h.is_contiguous() && kc.is_contiguous() && mix.is_contiguous(),
              "h, kc and mix must be contiguous.");
  return d;
}

void check_go(const torch::Tensor &go, const torch::Tensor &h, const FdcDims &d) {
  TORCH_CHECK(go.is_cuda(), "grad_out must be CUDA tensor.");
  TORCH_CHECK(go.dim() == 3, "grad_out must be [B,D,T], got ", go.sizes(), ".");
  TORCH_CHECK(go.size(0) == d.B, "grad_out B mismatch: grad_out=", go.size(0), ", h_full=", d.B, ".");
  TORCH_CHECK(go.size(1) == d.D, "grad_out D mismatch: grad_out=", go.size(1), ", h_full=", d.D, ".");
  TORCH_CHECK(go.size(2) == d.T, "grad_out T mismatch: grad_out=", go.size(2),
              ", kernel_chunk T=", d.T, ".");
  TORCH_CHECK(go.scalar_type() == h.scalar_type(), "grad_out dtype must equal h_full dtype.");
  TORCH_CHECK(go.device() == h.device(), "grad_out must be on the device of h.");
  TORCH_CHECK(go.is_contiguous(), "grad_out must be contiguous.");
}

using PlanKey = std::tuple<int, int, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                           int64_t>;
std::mutex g_mu;
std::map<PlanKey, int> g_fwd_cache, g_bwd_cache;

PlanKey make_key(const torch::Tensor &h, int64_t N, int64_t K, int64_t T, int64_t off,
                 int64_t dil) {
  return PlanKey{h.get_device(), dtype_code(h), h.size(0), h.size(1), h.size(2), T, N, K, off, dil};
}

int cached(std::map<PlanKey, int> &m, const PlanKey &k) {
  std::lock_guard<std::mutex> lk(g_mu);
  auto it = m.find(k);
  return it == m.end() ? -1 : it->second;
}

torch::Tensor fwd_run(const torch::Tensor &h, const torch::Tensor &kc, const torch::Tensor &mix,
                      const FdcDims &d, int64_t off, int64_t dil, int plan) {
  auto out = torch::empty({d.B, d.D, d.T}, h.options());
  const int rc = dudy_fdc_forward(h.data_ptr(), kc.data_ptr(), mix.data_ptr(), out.data_ptr(),
                                  d.B, d.D, d.L, d.T, d.N, d.K, off, dil, dtype_code(h), plan,
                                  stream_ptr());
  check_status(rc, "fused_dynamic_conv forward");
  return out;
}

std::vector<torch::Tensor> bwd_run(const torch::Tensor &go, const torch::Tensor &h,
                                   const torch::Tensor &kc, const torch::Tensor &mix,
                                   const FdcDims &d, int64_t off, int64_t dil, int plan) {
  auto gh = torch::empty_like(h);
  auto gk = torch::empty_like(kc);
  auto gm = torch::empty_like(mix);
  const int dt = dtype_code(h);
  const size_t ws_bytes =
      dudy_fdc_backward_workspace_size(d.B, d.D, d.L, d.T, d.N, d.K, off, dil, dt, plan);
  auto ws = torch::empty({(int64_t)std::max<size_t>(ws_bytes, 256)},
                         h.options().dtype(torch::kUInt8));
  const int rc = dudy_fdc_backward(go.data_ptr(), h.data_ptr(), kc.data_ptr(), mix.data_ptr(),
                                   gh.data_ptr(), gk.data_ptr(), gm.data_ptr(), ws.data_ptr(),
                                   (size_t)ws.numel(), d.B, d.D, d.L, d.T, d.N, d.K, off, dil, dt,
                                   plan, stream_ptr());
  check_status(rc, "fused_dynamic_conv backward");
  return {gh, gk, gm};
}

std::vector<int> candidate_plans(const torch::Tensor &h, const torch::Tensor &kc,
                                 const torch::Tensor &mix, const FdcDims &d, int64_t off,
                                 int64_t dil) {
  std::vector<int> c;
  const int dt = dtype_code(h);
  if (dudy_fdc_plan_available(DUDY_FDC_PLAN_TC, h.data_ptr(), kc.data_ptr(), mix.data_ptr(), d.B,
                              d.D, d.L, d.T, d.N, d.K, off, dil, dt))
    c.push_back(DUDY_FDC_PLAN_TC);
  c.push_back(DUDY_FDC_PLAN_SIMT);
  return c;
}

template <typename F>
float median_ms(F &&fn, int64_t repeat) {
  auto stream = at::cuda::getCurrentCUDAStream();
  fn();  // dry run
  std::vector<float> ms;
  cudaEvent_t a, b;
  cudaEventCreate(&a);
  cudaEventCreate(&b);
  for (int64_t i = 0; i < repeat; ++i) {
    cudaEventRecord(a, stream.stream());
    fn();
    cudaEventRecord(b, stream.stream());
    cudaEventSynchronize(b);
    float t = 0.f;
    cudaEventElapsedTime(&t, a, b);
    ms.push_back(t);
  }
  cudaEventDestroy(a);
  cudaEventDestroy(b);
  std::sort(ms.begin(), ms.end());
  return ms[ms.size() / 2];
}

torch::Tensor forward_chunk(torch::Tensor h, torch::Tensor kc, torch::Tensor mix, int64_t off,
                            int64_t dilation) {
  const FdcDims d = check_fdc(h, kc, mix, off, dilation);
  const c10::cuda::CUDAGuard guard(h.device());
  const int plan = cached(g_fwd_cache, make_key(h, d.N, d.K, d.T, off, dilation));
  if (debug_path())
    TORCH_WARN("[dudyconv] forward plan ", plan < 0 ? "auto" : dudy_fdc_plan_name(plan), " -> ",
               dudy_fdc_plan_name(dudy_fdc_default_plan(h.data_ptr(), kc.data_ptr(),
                                                        mix.data_ptr(), d.B, d.D, d.L, d.T, d.N,
                                                        d.K, off, dilation, dtype_code(h))));
  return fwd_run(h, kc, mix, d, off, dilation, plan);
}

int64_t forward_chunk_warmup(torch::Tensor h, torch::Tensor kc, torch::Tensor mix, int64_t off,
                             int64_t dilation, int64_t repeat) {
  TORCH_CHECK(repeat > 0, "repeat must be positive.");
  const FdcDims d = check_fdc(h, kc, mix, off, dilation);
  const c10::cuda::CUDAGuard guard(h.device());
  int best = -1;
  float best_ms = 1e30f;
  for (int p : candidate_plans(h, kc, mix, d, off, dilation)) {
    const float ms = median_ms([&] { fwd_run(h, kc, mix, d, off, dilation, p); }, repeat);
    if (debug_path()) TORCH_WARN("[dudyconv] forward warmup ", dudy_fdc_plan_name(p), ": ", ms, " ms");
    if (ms < best_ms) {
      best_ms = ms;
      best = p;
    }
  }
  std::lock_guard<std::mutex> lk(g_mu);
  g_fwd_cache[make_key(h, d.N, d.K, d.T, off, dilation)] = best;
  return best;
}

int64_t forward_chunk_cached_plan(torch::Tensor h, torch::Tensor kc, torch::Tensor mix,
                                  int64_t off, int64_t dilation) {
  const FdcDims d = check_fdc(h, kc, mix, off, dilation);
  return cached(g_fwd_cache, make_key(h, d.N, d.K, d.T, off, dilation));
}

void forward_chunk_clear_warmup_cache() {
  std::lock_guard<std::mutex> lk(g_mu);
  g_fwd_cache.clear();
}

std::string plan_name(int64_t plan_id) { return dudy_fdc_plan_name((int)plan_id); }

std::vector<torch::Tensor> backward_chunk(torch::Tensor go, torch::Tensor h, torch::Tensor kc,
                                          torch::Tensor mix, int64_t off, int64_t dilation) {
  const FdcDims d = check_fdc(h, kc, mix, off, dilation);
  check_go(go, h, d);
  const c10::cuda::CUDAGuard guard(h.device());
  const int plan = cached(g_bwd_cache, make_key(h, d.N, d.K, d.T, off, dilation));
  if (debug_path())
    TORCH_WARN("[dudyconv] backward plan ", plan < 0 ? "auto" : dudy_fdc_plan_name(plan));
  return bwd_run(go, h, kc, mix, d, off, dilation, plan);
}

int64_t backward_chunk_warmup(torch::Tensor go, torch::Tensor h, torch::Tensor kc,
                              torch::Tensor mix, int64_t off, int64_t dilation, int64_t repeat) {
  TORCH_CHECK(repeat > 0, "repeat must be positive.");
  const FdcDims d = check_fdc(h, kc, mix, off, dilation);
  check_go(go, h, d);
  const c10::cuda::CUDAGuard guard(h.device());
  int best = -1;
  float best_ms = 1e30f;
  for (int p : candidate_plans(h, kc, mix, d, off, dilation)) {
    const float ms = median_ms([&] { bwd_run(go, h, kc, mix, d, off, dilation, p); }, repeat);
    if (debug_path()) TORCH_WARN("[dudyconv] backward warmup ", dudy_fdc_plan_name(p), ": ", ms, " ms");
    if (ms < best_ms) {
      best_ms = ms;
      best = p;
    }
  }
  std::lock_guard<std::mutex> lk(g_mu);
  g_bwd_cache[make_key(h, d.N, d.K, d.T, off, dilation)] = best;
  return best;
}

int64_t backward_chunk_cached_plan(torch::Tensor h, torch::Tensor kc, int64_t off,
                                   int64_t dilation) {
  TORCH_CHECK(h.dim() == 3 && kc.dim() == 4, "h must be [B,D,L] and kc [B,K,N,T].");
  return cached(g_bwd_cache, make_key(h, kc.size(2), kc.size(1), kc.size(3), off, dilation));
}

void backward_chunk_clear_warmup_cache() {
  std::lock_guard<std::mutex> lk(g_mu);
  g_bwd_cache.clear();
}

// ---------------------------------------------------------------------------------------
// fused source conv (schemas of cuda_ops/fused_source_conv_mixed_ops.cpp:354-505)
// ---------------------------------------------------------------------------------------
struct FscmDims {
  int64_t B, D, L, C, S;
  bool has_bias;
};

FscmDims check_fscm(const torch::Tensor &x, const torch::Tensor &w, const torch::Tensor &bias,
                    const torch::Tensor &mw, const torch::Tensor &mb, int64_t off, int64_t T,
                    int64_t dil) {
  TORCH_CHECK(x.is_cuda() && w.is_cuda() && mw.is_cuda() && mb.is_cuda(),
              "fused_source_conv_mixed: tensors must be CUDA tensors.");
  TORCH_CHECK(x.dim() == 3, "x_norm must be [B,D,L], got ", x.sizes(), ".");
  TORCH_CHECK(w.dim() == 3, "weight must be [D,C,S], got ", w.sizes(), ".");
  TORCH_CHECK(mw.dim() == 2, "mix_weight must be [D,C], got ", mw.sizes(), ".");
  TORCH_CHECK(mb.dim() == 1, "mix_bias must be [D], got ", mb.sizes(), ".");
  FscmDims d{x.size(0), x.size(1), x.size(2), w.size(1), w.size(2),
             bias.defined() && bias.numel() > 0};
  TORCH_CHECK(w.size(0) == d.D, "weight D mismatch: weight=", w.size(0), ", x_norm=", d.D, ".");
  TORCH_CHECK(mw.size(0) == d.D && mw.size(1) == d.C, "mix_weight must be [D,C].");
  TORCH_CHECK(mb.size(0) == d.D, "mix_bias D mismatch: mix_bias=", mb.size(0), ", x_norm=", d.D, ".");
  if (d.has_bias) {
    TORCH_CHECK(bias.is_cuda(), "bias must be CUDA tensor when provided.");
    TORCH_CHECK(bias.dim() == 2 && bias.size(0) == d.D && bias.size(1) == d.C,
                "bias must be [D,C], got ", bias.sizes(), ".");
    TORCH_CHECK(bias.scalar_type() == x.scalar_type(), "bias dtype must equal x_norm dtype.");
    TORCH_CHECK(bias.is_contiguous(), "bias must be contiguous.");
  }
  dtype_code(x);
  TORCH_CHECK(w.scalar_type() == x.scalar_type(), "weight dtype must equal x_norm dtype.");
  TORCH_CHECK(mw.scalar_type() == x.scalar_type(), "mix_weight dtype must equal x_norm dtype.");
  TORCH_CHECK(mb.scalar_type() == x.scalar_type(), "mix_bias dtype must equal x_norm dtype.");
  TORCH_CHECK(off >= 0, "off must be non-negative.");
  TORCH_CHECK(T > 0, "T must be positive.");
  TORCH_CHECK(off + T <= d.L, "off + T must be <= L, got off=", off, ", T=", T, ", L=", d.L, ".");
  TORCH_CHECK(dil > 0, "dilation must be positive.");
  TORCH_CHECK(x.is_contiguous() && w.is_contiguous() && mw.is_contiguous() && mb.is_contiguous(),
              "fused_source_conv_mixed: tensors must be contiguous.");
  return d;
}

torch::Tensor fscm_fwd(const torch::Tensor &x, const torch::Tensor &w, const torch::Tensor &bias,
                       const torch::Tensor &mw, const torch::Tensor &mb, int64_t off, int64_t T,
                       int64_t dil, int64_t plan) {
  const FscmDims d = check_fscm(x, w, bias, mw, mb, off, T, dil);
  const c10::cuda::CUDAGuard guard(x.device());
  auto out = torch::empty({d.B, d.D, T}, x.options());
  const int rc = dudy_fscm_forward(x.data_ptr(), w.data_ptr(), d.has_bias ? bias.data_ptr() : nullptr,
                                   mw.data_ptr(), mb.data_ptr(), out.data_ptr(), d.B, d.D, d.L, d.C,
                                   d.S, off, T, dil, dtype_code(x), (int)plan, stream_ptr());
  check_status(rc, "fused_source_conv_mixed forward");
  return out;
}

std::vector<torch::Tensor> fscm_bwd(const torch::Tensor &go, const torch::Tensor &x,
                                    const torch::Tensor &w, const torch::Tensor &bias,
                                    const torch::Tensor &mw, const torch::Tensor &mb, int64_t off,
                                    int64_t T, int64_t dil, int64_t plan, int64_t tile_t) {
  const FscmDims d = check_fscm(x, w, bias, mw, mb, off, T, dil);
  TORCH_CHECK(go.is_cuda() && go.dim() == 3, "grad_out must be [B,D,T], got ", go.sizes(), ".");
  TORCH_CHECK(go.size(0) == d.B && go.size(1) == d.D && go.size(2) == T,
              "grad_out must be [B,D,T], got ", go.sizes(), ".");
  TORCH_CHECK(go.scalar_type() == x.scalar_type(), "grad_out dtype must equal x_norm dtype.");
  TORCH_CHECK(go.is_contiguous(), "grad_out must be contiguous.");
  const c10::cuda::CUDAGuard guard(x.device());
  auto gx = torch::empty_like(x);
  auto gw = torch::empty_like(w);
  auto gb = d.has_bias ? torch::empty_like(bias) : torch::empty({0}, x.options());
  auto gmw = torch::empty_like(mw);
  auto gmb = torch::empty_like(mb);
  const int dt = dtype_code(x);
  const size_t ws_bytes = dudy_fscm_backward_workspace_size(d.B, d.D, d.L, d.C, d.S, off, T, dil,
                                                            dt, (int)plan, tile_t);
  auto ws = torch::empty({(int64_t)std::max<size_t>(ws_bytes, 256)}, x.options().dtype(torch::kUInt8));
  const int rc = dudy_fscm_backward(
      go.data_ptr(), x.data_ptr(), w.data_ptr(), d.has_bias ? bias.data_ptr() : nullptr,
      mw.data_ptr(), mb.data_ptr(), gx.data_ptr(), gw.data_ptr(),
      d.has_bias ? gb.data_ptr() : nullptr, gmw.data_ptr(), gmb.data_ptr(), ws.data_ptr(),
      (size_t)ws.numel(), d.B, d.D, d.L, d.C, d.S, off, T, dil, dt, (int)plan, tile_t,
      stream_ptr());
  check_status(rc, "fused_source_conv_mixed backward");
  return {gx, gw, gb, gmw, gmb};
}

torch::Tensor fscm_forward_op(torch::Tensor x, torch::Tensor w, torch::Tensor bias,
                              torch::Tensor mw, torch::Tensor mb, int64_t off, int64_t T,
                              int64_t dil) {
  return fscm_fwd(x, w, bias, mw, mb, off, T, dil, DUDY_PLAN_AUTO);
}

torch::Tensor fscm_forward_plan_op(torch::Tensor x, torch::Tensor w, torch::Tensor bias,
                                   torch::Tensor mw, torch::Tensor mb, int64_t off, int64_t T,
                                   int64_t dil, int64_t plan) {
  TORCH_CHECK(dudy_fscm_forward_plan_legal((int)plan, x.size(1), w.size(1), w.size(2), off, dil),
              "fused_source_conv_mixed_forward_plan_cuda: illegal plan=", plan);
  return fscm_fwd(x, w, bias, mw, mb, off, T, dil, plan);
}

torch::Tensor fscm_forward_cached_plan_op(torch::Tensor x, torch::Tensor w, torch::Tensor bias,
                                          torch::Tensor mw, torch::Tensor mb, int64_t off,
                                          int64_t T, int64_t dil, int64_t cached_plan) {
  return fscm_forward_plan_op(x, w, bias, mw, mb, off, T, dil, cached_plan);
}

template <typename F>
float avg_ms(F &&fn, int64_t warmup_iters, int64_t bench_iters) {
  auto stream = at::cuda::getCurrentCUDAStream();
  for (int64_t i = 0; i < warmup_iters; ++i) fn();
  cudaEvent_t a, b;
  cudaEventCreate(&a);
  cudaEventCreate(&b);
  cudaEventRecord(a, stream.stream());
  for (int64_t i = 0; i < bench_iters; ++i) fn();
  cudaEventRecord(b, stream.stream());
  cudaEventSynchronize(b);
  float t = 0.f;
  cudaEventElapsedTime(&t, a, b);
  cudaEventDestroy(a);
  cudaEventDestroy(b);
  return t / (float)bench_iters;
}

int64_t fscm_forward_warmup_op(torch::Tensor x, torch::Tensor w, torch::Tensor bias,
                               torch::Tensor mw, torch::Tensor mb, int64_t off, int64_t T,
                               int64_t dil, int64_t warmup_iters, int64_t bench_iters) {
  TORCH_CHECK(warmup_iters >= 0, "fused_source_conv_mixed_forward_warmup_cuda: warmup_iters must be >= 0.");
  TORCH_CHECK(bench_iters > 0, "fused_source_conv_mixed_forward_warmup_cuda: bench_iters must be > 0.");
  check_fscm(x, w, bias, mw, mb, off, T, dil);
  const int64_t D = x.size(1), C = w.size(1), S = w.size(2);
  // candidate order of the reference (fused_source_conv_mixed_forward.cu:367-437)
  const int order[8] = {103, 101, 102, 100, 3, 1, 2, 0};
  int64_t best = -1;
  float best_ms = 1e30f;
  for (int p : order) {
    if (!dudy_fscm_forward_plan_legal(p, D, C, S, off, dil)) continue;
    const float ms = avg_ms([&] { fscm_fwd(x, w, bias, mw, mb, off, T, dil, p); }, warmup_iters, bench_iters);
    if (ms < best_ms) {
      best_ms = ms;
      best = p;
    }
  }
  return best;
}

std::vector<torch::Tensor> fscm_backward_op(torch::Tensor go, torch::Tensor x, torch::Tensor w,
                                            torch::Tensor bias, torch::Tensor mw, torch::Tensor mb,
                                            int64_t off, int64_t T, int64_t dil) {
  const int64_t tile = std::min<int64_t>(64, T);
  const int plan = dudy_fscm_backward_default_plan(x.size(0), x.size(1), x.size(2), w.size(1),
                                                   w.size(2), off, T, dil);
  return fscm_bwd(go, x, w, bias, mw, mb, off, T, dil, plan, plan == 0 ? 0 : tile);
}

std::vector<torch::Tensor> fscm_backward_plan_op(torch::Tensor go, torch::Tensor x,
                                                 torch::Tensor w, torch::Tensor bias,
                                                 torch::Tensor mw, torch::Tensor mb, int64_t off,
                                                 int64_t T, int64_t dil, int64_t plan,
                                                 int64_t tile_t) {
  TORCH_CHECK(dudy_fscm_backward_plan_legal((int)plan, w.size(1), w.size(2), tile_t),
              "fused_source_conv_mixed_backward_plan_cuda: illegal plan=", plan, ", tile_t=", tile_t);
  return fscm_bwd(go, x, w, bias, mw, mb, off, T, dil, plan, tile_t);
}

int64_t pack_plan(int64_t plan, int64_t tile_t) {
  const uint64_t p = (uint64_t)(uint32_t)plan, t = (uint64_t)(uint32_t)tile_t;
  return (int64_t)(p | (t << 32));
}
int64_t unpack_plan(int64_t packed) { return (int64_t)((uint64_t)packed & 0xffffffffull); }
int64_t unpack_tile(int64_t packed) { return (int64_t)(((uint64_t)packed >> 32) & 0xffffffffull); }

std::vector<torch::Tensor> fscm_backward_cached_plan_op(torch::Tensor go, torch::Tensor x,
                                                        torch::Tensor w, torch::Tensor bias,
                                                        torch::Tensor mw, torch::Tensor mb,
                                                        int64_t off, int64_t T, int64_t dil,
                                                        int64_t cached_plan) {
  const int64_t plan = unpack_plan(cached_plan);
  const int64_t tile = plan == 0 ? 0 : unpack_tile(cached_plan);
  return fscm_backward_plan_op(go, x, w, bias, mw, mb, off, T, dil, plan, tile);
}

int64_t fscm_backward_warmup_op(torch::Tensor go, torch::Tensor x, torch::Tensor w,
                                torch::Tensor bias, torch::Tensor mw, torch::Tensor mb,
                                int64_t off, int64_t T, int64_t dil, int64_t warmup_iters,
                                int64_t bench_iters) {
  TORCH_CHECK(warmup_iters >= 0, "fused_source_conv_mixed_backward_warmup_cuda: warmup_iters must be >= 0.");
  TORCH_CHECK(bench_iters > 0, "fused_source_conv_mixed_backward_warmup_cuda: bench_iters must be > 0.");
  check_fscm(x, w, bias, mw, mb, off, T, dil);
  const int64_t C = w.size(1), S = w.size(2);
  // candidates of the reference (fused_source_conv_mixed_backward.cu:395-466)
  std::vector<std::pair<int, int64_t>> cands{{0, 0}};
  if (C <= 64 && S <= 8) {
    for (int64_t t : {64, 128, 256}) {
      const int64_t tt = (t > T) ? T : t;
      cands.push_back({1, tt});
      cands.push_back({2, tt});
    }
  }
  int best = 0;
  int64_t best_tile = 0;
  float best_ms = 1e30f;
  for (auto &c : cands) {
    const float ms = avg_ms([&] { fscm_bwd(go, x, w, bias, mw, mb, off, T, dil, c.first, c.second); },
                            warmup_iters, bench_iters);
    if (ms < best_ms) {
      best_ms = ms;
      best = c.first;
      best_tile = c.second;
    }
  }
  return pack_plan(best, best == 0 ? 0 : best_tile);
}

std::vector<torch::Tensor> fscm_backward_atomic_op(torch::Tensor go, torch::Tensor x,
                                                   torch::Tensor w, torch::Tensor bias,
                                                   torch::Tensor mw, torch::Tensor mb, int64_t off,
                                                   int64_t T, int64_t dil) {
  return fscm_bwd(go, x, w, bias, mw, mb, off, T, dil, 0, 0);
}

std::vector<torch::Tensor> fscm_backward_per_d_reduce_op(torch::Tensor go, torch::Tensor x,
                                                         torch::Tensor w, torch::Tensor bias,
                                                         torch::Tensor mw, torch::Tensor mb,
                                                         int64_t off, int64_t T, int64_t dil,
                                                         int64_t tile_t) {
  return fscm_backward_plan_op(go, x, w, bias, mw, mb, off, T, dil, 1, tile_t);
}

std::vector<torch::Tensor> fscm_backward_gather_x_op(torch::Tensor go, torch::Tensor x,
                                                     torch::Tensor w, torch::Tensor bias,
                                                     torch::Tensor mw, torch::Tensor mb,
                                                     int64_t off, int64_t T, int64_t dil,
                                                     int64_t tile_t) {
  return fscm_backward_plan_op(go, x, w, bias, mw, mb, off, T, dil, 2, tile_t);
}

// ---------------------------------------------------------------------------------------
// kernel generator tail: logits [B, N*K, T] -> kernel_chunk [B, K, N, T] (softmax over K,
// flip), and its backward; no counterpart in the reference's binding (the reference runs
// StreamingKernelGenConv1d._logits_to_kernel in PyTorch, backbone_dil_unshared.py:1821-1900)
// ---------------------------------------------------------------------------------------
torch::Tensor logits_to_kernel(torch::Tensor logits, int64_t num_kernels, int64_t kernel_size) {
  TORCH_CHECK(logits.is_cuda(), "logits must be CUDA tensor.");
  TORCH_CHECK(logits.dim() == 3, "logits must be [B,N*K,T], got ", logits.sizes(), ".");
  TORCH_CHECK(num_kernels > 0 && kernel_size > 0, "num_kernels and kernel_size must be positive.");
  TORCH_CHECK(logits.size(1) == num_kernels * kernel_size, "logits channels must be N*K=",
              num_kernels * kernel_size, ", got ", logits.size(1), ".");
  TORCH_CHECK(logits.is_contiguous(), "logits must be contiguous.");
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t B = logits.size(0), T = logits.size(2);
  auto kc = torch::empty({B, kernel_size, num_kernels, T}, logits.options());
  check_status(dudy_logits_to_kernel(logits.data_ptr(), kc.data_ptr(), B, num_kernels,
                                     kernel_size, T, dtype_code(logits), stream_ptr()),
               "logits_to_kernel");
  return kc;
}

torch::Tensor logits_to_kernel_backward(torch::Tensor kc, torch::Tensor grad_kc) {
  TORCH_CHECK(kc.is_cuda() && grad_kc.is_cuda(), "kc and grad_kc must be CUDA tensors.");
  TORCH_CHECK(kc.dim() == 4 && grad_kc.sizes() == kc.sizes(),
              "kc and grad_kc must both be [B,K,N,T].");
  TORCH_CHECK(grad_kc.scalar_type() == kc.scalar_type(), "grad_kc dtype must equal kc dtype.");
  TORCH_CHECK(kc.is_contiguous() && grad_kc.is_contiguous(), "kc and grad_kc must be contiguous.");
  const c10::cuda::CUDAGuard guard(kc.device());
  const int64_t B = kc.size(0), K = kc.size(1), N = kc.size(2), T = kc.size(3);
  auto gl = torch::empty({B, N * K, T}, kc.options());
  check_status(dudy_logits_to_kernel_backward(kc.data_ptr(), grad_kc.data_ptr(), gl.data_ptr(),
                                              B, N, K, T, dtype_code(kc), stream_ptr()),
               "logits_to_kernel_backward");
  return gl;
}

// ---------------------------------------------------------------------------------------
// state-space block (no counterpart in the reference): short causal conv, selective scan, and
// the norms, gate and residual between blocks. Optional tensors come as None.
// ---------------------------------------------------------------------------------------
using OptTensor = c10::optional<torch::Tensor>;

const void *opt_ptr(const OptTensor &t) { return t.has_value() ? t->data_ptr() : nullptr; }

OptTensor contig(const OptTensor &t) {
  return t.has_value() ? OptTensor(t->contiguous()) : t;
}

bool differentiated(const OptTensor &t) { return t.has_value() && t->requires_grad(); }

template <typename... Ts>
bool wants_grad(const Ts &...ts) {
  return at::GradMode::is_enabled() && (differentiated(ts) || ...);
}

// An output without a tangent would count inputs that carry one as constants.
template <typename... Ts>
void refuse_tangents(const char *what, const Ts &...ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  auto dual = [](const OptTensor &t) { return t.has_value() && t->_fw_grad(0).defined(); };
  TORCH_CHECK(!(dual(ts) || ...), what, " has no forward-mode derivative.");
}

// autograd's saved tensors: what was None comes back undefined
torch::Tensor or_undefined(const OptTensor &t) { return t.has_value() ? *t : torch::Tensor(); }
OptTensor or_none(const torch::Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// A kernel wrote t through its pointer: a graph that kept t for its backward must not use it now.
// (Tensors made in inference mode have no version and are kept by none.)
void written(const torch::Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// in a backward that is itself being recorded
void refuse_twice(const char *what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " cannot be differentiated twice.");
}

// A [..] tensor of `like`'s device and of type `dt`, with the given sizes
void check_like(const torch::Tensor &t, const char *name, at::IntArrayRef sizes,
                at::ScalarType dt, const torch::Tensor &like) {
  TORCH_CHECK(t.is_cuda(), name, " must be CUDA tensor.");
  TORCH_CHECK(t.device() == like.device(), "all tensors must be on the same device.");
  TORCH_CHECK(t.sizes() == sizes, name, " must be ", sizes, ", got ", t.sizes(), ".");
  TORCH_CHECK(t.scalar_type() == dt, name, " must be ", dt, ", got ", t.scalar_type(), ".");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous.");
}

void check_like(const OptTensor &t, const char *name, at::IntArrayRef sizes, at::ScalarType dt,
                const torch::Tensor &like) {
  if (t.has_value()) check_like(*t, name, sizes, dt, like);
}

// An output or scratch, straight from the caching allocator: through the dispatcher each cost
// twice as much, and a backward makes up to ten.
torch::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const torch::Tensor &like) {
  return torch::Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

torch::Tensor fresh_like(const torch::Tensor &t) { return fresh(t.sizes(), t.scalar_type(), t); }

torch::Tensor scratch(size_t bytes, const torch::Tensor &like) {
  return fresh({(int64_t)std::max<size_t>(bytes, 16)}, torch::kUInt8, like);
}

torch::Tensor floats(at::IntArrayRef sizes, const torch::Tensor &like) {
  return fresh(sizes, torch::kFloat32, like);
}

void check_seq(const torch::Tensor &x, const char *name) {
  TORCH_CHECK(x.is_cuda(), name, " must be CUDA tensor.");
  TORCH_CHECK(x.dim() == 3, name, " must be [B,D,L], got ", x.sizes(), ".");
  TORCH_CHECK(x.is_contiguous(), name, " must be contiguous.");
  TORCH_CHECK(x.numel() > 0, "B, D and L must be positive.");
  dtype_code(x);
}

void check_short_conv(const torch::Tensor &x, const torch::Tensor &w, const OptTensor &bias,
                      const OptTensor &state, const OptTensor &lengths) {
  check_seq(x, "x");
  TORCH_CHECK(w.dim() == 2, "weight must be [D,S], got ", w.sizes(), ".");
  const int64_t B = x.size(0), D = x.size(1), S = w.size(1);
  TORCH_CHECK(S >= 2 && S <= DUDY_SHORT_CONV_MAX_TAPS, "S must be between 2 and ",
              DUDY_SHORT_CONV_MAX_TAPS, ", got ", S, ".");
  check_like(w, "weight", {D, S}, x.scalar_type(), x);
  check_like(bias, "bias", {D}, x.scalar_type(), x);
  check_like(state, "initial_state", {B, D, S - 1}, x.scalar_type(), x);
  check_like(lengths, "lengths", {B}, at::kInt, x);
}

std::vector<torch::Tensor> short_conv_forward(torch::Tensor x, torch::Tensor w, OptTensor bias,
                                              OptTensor state, OptTensor lengths, bool silu,
                                              bool want_final) {
  check_short_conv(x, w, bias, state, lengths);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t B = x.size(0), D = x.size(1), L = x.size(2), S = w.size(1);
  std::vector<torch::Tensor> out{fresh_like(x)};
  if (want_final) out.push_back(fresh({B, D, S - 1}, x.scalar_type(), x));
  check_status(dudy_short_conv_forward(
                   x.data_ptr(), w.data_ptr(), opt_ptr(bias), opt_ptr(state),
                   (const int32_t *)opt_ptr(lengths), out[0].data_ptr(),
                   want_final ? out[1].data_ptr() : nullptr, B, D, L, S, silu, dtype_code(x),
                   stream_ptr()),
               "fused_short_conv forward");
  return out;
}

// grad_x, grad_weight, grad_bias (empty without a bias), grad_state (empty unless wanted)
std::vector<torch::Tensor> short_conv_backward(torch::Tensor go, OptTensor gfinal,
                                               torch::Tensor x, torch::Tensor w, OptTensor bias,
                                               OptTensor state, OptTensor lengths, bool silu,
                                               bool want_state) {
  check_short_conv(x, w, bias, state, lengths);
  const int64_t B = x.size(0), D = x.size(1), L = x.size(2), S = w.size(1);
  check_like(go, "grad_out", x.sizes(), x.scalar_type(), x);
  check_like(gfinal, "grad_final_state", {B, D, S - 1}, x.scalar_type(), x);
  const c10::cuda::CUDAGuard guard(x.device());
  auto gx = fresh_like(x), gw = fresh_like(w);
  auto gb = fresh({bias.has_value() ? D : 0}, x.scalar_type(), x);
  auto gs = want_state ? fresh({B, D, S - 1}, x.scalar_type(), x) : fresh({0}, x.scalar_type(), x);
  const int dt = dtype_code(x);
  auto ws = scratch(dudy_short_conv_backward_workspace_size(B, D, L, S, dt), x);
  check_status(dudy_short_conv_backward(
                   go.data_ptr(), opt_ptr(gfinal), x.data_ptr(), w.data_ptr(), opt_ptr(bias),
                   opt_ptr(state), (const int32_t *)opt_ptr(lengths), gx.data_ptr(),
                   gw.data_ptr(), bias.has_value() ? gb.data_ptr() : nullptr,
                   want_state ? gs.data_ptr() : nullptr, ws.data_ptr(), (size_t)ws.numel(), B, D,
                   L, S, silu, dt, stream_ptr()),
               "fused_short_conv backward");
  return {gx, gw, gb, gs};
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct ShortConvFn : public torch::autograd::Function<ShortConvFn> {
  static variable_list forward(AutogradContext *ctx, torch::Tensor x, torch::Tensor w,
                               OptTensor bias, OptTensor state, OptTensor lengths, bool silu,
                               bool want_final) {
    // asked before the copies: made without gradients, they no longer say what was given
    const bool want_state = differentiated(state);
    x = x.contiguous();
    w = w.contiguous();
    bias = contig(bias);
    state = contig(state);
    lengths = contig(lengths);
    auto out = short_conv_forward(x, w, bias, state, lengths, silu, want_final);
    ctx->save_for_backward(
        {x, w, or_undefined(bias), or_undefined(state), or_undefined(lengths)});
    ctx->saved_data["silu"] = silu;
    ctx->saved_data["want_state"] = want_state;
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    refuse_twice("fused_short_conv");
    const auto v = ctx->get_saved_variables();
    variable_list none(7);
    const bool final_grad = g.size() > 1 && g[1].defined();
    if (!g[0].defined() && !final_grad) return none;
    auto go = g[0].defined() ? g[0].contiguous() : torch::zeros_like(v[0]);
    auto r = short_conv_backward(go, final_grad ? OptTensor(g[1].contiguous()) : OptTensor(), v[0],
                                 v[1], or_none(v[2]), or_none(v[3]), or_none(v[4]),
                                 ctx->saved_data["silu"].toBool(),
                                 ctx->saved_data["want_state"].toBool());
    for (int i = 0; i < 4; ++i)
      if (i < 2 || r[i].numel() > 0) none[i] = r[i];
    return none;
  }
};

// out and, where wanted, the final state; recorded for the backward where an input asks for it
std::vector<torch::Tensor> short_conv(torch::Tensor x, torch::Tensor w, OptTensor bias,
                                      OptTensor state, OptTensor lengths, bool silu,
                                      bool want_final) {
  refuse_tangents("fused_short_conv", x, w, bias, state);
  if (wants_grad(x, w, bias, state))
    return ShortConvFn::apply(x, w, bias, state, lengths, silu, want_final);
  return short_conv_forward(x.contiguous(), w.contiguous(), contig(bias), contig(state),
                            contig(lengths), silu, want_final);
}

torch::Tensor short_conv_step(torch::Tensor x, torch::Tensor state, torch::Tensor w,
                              OptTensor bias, bool silu) {
  refuse_tangents("fused_short_conv_step", x, state, w, bias);
  TORCH_CHECK(!wants_grad(x, state, w, bias),
              "fused_short_conv_step has no backward: call it under torch.no_grad().");
  x = x.contiguous();
  w = w.contiguous();
  bias = contig(bias);
  TORCH_CHECK(x.is_cuda(), "x must be CUDA tensor.");
  TORCH_CHECK(x.dim() == 2 && x.numel() > 0, "x must be [B,D], got ", x.sizes(), ".");
  TORCH_CHECK(x.is_contiguous(), "x must be contiguous.");
  TORCH_CHECK(w.dim() == 2, "weight must be [D,S], got ", w.sizes(), ".");
  const int64_t B = x.size(0), D = x.size(1), S = w.size(1);
  const int dt = dtype_code(x);
  check_like(w, "weight", {D, S}, x.scalar_type(), x);
  check_like(bias, "bias", {D}, x.scalar_type(), x);
  check_like(state, "conv_state", {B, D, S - 1}, x.scalar_type(), x);
  const c10::cuda::CUDAGuard guard(x.device());
  auto out = fresh_like(x);
  check_status(dudy_short_conv_step(x.data_ptr(), state.data_ptr(), w.data_ptr(), opt_ptr(bias),
                                    out.data_ptr(), B, D, S, silu, dt, stream_ptr()),
               "fused_short_conv step");
  written(state);
  return out;
}

struct ScanDims {
  int64_t B, D, L, N, G;
};

// u is [B,D,L] (L given) or [B,D] (L = 0: one token)
ScanDims check_scan(const torch::Tensor &u, const torch::Tensor &delta, const torch::Tensor &A,
                    const torch::Tensor &Bm, const torch::Tensor &Cm, const OptTensor &skip,
                    const OptTensor &bias, bool token) {
  if (token) {
    TORCH_CHECK(u.is_cuda(), "u must be CUDA tensor.");
    TORCH_CHECK(u.dim() == 2 && u.numel() > 0, "u must be [B,D], got ", u.sizes(), ".");
    TORCH_CHECK(u.is_contiguous(), "u must be contiguous.");
    dtype_code(u);
  } else {
    check_seq(u, "u");
  }
  TORCH_CHECK(A.dim() == 2, "A must be [D,N], got ", A.sizes(), ".");
  TORCH_CHECK(Bm.dim() == u.dim() + 1, token ? "B must be [B,G,N], got " : "B must be [B,G,N,L], got ",
              Bm.sizes(), ".");
  const ScanDims d{u.size(0), u.size(1), token ? 1 : u.size(2), A.size(1), Bm.size(1)};
  TORCH_CHECK(d.N >= 1 && d.N <= DUDY_SCAN_MAX_STATE, "N must be between 1 and ",
              DUDY_SCAN_MAX_STATE, ", got ", d.N, ".");
  TORCH_CHECK(d.G > 0 && d.D % d.G == 0, "D must be a multiple of the number of groups, got D=",
              d.D, ", G=", d.G, ".");
  const auto dt = u.scalar_type();
  check_like(delta, "delta", u.sizes(), dt, u);
  check_like(A, "A", {d.D, d.N}, at::kFloat, u);
  std::vector<int64_t> bc{d.B, d.G, d.N};
  if (!token) bc.push_back(d.L);
  check_like(Bm, "B", bc, dt, u);
  check_like(Cm, "C", bc, dt, u);
  check_like(skip, "skip", {d.D}, at::kFloat, u);
  check_like(bias, "delta_bias", {d.D}, at::kFloat, u);
  return d;
}

// y, final_state (empty unless wanted), checkpoints (empty unless wanted)
std::vector<torch::Tensor> selective_scan_forward(torch::Tensor u, torch::Tensor delta,
                                                  torch::Tensor A, torch::Tensor Bm,
                                                  torch::Tensor Cm, OptTensor skip,
                                                  OptTensor bias, OptTensor state,
                                                  OptTensor lengths, bool softplus,
                                                  bool want_final, bool want_ckpt) {
  const ScanDims d = check_scan(u, delta, A, Bm, Cm, skip, bias, false);
  check_like(state, "initial_state", {d.B, d.D, d.N}, at::kFloat, u);
  check_like(lengths, "lengths", {d.B}, at::kInt, u);
  const c10::cuda::CUDAGuard guard(u.device());
  const int dt = dtype_code(u);
  auto y = fresh_like(u);
  auto fin = want_final ? floats({d.B, d.D, d.N}, u) : torch::Tensor();
  auto ck = want_ckpt
                ? scratch(dudy_selective_scan_checkpoint_bytes(d.B, d.D, d.L, d.N, d.G, dt), u)
                : torch::Tensor();
  const size_t ws_bytes =
      dudy_selective_scan_forward_workspace_size(d.B, d.D, d.L, d.N, d.G, dt);
  auto ws = ws_bytes ? scratch(ws_bytes, u) : torch::Tensor();
  check_status(dudy_selective_scan_forward(
                   u.data_ptr(), delta.data_ptr(), (const float *)A.data_ptr(), Bm.data_ptr(),
                   Cm.data_ptr(), (const float *)opt_ptr(skip), (const float *)opt_ptr(bias),
                   (const float *)opt_ptr(state), (const int32_t *)opt_ptr(lengths), y.data_ptr(),
                   want_final ? (float *)fin.data_ptr() : nullptr,
                   want_ckpt ? (float *)ck.data_ptr() : nullptr,
                   ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, d.B, d.D, d.L, d.N, d.G,
                   softplus, dt, stream_ptr()),
               "fused_selective_scan forward");
  return {y, fin, ck};
}

// grad u, delta, A, B, C, skip, delta_bias, state (undefined where there is no such input)
std::vector<torch::Tensor> selective_scan_backward(torch::Tensor go, OptTensor gfinal,
                                                   torch::Tensor u, torch::Tensor delta,
                                                   torch::Tensor A, torch::Tensor Bm,
                                                   torch::Tensor Cm, OptTensor skip,
                                                   OptTensor bias, torch::Tensor ckpt,
                                                   OptTensor lengths, bool softplus,
                                                   bool want_state) {
  const ScanDims d = check_scan(u, delta, A, Bm, Cm, skip, bias, false);
  check_like(go, "grad_out", u.sizes(), u.scalar_type(), u);
  check_like(gfinal, "grad_final_state", {d.B, d.D, d.N}, at::kFloat, u);
  check_like(lengths, "lengths", {d.B}, at::kInt, u);
  const int dt = dtype_code(u);
  TORCH_CHECK(ckpt.is_cuda() && ckpt.device() == u.device() &&
                  (size_t)ckpt.nbytes() >=
                      dudy_selective_scan_checkpoint_bytes(d.B, d.D, d.L, d.N, d.G, dt),
              "checkpoints do not belong to these inputs.");
  const c10::cuda::CUDAGuard guard(u.device());
  auto gu = fresh_like(u), gd = fresh_like(u), gA = fresh_like(A);
  auto gB = fresh_like(Bm), gC = fresh_like(Cm);
  auto gs = skip.has_value() ? floats({d.D}, u) : torch::Tensor();
  auto gb = bias.has_value() ? floats({d.D}, u) : torch::Tensor();
  auto gst = want_state ? floats({d.B, d.D, d.N}, u) : torch::Tensor();
  auto ws = scratch(dudy_selective_scan_backward_workspace_size(d.B, d.D, d.L, d.N, d.G, dt), u);
  auto fp = [](const torch::Tensor &t) { return t.defined() ? (float *)t.data_ptr() : nullptr; };
  check_status(dudy_selective_scan_backward(
                   go.data_ptr(), (const float *)opt_ptr(gfinal), u.data_ptr(), delta.data_ptr(),
                   (const float *)A.data_ptr(), Bm.data_ptr(), Cm.data_ptr(),
                   (const float *)opt_ptr(skip), (const float *)opt_ptr(bias),
                   (const float *)ckpt.data_ptr(), (const int32_t *)opt_ptr(lengths),
                   gu.data_ptr(), gd.data_ptr(), (float *)gA.data_ptr(), gB.data_ptr(),
                   gC.data_ptr(), fp(gs), fp(gb), fp(gst), ws.data_ptr(), (size_t)ws.numel(), d.B,
                   d.D, d.L, d.N, d.G, softplus, dt, stream_ptr()),
               "fused_selective_scan backward");
  return {gu, gd, gA, gB, gC, gs, gb, gst};
}

// [B,N,L] (or [B,N] of one token) is one group
torch::Tensor grouped(const torch::Tensor &t, int64_t dims) {
  return (t.dim() == dims - 1 ? t.unsqueeze(1) : t).contiguous();
}

struct SelectiveScanFn : public torch::autograd::Function<SelectiveScanFn> {
  static variable_list forward(AutogradContext *ctx, torch::Tensor u, torch::Tensor delta,
                               torch::Tensor A, torch::Tensor Bm, torch::Tensor Cm,
                               OptTensor skip, OptTensor bias, OptTensor state,
                               OptTensor lengths, bool softplus, bool want_final) {
    const bool b3 = Bm.dim() == 3, c3 = Cm.dim() == 3;
    const bool want_state = differentiated(state);  // before the copies, as in the conv
    u = u.contiguous();
    delta = delta.contiguous();
    A = A.contiguous();
    Bm = grouped(Bm, 4);
    Cm = grouped(Cm, 4);
    skip = contig(skip);
    bias = contig(bias);
    state = contig(state);
    lengths = contig(lengths);
    auto r = selective_scan_forward(u, delta, A, Bm, Cm, skip, bias, state, lengths, softplus,
                                    want_final, true);
    ctx->save_for_backward({u, delta, A, Bm, Cm, or_undefined(skip), or_undefined(bias), r[2],
                            or_undefined(lengths)});
    ctx->saved_data["softplus"] = softplus;
    ctx->saved_data["want_state"] = want_state;
    ctx->saved_data["b3"] = b3;
    ctx->saved_data["c3"] = c3;
    ctx->set_materialize_grads(false);
    return want_final ? variable_list{r[0], r[1]} : variable_list{r[0]};
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    refuse_twice("fused_selective_scan");
    const auto v = ctx->get_saved_variables();
    variable_list out(11);
    const bool final_grad = g.size() > 1 && g[1].defined();
    if (!g[0].defined() && !final_grad) return out;
    auto go = g[0].defined() ? g[0].contiguous() : torch::zeros_like(v[0]);
    auto r = selective_scan_backward(
        go, final_grad ? OptTensor(g[1].contiguous()) : OptTensor(), v[0], v[1], v[2], v[3], v[4],
        or_none(v[5]), or_none(v[6]), v[7], or_none(v[8]), ctx->saved_data["softplus"].toBool(),
        ctx->saved_data["want_state"].toBool());
    for (size_t i = 0; i < r.size(); ++i) out[i] = r[i];
    if (ctx->saved_data["b3"].toBool()) out[3] = out[3].squeeze(1);
    if (ctx->saved_data["c3"].toBool()) out[4] = out[4].squeeze(1);
    return out;
  }
};

// y and, where wanted, the final state
std::vector<torch::Tensor> selective_scan(torch::Tensor u, torch::Tensor delta, torch::Tensor A,
                                          torch::Tensor Bm, torch::Tensor Cm, OptTensor skip,
                                          OptTensor bias, OptTensor state, OptTensor lengths,
                                          bool softplus, bool want_final) {
  refuse_tangents("fused_selective_scan", u, delta, A, Bm, Cm, skip, bias, state);
  if (wants_grad(u, delta, A, Bm, Cm, skip, bias, state))
    return SelectiveScanFn::apply(u, delta, A, Bm, Cm, skip, bias, state, lengths, softplus,
                                  want_final);
  auto r = selective_scan_forward(u.contiguous(), delta.contiguous(), A.contiguous(),
                                  grouped(Bm, 4), grouped(Cm, 4), contig(skip), contig(bias),
                                  contig(state), contig(lengths), softplus, want_final, false);
  r.resize(want_final ? 2 : 1);
  return r;
}

torch::Tensor selective_scan_step(torch::Tensor u, torch::Tensor delta, torch::Tensor A,
                                  torch::Tensor Bm, torch::Tensor Cm, torch::Tensor state,
                                  OptTensor skip, OptTensor bias, bool softplus) {
  refuse_tangents("fused_selective_scan_step", u, delta, A, Bm, Cm, state, skip, bias);
  TORCH_CHECK(!wants_grad(u, delta, A, Bm, Cm, state, skip, bias),
              "fused_selective_scan_step has no backward: call it under torch.no_grad().");
  u = u.contiguous();
  delta = delta.contiguous();
  A = A.contiguous();
  Bm = grouped(Bm, 3);
  Cm = grouped(Cm, 3);
  skip = contig(skip);
  bias = contig(bias);
  const ScanDims d = check_scan(u, delta, A, Bm, Cm, skip, bias, true);
  check_like(state, "state", {d.B, d.D, d.N}, at::kFloat, u);
  const c10::cuda::CUDAGuard guard(u.device());
  auto y = fresh_like(u);
  check_status(dudy_selective_scan_step(
                   u.data_ptr(), delta.data_ptr(), (const float *)A.data_ptr(), Bm.data_ptr(),
                   Cm.data_ptr(), (const float *)opt_ptr(skip), (const float *)opt_ptr(bias),
                   (float *)state.data_ptr(), y.data_ptr(), d.B, d.D, d.N, d.G, softplus,
                   dtype_code(u), stream_ptr()),
               "fused_selective_scan step");
  written(state);
  return y;
}

void check_block_norm(const torch::Tensor &x, const torch::Tensor &residual,
                      const OptTensor &gate, const torch::Tensor &w1, const OptTensor &b1,
                      const OptTensor &scale, const torch::Tensor &w2, const OptTensor &b2) {
  check_seq(x, "x");
  const auto dt = x.scalar_type();
  TORCH_CHECK(residual.scalar_type() == dt || residual.scalar_type() == at::kFloat,
              "residual must be of x's type or float32, got ", residual.scalar_type(), ".");
  check_like(residual, "residual", x.sizes(), residual.scalar_type(), x);
  check_like(gate, "gate", x.sizes(), dt, x);
  const int64_t D = x.size(1);
  check_like(w1, "post_weight", {D}, dt, x);
  check_like(b1, "post_bias", {D}, dt, x);
  check_like(scale, "scale", {D}, dt, x);
  check_like(w2, "pre_weight", {D}, dt, x);
  check_like(b2, "pre_bias", {D}, dt, x);
}

// y, residual_out, stats (undefined unless wanted)
std::vector<torch::Tensor> block_norm_forward(torch::Tensor x, torch::Tensor residual,
                                              OptTensor gate, torch::Tensor w1, OptTensor b1,
                                              OptTensor scale, torch::Tensor w2, OptTensor b2,
                                              bool layer, double eps, bool want_stats) {
  check_block_norm(x, residual, gate, w1, b1, scale, w2, b2);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t B = x.size(0), D = x.size(1), L = x.size(2);
  auto y = fresh_like(x), rout = fresh_like(residual);
  auto stats = want_stats ? floats({4, B, L}, x) : torch::Tensor();
  check_status(dudy_block_norm_forward(
                   x.data_ptr(), opt_ptr(gate), residual.data_ptr(), w1.data_ptr(), opt_ptr(b1),
                   opt_ptr(scale), w2.data_ptr(), opt_ptr(b2), y.data_ptr(), rout.data_ptr(),
                   want_stats ? (float *)stats.data_ptr() : nullptr, B, D, L, layer, (float)eps,
                   dtype_code(x), dtype_code(residual), stream_ptr()),
               "fused_gated_residual_norm forward");
  return {y, rout, stats};
}

// grad x, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias (undefined where
// there is no such input)
std::vector<torch::Tensor> block_norm_backward(torch::Tensor gy, OptTensor grout,
                                               torch::Tensor x, torch::Tensor residual,
                                               OptTensor gate, torch::Tensor w1, OptTensor b1,
                                               OptTensor scale, torch::Tensor w2, OptTensor b2,
                                               torch::Tensor stats, bool layer) {
  check_block_norm(x, residual, gate, w1, b1, scale, w2, b2);
  const int64_t B = x.size(0), D = x.size(1), L = x.size(2);
  check_like(gy, "grad_y", x.sizes(), x.scalar_type(), x);
  check_like(grout, "grad_residual_out", x.sizes(), residual.scalar_type(), x);
  check_like(stats, "stats", {4, B, L}, at::kFloat, x);
  const c10::cuda::CUDAGuard guard(x.device());
  auto like = [](const OptTensor &t) {
    return t.has_value() ? fresh_like(*t) : torch::Tensor();
  };
  auto ptr = [](const torch::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; };
  auto gx = fresh_like(x), gr = fresh_like(residual), gg = like(gate);
  auto gw1 = fresh_like(w1), gb1 = like(b1), gsc = like(scale);
  auto gw2 = fresh_like(w2), gb2 = like(b2);
  const int dt = dtype_code(x), rdt = dtype_code(residual);
  auto ws = scratch(dudy_block_norm_backward_workspace_size(B, D, L, dt, rdt), x);
  check_status(dudy_block_norm_backward(
                   gy.data_ptr(), opt_ptr(grout), x.data_ptr(), opt_ptr(gate),
                   residual.data_ptr(), w1.data_ptr(), opt_ptr(b1), opt_ptr(scale),
                   w2.data_ptr(), (const float *)stats.data_ptr(), gx.data_ptr(), ptr(gg),
                   gr.data_ptr(), gw1.data_ptr(), ptr(gb1), ptr(gsc), gw2.data_ptr(), ptr(gb2),
                   ws.data_ptr(), (size_t)ws.numel(), B, D, L, layer, dt, rdt, stream_ptr()),
               "fused_gated_residual_norm backward");
  return {gx, gr, gg, gw1, gb1, gsc, gw2, gb2};
}

struct BlockNormFn : public torch::autograd::Function<BlockNormFn> {
  static variable_list forward(AutogradContext *ctx, torch::Tensor x, torch::Tensor residual,
                               OptTensor gate, torch::Tensor w1, OptTensor b1, OptTensor scale,
                               torch::Tensor w2, OptTensor b2, bool layer, double eps) {
    x = x.contiguous();
    residual = residual.contiguous();
    gate = contig(gate);
    w1 = w1.contiguous();
    b1 = contig(b1);
    scale = contig(scale);
    w2 = w2.contiguous();
    b2 = contig(b2);
    auto r = block_norm_forward(x, residual, gate, w1, b1, scale, w2, b2, layer, eps, true);
    ctx->save_for_backward({x, residual, or_undefined(gate), w1, or_undefined(b1),
                            or_undefined(scale), w2, or_undefined(b2), r[2]});
    ctx->saved_data["layer"] = layer;
    ctx->set_materialize_grads(false);
    return {r[0], r[1]};
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    refuse_twice("fused_gated_residual_norm");
    const auto v = ctx->get_saved_variables();
    variable_list out(10);
    if (!g[0].defined() && !g[1].defined()) return out;
    auto gy = g[0].defined() ? g[0].contiguous() : torch::zeros_like(v[0]);
    auto r = block_norm_backward(gy, g[1].defined() ? OptTensor(g[1].contiguous()) : OptTensor(),
                                 v[0], v[1], or_none(v[2]), v[3], or_none(v[4]), or_none(v[5]),
                                 v[6], or_none(v[7]), v[8], ctx->saved_data["layer"].toBool());
    for (size_t i = 0; i < r.size(); ++i) out[i] = r[i];
    return out;
  }
};

// y, residual_out
std::vector<torch::Tensor> block_norm(torch::Tensor x, torch::Tensor residual, OptTensor gate,
                                      torch::Tensor w1, OptTensor b1, OptTensor scale,
                                      torch::Tensor w2, OptTensor b2, bool layer, double eps) {
  refuse_tangents("fused_gated_residual_norm", x, residual, gate, w1, b1, scale, w2, b2);
  if (wants_grad(x, residual, gate, w1, b1, scale, w2, b2))
    return BlockNormFn::apply(x, residual, gate, w1, b1, scale, w2, b2, layer, eps);
  auto r = block_norm_forward(x.contiguous(), residual.contiguous(), contig(gate),
                              w1.contiguous(), contig(b1), contig(scale), w2.contiguous(),
                              contig(b2), layer, eps, false);
  r.resize(2);
  return r;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "dudyconv_b200: B200 (sm_100a) fused dynamic conv / fused source conv";
  m.def("forward_chunk", &forward_chunk, "Fused dynamic convolution forward chunk",
        py::arg("h"), py::arg("kc"), py::arg("mix"), py::arg("off"), py::arg("dilation"));
  m.def("forward_chunk_warmup", &forward_chunk_warmup, "Forward plan warmup / autotune",
        py::arg("h"), py::arg("kc"), py::arg("mix"), py::arg("off"), py::arg("dilation"),
        py::arg("repeat") = 3);
  m.def("forward_chunk_cached_plan", &forward_chunk_cached_plan, "Cached forward plan (-1 if none)",
        py::arg("h"), py::arg("kc"), py::arg("mix"), py::arg("off"), py::arg("dilation"));
  m.def("forward_chunk_clear_warmup_cache", &forward_chunk_clear_warmup_cache,
        "Clear the forward plan cache");
  m.def("forward_plan_name", &plan_name, "Forward plan name", py::arg("plan_id"));
  m.def("backward_chunk", &backward_chunk, "Fused dynamic convolution backward chunk",
        py::arg("go"), py::arg("h"), py::arg("kc"), py::arg("mix"), py::arg("off"),
        py::arg("dilation"));
  m.def("backward_chunk_warmup", &backward_chunk_warmup, "Backward plan warmup / autotune",
        py::arg("go"), py::arg("h"), py::arg("kc"), py::arg("mix"), py::arg("off"),
        py::arg("dilation"), py::arg("repeat") = 3);
  m.def("backward_chunk_cached_plan", &backward_chunk_cached_plan,
        "Cached backward plan (-1 if none)", py::arg("h"), py::arg("kc"), py::arg("off"),
        py::arg("dilation"));
  m.def("backward_chunk_clear_warmup_cache", &backward_chunk_clear_warmup_cache,
        "Clear the backward plan cache");
  m.def("backward_plan_name", &plan_name, "Backward plan name", py::arg("plan_id"));
  m.def("library_version", [] { return std::string(dudy_version()); });
  m.def("device_error", [](bool reset) { return dudy_device_error(reset ? 1 : 0); },
        py::arg("reset") = false);
  m.def("logits_to_kernel", &logits_to_kernel,
        "Kernel generator tail: softmax over K, flip, [B,N*K,T] -> [B,K,N,T]",
        py::arg("logits"), py::arg("num_kernels"), py::arg("kernel_size"));
  m.def("logits_to_kernel_backward", &logits_to_kernel_backward,
        "Backward of logits_to_kernel from its output kc and grad_kc", py::arg("kc"),
        py::arg("grad_kc"));
  m.def("short_conv", &short_conv, "Short causal depthwise conv", py::arg("x"),
        py::arg("weight"), py::arg("bias"), py::arg("state"), py::arg("lengths"), py::arg("silu"),
        py::arg("want_final"));
  m.def("short_conv_step", &short_conv_step, "Short causal depthwise conv, one token",
        py::arg("x"), py::arg("state"), py::arg("weight"), py::arg("bias"), py::arg("silu"));
  m.def("selective_scan", &selective_scan, "Selective scan", py::arg("u"), py::arg("delta"),
        py::arg("A"), py::arg("B"), py::arg("C"), py::arg("skip"), py::arg("delta_bias"),
        py::arg("state"), py::arg("lengths"), py::arg("softplus"), py::arg("want_final"));
  m.def("selective_scan_step", &selective_scan_step, "Selective scan, one token", py::arg("u"),
        py::arg("delta"), py::arg("A"), py::arg("B"), py::arg("C"), py::arg("state"),
        py::arg("skip"), py::arg("delta_bias"), py::arg("softplus"));
  m.def("block_norm", &block_norm, "Gate, norms and residual between blocks", py::arg("x"),
        py::arg("residual"), py::arg("gate"), py::arg("post_weight"), py::arg("post_bias"),
        py::arg("scale"), py::arg("pre_weight"), py::arg("pre_bias"), py::arg("layer"),
        py::arg("eps"));
}

TORCH_LIBRARY(fused_source_conv_mixed, m) {
  m.def("forward(Tensor x_norm, Tensor weight, Tensor bias, Tensor mix_weight, Tensor mix_bias, "
        "int off, int T, int dilation) -> Tensor");
  m.def("forward_plan(Tensor x_norm, Tensor weight, Tensor bias, Tensor mix_weight, "
        "Tensor mix_bias, int off, int T, int dilation, int plan) -> Tensor");
  m.def("forward_cached_plan(Tensor x_norm, Tensor weight, Tensor bias, Tensor mix_weight, "
        "Tensor mix_bias, int off, int T, int dilation, int cached_plan) -> Tensor");
  m.def("forward_warmup(Tensor x_norm, Tensor weight, Tensor bias, Tensor mix_weight, "
        "Tensor mix_bias, int off, int T, int dilation, int warmup_iters, int bench_iters) -> int");
  m.def("backward(Tensor grad_out, Tensor x_norm, Tensor weight, Tensor bias, Tensor mix_weight, "
        "Tensor mix_bias, int off, int T, int dilation) -> Tensor[]");
  m.def("backward_plan(Tensor grad_out, Tensor x_norm, Tensor weight, Tensor bias, "
        "Tensor mix_weight, Tensor mix_bias, int off, int T, int dilation, int plan, int tile_t) "
        "-> Tensor[]");
  m.def("backward_cached_plan(Tensor grad_out, Tensor x_norm, Tensor weight, Tensor bias, "
        "Tensor mix_weight, Tensor mix_bias, int off, int T, int dilation, int cached_plan) "
        "-> Tensor[]");
  m.def("backward_warmup(Tensor grad_out, Tensor x_norm, Tensor weight, Tensor bias, "
        "Tensor mix_weight, Tensor mix_bias, int off, int T, int dilation, int warmup_iters, "
        "int bench_iters) -> int");
  m.def("backward_pack_cached_plan(int plan, int tile_t) -> int");
  m.def("backward_cached_plan_get_plan(int cached_plan) -> int");
  m.def("backward_cached_plan_get_tile_t(int cached_plan) -> int");
  m.def("backward_atomic(Tensor grad_out, Tensor x_norm, Tensor weight, Tensor bias, "
        "Tensor mix_weight, Tensor mix_bias, int off, int T, int dilation) -> Tensor[]");
  m.def("backward_per_d_reduce(Tensor grad_out, Tensor x_norm, Tensor weight, Tensor bias, "
        "Tensor mix_weight, Tensor mix_bias, int off, int T, int dilation, int tile_t) -> Tensor[]");
  m.def("backward_gather_x(Tensor grad_out, Tensor x_norm, Tensor weight, Tensor bias, "
        "Tensor mix_weight, Tensor mix_bias, int off, int T, int dilation, int tile_t) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(fused_source_conv_mixed, CUDA, m) {
  m.impl("forward", TORCH_FN(fscm_forward_op));
  m.impl("forward_plan", TORCH_FN(fscm_forward_plan_op));
  m.impl("forward_cached_plan", TORCH_FN(fscm_forward_cached_plan_op));
  m.impl("forward_warmup", TORCH_FN(fscm_forward_warmup_op));
  m.impl("backward", TORCH_FN(fscm_backward_op));
  m.impl("backward_plan", TORCH_FN(fscm_backward_plan_op));
  m.impl("backward_cached_plan", TORCH_FN(fscm_backward_cached_plan_op));
  m.impl("backward_warmup", TORCH_FN(fscm_backward_warmup_op));
  m.impl("backward_atomic", TORCH_FN(fscm_backward_atomic_op));
  m.impl("backward_per_d_reduce", TORCH_FN(fscm_backward_per_d_reduce_op));
  m.impl("backward_gather_x", TORCH_FN(fscm_backward_gather_x_op));
}

TORCH_LIBRARY_IMPL(fused_source_conv_mixed, CompositeExplicitAutograd, m) {
  m.impl("backward_pack_cached_plan", TORCH_FN(pack_plan));
  m.impl("backward_cached_plan_get_plan", TORCH_FN(unpack_plan));
  m.impl("backward_cached_plan_get_tile_t", TORCH_FN(unpack_tile));
}
