// rowvec.cuh -- what the [B, D, L] row kernels of the state-space block share: eight
// consecutive positions of a row at a time, asynchronous copies into shared memory, the
// activations, and the host-side checks of their C entry points.
#pragma once

#include "common.cuh"

namespace dudy {

// ---- eight positions of a row ------------------------------------------------------------
// 16-bit rows: one 16-byte access, fp32 rows: two. `p` is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void row_load8(const T *p, float (&v)[8]) {
  const uint4 q = *reinterpret_cast<const uint4 *>(p);
  const T *e = reinterpret_cast<const T *>(&q);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = Elem<T>::to_f(e[i]);
}
template <>
__device__ __forceinline__ void row_load8<float>(const float *p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4 *>(p);
  const float4 b = *reinterpret_cast<const float4 *>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

template <typename T>
__device__ __forceinline__ void row_store8(T *p, const float (&v)[8]) {
  uint4 q;
  T *e = reinterpret_cast<T *>(&q);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = Elem<T>::from_f(v[i]);
  *reinterpret_cast<uint4 *>(p) = q;
}
template <>
__device__ __forceinline__ void row_store8<float>(float *p, const float (&v)[8]) {
  *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4 *>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}

// Positions [t, t+8) of a row, zero at and after `end` (what lies there is not read).
template <typename T, bool VEC>
__device__ __forceinline__ void row_load8_until(const T *row, int64_t t, int64_t end,
                                                float (&v)[8]) {
  if (VEC && t + 8 <= end) {
    row_load8(row + t, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = t + i < end ? ldf(row + t + i) : 0.f;
}

template <typename T, bool VEC>
__device__ __forceinline__ void row_store8_until(T *row, int64_t t, int64_t end,
                                                 const float (&v)[8]) {
  if (VEC && t + 8 <= end) {
    row_store8(row + t, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (t + i < end) stf(row + t + i, v[i]);
}

// ---- activations --------------------------------------------------------------------------
// 1 / (1 + exp(-v)); 16-bit tensors use the fast exponential and division (relative error
// about 2^-21, far below the rounding of the result), fp32 tensors the accurate ones.
template <typename T>
__device__ __forceinline__ float sigmoid_for(float v) {
  return __fdividef(1.f, 1.f + __expf(-v));
}
template <>
__device__ __forceinline__ float sigmoid_for<float>(float v) {
  return 1.f / (1.f + expf(-v));
}

// ---- asynchronous 16-byte copies into shared memory ------------------------------------------
__device__ __forceinline__ void cp_async16(void *smem, const void *gmem) {
  const uint32_t s = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(gmem) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---- host side ------------------------------------------------------------------------------
inline bool aligned_to_16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline int refuse(const std::string &msg, int status = DUDY_ERR_INVALID) {
  set_error(msg);
  return status;
}

inline bool dtype_known(int dtype) {
  return dtype == DUDY_DTYPE_F32 || dtype == DUDY_DTYPE_F16 || dtype == DUDY_DTYPE_BF16;
}

inline int require_sm100() {
  if (device_cc() == 100) return DUDY_OK;
  return refuse("current CUDA device is not an sm_100 (B200-class) GPU; this library is built "
                "for sm_100a only", DUDY_ERR_DEVICE);
}

inline int require_workspace(const void *ws, size_t got, size_t need) {
  if (need == 0 || (ws && got >= need)) return DUDY_OK;
  return refuse("workspace too small: need " + std::to_string(need) + " bytes, got " +
                std::to_string(ws ? got : 0), DUDY_ERR_WORKSPACE);
}

}  // namespace dudy
