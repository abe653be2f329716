// rowvec.cuh -- what the [B, D, L] row kernels of the state-space block share: eight
// consecutive positions of a row at a time, asynchronous copies into shared memory, the
// activations, and the host-side checks of their C entry points.
#pragma once

#include "common.cuh"

namespace dudy {

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// two neighbouring 16-bit elements of one word
__device__ __forceinline__ float2 pair_of(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
__device__ __forceinline__ float2 pair_of(uint32_t w, __nv_bfloat16) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w));
}
__device__ __forceinline__ uint32_t word_of(float2 v, __half) {
  const __half2 h = __float22half2_rn(v);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t word_of(float2 v, __nv_bfloat16) {
  const __nv_bfloat162 h = __float22bfloat162_rn(v);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// ---- eight positions of a row ------------------------------------------------------------
// 2 N 16-bit elements from an address that need not be that of a word (rows of odd length): words
// where it is, else the words between and an element at each end.
template <int N>
__device__ __forceinline__ void load_halves(uint32_t *w, const uint16_t *h) {
  if ((reinterpret_cast<uintptr_t>(h) & 2u) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t *>(h)[i];
  } else {
    uint32_t m[N + 1];
    m[0] = (uint32_t)h[0] << 16;
#pragma unroll
    for (int i = 1; i < N; ++i) m[i] = reinterpret_cast<const uint32_t *>(h - 1)[i];
    m[N] = h[2 * N - 1];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __funnelshift_r(m[i], m[i + 1], 16);
  }
}
template <int N>
__device__ __forceinline__ void store_halves(uint16_t *h, const uint32_t *w) {
  if ((reinterpret_cast<uintptr_t>(h) & 2u) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<uint32_t *>(h)[i] = w[i];
  } else {
    h[0] = (uint16_t)w[0];
#pragma unroll
    for (int i = 1; i < N; ++i)
      reinterpret_cast<uint32_t *>(h - 1)[i] = __funnelshift_r(w[i - 1], w[i], 16);
    h[2 * N - 1] = (uint16_t)(w[N - 1] >> 16);
  }
}

// Kept in whole 32-bit words from the load on, also where the elements are loaded one by one: the
// conversion waits until it is asked for, so loads that come early stay in flight.
template <typename T>
struct RowEight {
  static constexpr int kW = 2 * sizeof(T);
  uint32_t w[kW];
  // row[t .. t+8), zero at and behind `end`, which is not read. `vec`: rows and t start on eight
  // elements.
  __device__ __forceinline__ void load(const T *row, int t, int end, bool vec) {
    if (vec && t + 8 <= end) {
#pragma unroll
      for (int i = 0; i < kW / 4; ++i) {
        const uint4 q = reinterpret_cast<const uint4 *>(row + t)[i];
        w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = t + i < end ? reinterpret_cast<const uint32_t *>(row)[t + i] : 0u;
    } else if (t + 8 <= end) {
      load_halves<4>(w, reinterpret_cast<const uint16_t *>(row + t));
    } else {
      const uint16_t *h = reinterpret_cast<const uint16_t *>(row);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = (t + 2 * i < end ? (uint32_t)h[t + 2 * i] : 0u) |
               (t + 2 * i + 1 < end ? (uint32_t)h[t + 2 * i + 1] << 16 : 0u);
    }
  }
  __device__ __forceinline__ float2 pair(int i) const {
    if constexpr (sizeof(T) == 4)
      return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else
      return pair_of(w[i], T());
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = pair(i);
      v[2 * i] = p.x;
      v[2 * i + 1] = p.y;
    }
  }
};

// row[t .. t+8) = v, before `end`
template <typename T>
__device__ __forceinline__ void row_store8(T *row, int t, int end, const float (&v)[8], bool vec) {
  if (vec && t + 8 <= end) {
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4 *>(row + t)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4 *>(row + t)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4 *>(row + t) =
          make_uint4(word_of(make_float2(v[0], v[1]), T()), word_of(make_float2(v[2], v[3]), T()),
                     word_of(make_float2(v[4], v[5]), T()), word_of(make_float2(v[6], v[7]), T()));
    }
  } else if (sizeof(T) == 2 && t + 8 <= end) {
    if constexpr (sizeof(T) == 2) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = word_of(make_float2(v[2 * i], v[2 * i + 1]), T());
      store_halves<4>(reinterpret_cast<uint16_t *>(row + t), w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (t + i < end) stf(row + t + i, v[i]);
  }
}

// ---- four positions of a row, as they lie in memory --------------------------------------------
template <typename T>
struct RowFour;
template <>
struct RowFour<float> {
  uint32_t w[4];
  __device__ __forceinline__ float get(int i) const { return __uint_as_float(w[i]); }
  __device__ __forceinline__ void load_all(const float *p) {
    const uint4 q = *reinterpret_cast<const uint4 *>(p);
    w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
  }
  __device__ __forceinline__ void load_shifted(const float *p, int) { load_all(p); }
};
template <typename T>
struct RowFour {
  uint32_t w[2];
  __device__ __forceinline__ float get(int i) const {
    const uint16_t h = (uint16_t)(w[i >> 1] >> (i & 1 ? 16 : 0));
    return Elem<T>::to_f(*reinterpret_cast<const T *>(&h));
  }
  __device__ __forceinline__ void load_all(const T *p) {
    const uint2 q = *reinterpret_cast<const uint2 *>(p);
    w[0] = q.x; w[1] = q.y;
  }
  // p[sh .. sh + 4), sh 0 or 1, from six elements
  __device__ __forceinline__ void load_shifted(const T *p, int sh) {
    const uint32_t *q = reinterpret_cast<const uint32_t *>(p);
    const uint32_t a = q[0], b = q[1], c = q[2];
    w[0] = __funnelshift_r(a, b, 16 * sh);
    w[1] = __funnelshift_r(b, c, 16 * sh);
  }
  __device__ __forceinline__ void set(const float (&v)[4]) {
    w[0] = word_of(make_float2(v[0], v[1]), T());
    w[1] = word_of(make_float2(v[2], v[3]), T());
  }
  __device__ __forceinline__ void store_all(T *p) const {
    *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
  }
};

// row[t .. t+4) = v, before `end`
template <typename T>
__device__ __forceinline__ void row_store4(T *row, int64_t t, int64_t end, const float (&v)[4],
                                           bool vec) {
  if (vec && t + 4 <= end) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4 *>(row + t) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      RowFour<T> f;
      f.set(v);
      f.store_all(row + t);
    }
  } else if (sizeof(T) == 2 && t + 4 <= end) {
    if constexpr (sizeof(T) == 2) {
      RowFour<T> f;
      f.set(v);
      store_halves<2>(reinterpret_cast<uint16_t *>(row + t), f.w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (t + i < end) stf(row + t + i, v[i]);
  }
}

// row[t], row[t+1] = v, before `end`
template <typename T>
__device__ __forceinline__ void row_store2(T *row, int64_t t, int64_t end, const float (&v)[2],
                                           bool vec) {
  if (vec && t + 2 <= end) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float2 *>(row + t) = make_float2(v[0], v[1]);
    } else {
      *reinterpret_cast<uint32_t *>(row + t) = word_of(make_float2(v[0], v[1]), T());
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (t + i < end) stf(row + t + i, v[i]);
  }
}

// ---- activations --------------------------------------------------------------------------
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 1 / (1 + exp(-v)); 16-bit tensors use the fast exponential and reciprocal (relative error
// about 2^-21, far below the rounding of the result), fp32 tensors the accurate ones.
template <typename T>
__device__ __forceinline__ float sigmoid_for(float v) {
  return rcp(1.f + ex2(-1.4426950408889634f * v));
}
template <>
__device__ __forceinline__ float sigmoid_for<float>(float v) {
  return 1.f / (1.f + expf(-v));
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 neg2(float2 a) { return make_float2(-a.x, -a.y); }

template <typename T>
__device__ __forceinline__ float2 sigmoid2(float2 v) {
  if constexpr (sizeof(T) == 4) {
    return make_float2(sigmoid_for<T>(v.x), sigmoid_for<T>(v.y));
  } else {
    const float2 e = mul2(v, both(-1.4426950408889634f));
    const float2 d = add2(make_float2(ex2(e.x), ex2(e.y)), both(1.f));
    return make_float2(rcp(d.x), rcp(d.y));
  }
}

// ---- sums across lanes ------------------------------------------------------------------------
// Sums of n values each over the lanes that differ in the bits [STRIDE, STRIDE * LANES) of the
// lane number. While there are several values, half of them go to the partner lane and half
// come from it, so a stage costs n / 2 shuffles; afterwards lane l of the group (its number in
// those bits) holds the sums of values l * n / LANES .. , or, with more lanes than n / KEEP
// values, all lanes that agree in the upper bits hold the same KEEP values.
template <int STRIDE, int LANES, int N, int KEEP = 1>
struct Scatter {
  static constexpr int kLeft = LANES == 1 || N == KEEP ? N : Scatter<STRIDE, LANES / 2, N / 2, KEEP>::kLeft;
  static __device__ __forceinline__ void sum(float *v, int lane) {
    if constexpr (LANES > 1) {
      constexpr int o = STRIDE * LANES / 2;
      if constexpr (N > KEEP) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          const float send = up ? v[i] : v[i + N / 2];
          const float keep = up ? v[i + N / 2] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
        Scatter<STRIDE, LANES / 2, N / 2, KEEP>::sum(v, lane);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
        Scatter<STRIDE, LANES / 2, N, KEEP>::sum(v, lane);
      }
    }
  }
};
template <int STRIDE, int N, int KEEP>
struct Scatter<STRIDE, 1, N, KEEP> {
  static constexpr int kLeft = N;
  static __device__ __forceinline__ void sum(float *, int) {}
};

// The sum of p[i * stride], i < parts, of one of 32 columns a block of ROWS x 32 threads works on:
// each row of threads takes every ROWS-th part, and the rows' sums are added in order. Returned to
// row 0 (threadIdx.x < 32).
template <int ROWS>
__device__ __forceinline__ float column_sum(const float *p, int64_t parts, int64_t stride, bool in,
                                            float (*red)[32]) {
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  float v = 0.f;
  if (in) {
#pragma unroll 4
    for (int64_t i = ty; i < parts; i += ROWS) v += p[i * stride];
  }
  __syncthreads();
  red[ty][tx] = v;
  __syncthreads();
  v = 0.f;
  if (ty == 0) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) v += red[i][tx];
  }
  return v;
}

// ---- asynchronous 16-byte copies into shared memory ------------------------------------------
__device__ __forceinline__ void cp_async16(void *smem, const void *gmem) {
  const uint32_t s = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(gmem) : "memory");
}
// `bytes` of four, the rest zero
__device__ __forceinline__ void cp_async4(void *smem, const void *gmem, int bytes) {
  const uint32_t s = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(s), "l"(gmem), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

inline int require_apart(const void *state, const void *final_state) {
  if (!state || state != final_state) return DUDY_OK;
  return refuse("final_state must not be the initial state's memory.");
}

inline int require_workspace(const void *ws, size_t got, size_t need) {
  if (need == 0 || (ws && got >= need)) return DUDY_OK;
  return refuse("workspace too small: need " + std::to_string(need) + " bytes, got " +
                std::to_string(ws ? got : 0), DUDY_ERR_WORKSPACE);
}

}  // namespace dudy
