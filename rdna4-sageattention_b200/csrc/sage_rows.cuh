// Shared by the row-wise kernels (rotary positions, the paged K/V cache): 8-channel loads and stores of 16-bit
// rows, argument checks and the launch status.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "../../include/sage_b200.h"
#include "sage_internal.h"

namespace sage {

__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8], __nv_bfloat16) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {   // a bf16 is the upper half of a float
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8], __half) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 8 consecutive channels (16 bytes, aligned) of a 16-bit row.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  float y[8];
  unpack8(*reinterpret_cast<const uint4*>(p), y, T());
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = y[i];
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2(x[0], x[1], T()), pack2(x[2], x[3], T()), pack2(x[4], x[5], T()),
                                            pack2(x[6], x[7], T()));
}

inline int check_rows(int dtype, int B, int S, int H, int D) {
  if (dtype != SAGE_BF16 && dtype != SAGE_F16) {
    set_error("dtype %d (SAGE_BF16 or SAGE_F16 required)", dtype);
    return SAGE_ERR_UNSUPPORTED;
  }
  if (D != 64 && D != 96 && D != 128 && D != 256) {
    set_error("head_dim %d (supported 64, 96, 128, 256)", D);
    return SAGE_ERR_UNSUPPORTED;
  }
  if (B <= 0 || S <= 0 || H <= 0) {
    set_error("empty tensor (B=%d S=%d H=%d)", B, S, H);
    return SAGE_ERR_UNSUPPORTED;
  }
  return SAGE_OK;
}

inline int check_rows_pointer(const void* p, int64_t sb, int64_t ss, int64_t sh, const char* name) {
  if (p == nullptr || (reinterpret_cast<uintptr_t>(p) & 15u) || (sb & 7) || (ss & 7) || (sh & 7)) {
    set_error("%s: pointer and (batch, seq, head) strides must be 16-byte aligned", name);
    return SAGE_ERR_INVALID;
  }
  return SAGE_OK;
}

inline Strides3 strides3(const int64_t (&st)[3]) { return Strides3{st[0], st[1], st[2]}; }

inline int check_rows_pointer(const void* p, const int64_t (&st)[3], const char* name) {
  return check_rows_pointer(p, st[0], st[1], st[2], name);
}

inline int launch_result(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return SAGE_OK;
  set_error("%s: %s", what, cudaGetErrorString(e));
  return SAGE_ERR_LAUNCH;
}

// f(integral_constant<int, D>) for the checked head dim.
template <typename F>
inline int by_head_dim(int D, F&& f) {
  switch (D) {
    case 64: return f(std::integral_constant<int, 64>());
    case 96: return f(std::integral_constant<int, 96>());
    case 128: return f(std::integral_constant<int, 128>());
    default: return f(std::integral_constant<int, 256>());
  }
}

}  // namespace sage
