// What the kernels of the sequence-model operators (adamw.cu, residual_norm.cu, recurrence.cu) share: the element
// types of their tensors, and the checks of their entry points.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/fbfftconv.h"
#include "kernels.h"

namespace fbfft {

constexpr bool known_type(int t) { return t == FBFFTCONV_FLOAT32 || t == FBFFTCONV_BFLOAT16 || t == FBFFTCONV_FLOAT16; }
constexpr int type_bytes(int t) { return t == FBFFTCONV_FLOAT32 ? 4 : 2; }

// Values are computed in fp32 and rounded to nearest once, where they are stored.
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// Two neighbouring 16-bit values in one register, the lower address in the lower half.
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t u);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// report_error with a format.
inline int op_fail(int code, const char* fmt, ...) {
  char buf[384];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return report_error(code, buf);
}

inline int op_cuda_fail(cudaError_t e, const char* what) {
  cudaGetLastError();  // reported here; the next call must not report it again
  return op_fail(FBFFTCONV_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// Makes `device` current for the scope of a call.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    error_ = cudaGetDevice(&before_);
    if (error_ == cudaSuccess && before_ != device) {
      error_ = cudaSetDevice(device);
      switched_ = error_ == cudaSuccess;
    }
  }
  ~OnDevice() {
    if (switched_) cudaSetDevice(before_);
  }
  cudaError_t error() const { return error_; }

 private:
  int before_ = -1;
  bool switched_ = false;
  cudaError_t error_;
};

inline int resolve_device(int device, int* out) {
  if (device >= 0) {
    *out = device;
    return FBFFTCONV_OK;
  }
  const cudaError_t e = cudaGetDevice(out);
  return e == cudaSuccess ? FBFFTCONV_OK : op_cuda_fail(e, "cudaGetDevice");
}

inline bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

#define OP_TRY(expr)                     \
  do {                                   \
    const int rc_ = (expr);              \
    if (rc_ != FBFFTCONV_OK) return rc_; \
  } while (0)

}  // namespace fbfft
