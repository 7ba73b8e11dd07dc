// Shared by the transformer-layer kernels (matrix products with an epilogue, layer norm): element
// conversion, activations and their derivatives, and the host-side device scope.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "dcn_b200.h"

namespace dcn {

// Records `msg` as the calling thread's dcn_last_error() text and returns `code`.
int set_error(int code, const char *msg);

// One matrix product  out[i, j] = epilogue(sum_k A[i, k] * B[j, k]),  i < m, j < n, k < kk.
// An operand lies in memory either with k contiguous (rows of k, row stride ld) or, when its
// *_mn flag is set, with i (or j) contiguous (rows of i, one per k, row stride ld).
struct GemmArgs {
  const void *a, *b;
  long long lda, ldb;
  bool a_mn, b_mn;
  long long m, n, kk;
  // epilogue, in this order, in fp32: v = acc + bias[j]; `saved` keeps what the activation's
  // derivative needs of v; v = act(v); v *= slope_act'(slope); v += res[i, j]
  const void *bias;
  int act;
  void *saved;
  const void *slope;
  int slope_act;
  const void *res;
  long long ldr;
  void *out;       // element type of the operands, row stride n
  // row sums of A over k, [m] (the bias gradient, when A is the transposed output gradient)
  void *row_sum;
};

template <typename T> struct ElemOf;
template <> struct ElemOf<float> {
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};
template <> struct ElemOf<__nv_bfloat16> {
  static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};
template <> struct ElemOf<__half> {
  static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};

// 0.5 * (1 + erf(z / sqrt 2)), the normal distribution function; through erfc so that the
// lower tail keeps its relative accuracy
__device__ __forceinline__ float normal_cdf(float z) { return 0.5f * erfcf(-0.70710678118654752f * z); }

__device__ __forceinline__ float act_value(int act, float z) {
  // a NaN stays a NaN in both
  if (act == DCN_ACT_RELU) return z < 0.f ? 0.f : z;
  if (act == DCN_ACT_GELU) return z * normal_cdf(z);
  return z;
}
// d gelu / dz = cdf(z) + z pdf(z)
__device__ __forceinline__ float gelu_slope(float z) {
  return normal_cdf(z) + z * 0.39894228040143268f * expf(-0.5f * z * z);
}
// The bit that relu's backward pass keeps of z: the gradient passes unless z <= 0.
__device__ __forceinline__ bool relu_bit(float z) { return !(z <= 0.f); }

// Makes `device` current for the lifetime of the object and restores the caller's device.
struct LayerDeviceScope {
  int prev = -1;
  bool switched = false;
  cudaError_t err;
  explicit LayerDeviceScope(int device) {
    err = cudaGetDevice(&prev);
    if (err == cudaSuccess && prev != device) {
      err = cudaSetDevice(device);
      switched = err == cudaSuccess;
    }
  }
  ~LayerDeviceScope() {
    if (switched) cudaSetDevice(prev);
  }
};

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace dcn
