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
  // with slope_act: fp32 column sums of v (before the residual and the rounding) over every 32 rows,
  // [ceil(m / 32)][n]
  float *col_part;
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

// Phi(z) = 0.5 * (1 + erf(z / sqrt 2)) and phi(z), the normal distribution function and density.
//
// kExact (fp32 tensors): through erfcf, so that the lower tail keeps its relative accuracy.
// Otherwise (16-bit tensors): erfc(x) = t (a1 + t (a2 + t (a3 + t (a4 + t a5)))) exp(-x^2),
// t = 1 / (1 + p x), x >= 0 (Abramowitz and Stegun 7.1.26, absolute error below 1.5e-7, a fiftieth of
// half a step of fp16 at 1).  It takes two special-function instructions and a dozen others, and
// the exponential is the density's too; with erfcf the epilogue of a 128 x 256 tile took longer than
// 16 steps of its main loop (4096 x 1024 x 2048 fp16 forward: 57 us).
template <bool kExact>
__device__ __forceinline__ void normal(float z, float *cdf, float *density) {
  if constexpr (kExact) {
    *cdf = 0.5f * erfcf(-0.70710678118654752f * z);
    *density = 0.39894228040143268f * expf(-0.5f * z * z);
  } else {
    const float x = fabsf(z) * 0.70710678118654752f;
    const float e = __expf(-x * x);
    const float t = __fdividef(1.f, fmaf(0.3275911f, x, 1.f));
    const float q = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f),
                             0.254829592f);
    const float tail = 0.5f * q * e;   // Phi(-|z|)
    *cdf = z < 0.f ? tail : 1.f - tail;
    *density = 0.39894228040143268f * e;
  }
}
template <bool kExact>
__device__ __forceinline__ float gelu_value(float z) {
  float cdf, density;
  normal<kExact>(z, &cdf, &density);
  // far out z * Phi(z) is -inf * 0; below -40 nothing is left of it in any type
  return z < -40.f ? -0.f : z * cdf;
}
// d gelu / dz = Phi(z) + z phi(z)
template <bool kExact>
__device__ __forceinline__ float gelu_slope(float z) {
  float cdf, density;
  normal<kExact>(z, &cdf, &density);
  return fabsf(z) > 40.f ? (z > 0.f ? 1.f : 0.f) : fmaf(z, density, cdf);
}
// A NaN stays a NaN.
__device__ __forceinline__ float relu_value(float z) {
  float v;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(v) : "f"(z));
  return v;
}
// The bit that relu's backward pass keeps of z: the gradient passes unless z <= 0.
__device__ __forceinline__ bool relu_bit(float z) { return !(z <= 0.f); }

// Programmatic dependent launch.  A kernel launched with launch_pdl may start while the kernel before it
// in the stream still runs: everything up to pdl_wait (barriers, tensor memory) overlaps that kernel's
// tail.  pdl_wait returns when all earlier work of the stream is done and visible, so it stands in
// front of the first access to global memory of every thread.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// cluster: blocks of a thread-block cluster (1: none).
template <typename... P, typename... A>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, int cluster,
                       const A &...args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = block;
  c.dynamicSmemBytes = smem;
  c.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  c.attrs = attr;
  c.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&c, kernel, P(args)...);
}

// Makes `device` current for the lifetime of the object and restores the caller's device.  Also binds the
// device's context to the calling thread where no runtime call has done so yet (an autograd thread's
// first call): the tensor-map encoder is a driver call and would fail without one.
struct LayerDeviceScope {
  int prev = -1;
  bool switched = false;
  cudaError_t err;
  explicit LayerDeviceScope(int device) {
    err = cudaGetDevice(&prev);
    if (err == cudaSuccess) err = cudaSetDevice(device);
    switched = err == cudaSuccess && prev != device;
  }
  ~LayerDeviceScope() {
    if (switched) cudaSetDevice(prev);
  }
};

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace dcn
