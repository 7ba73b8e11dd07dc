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
  // column sums of other partial rows [join_parts][m] to join on the way, with a product whose parts are joined
  const float *join_part;
  int join_parts;
  void *join_out;
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

// Phi and phi: the normal distribution function and density.  gelu(z) = z Phi(z), its derivative
// Phi(z) + z phi(z).
//
// fp32 tensors (kFine): Phi(-a) = e^(-a^2 / 2) q(s), s = 1 / (1 + 0.23 a), q a polynomial of degree 8, fitted
// here (iteratively reweighted least squares on 0 <= a <= 14) for relative error: 5e-8, with fp32's roundings
// 5e-7, and 7e-8 absolute in a Phi(-a).  With erfcf and expf the epilogue took longer than the product
// (35642 x 256 x 1024: 245 us, without gelu 108).
//
// 16-bit tensors: Phi(-a) = 2^p(a), a = |z|, p a polynomial of degree 7, fitted here (iteratively reweighted
// least squares on [0, 6]) so that the error of a Phi(-a) is a fixed share of half a step of fp16: at most
// 0.0073 of it, 9.3e-7 absolute; beyond 6 p falls to -274 at 20, where a is cut off.  Then
// gelu(z) = max(z, 0) - a Phi(-a): one special-function instruction and, two elements at a time, four and a
// half multiply-adds an element, no branch and no cancellation.
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (x0, x1) += (y0, y1) in one instruction
__device__ __forceinline__ void add2(float &x0, float &x1, float y0, float y1) {
  asm("{\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%0, %1};\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "add.rn.f32x2 a, a, b;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x0), "+f"(x1)
      : "f"(y0), "f"(y1));
}
// (a0, a1) += (x0, x1) * (y0, y1)
__device__ __forceinline__ void fma2_to(float &a0, float &a1, float x0, float x1, float y0, float y1) {
  asm("{\n\t.reg .b64 a, b, c;\n\t"
      "mov.b64 a, {%2, %3};\n\t"
      "mov.b64 b, {%4, %5};\n\t"
      "mov.b64 c, {%0, %1};\n\t"
      "fma.rn.f32x2 c, a, b, c;\n\t"
      "mov.b64 {%0, %1}, c;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(x0), "f"(x1), "f"(y0), "f"(y1));
}
// (x0, x1) * (y0, y1) + (z, z), each rounded to nearest
__device__ __forceinline__ void fma2(float &x0, float &x1, float y0, float y1, float z) {
  asm("{\n\t.reg .b64 a, b, c;\n\t"
      "mov.b64 a, {%0, %1};\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "mov.b64 c, {%4, %4};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x0), "+f"(x1)
      : "f"(y0), "f"(y1), "f"(z));
}
// Phi(-a0), Phi(-a1), 0 <= a <= 20
template <bool kFine>
__device__ __forceinline__ void tails(float a0, float a1, float &t0, float &t1) {
  if constexpr (kFine) {
    constexpr float c[9] = {-2.7761721867136657e-05f, 0.09237844496965408f, 0.08576300740242004f, 0.11951372772455215f,
                            -0.032919447869062424f, 0.3014717698097229f, -0.2781260907649994f, 0.2904137372970581f,
                            -0.07846737653017044f};
    float s0, s1;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s0) : "f"(fmaf(a0, 0.23f, 1.f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s1) : "f"(fmaf(a1, 0.23f, 1.f)));
    t0 = t1 = c[8];
#pragma unroll
    for (int i = 7; i >= 0; --i) fma2(t0, t1, s0, s1, c[i]);
    t0 *= exp2_approx(-0.72134752044448170f * (a0 * a0));
    t1 *= exp2_approx(-0.72134752044448170f * (a1 * a1));
    return;
  }
  constexpr float c[8] = {-0.9999973773956299f, -1.151201844215393f, -0.4586567282676697f, -0.053682103753089905f,
                          0.008319714106619358f, -0.0008661015890538692f, 5.079910988570191e-05f,
                          -1.131071940108086e-06f};
  t0 = t1 = c[7];
#pragma unroll
  for (int i = 6; i >= 0; --i) fma2(t0, t1, a0, a1, c[i]);
  t0 = exp2_approx(t0);
  t1 = exp2_approx(t1);
}
__device__ __forceinline__ float relu_value(float z);
// z clipped to +-20, a NaN kept
__device__ __forceinline__ float clip20(float z) {
  float v;
  asm("min.NaN.f32 %0, %1, 0f41A00000;\n\tmax.NaN.f32 %0, %0, 0fC1A00000;" : "=f"(v) : "f"(z));
  return v;
}
__device__ __forceinline__ float slope_from(float clipped, float tail) {
  const float density = 0.39894228040143268f * exp2_approx(-0.72134752044448170f * clipped * clipped);
  return fmaf(clipped, density, clipped > 0.f ? 1.f - tail : tail);
}

// Two values of gelu; two derivatives; both (s: the derivatives).
template <bool kFine>
__device__ __forceinline__ void gelu_values(float &v0, float &v1) {
  const float a0 = fminf(fabsf(v0), 20.f), a1 = fminf(fabsf(v1), 20.f);
  float t0, t1;
  tails<kFine>(a0, a1, t0, t1);
  v0 = fmaf(-a0, t0, relu_value(v0));
  v1 = fmaf(-a1, t1, relu_value(v1));
}
template <bool kFine>
__device__ __forceinline__ void gelu_both(float &v0, float &v1, float &s0, float &s1) {
  const float c0 = clip20(v0), c1 = clip20(v1);
  float t0, t1;
  tails<kFine>(fabsf(c0), fabsf(c1), t0, t1);
  v0 = fmaf(-fabsf(c0), t0, relu_value(v0));
  v1 = fmaf(-fabsf(c1), t1, relu_value(v1));
  s0 = slope_from(c0, t0);
  s1 = slope_from(c1, t1);
}
template <bool kFine>
__device__ __forceinline__ void gelu_slopes(float &v0, float &v1) {
  const float c0 = clip20(v0), c1 = clip20(v1);
  float t0, t1;
  tails<kFine>(fabsf(c0), fabsf(c1), t0, t1);
  v0 = slope_from(c0, t0);
  v1 = slope_from(c1, t1);
}
template <bool kFine>
__device__ __forceinline__ float gelu_value(float z) {
  float other = z;
  gelu_values<kFine>(z, other);
  return z;
}
template <bool kFine>
__device__ __forceinline__ float gelu_slope(float z) {
  float other = z;
  gelu_slopes<kFine>(z, other);
  return z;
}

// What is kept of gelu for the backward pass: the derivative.  fp32 tensors keep it as it is.  For 16-bit ones
// it is a code of 16 bits, for a few instructions each way instead of the derivative's twenty in the backward
// pass:
//   0 .. 36995      the derivative in steps of 2^-15 (it is at most 1.1290; 0 and 1 are exact): within 2^-16, a
//                   sixteenth of half a step of fp16 at 1
//   37376 .. 65057  negative ones (at least -0.1290) as a float of ten mantissa bits from -2^-30 on: within 2^-11
//                   of the derivative, down to where z is -6.6.  In the steps of 2^-15 it would be 3 % off at z = -4
//                   and zero from -5 on, and such a unit would no longer learn.
//   65535           NaN
// Between 0 and -2^-30 it is 0.
constexpr uint32_t kNegativeCode = 0x9200u;   // -2^-30
// the code: the low 16 bits.  1.5 * 2^23 + q has q in the low bits of its pattern; a NaN comes out of the
// multiply-add as 0x7fffffff.  0xB0800000, the pattern of -2^-30, shifted by 13 ends in 0x8400.
__device__ __forceinline__ uint32_t slope_code(float slope) {
  const uint32_t fixed = __float_as_uint(fmaf(slope, 32768.f, 12582912.f));
  const uint32_t floating = (__float_as_uint(slope) + (((kNegativeCode - 0x8400u) << 13) + 0x1000u)) >> 13;
  return slope <= -9.31322574615478515625e-10f ? floating : fixed;
}
__device__ __forceinline__ uint32_t slope_codes(float lo, float hi) {
  return __byte_perm(slope_code(lo), slope_code(hi), 0x5410);
}
// pattern: 0x4B400000, which is 1.5 * 2^23, with the code in its low 16 bits
__device__ __forceinline__ float slope_of(uint32_t pattern) {
  const float fixed = fmaf(__uint_as_float(pattern), 1.f / 32768.f, -384.f);   // exact
  const float floating = __uint_as_float((pattern << 13) + (0xB0800000u - (kNegativeCode << 13)));
  const float v = pattern >= (0x4B400000u | kNegativeCode) ? floating : fixed;
  return v < -0.15f ? __uint_as_float(0x7fffffffu) : v;
}
__device__ __forceinline__ float slope_of_low(uint32_t codes) { return slope_of(__byte_perm(codes, 0x4B400000u, 0x7610)); }
__device__ __forceinline__ float slope_of_high(uint32_t codes) { return slope_of(__byte_perm(codes, 0x4B400000u, 0x7632)); }
// A NaN stays a NaN.
__device__ __forceinline__ float relu_value(float z) {
  float v;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(v) : "f"(z));
  return v;
}
// The bit that relu's backward pass keeps of z: the gradient passes unless z <= 0.
__device__ __forceinline__ bool relu_bit(float z) { return !(z <= 0.f); }

// The sum of `parts` values `stride` apart, from p on, for each of C neighbouring columns: a block of NT
// threads, NT / C to a column (threadIdx.x % C), joined in an order that does not change.  The result is in
// the first C threads.  Eight columns while they are few: all that counts then is latency (444 rows of 512
// columns 7.8 us with 32 columns to a block); with many the blocks are enough anyway.
template <int NT, int C>
__device__ __forceinline__ float column_join(const float *p, int parts, long long stride, bool live) {
  constexpr int W = NT / 32, L = 32 / C, kInFlight = NT == 1024 ? 4 : 8;   // warps; lanes of a warp to a column
  static_assert((C == 8 || C == 32) && W % L == 0, "whole warps");
  __shared__ float s[W][C];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float v = 0.f;
  if (live) {
#pragma unroll kInFlight
    for (int q = threadIdx.x / C; q < parts; q += NT / C) v += p[q * stride];
  }
#pragma unroll
  for (int d = C; d < 32; d *= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  if (lane < C) s[warp][lane] = v;
  __syncthreads();
  if (warp) return 0.f;
  v = 0.f;
#pragma unroll
  for (int q = 0; q < W / L; ++q) v += s[lane / C * (W / L) + q][lane % C];
#pragma unroll
  for (int d = C; d < 32; d *= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
inline int join_columns(long long cols) { return cols <= 2048 ? 8 : 32; }

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
