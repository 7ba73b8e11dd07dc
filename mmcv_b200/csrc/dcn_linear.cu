// C entries of the matrix product with bias, activation and residual in its epilogue, forward and
// backward: argument checks, workspace layout, and the sequence of kernels of each pass.
//   forward   y = act(x W^T + b) + r                       one product
//   backward  gz = gy * act'(z)                            element-wise, only with an activation
//             gx = gz W  (times the derivative of the activation before, plus gx_add)
//             gW = gz^T x,  gb = column sums of gz
#include "dcn_layers.cuh"

namespace dcn {

cudaError_t launch_gemm_simple(const GemmArgs &g, int dtype, cudaStream_t s);

namespace {

size_t up256(size_t v) { return (v + 255) / 256 * 256; }
size_t esize(int dtype) { return dtype == DCN_DTYPE_F32 ? 4 : 2; }

// gz = gy * act'(z), dense [rows, cols]; one thread per element, rows in blockIdx.y strides
template <typename T>
__global__ void __launch_bounds__(256) linear_gz(const T *__restrict__ gy, long long ldgy, const void *saved,
                                                 int act, long long rows, long long cols, T *__restrict__ gz) {
  const long long words = (cols + 31) / 32;
  for (long long idx = blockIdx.x * 256LL + threadIdx.x; idx < rows * cols; idx += gridDim.x * 256LL) {
    const long long r = idx / cols, c = idx - r * cols;
    float v = ElemOf<T>::to(gy[r * ldgy + c]);
    if (act == DCN_ACT_RELU)
      v = ((((const uint32_t *)saved)[r * words + c / 32] >> (c & 31)) & 1u) ? v : 0.f;
    else
      v *= gelu_slope(ElemOf<T>::to(((const T *)saved)[idx]));
    gz[idx] = ElemOf<T>::from(v);
  }
}

// gb[c] = sum_r gz[r, c] where the product that could carry it is not run: a block owns 32 columns
template <typename T>
__global__ void __launch_bounds__(1024) linear_column_sum(const T *__restrict__ gz, long long ld, long long rows,
                                                          long long cols, T *__restrict__ gb) {
  __shared__ float part[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long long c = blockIdx.x * 32LL + tx;
  float s = 0.f;
  if (c < cols)
    for (long long r = ty; r < rows; r += 32) s += ElemOf<T>::to(gz[r * ld + c]);
  part[ty][tx] = s;
  __syncthreads();
  for (int d = 16; d > 0; d >>= 1) {
    if (ty < d) part[ty][tx] += part[ty + d][tx];
    __syncthreads();
  }
  if (ty == 0 && c < cols) gb[c] = ElemOf<T>::from(part[0][tx]);
}

template <typename T>
cudaError_t run_gz(const void *gy, long long ldgy, const void *saved, int act, long long rows, long long cols,
                   void *gz, cudaStream_t s) {
  const long long blocks = (rows * cols + 255) / 256;
  linear_gz<T><<<(int)(blocks < 148 * 32 ? blocks : 148 * 32), 256, 0, s>>>((const T *)gy, ldgy, saved, act, rows,
                                                                            cols, (T *)gz);
  return cudaGetLastError();
}
template <typename T>
cudaError_t run_column_sum(const void *gz, long long ld, long long rows, long long cols, void *gb, cudaStream_t s) {
  linear_column_sum<T><<<(int)((cols + 31) / 32), 1024, 0, s>>>((const T *)gz, ld, rows, cols, (T *)gb);
  return cudaGetLastError();
}

int check_sizes(int32_t dtype, int32_t act, int64_t rows, int64_t cin, int64_t cout) {
  if (dtype != DCN_DTYPE_F32 && dtype != DCN_DTYPE_BF16 && dtype != DCN_DTYPE_F16)
    return set_error(DCN_ERR_UNSUPPORTED, "linear: fp32, bf16 and fp16 tensors only");
  if (act != DCN_ACT_NONE && act != DCN_ACT_RELU && act != DCN_ACT_GELU)
    return set_error(DCN_ERR_ARG, "linear: unknown activation");
  if (rows < 0 || cin <= 0 || cout <= 0)
    return set_error(DCN_ERR_ARG, "linear: cin and cout must be positive, rows must not be negative");
  const int64_t most = 2147483647LL - 1024;   // coordinates are 32-bit, element offsets 64-bit
  if (rows > most || cin > (1 << 20) || cout > (1 << 20))
    return set_error(DCN_ERR_UNSUPPORTED, "linear: at most 2^31 rows and 2^20 channels");
  return DCN_OK;
}

int cuda_error(cudaError_t e) { return set_error(DCN_ERR_CUDA, cudaGetErrorString(e)); }

}  // namespace
}  // namespace dcn

using namespace dcn;

extern "C" {

int dcn_linear_workspace_bytes(int32_t dtype, int64_t rows, int64_t cin, int64_t cout, int64_t alignment,
                               size_t *bytes) {
  if (!bytes) return set_error(DCN_ERR_ARG, "linear: bytes is NULL");
  int rc = check_sizes(dtype, DCN_ACT_NONE, rows, cin, cout);
  if (rc) return rc;
  (void)alignment;
  *bytes = 0;
  return DCN_OK;
}

int dcn_linear_forward(const void *x, int64_t ldx, const void *weight, int64_t ldw, const void *bias,
                       const void *residual, int64_t ldr, void *y, void *saved, int32_t dtype, int32_t act,
                       int64_t rows, int64_t cin, int64_t cout, int32_t device, void *workspace,
                       size_t workspace_bytes, void *stream) {
  int rc = check_sizes(dtype, act, rows, cin, cout);
  if (rc) return rc;
  if (rows == 0) return DCN_OK;
  if (!x || !weight || !y) return set_error(DCN_ERR_ARG, "linear: x, weight and y must be non-NULL");
  if (ldx < cin || ldw < cin || (residual && ldr < cout))
    return set_error(DCN_ERR_ARG, "linear: a row stride is smaller than the row");
  LayerDeviceScope scope(device);
  if (scope.err != cudaSuccess) return cuda_error(scope.err);
  GemmArgs g = {};
  g.a = x; g.lda = ldx; g.b = weight; g.ldb = ldw;
  g.m = rows; g.n = cout; g.kk = cin;
  g.bias = bias; g.act = act; g.saved = saved; g.res = residual; g.ldr = ldr; g.out = y;
  cudaError_t e = launch_gemm_simple(g, dtype, (cudaStream_t)stream);
  return e == cudaSuccess ? DCN_OK : cuda_error(e);
}

int dcn_linear_backward_workspace_bytes(int32_t dtype, int32_t act, int64_t rows, int64_t cin, int64_t cout,
                                        int64_t alignment, int32_t want_gx, int32_t want_gw, size_t *bytes) {
  if (!bytes) return set_error(DCN_ERR_ARG, "linear: bytes is NULL");
  int rc = check_sizes(dtype, act, rows, cin, cout);
  if (rc) return rc;
  (void)alignment; (void)want_gx; (void)want_gw;
  *bytes = act == DCN_ACT_NONE ? 0 : up256((size_t)rows * cout * esize(dtype));
  return DCN_OK;
}

int dcn_linear_backward(const void *gy, int64_t ldgy, const void *x, int64_t ldx, const void *weight,
                        int64_t ldw, const void *saved, const void *in_saved, const void *gx_add, void *gx,
                        void *gw, void *gb, int32_t dtype, int32_t act, int32_t in_act, int64_t rows,
                        int64_t cin, int64_t cout, int32_t device, void *workspace, size_t workspace_bytes,
                        void *stream) {
  int rc = check_sizes(dtype, act, rows, cin, cout);
  if (!rc) rc = check_sizes(dtype, in_act, rows, cin, cout);
  if (rc) return rc;
  LayerDeviceScope scope(device);
  if (scope.err != cudaSuccess) return cuda_error(scope.err);
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e = cudaSuccess;
  if (rows == 0) {
    if (gw) e = cudaMemsetAsync(gw, 0, (size_t)cin * cout * esize(dtype), s);
    if (e == cudaSuccess && gb) e = cudaMemsetAsync(gb, 0, (size_t)cout * esize(dtype), s);
    return e == cudaSuccess ? DCN_OK : cuda_error(e);
  }
  if (!gy || (gx && !weight) || (gw && !x) || (act != DCN_ACT_NONE && !saved) ||
      (gx && in_act != DCN_ACT_NONE && !in_saved))
    return set_error(DCN_ERR_ARG, "linear backward: a needed pointer is NULL");
  if (ldgy < cout || (gw && ldx < cin) || (gx && ldw < cin))
    return set_error(DCN_ERR_ARG, "linear backward: a row stride is smaller than the row");
  size_t need = 0;
  dcn_linear_backward_workspace_bytes(dtype, act, rows, cin, cout, 0, gx != nullptr, gw != nullptr, &need);
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255)))
    return set_error(DCN_ERR_WORKSPACE, "linear backward: workspace missing, too small or misaligned");
  if (!gx && !gw && !gb) return DCN_OK;
  const void *gz = gy;
  long long ldgz = ldgy;
  if (act != DCN_ACT_NONE) {
    if (dtype == DCN_DTYPE_F32) e = run_gz<float>(gy, ldgy, saved, act, rows, cout, workspace, s);
    else if (dtype == DCN_DTYPE_BF16) e = run_gz<__nv_bfloat16>(gy, ldgy, saved, act, rows, cout, workspace, s);
    else e = run_gz<__half>(gy, ldgy, saved, act, rows, cout, workspace, s);
    if (e != cudaSuccess) return cuda_error(e);
    gz = workspace;
    ldgz = cout;
  }
  if (gx) {
    GemmArgs g = {};
    g.a = gz; g.lda = ldgz; g.b = weight; g.ldb = ldw; g.b_mn = true;
    g.m = rows; g.n = cin; g.kk = cout;
    g.slope = in_saved; g.slope_act = in_act; g.res = gx_add; g.ldr = cin; g.out = gx;
    e = launch_gemm_simple(g, dtype, s);
    if (e != cudaSuccess) return cuda_error(e);
  }
  if (gw) {
    GemmArgs g = {};
    g.a = gz; g.lda = ldgz; g.a_mn = true; g.b = x; g.ldb = ldx; g.b_mn = true;
    g.m = cout; g.n = cin; g.kk = rows;
    g.out = gw; g.row_sum = gb;
    e = launch_gemm_simple(g, dtype, s);
    if (e != cudaSuccess) return cuda_error(e);
  } else if (gb) {
    if (dtype == DCN_DTYPE_F32) e = run_column_sum<float>(gz, ldgz, rows, cout, gb, s);
    else if (dtype == DCN_DTYPE_BF16) e = run_column_sum<__nv_bfloat16>(gz, ldgz, rows, cout, gb, s);
    else e = run_column_sum<__half>(gz, ldgz, rows, cout, gb, s);
    if (e != cudaSuccess) return cuda_error(e);
  }
  return DCN_OK;
}

}  // extern "C"
