// C entries of the matrix product with bias, activation and residual in its epilogue, forward and
// backward: argument checks, workspace layout, and the sequence of kernels of each pass.
//   forward   y = act(x W^T + b) + r                       one product
//   backward  gz = gy * act'(z)                            element-wise, only with an activation
//             gx = gz W  (times the derivative of the activation before, plus gx_add)
//             gW = gz^T x,  gb = column sums of gz
// Column sums of gx on its way through that derivative (the bias gradient of the layer before) are taken
// from the epilogue's fp32 values: gx itself is rounded to the tensors' type.
// Few rows and small fp32 or unaligned problems have kernels of their own, which read everything where and as
// it lies (dcn_linear_rows, dcn_gemm_simt).  For the tensor cores, 16-bit operands whose rows start on 16
// bytes are read where they lie; others are first copied to rows that do, and fp32 operands are split into
// three bf16 planes (dcn_gemm_stage, both).
#include "dcn_gemm.cuh"

namespace dcn {

namespace {

size_t up256(size_t v) { return (v + 255) / 256 * 256; }
size_t esize(int dtype) { return dtype == DCN_DTYPE_F32 ? 4 : 2; }
int planes_of(int dtype) { return dtype == DCN_DTYPE_F32 ? 3 : 1; }
long long pitch_of(long long cols) { return (cols + 7) / 8 * 8; }
size_t plane_bytes(int dtype, long long rows, long long cols) {
  return up256((size_t)planes_of(dtype) * rows * pitch_of(cols) * 2);
}

// Byte offsets of a pass's scratch tensors; total in `bytes`.
struct Layout {
  size_t gz = 0, x = 0, w = 0, part = 0, row_part = 0, sums = 0, gx_sums = 0, bytes = 0;
  bool stage_gz = false, stage_x = false, stage_w = false;
  bool rows = false, simt = false;   // nothing staged: dcn_linear_rows, dcn_gemm_simt
  GemmPlan gx_plan = {}, gw_plan = {};
};
size_t take(Layout *l, size_t n) {
  const size_t at = l->bytes;
  l->bytes += up256(n);
  return at;
}
bool needs_stage(int dtype, int64_t alignment) { return dtype == DCN_DTYPE_F32 || (alignment & 15) != 0; }

// Which kernel a pass runs on; depends on sizes, type and alignment only, so that the workspace query and
// the call agree and a call that keeps something for the backward pass gives the same bits as one that
// does not.
//
// Times in us of one call among others, here / tensor cores with their staging pass:
//   dcn_linear_rows   1 x 256 x 1024 bf16 2.0 / 5.0, fp32 2.1 / 9.2; 8 x 1024 x 1024 bf16 4.7 / 8.5, fp32
//                     5.5 / 16; 8 x 4096 x 1024 bf16 10.5 / 11.9, fp32 16 / 41; but 8 x 1024 x 4096 bf16
//                     10.9 / 9.0, 4 x 4096 x 4096 21 / 21, 1 x 2048 x 16384 26 / 22 (fp32 32 / 108)
//   dcn_gemm_simt     forward, fp32: 300 x 256 x 256 7.9 / 10.8, 600 x 256 x 256 11.2 / 10.9; backward, fp32:
//                     300 x 256 x 256 9.1 / 25, 600 x 256 x 256 19 / 27
// and its one launch takes the place of two to six.  16-bit operands that need no staging stay on the tensor
// cores (32 x 256 x 256 bf16 backward: 10.7 / 9.7).
bool forward_rows(int dtype, long long rows, long long cout, int64_t alignment) {
  if (needs_stage(dtype, alignment) || cout <= 8 * 148) return rows <= 8;
  return rows <= 4 && cout <= 32 * 148;
}
// rows as whole tiles
double products(long long rows, long long cin, long long cout) {
  return (double)((rows + 31) / 32 * 32) * (double)cin * (double)cout;
}
bool forward_simt(int dtype, long long rows, long long cin, long long cout) {
  return dtype == DCN_DTYPE_F32 && cin <= 1024 && products(rows, cin, cout) <= 1 << 25;
}
// a block walks all of cout (for gx) or of the rows (for gw): long walks are slow
bool backward_simt(int dtype, long long rows, long long cin, long long cout, int64_t alignment) {
  return needs_stage(dtype, alignment) && rows <= 640 && cout <= 640 && products(rows, cin, cout) <= 1 << 25;
}

Layout forward_layout(int dtype, long long rows, long long cin, long long cout, int64_t alignment) {
  Layout l;
  l.rows = forward_rows(dtype, rows, cout, alignment);
  l.simt = !l.rows && forward_simt(dtype, rows, cin, cout);
  if (l.rows || l.simt) return l;
  l.stage_x = l.stage_w = needs_stage(dtype, alignment);
  if (l.stage_x) {
    l.x = take(&l, plane_bytes(dtype, rows, cin));
    l.w = take(&l, plane_bytes(dtype, cout, cin));
  }
  return l;
}

Layout backward_layout(int dtype, int act, long long rows, long long cin, long long cout, int64_t alignment,
                       bool want_gx, bool want_gw, bool want_gb, bool want_gx_sum) {
  Layout l;
  if (want_gx_sum) l.gx_sums = take(&l, (size_t)((rows + 31) / 32) * cin * 4);
  l.simt = backward_simt(dtype, rows, cin, cout, alignment);
  if (l.simt) return l;
  const bool stage = needs_stage(dtype, alignment);
  l.stage_gz = stage || act != DCN_ACT_NONE || (want_gb && !want_gw);   // the last: for its column sums
  l.stage_x = stage && want_gw;
  l.stage_w = stage && want_gx;
  if (l.stage_gz) l.gz = take(&l, plane_bytes(dtype, rows, cout));
  if (l.stage_x) l.x = take(&l, plane_bytes(dtype, rows, cin));
  if (l.stage_w) l.w = take(&l, plane_bytes(dtype, cout, cin));
  if (want_gx) l.gx_plan = plan_gemm(planes_of(dtype), rows, cin, cout, false);
  if (want_gw) {
    l.gw_plan = plan_gemm(planes_of(dtype), cout, cin, rows, true);
    l.part = take(&l, l.gw_plan.part_bytes);
    l.row_part = take(&l, l.gw_plan.row_part_bytes);
  }
  if (l.stage_gz) l.sums = take(&l, (size_t)stage_slabs(rows, cout) * cout * 4);
  return l;
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
  *bytes = forward_layout(dtype, rows, cin, cout, alignment).bytes;
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
  if (act == DCN_ACT_GELU && !aligned16(saved)) return set_error(DCN_ERR_ARG, "linear: saved must be 16-byte aligned");
  LayerDeviceScope scope(device);
  if (scope.err != cudaSuccess) return cuda_error(scope.err);
  cudaStream_t s = (cudaStream_t)stream;
  const int64_t es = (int64_t)esize(dtype);
  const int64_t alignment = (int64_t)(uintptr_t)x | (int64_t)(uintptr_t)weight | ((ldx | ldw) * es);
  const Layout l = forward_layout(dtype, rows, cin, cout, alignment);
  if (l.bytes && (!workspace || workspace_bytes < l.bytes || ((uintptr_t)workspace & 255)))
    return set_error(DCN_ERR_WORKSPACE, "linear: workspace missing, too small or misaligned");
  uint8_t *ws = (uint8_t *)workspace;
  cudaError_t e = cudaSuccess;
  GemmArgs g = {};
  g.a = x; g.lda = ldx; g.b = weight; g.ldb = ldw;
  g.m = rows; g.n = cout; g.kk = cin;
  g.bias = bias; g.act = act; g.saved = saved; g.res = residual; g.ldr = ldr; g.out = y;
  if (l.rows || l.simt) {
    SimtJobs jobs = {};
    if (l.simt) jobs.job[0] = simt_job(g, nullptr, DCN_ACT_NONE);
    e = l.simt ? launch_gemm_simt(jobs, dtype, s) : launch_linear_rows(g, dtype, s);
    return e == cudaSuccess ? DCN_OK : cuda_error(e);
  }
  if (l.stage_x) {
    StageJobs jobs = {};
    add_stage(&jobs, x, ldx, nullptr, DCN_ACT_NONE, rows, cin, dtype, ws + l.x, nullptr);
    add_stage(&jobs, weight, ldw, nullptr, DCN_ACT_NONE, cout, cin, dtype, ws + l.w, nullptr);
    e = launch_gemm_stage(jobs, dtype, s);
    if (e != cudaSuccess) return cuda_error(e);
    g.a = ws + l.x;
    g.b = ws + l.w;
    g.lda = g.ldb = pitch_of(cin);
  }
  e = launch_gemm_tc(g, plan_gemm(planes_of(dtype), rows, cout, cin, false), dtype, nullptr, nullptr, s);
  return e == cudaSuccess ? DCN_OK : cuda_error(e);
}

int dcn_linear_backward_workspace_bytes(int32_t dtype, int32_t act, int64_t rows, int64_t cin, int64_t cout,
                                        int64_t alignment, int32_t want_gx, int32_t want_gw, int32_t want_gb,
                                        size_t *bytes) {
  if (!bytes) return set_error(DCN_ERR_ARG, "linear: bytes is NULL");
  int rc = check_sizes(dtype, act, rows, cin, cout);
  if (rc) return rc;
  *bytes = rows ? backward_layout(dtype, act, rows, cin, cout, alignment, want_gx != 0, want_gw != 0, want_gb != 0,
                                  want_gx == 2).bytes : 0;
  return DCN_OK;
}

int dcn_linear_backward(const void *gy, int64_t ldgy, const void *x, int64_t ldx, const void *weight,
                        int64_t ldw, const void *saved, const void *in_saved, const void *gx_add, void *gx,
                        void *gx_sum, void *gw, void *gb, int32_t dtype, int32_t act, int32_t in_act, int64_t rows,
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
    if (e == cudaSuccess && gx_sum) e = cudaMemsetAsync(gx_sum, 0, (size_t)cin * esize(dtype), s);
    return e == cudaSuccess ? DCN_OK : cuda_error(e);
  }
  if (!gy || (gx && !weight) || (gw && !x) || (act != DCN_ACT_NONE && !saved) ||
      (gx && in_act != DCN_ACT_NONE && !in_saved))
    return set_error(DCN_ERR_ARG, "linear backward: a needed pointer is NULL");
  if (gx_sum && (!gx || gx_add || in_act == DCN_ACT_NONE))
    return set_error(DCN_ERR_ARG, "linear backward: gx_sum goes with gx and in_act, without gx_add");
  if (ldgy < cout || (gw && ldx < cin) || (gx && ldw < cin))
    return set_error(DCN_ERR_ARG, "linear backward: a row stride is smaller than the row");
  if ((act == DCN_ACT_GELU && !aligned16(saved)) || (in_act == DCN_ACT_GELU && !aligned16(in_saved)))
    return set_error(DCN_ERR_ARG, "linear backward: saved and in_saved must be 16-byte aligned");
  if (!gx && !gw && !gb) return DCN_OK;
  const int64_t es = (int64_t)esize(dtype);
  const int64_t alignment = (int64_t)(uintptr_t)gy | (gw ? (int64_t)(uintptr_t)x | ldx * es : 0) |
                            (gx ? (int64_t)(uintptr_t)weight | ldw * es : 0) | ldgy * es;
  const Layout l = backward_layout(dtype, act, rows, cin, cout, alignment, gx != nullptr, gw != nullptr, gb != nullptr,
                                   gx_sum != nullptr);
  if (l.bytes && (!workspace || workspace_bytes < l.bytes || ((uintptr_t)workspace & 255)))
    return set_error(DCN_ERR_WORKSPACE, "linear backward: workspace missing, too small or misaligned");
  uint8_t *ws = (uint8_t *)workspace;
  if (l.simt) {
    SimtJobs jobs = {};
    float *gx_part = gx_sum ? (float *)(ws + l.gx_sums) : nullptr;
    if (gx) {
      GemmArgs g = {};
      g.a = gy; g.lda = ldgy; g.b = weight; g.ldb = ldw; g.b_mn = true;
      g.m = rows; g.n = cin; g.kk = cout;
      g.slope = in_saved; g.slope_act = in_act; g.res = gx_add; g.ldr = cin; g.out = gx; g.col_part = gx_part;
      jobs.job[0] = simt_job(g, saved, act);
    }
    if (gw || gb) {
      GemmArgs g = {};
      g.a = gy; g.lda = ldgy; g.a_mn = true; g.b = x; g.ldb = ldx; g.b_mn = true;
      g.m = cout; g.n = cin; g.kk = rows;
      g.out = gw; g.row_sum = gb;
      jobs.job[1] = simt_job(g, saved, act);
    }
    e = launch_gemm_simt(jobs, dtype, s);
    if (e == cudaSuccess && gx_sum) e = launch_column_reduce(gx_part, (int)((rows + 31) / 32), cin, dtype, gx_sum, s);
    return e == cudaSuccess ? DCN_OK : cuda_error(e);
  }
  const void *gz = gy, *xs = x, *wt = weight;
  long long ldgz = ldgy, ldxs = ldx, ldwt = ldw;
  // the bias gradient: column sums of the staging pass, taken before gz is rounded, where there is one,
  // else row sums of the weight gradient's A operand
  const bool sums = gb && l.stage_gz;
  StageJobs jobs = {};
  if (l.stage_gz) {
    add_stage(&jobs, gy, ldgy, saved, act, rows, cout, dtype, ws + l.gz, sums ? (float *)(ws + l.sums) : nullptr);
    gz = ws + l.gz;
    ldgz = pitch_of(cout);
  }
  if (l.stage_x) {
    add_stage(&jobs, x, ldx, nullptr, DCN_ACT_NONE, rows, cin, dtype, ws + l.x, nullptr);
    xs = ws + l.x;
    ldxs = pitch_of(cin);
  }
  if (l.stage_w) {
    add_stage(&jobs, weight, ldw, nullptr, DCN_ACT_NONE, cout, cin, dtype, ws + l.w, nullptr);
    wt = ws + l.w;
    ldwt = pitch_of(cin);
  }
  e = launch_gemm_stage(jobs, dtype, s);
  const bool joined = sums && gw && l.gw_plan.splits > 1;   // by the launch that joins the weight gradient's parts
  if (e == cudaSuccess && sums && !joined)
    e = launch_column_reduce((const float *)(ws + l.sums), stage_slabs(rows, cout), cout, dtype, gb, s);
  if (e != cudaSuccess) return cuda_error(e);
  if (gx) {
    GemmArgs g = {};
    g.a = gz; g.lda = ldgz; g.b = wt; g.ldb = ldwt; g.b_mn = true;
    g.m = rows; g.n = cin; g.kk = cout;
    g.slope = in_saved; g.slope_act = in_act; g.res = gx_add; g.ldr = cin; g.out = gx;
    g.col_part = gx_sum ? (float *)(ws + l.gx_sums) : nullptr;
    e = launch_gemm_tc(g, l.gx_plan, dtype, nullptr, nullptr, s);
    if (e == cudaSuccess && gx_sum) e = launch_column_reduce(g.col_part, (int)((rows + 31) / 32), cin, dtype, gx_sum, s);
    if (e != cudaSuccess) return cuda_error(e);
  }
  if (gw) {
    GemmArgs g = {};
    g.a = gz; g.lda = ldgz; g.a_mn = true; g.b = xs; g.ldb = ldxs; g.b_mn = true;
    g.m = cout; g.n = cin; g.kk = rows;
    g.out = gw; g.row_sum = sums ? nullptr : gb;
    if (joined) {
      g.join_part = (const float *)(ws + l.sums);
      g.join_parts = stage_slabs(rows, cout);
      g.join_out = gb;
    }
    e = launch_gemm_tc(g, l.gw_plan, dtype, (float *)(ws + l.part), (float *)(ws + l.row_part), s);
    if (e != cudaSuccess) return cuda_error(e);
  }
  return DCN_OK;
}

int dcn_linear_read_status(int32_t device, void *stream, int32_t *status) {
  if (!status) return set_error(DCN_ERR_ARG, "linear: status is NULL");
  LayerDeviceScope scope(device);
  if (scope.err != cudaSuccess) return cuda_error(scope.err);
  const cudaError_t e = read_gemm_status((cudaStream_t)stream, status);
  return e == cudaSuccess ? DCN_OK : cuda_error(e);
}

}  // extern "C"
