// Interface between the linear layer's C entries and the tensor-core product.
#pragma once

#include <cuda.h>

#include "dcn_layers.cuh"

namespace dcn {

// How a product is cut up; depends on sizes and type only, so that the workspace query and the call agree.
struct GemmPlan {
  int bn;          // columns of an output tile
  int cg;          // blocks that share a tile: 1 (128 rows) or a cluster of 2 (256 rows)
  int ks;          // blocks of a cluster that share a tile's sum over k, joined in shared memory (cg = 1, bn = 64)
  int splits;      // ranges of k, each with fp32 parts of its own in memory
  int kb_total, kb_split;   // 64-value blocks of k, in all and in a range
  long long ldp;   // row stride of the fp32 parts, elements
  size_t part_bytes, row_part_bytes;   // 0 without splits
};
GemmPlan plan_gemm(int planes, long long m, long long n, long long k, bool weight_gradient);

// 16 bytes of kept derivatives (of tensors of type T) as floats
template <typename T>
__device__ __forceinline__ void unpack_slopes(const uint4 &u, float *v) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[i] = __uint_as_float(w[i]);
    } else {
      v[2 * i] = slope_of_low(w[i]);
      v[2 * i + 1] = slope_of_high(w[i]);
    }
  }
}

template <typename T>
__device__ __forceinline__ void keep_slope(void *saved, long long at, float slope) {
  if constexpr (sizeof(T) == 4) ((float *)saved)[at] = slope;
  else ((uint16_t *)saved)[at] = (uint16_t)slope_code(slope);
}

// One launch of the tensor-core kernel.
struct alignas(64) GemmTc {
  CUtensorMap a, b, out, res, aux;
  GemmArgs g;
  int m, n;                        // of g
  int tiles_m, tiles_n, splits, kb_total, kb_split;
  int step_n, step_m, step_s;      // a block's stride through the items, in column tiles, row tiles and ranges
  int ks;
  int stages;
  int out_tma, res_tma;            // 0: element by element
  int bias16;                      // the bias starts on 16 bytes
  long long ldz;                   // row stride of kept derivatives: a multiple of 8
  float *row_part;                 // [splits][m], with splits > 1
  unsigned long long wait_limit_ns;
};

// One tensor type each (dcn_gemm_tc.cuh).
cudaError_t run_gemm_bf16(GemmTc &p, int bn, int cg, bool parts, cudaStream_t s);
cudaError_t run_gemm_f16(GemmTc &p, int bn, int cg, bool parts, cudaStream_t s);
cudaError_t run_gemm_f32(GemmTc &p, int bn, int cg, bool parts, cudaStream_t s);
cudaError_t read_gemm_status_bf16(cudaStream_t s, int *status);
cudaError_t read_gemm_status_f16(cudaStream_t s, int *status);
cudaError_t read_gemm_status_f32(cudaStream_t s, int *status);

// g.a / g.b point at 16-bit planes [planes][rows][ld] whose rows start on 16 bytes; g.out, g.res, g.saved
// and g.slope have the tensors' own `dtype`.  part / row_part: the plan's scratch.
cudaError_t launch_gemm_tc(const GemmArgs &g, const GemmPlan &plan, int dtype, float *part, float *row_part,
                           cudaStream_t s);

// The forward product for m <= 8 (g.a, g.b in the tensors' own type, k contiguous, any row stride).
cudaError_t launch_linear_rows(const GemmArgs &g, int dtype, cudaStream_t s);

// Up to two products in one launch, operands in the tensors' own type as they lie (dcn_gemm_simt.cu).
// a_saved / a_act: A is multiplied by that derivative, [rows of the tensor][its columns], as it is loaded.
// g.row_sum without g.out: the row sums alone.
struct SimtJob {
  GemmArgs g;
  const void *a_saved;
  int a_act;
  int tiles_n, tiles;
};
struct SimtJobs {
  SimtJob job[2];   // no tiles: nothing to do
};
SimtJob simt_job(const GemmArgs &g, const void *a_saved, int a_act);
cudaError_t launch_gemm_simt(const SimtJobs &jobs, int dtype, cudaStream_t s);

// Element-wise pass in front of a product: v = src * act'(saved), written as the planes that the
// product reads ([planes][rows][pitch], pitch: cols rounded up to 8).  With `sums`, [stage_slabs][cols] fp32
// column sums of v as well.
struct StageJob {
  const void *src, *saved;
  void *dst;
  float *sums;
  long long ld, rows, cols, pitch;
  int act;
  int vec_src;                // rows start on 16 bytes
  int log_tx, gx, gy, first;  // threads along a row, blocks along a row, slabs of rows, the first block
};
struct StageJobs {
  StageJob job[3];
  int count, blocks;
};
void add_stage(StageJobs *jobs, const void *src, long long ld, const void *saved, int act, long long rows, long long cols,
               int dtype, void *planes, float *sums);
cudaError_t launch_gemm_stage(StageJobs &jobs, int dtype, cudaStream_t s);
int stage_slabs(long long rows, long long cols);
// out[c] = sum over `parts` rows of part [parts][cols]
cudaError_t launch_column_reduce(const float *part, int parts, long long cols, int dtype, void *out, cudaStream_t s);

// The first bounded wait that ran out on the current device since the last reading (0: none);
// waits for `s`.
cudaError_t read_gemm_status(cudaStream_t s, int *status);

}  // namespace dcn
