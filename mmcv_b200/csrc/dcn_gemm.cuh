// Interface between the linear layer's C entries and the tensor-core product.
#pragma once

#include "dcn_layers.cuh"

namespace dcn {

// How a product is cut up; depends on sizes and type only, so that the workspace query and the call agree.
struct GemmPlan {
  int bn;          // columns of an output tile
  int cg;          // blocks that share a tile: 1 (128 rows) or a cluster of 2 (256 rows)
  int splits;      // ranges of k, each with fp32 parts of its own
  int kb_total, kb_split;   // 64-value blocks of k, in all and in a range
  long long ldp;   // row stride of the fp32 parts, elements
  size_t part_bytes, row_part_bytes;   // 0 without splits
};
GemmPlan plan_gemm(int planes, long long m, long long n, long long k, bool weight_gradient);

// g.a / g.b point at 16-bit planes [planes][rows][ld] whose rows start on 16 bytes; g.out, g.res, g.saved
// and g.slope have the tensors' own `dtype`.  part / row_part: the plan's scratch.
cudaError_t launch_gemm_tc(const GemmArgs &g, const GemmPlan &plan, int dtype, float *part, float *row_part,
                           cudaStream_t s);

// Element-wise pass in front of a product: v = src * act'(saved), written as the planes that the
// product reads ([planes][rows][pitch], pitch a multiple of 8).  With `sums`, [slabs][cols] fp32
// column sums of v as well; returns the number of slabs through *slabs.
cudaError_t launch_gemm_stage(const void *src, long long ld, const void *saved, int act, long long rows,
                              long long cols, int dtype, void *planes, long long pitch, float *sums, int *slabs,
                              cudaStream_t s);
int stage_slabs(long long rows, long long cols);
// out[c] = sum over `parts` rows of part [parts][cols]
cudaError_t launch_column_reduce(const float *part, int parts, long long cols, int dtype, void *out, cudaStream_t s);

// The first bounded wait that ran out on the current device since the last reading (0: none);
// waits for `s`.
cudaError_t read_gemm_status(cudaStream_t s, int *status);

}  // namespace dcn
