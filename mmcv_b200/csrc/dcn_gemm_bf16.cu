// The tensor-core products of bf16 tensors.
#include "dcn_gemm_tc.cuh"

namespace dcn {

cudaError_t run_gemm_bf16(GemmTc &p, int bn, int cg, bool parts, cudaStream_t s) {
  return run_order<__nv_bfloat16, __nv_bfloat16, 1>(p, bn, cg, parts, s);
}
cudaError_t read_gemm_status_bf16(cudaStream_t s, int *status) { return read_status(s, status); }

}  // namespace dcn
