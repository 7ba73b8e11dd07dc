// The tensor-core products of fp32 tensors, as three bf16 planes.
#include "dcn_gemm_tc.cuh"

namespace dcn {

cudaError_t run_gemm_f32(GemmTc &p, int bn, int cg, bool parts, cudaStream_t s) {
  return run_order<__nv_bfloat16, float, 3>(p, bn, cg, parts, s);
}
cudaError_t read_gemm_status_f32(cudaStream_t s, int *status) { return read_status(s, status); }

}  // namespace dcn
