// The tensor-core products of fp16 tensors.
#include "dcn_gemm_tc.cuh"

namespace dcn {

cudaError_t run_gemm_f16(GemmTc &p, int bn, int cg, bool parts, cudaStream_t s) {
  return run_order<__half, __half, 1>(p, bn, cg, parts, s);
}
cudaError_t read_gemm_status_f16(cudaStream_t s, int *status) { return read_status(s, status); }

}  // namespace dcn
