// Matrix product with an epilogue on the SIMT cores: any size, stride, alignment and type.
// out[i, j] = epilogue(sum_k A[i, k] * B[j, k]); 64 x 64 tiles, 16 values of k per step, fp32.
#include "dcn_layers.cuh"

namespace dcn {
namespace {

constexpr int kT = 64, kK = 16;

template <typename T>
__global__ void __launch_bounds__(256) gemm_simple(const GemmArgs g) {
  __shared__ float as[kK][kT + 1], bs[kK][kT + 1];
  const T *A = (const T *)g.a, *B = (const T *)g.b;
  const long long i0 = (long long)blockIdx.x * kT, j0 = (long long)blockIdx.y * kT;
  const int t = threadIdx.x, tx = t & 15, ty = t >> 4;
  float acc[4][4] = {}, rs[4] = {};
  for (long long k0 = 0; k0 < g.kk; k0 += kK) {
    for (int e = t; e < kT * kK; e += 256) {
      // the index that is contiguous in memory runs fastest
      const int ka = g.a_mn ? e / kT : e % kK, ia = g.a_mn ? e % kT : e / kK;
      const int kb = g.b_mn ? e / kT : e % kK, jb = g.b_mn ? e % kT : e / kK;
      as[ka][ia] = (k0 + ka < g.kk && i0 + ia < g.m)
                       ? ElemOf<T>::to(A[g.a_mn ? (k0 + ka) * g.lda + i0 + ia : (i0 + ia) * g.lda + k0 + ka]) : 0.f;
      bs[kb][jb] = (k0 + kb < g.kk && j0 + jb < g.n)
                       ? ElemOf<T>::to(B[g.b_mn ? (k0 + kb) * g.ldb + j0 + jb : (j0 + jb) * g.ldb + k0 + kb]) : 0.f;
    }
    __syncthreads();
    float part[4][4] = {}, prs[4] = {};   // a step's sums apart: long sums lose less
#pragma unroll
    for (int k = 0; k < kK; ++k) {
      float av[4], bv[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) { av[r] = as[k][ty * 4 + r]; bv[r] = bs[k][tx * 4 + r]; }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        prs[r] += av[r];
#pragma unroll
        for (int c = 0; c < 4; ++c) part[r][c] = fmaf(av[r], bv[c], part[r][c]);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      rs[r] += prs[r];
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[r][c] += part[r][c];
    }
    __syncthreads();
  }
  const long long words = (g.n + 31) / 32;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const long long i = i0 + ty * 4 + r;
    uint32_t bits = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const long long j = j0 + tx * 4 + c;
      if (i >= g.m || j >= g.n) continue;
      float v = acc[r][c] + (g.bias ? ElemOf<T>::to(((const T *)g.bias)[j]) : 0.f);
      if (g.saved) {
        if (g.act == DCN_ACT_RELU) bits |= (uint32_t)relu_bit(v) << ((tx * 4 + c) & 31);
        if (g.act == DCN_ACT_GELU) ((T *)g.saved)[i * g.n + j] = ElemOf<T>::from(v);
      }
      v = act_value(g.act, v);
      if (g.slope_act == DCN_ACT_RELU && !((((const uint32_t *)g.slope)[i * words + j / 32] >> (j & 31)) & 1u)) v = 0.f;
      if (g.slope_act == DCN_ACT_GELU) v *= gelu_slope(ElemOf<T>::to(((const T *)g.slope)[i * g.n + j]));
      if (g.res) v += ElemOf<T>::to(((const T *)g.res)[i * g.ldr + j]);
      ((T *)g.out)[i * g.n + j] = ElemOf<T>::from(v);
    }
    if (g.saved && g.act == DCN_ACT_RELU) {   // the eight threads of a 32-column word are neighbouring lanes
      for (int d = 1; d < 8; d <<= 1) bits |= __shfl_xor_sync(0xffffffffu, bits, d);
      const long long w = (j0 + tx * 4) / 32;
      if ((tx & 7) == 0 && i < g.m && w < words) ((uint32_t *)g.saved)[i * words + w] = bits;
    }
    if (g.row_sum && blockIdx.y == 0 && tx == 0 && i < g.m) ((T *)g.row_sum)[i] = ElemOf<T>::from(rs[r]);
  }
}

}  // namespace

cudaError_t launch_gemm_simple(const GemmArgs &g, int dtype, cudaStream_t s) {
  const dim3 grid((unsigned)((g.m + kT - 1) / kT), (unsigned)((g.n + kT - 1) / kT));
  if (dtype == DCN_DTYPE_F32) gemm_simple<float><<<grid, 256, 0, s>>>(g);
  else if (dtype == DCN_DTYPE_BF16) gemm_simple<__nv_bfloat16><<<grid, 256, 0, s>>>(g);
  else gemm_simple<__half><<<grid, 256, 0, s>>>(g);
  return cudaGetLastError();
}

}  // namespace dcn
