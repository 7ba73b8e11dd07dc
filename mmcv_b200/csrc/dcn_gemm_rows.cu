// The forward product for up to eight rows (a token, a few queries):
//   y[r, n] = act(sum_k x[r, k] w[n, k] + b[n]) + res[r, n]
// What counts is the weight's way through the chip once and the latency of few waves of loads, so nothing is
// staged and no tensor core is asked: a warp owns a column, or a half or quarter of its k (KP = 2, 4: as many
// times the blocks, and that part of the turns), its lanes lie along k, 16 bytes of the weight each and four
// loads in flight, and x comes from L1.  The R sums of a warp are joined by exchanges in which each lane gives
// away the half that its partner keeps, the warps of a column in order.  More columns to a warp were slower
// (1 x 4096 x 4096 bf16: one 11.5 us, two 17.8, four 31.7).  Bound: memory (the weight), or the launch.
// Measured against the other kernels: forward_rows in dcn_linear.cu.
#include "dcn_gemm.cuh"

namespace dcn {
namespace {

// V elements of T as floats: 16 bytes at once where `whole`, else those below `left`, the others zero
template <typename T, int V>
__device__ __forceinline__ uint4 load16(const T *p, int left) {
  if (V > 1 && left >= V) return __ldg(reinterpret_cast<const uint4 *>(p));
  uint4 u = make_uint4(0, 0, 0, 0);
  T *e = reinterpret_cast<T *>(&u);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < left) e[i] = p[i];
  return u;
}
template <typename T, int V>
__device__ __forceinline__ void floats(const uint4 &u, float (&o)[V]) {
  const T *e = reinterpret_cast<const T *>(&u);
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = ElemOf<T>::to(e[i]);
}

template <typename T, int V, int R, int KP>
__global__ void __launch_bounds__(1024) dcn_linear_rows(const GemmArgs g) {
  constexpr int U = 4, CB = 32 / KP;    // chunks of k in flight; columns of a block
  __shared__ uint32_t bits[R];
  __shared__ float join[KP > 1 ? KP : 1][CB][R];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = warp % CB, part = warp / CB;
  const int m = (int)g.m, n = (int)g.n, kk = (int)g.kk;
  const int j = blockIdx.x * CB + col;
  const bool keep_bits = g.act == DCN_ACT_RELU && g.saved;
  pdl_wait();
  pdl_launch();
  if (keep_bits) {
    if (threadIdx.x < R) bits[threadIdx.x] = 0u;
    __syncthreads();
  }
  const T *w = (const T *)g.b + (long long)min(j, n - 1) * g.ldb, *x = (const T *)g.a;
  float acc[R] = {};
  for (int k0 = (part * 32 + lane) * V; k0 < kk; k0 += 32 * V * KP * U) {
    uint4 wu[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * 32 * V * KP;
      wu[u] = make_uint4(0, 0, 0, 0);
      if (k < kk) wu[u] = load16<T, V>(w + k, kk - k);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * 32 * V * KP;
      if (k >= kk) break;
      float wv[V];
      floats<T, V>(wu[u], wv);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float xv[V];
        floats<T, V>(load16<T, V>(x + min(r, m - 1) * g.lda + k, kk - k), xv);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[r] = fmaf(xv[i], wv[i], acc[r]);
      }
    }
  }
  // lane / (32 / R) ends up with the sum acc[lane / (32 / R)] over the warp
  int have = R;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    if (have > 1) {
      have /= 2;
      const bool up = (lane & d) != 0;
#pragma unroll
      for (int i = 0; i < have; ++i) {
        const float give = up ? acc[i] : acc[i + have], keep = up ? acc[i + have] : acc[i];
        acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, d);
      }
    } else {
      acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], d);
    }
  }
  const int r = lane / (32 / R);
  const bool mine = lane % (32 / R) == 0;
  float v = acc[0];
  if constexpr (KP > 1) {
    if (mine) join[part][col][r] = v;
    __syncthreads();
    if (part == 0) {
      v = join[0][col][r];
#pragma unroll
      for (int q = 1; q < KP; ++q) v += join[q][col][r];
    }
  }
  if (part == 0 && mine && j < n && r < m) {
    constexpr bool kFine = sizeof(T) == 4;
    if (g.bias) v += ElemOf<T>::to(((const T *)g.bias)[j]);
    if (g.act == DCN_ACT_RELU) {
      if (keep_bits && relu_bit(v)) atomicOr(&bits[r], 1u << col);
      v = relu_value(v);
    } else if (g.act == DCN_ACT_GELU) {
      if (g.saved) keep_slope<T>(g.saved, r * ((g.n + 7) / 8 * 8) + j, gelu_slope<kFine>(v));
      v = gelu_value<kFine>(v);
    }
    if (g.res) v += ElemOf<T>::to(((const T *)g.res)[r * g.ldr + j]);
    ((T *)g.out)[r * g.n + j] = ElemOf<T>::from(v);
  }
  if (keep_bits) {   // a block's columns are a word of the bits, or a half or byte of one
    __syncthreads();
    if ((int)threadIdx.x < m) {
      uint32_t *row = (uint32_t *)g.saved + threadIdx.x * ((g.n + 31) / 32);
      if constexpr (CB == 32) row[blockIdx.x] = bits[threadIdx.x];
      else if constexpr (CB == 16) ((uint16_t *)row)[blockIdx.x] = (uint16_t)bits[threadIdx.x];
      else ((uint8_t *)row)[blockIdx.x] = (uint8_t)bits[threadIdx.x];
    }
  }
}

template <typename T, int V, int R>
cudaError_t run_rows(const GemmArgs &g, cudaStream_t s) {
  // parts of k while the blocks that come of it have an SM each (1 x 4096 x 1024 bf16: quarters 3.6 us, whole
  // columns 8.8; 1 x 1024 x 4096: 7.2, 3.4)
  if (g.n <= 8 * 148) return launch_pdl(dcn_linear_rows<T, V, R, 4>, (unsigned)((g.n + 7) / 8), 1024, 0, s, 1, g);
  if (g.n <= 16 * 148) return launch_pdl(dcn_linear_rows<T, V, R, 2>, (unsigned)((g.n + 15) / 16), 1024, 0, s, 1, g);
  return launch_pdl(dcn_linear_rows<T, V, R, 1>, (unsigned)((g.n + 31) / 32), 1024, 0, s, 1, g);
}
template <typename T, int V>
cudaError_t run_v(const GemmArgs &g, cudaStream_t s) {
  if (g.m == 1) return run_rows<T, V, 1>(g, s);
  if (g.m == 2) return run_rows<T, V, 2>(g, s);
  if (g.m <= 4) return run_rows<T, V, 4>(g, s);
  return run_rows<T, V, 8>(g, s);
}
template <typename T>
cudaError_t run(const GemmArgs &g, cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  if (aligned16(g.a) && aligned16(g.b) && (g.lda % V == 0 || g.m == 1) && (g.ldb % V == 0 || g.n == 1)) return run_v<T, V>(g, s);
  return run_v<T, 1>(g, s);
}

}  // namespace

cudaError_t launch_linear_rows(const GemmArgs &g, int dtype, cudaStream_t s) {
  if (dtype == DCN_DTYPE_F32) return run<float>(g, s);
  if (dtype == DCN_DTYPE_BF16) return run<__nv_bfloat16>(g, s);
  return run<__half>(g, s);
}

}  // namespace dcn
