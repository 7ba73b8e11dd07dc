// The forward product for up to eight rows (a token, a few queries):
//   y[r, n] = act(sum_k x[r, k] w[n, k] + b[n]) + res[r, n]
// What counts is the weight's way through the chip once and the latency of a single wave of loads, so
// nothing is staged and no tensor core is asked: a warp owns NC columns, its lanes lie along k, 16 bytes
// of the weight each, and x comes from L1.  The NC * R sums of a warp are joined by exchanges in which
// each lane gives away the half that its partner keeps.  A block has 32 columns, so that it owns whole
// words of relu's kept bits.  Bound: memory (the weight), or the launch.
// Measured against the tensor-core kernel (its tiles are 128 rows): see run_rows.
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

template <typename T, int V, int R, int NC>
__global__ void __launch_bounds__(1024 / NC) dcn_linear_rows(const GemmArgs g) {
  constexpr int U = 4 / NC;             // chunks of k in flight: four loads of the weight in all
  constexpr int N = NC * R;
  __shared__ uint32_t bits[R];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int m = (int)g.m, n = (int)g.n, kk = (int)g.kk;
  const int j0 = blockIdx.x * 32 + warp * NC;
  const T *w = (const T *)g.b, *x = (const T *)g.a;
  const bool keep_bits = g.act == DCN_ACT_RELU && g.saved;
  pdl_wait();
  pdl_launch();
  if (keep_bits) {
    if (threadIdx.x < R) bits[threadIdx.x] = 0u;
    __syncthreads();
  }
  float acc[N] = {};
  if (j0 < n) {
    for (int k0 = lane * V; k0 < kk; k0 += 32 * V * U) {
      uint4 wu[U][NC];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int k = k0 + u * 32 * V;
          wu[u][c] = make_uint4(0, 0, 0, 0);
          if (k < kk) wu[u][c] = load16<T, V>(w + min(j0 + c, n - 1) * g.ldb + k, kk - k);
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * 32 * V;
        if (k >= kk) break;
        float wv[NC][V];
#pragma unroll
        for (int c = 0; c < NC; ++c) floats<T, V>(wu[u][c], wv[c]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float xv[V];
          floats<T, V>(load16<T, V>(x + min(r, m - 1) * g.lda + k, kk - k), xv);
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) acc[c * R + r] = fmaf(xv[i], wv[c][i], acc[c * R + r]);
        }
      }
    }
  }
  // lane / (32 / N) ends up with the sum acc[lane / (32 / N)] over the warp
  int have = N;
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
  const int idx = lane / (32 / N), c = idx / R, r = idx % R, j = j0 + c;
  if (lane % (32 / N) == 0 && j < n && r < m) {
    constexpr bool kFine = sizeof(T) == 4;
    float v = acc[0];
    if (g.bias) v += ElemOf<T>::to(((const T *)g.bias)[j]);
    if (g.act == DCN_ACT_RELU) {
      if (keep_bits && relu_bit(v)) atomicOr(&bits[r], 1u << (j & 31));
      v = relu_value(v);
    } else if (g.act == DCN_ACT_GELU) {
      if (g.saved) keep_slope<T>(g.saved, r * ((g.n + 7) / 8 * 8) + j, gelu_slope<kFine>(v));
      v = gelu_value<kFine>(v);
    }
    if (g.res) v += ElemOf<T>::to(((const T *)g.res)[r * g.ldr + j]);
    ((T *)g.out)[r * g.n + j] = ElemOf<T>::from(v);
  }
  if (keep_bits) {
    __syncthreads();
    if ((int)threadIdx.x < m) ((uint32_t *)g.saved)[threadIdx.x * ((g.n + 31) / 32) + blockIdx.x] = bits[threadIdx.x];
  }
}

template <typename T, int V, int R>
cudaError_t run_rows(const GemmArgs &g, cudaStream_t s) {
  const unsigned blocks = (unsigned)((g.n + 31) / 32);
  // one column a warp while the blocks do not fill the SMs: a column's loads are then spread over more of them
  if (blocks < 148) return launch_pdl(dcn_linear_rows<T, V, R, 1>, blocks, 1024, 0, s, 1, g);
  return launch_pdl(dcn_linear_rows<T, V, R, 4>, blocks, 256, 0, s, 1, g);
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
