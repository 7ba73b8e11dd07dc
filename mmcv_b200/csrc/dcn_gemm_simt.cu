// Matrix products of small problems on the ordinary cores, operands read where and as they lie:
//   out[i, j] = epilogue(sum_k A[i, k] * B[j, k])
// The tensor-core kernel wants operands whose rows start on 16 bytes and fp32 as three planes, so small
// fp32 and odd-sized problems spend their time on the passes that write those, and a backward pass is
// four to seven launches of a few microseconds.  Here a forward product is one launch and a backward pass
// (both of its products, the bias gradient and the activation's derivative) is one as well: the derivative
// is applied to the gradient while a tile is loaded, in fp32 and unrounded.
//
// A block of 256 threads computes 32 x 32 results over 64 values of k at a time: four groups of 64 threads
// take 16 of them each, 4 x 4 results to a thread, and are added in order at the end.  The next 64 values
// are in registers while these are multiplied.  Bound: with few tiles the chain of loads (1.2 us for 64 values of
// k), else the shared-memory reads and FMAs of the 4 x 4 step.  300 x 256 x 256 fp32: forward 7.9 us, backward 9.1;
// backward_simt in dcn_linear.cu has the other kernels' times.
#include "dcn_gemm.cuh"

namespace dcn {
namespace {

constexpr int kTile = 32, kStep = 64, kPitch = kTile + 4;   // (k + i) pitch: 16-byte rows, no bank conflicts

// act'(z) from what the forward pass kept at [r, c] of [rows, cols]
template <typename T>
__device__ __forceinline__ float slope_at(const void *saved, int act, long long r, long long c, long long cols) {
  if (act == DCN_ACT_RELU)
    return (((const uint32_t *)saved)[r * ((cols + 31) / 32) + (c >> 5)] >> (c & 31)) & 1u ? 1.f : 0.f;
  const long long at = r * ((cols + 7) / 8 * 8) + c;
  if constexpr (sizeof(T) == 4) return ((const float *)saved)[at];
  else return slope_of_low(((const uint16_t *)saved)[at]);
}
// g * act'(z); relu drops g where the bit is off, whatever g is
template <typename T>
__device__ __forceinline__ float through(float g, const void *saved, int act, long long r, long long c, long long cols) {
  const float s = slope_at<T>(saved, act, r, c, cols);
  return act == DCN_ACT_RELU ? (s != 0.f ? g : 0.f) : g * s;
}

// Eight elements of a 32 x 64 (index x k) piece of an operand to a thread: neighbouring lanes along whichever
// index is contiguous in memory (along k: eight by four, so that the writes to shared memory, k-major, do not
// meet on a bank).
__device__ __forceinline__ void place(bool mn, int e, int &i, int &k) {
  const int t = threadIdx.x;
  if (mn) {
    i = t & 31;
    k = (t >> 5) + e * 8;
  } else {
    k = (t & 7) + (e & 7) * 8;
    i = (t >> 3) & 31;
  }
}

template <typename T>
__device__ void tile_product(const SimtJob &p, int tile, float *smem) {
  const GemmArgs &g = p.g;
  const int t = threadIdx.x, tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
  const long long i0 = (long long)tm * kTile;
  const int j0 = tn * kTile;
  const int m = (int)min((long long)kTile, g.m - i0), n = g.out ? (int)min((long long)kTile, g.n - j0) : 0;
  float *as = smem, *bs = smem + kStep * kPitch;
  const T *a = (const T *)g.a + (g.a_mn ? i0 : i0 * g.lda), *b = (const T *)g.b + (g.b_mn ? j0 : j0 * g.ldb);
  const long long ai = g.a_mn ? 1 : g.lda, ak = g.a_mn ? g.lda : 1, bj = g.b_mn ? 1 : g.ldb, bk = g.b_mn ? g.ldb : 1;
  const bool sums = g.row_sum && tn == 0;
  float ra[8], rb[8];
  auto fetch = [&](long long k0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      int i, k;
      place(g.a_mn, e, i, k);
      ra[e] = i < m && k0 + k < g.kk ? ElemOf<T>::to(a[i * ai + (k0 + k) * ak]) : 0.f;
      place(g.b_mn, e, i, k);
      rb[e] = i < n && k0 + k < g.kk ? ElemOf<T>::to(b[i * bj + (k0 + k) * bk]) : 0.f;
    }
    if (p.a_act != DCN_ACT_NONE) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        int i, k;
        place(g.a_mn, e, i, k);
        if (i < m && k0 + k < g.kk)
          ra[e] = g.a_mn ? through<T>(ra[e], p.a_saved, p.a_act, k0 + k, i0 + i, g.m)
                         : through<T>(ra[e], p.a_saved, p.a_act, i0 + i, k0 + k, g.kk);
      }
    }
  };
  const int grp = t >> 6, tx = t & 7, ty = (t >> 3) & 7;
  float acc[4][4] = {};
  float row = 0.f;
  fetch(0);
  for (long long k0 = 0; k0 < g.kk; k0 += kStep) {
    __syncthreads();   // the last step's values have been used
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      int i, k;
      place(g.a_mn, e, i, k);
      as[k * kPitch + i] = ra[e];
      place(g.b_mn, e, i, k);
      bs[k * kPitch + i] = rb[e];
    }
    __syncthreads();
    if (k0 + kStep < g.kk) fetch(k0 + kStep);
    if (sums) {
#pragma unroll
      for (int k = 0; k < 8; ++k) row += as[((t >> 5) * 8 + k) * kPitch + (t & 31)];
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float4 av = *reinterpret_cast<const float4 *>(as + (grp * 16 + k) * kPitch + ty * 4);
      const float4 bv = *reinterpret_cast<const float4 *>(bs + (grp * 16 + k) * kPitch + tx * 4);
      const float x[4] = {av.x, av.y, av.z, av.w}, y[4] = {bv.x, bv.y, bv.z, bv.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
    }
  }
  if (sums) {   // eight threads to a row, in order
    __syncthreads();
    smem[t] = row;
    __syncthreads();
    if (t < m) {
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) s += smem[q * 32 + t];
      ((T *)g.row_sum)[i0 + t] = ElemOf<T>::from(s);
    }
  }
  if (!g.out) return;
  // [group][32][32]; the four groups are added in order, a warp to a row, its lanes along the columns
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<float4 *>(smem + grp * kTile * kTile + (ty * 4 + i) * 32 + tx * 4) =
        make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
  __syncthreads();
  const int c = t & 31, j = j0 + c;
  const bool col = c < n;
  const float bias = g.bias && col ? ElemOf<T>::to(((const T *)g.bias)[j]) : 0.f;
  float sum = 0.f;
#pragma unroll
  for (int r = t >> 5; r < kTile; r += 8) {
    const long long i = i0 + r;
    const bool in = r < m && col;
    const float *s = smem + r * 32 + c;
    float v = s[0];
#pragma unroll
    for (int q = 1; q < 4; ++q) v += s[q * kTile * kTile];
    v += bias;
    if (g.act == DCN_ACT_RELU) {
      if (g.saved) {
        const uint32_t bits = __ballot_sync(0xffffffffu, in && relu_bit(v));
        if (c == 0 && r < m) ((uint32_t *)g.saved)[i * ((g.n + 31) / 32) + tn] = bits;
      }
      v = relu_value(v);
    } else if (g.act == DCN_ACT_GELU) {
      if (g.saved && in) keep_slope<T>(g.saved, i * ((g.n + 7) / 8 * 8) + j, gelu_slope<sizeof(T) == 4>(v));
      v = gelu_value<sizeof(T) == 4>(v);
    }
    if (!in) continue;
    if (g.slope_act != DCN_ACT_NONE) v = through<T>(v, g.slope, g.slope_act, i, j, g.n);
    if (g.res) v += ElemOf<T>::to(((const T *)g.res)[i * g.ldr + j]);
    sum += v;
    ((T *)g.out)[i * g.n + j] = ElemOf<T>::from(v);
  }
  if (g.col_part) {
    __syncthreads();
    smem[t] = sum;
    __syncthreads();
    if (t < n) {
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) s += smem[q * 32 + t];
      g.col_part[tm * g.n + j0 + t] = s;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) dcn_gemm_simt(const __grid_constant__ SimtJobs jobs) {
  __shared__ __align__(16) float smem[2 * kStep * kPitch];
  static_assert(2 * kStep * kPitch >= 4 * kTile * kTile, "the groups' results");
  pdl_wait();
  pdl_launch();
  const int first = jobs.job[0].tiles;
  if ((int)blockIdx.x < first) tile_product<T>(jobs.job[0], blockIdx.x, smem);
  else tile_product<T>(jobs.job[1], blockIdx.x - first, smem);
}

template <typename T>
cudaError_t run(const SimtJobs &jobs, cudaStream_t s) {
  return launch_pdl(dcn_gemm_simt<T>, (unsigned)(jobs.job[0].tiles + jobs.job[1].tiles), 256, 0, s, 1, jobs);
}

}  // namespace

SimtJob simt_job(const GemmArgs &g, const void *a_saved, int a_act) {
  SimtJob p = {};
  p.g = g;
  p.a_saved = a_saved;
  p.a_act = a_act;
  p.tiles_n = g.out ? (int)((g.n + kTile - 1) / kTile) : 1;
  p.tiles = (int)((g.m + kTile - 1) / kTile) * p.tiles_n;
  return p;
}

cudaError_t launch_gemm_simt(const SimtJobs &jobs, int dtype, cudaStream_t s) {
  if (dtype == DCN_DTYPE_F32) return run<float>(jobs, s);
  if (dtype == DCN_DTYPE_BF16) return run<__nv_bfloat16>(jobs, s);
  return run<__half>(jobs, s);
}

}  // namespace dcn
