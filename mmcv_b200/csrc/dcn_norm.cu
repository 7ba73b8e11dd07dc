// Layer norm over the last dimension, forward and backward.
//
//   forward   m = mean(x), d = x - m, c = mean(d), var = mean(d^2) - c^2, rstd = 1 / sqrt(var + eps)
//             n = (d - c) rstd,  y = n w + b
//   backward  g = gy w,  gx = rstd (g - mean(g) - n mean(g n)),  gw = sum_rows gy n,  gb = sum_rows gy
//
// m is rounded to fp32; c is what that rounding (and the rounding of the sum) left out.  With it a
// row whose mean is large against its spread keeps its digits: the variance is taken around m + c,
// never as a difference of large squares.  The statistics kept for the backward pass are m, c, rstd.
//
// Both passes read each tensor once: a row (up to 8192 columns) lives in the registers of a group of G
// threads, 4 to 256, E elements to a thread, loaded 16 bytes at a time (one element at a time where sizes or
// alignment forbid it).  Bound: memory for fp32 (35642 x 256 forward 11.7 us, its bytes 11.1 at the copy rate),
// instructions and the latency of short rows for 16 bits (bf16 8.6 us, bytes 5.6; 64 % of the issue slots).
// The backward pass keeps gw and gb in registers over all rows that a group takes, adds the groups of
// a block in order, writes one partial row per block, and a second kernel adds those in order: the
// result does not depend on when blocks run (35642 x 256 bf16: 17.6 us with both kernels, 11.8 for gx alone,
// bytes 8.3).
#include <cstdint>
#include <type_traits>

#include "dcn_layers.cuh"

namespace dcn {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPartials = 148 * 4;

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T *p, float (&o)[V]) {
  if constexpr (V == 1) {
    o[0] = ElemOf<T>::to(*p);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 v = *reinterpret_cast<const float4 *>(p + i);
      o[i] = v.x; o[i + 1] = v.y; o[i + 2] = v.z; o[i + 3] = v.w;
    }
  } else {
    static_assert(V == 8, "sixteen bytes");
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        o[2 * i] = __uint_as_float(w[i] << 16);
        o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        o[2 * i] = f.x;
        o[2 * i + 1] = f.y;
      }
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T *p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = ElemOf<T>::from(v[0]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4)
      *reinterpret_cast<float4 *>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      T lo = ElemOf<T>::from(v[2 * i]), hi = ElemOf<T>::from(v[2 * i + 1]);
      w[i] = (uint32_t)*reinterpret_cast<uint16_t *>(&lo) | ((uint32_t)*reinterpret_cast<uint16_t *>(&hi) << 16);
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// V weights (or biases) from either type; `none` where there is no tensor.
template <typename T, int V>
__device__ __forceinline__ void load_param(const void *p, bool f32, long long at, float none, float (&o)[V]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = none;
  } else if (f32) {
    load_vec<float, V>((const float *)p + at, o);
  } else {
    load_vec<T, V>((const T *)p + at, o);
  }
}

// Sums of N values over the G threads of a group; every thread gets them.  A group of several warps meets on
// a barrier of its own.
template <int G>
__device__ __forceinline__ void group_barrier() {
  if constexpr (G >= kThreads) __syncthreads();
  else asm volatile("bar.sync %0, %1;" ::"r"(1 + (int)threadIdx.x / G), "n"(G) : "memory");
}
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float *smem) {
  static_assert(N <= 2, "a warp's place in smem");
#pragma unroll
  for (int d = (G < 32 ? G : 32) / 2; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], d);
  if constexpr (G > 32) {
    const int warp = threadIdx.x >> 5, first = (int)threadIdx.x / G * (G / 32);
    group_barrier<G>();   // the values of an earlier call have been read
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) smem[warp * 2 + i] = v[i];   // a warp's place is the same for every N: groups do not wait for one another
    group_barrier<G>();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.f;
#pragma unroll
      for (int w = 0; w < G / 32; ++w) v[i] += smem[(first + w) * 2 + i];
    }
  }
}

// V elements at a time, two to an instruction: bf16 rows are bound by instructions before memory (35642 x 256
// forward 9.5 us one by one).  Sums go to two places, even and odd.
template <int V>
__device__ __forceinline__ void sum_to(float (&s)[2], const float (&x)[V]) {
  if constexpr (V == 1) s[0] += x[0];
  else
#pragma unroll
    for (int e = 0; e < V; e += 2) add2(s[0], s[1], x[e], x[e + 1]);
}
template <int V>
__device__ __forceinline__ void dot_to(float (&s)[2], const float (&x)[V], const float (&y)[V]) {
  if constexpr (V == 1) s[0] = fmaf(x[0], y[0], s[0]);
  else
#pragma unroll
    for (int e = 0; e < V; e += 2) fma2_to(s[0], s[1], x[e], x[e + 1], y[e], y[e + 1]);
}
template <int V>   // x + c
__device__ __forceinline__ void shift(float (&x)[V], float c) {
  if constexpr (V == 1) x[0] += c;
  else
#pragma unroll
    for (int e = 0; e < V; e += 2) add2(x[e], x[e + 1], c, c);
}
template <int V>   // x * f + c
__device__ __forceinline__ void affine(float (&x)[V], float f, float c) {
  if constexpr (V == 1) x[0] = fmaf(x[0], f, c);
  else
#pragma unroll
    for (int e = 0; e < V; e += 2) fma2(x[e], x[e + 1], f, f, c);
}
template <int V>   // a + x
__device__ __forceinline__ void accumulate(float (&a)[V], const float (&x)[V]) {
  if constexpr (V == 1) a[0] += x[0];
  else
#pragma unroll
    for (int e = 0; e < V; e += 2) add2(a[e], a[e + 1], x[e], x[e + 1]);
}
template <int V>   // x * y
__device__ __forceinline__ void multiply(float (&x)[V], const float (&y)[V]) {
  if constexpr (V == 1) x[0] *= y[0];
  else
#pragma unroll
    for (int e = 0; e < V; e += 2) fma2(x[e], x[e + 1], y[e], y[e + 1], -0.f);
}
template <int V>   // a + x * y
__device__ __forceinline__ void multiply_add(float (&a)[V], const float (&x)[V], const float (&y)[V]) {
  if constexpr (V == 1) a[0] = fmaf(x[0], y[0], a[0]);
  else
#pragma unroll
    for (int e = 0; e < V; e += 2) fma2_to(a[e], a[e + 1], x[e], x[e + 1], y[e], y[e + 1]);
}

struct NormArgs {
  const void *x, *gy, *w, *b;
  void *y;
  float *stats;        // [3][rows]: m, c, rstd
  float *part;         // [gridDim.x][2][cols]: a block's sums for gw and gb
  long long ldx, ldgy, rows;
  int cols;
  bool wf32;
  float eps;
};

// A thread's part of a row as it lies in memory.
template <typename T, int V, int NV>
struct Loads {
  uint4 q[V == 1 ? 1 : NV];
  T e[V == 1 ? NV : 1];
  template <int G>
  __device__ __forceinline__ void get(const T *p, int t, int cols) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + t) * V;
      if (c < cols) {
        if constexpr (V == 1) e[i] = p[c];
        else q[i] = *reinterpret_cast<const uint4 *>(p + c);
      }
    }
  }
  __device__ __forceinline__ void unpack(int i, float (&o)[V]) const {
    if constexpr (V == 1) o[0] = ElemOf<T>::to(e[i]);
    else load_vec<T, V>(reinterpret_cast<const T *>(&q[i]), o);
  }
};

template <typename T, int V, int E, int G>
__global__ void __launch_bounds__(kThreads) norm_forward(const NormArgs a) {
  constexpr int NV = E / V;
  __shared__ float red[kThreads / 32 * 2];
  const int t = threadIdx.x % G;
  long long row = blockIdx.x * (long long)(kThreads / G) + threadIdx.x / G;
  pdl_wait();
  pdl_launch();
  const bool live = row < a.rows;   // a warp may hold several rows: all lanes go through the sums
  if (!live) row = a.rows - 1;
  const T *x = (const T *)a.x + row * a.ldx;
  float v[NV][V];
  float s2[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + t) * V;
    if (c < a.cols) {
      load_vec<T, V>(x + c, v[i]);
      sum_to(s2, v[i]);
    }
  }
  float s[1] = {s2[0] + s2[1]};
  group_sum<G>(s, red);
  const float inv = 1.f / (float)a.cols, m = s[0] * inv;
  float d1[2] = {0.f, 0.f}, d2[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + t) * V;
    if (c < a.cols) {
      shift(v[i], -m);
      sum_to(d1, v[i]);
      dot_to(d2, v[i], v[i]);
    }
  }
  float q[2] = {d1[0] + d1[1], d2[0] + d2[1]};
  group_sum<G>(q, red);
  const float corr = q[0] * inv;
  const float rstd = 1.f / sqrtf(fmaxf(q[1] * inv - corr * corr, 0.f) + a.eps);
  // fmaxf drops a NaN; m carries it into every element of the row all the same
  if (!live) return;
  T *y = (T *)a.y + row * a.cols;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + t) * V;
    if (c < a.cols) {
      float w[V], b[V];
      load_param<T, V>(a.w, a.wf32, c, 1.f, w);
      load_param<T, V>(a.b, a.wf32, c, 0.f, b);
      affine(v[i], rstd, -corr * rstd);
      multiply_add(b, v[i], w);
      store_vec<T, V>(y + c, b);
    }
  }
  if (a.stats && t == 0) {
    a.stats[row] = m;
    a.stats[a.rows + row] = corr;
    a.stats[2 * a.rows + row] = rstd;
  }
}

// Blocks that share an SM: a thread holds 4 E sums and values and the loads of its next row.
template <int V, int E>
constexpr int kResident = E <= 8 ? 3 : V > 1 && E <= 16 ? 2 : 1;

template <typename T, int V, int E, int G, bool kParams>
__global__ void __launch_bounds__(kThreads, kResident<V, E>) norm_backward(const NormArgs a) {
  constexpr int NV = E / V, RPB = kThreads / G;
  constexpr bool kAhead = V > 1 && E <= 16;   // the next row's loads run under this row's sums
  __shared__ float red[kThreads / 32 * 2];
  __shared__ float cols_s[kParams && RPB > 1 ? RPB * 2 * G * E : 1];
  const int t = threadIdx.x % G;
  const float inv = 1.f / (float)a.cols;
  float gw[kParams ? NV : 1][V] = {}, gb[kParams ? NV : 1][V] = {};
  pdl_wait();
  pdl_launch();
  const T *xs = (const T *)a.x, *gys = (const T *)a.gy;
  const long long step = (long long)gridDim.x * RPB;
  Loads<T, V, NV> nx, ng;
  auto get = [&](long long r) {
    nx.template get<G>(xs + r * a.ldx, t, a.cols);
    ng.template get<G>(gys + r * a.ldgy, t, a.cols);
  };
  long long row = blockIdx.x * (long long)RPB + threadIdx.x / G;
  if (kAhead && row < a.rows) get(row);
  for (; row < a.rows; row += step) {
    if (!kAhead) get(row);
    const float m = a.stats[row], corr = a.stats[a.rows + row], rstd = a.stats[2 * a.rows + row];
    float n[NV][V], g[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * G + t) * V < a.cols) {
        nx.unpack(i, n[i]);
        ng.unpack(i, g[i]);
      }
    if (kAhead && row + step < a.rows) get(row + step);
    float sg[2] = {0.f, 0.f}, sn[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + t) * V;
      if (c < a.cols) {
        float w[V];
        load_param<T, V>(a.w, a.wf32, c, 1.f, w);
        shift(n[i], -m);
        affine(n[i], rstd, -corr * rstd);
        if constexpr (kParams) {
          multiply_add(gw[i], g[i], n[i]);
          accumulate(gb[i], g[i]);
        }
        multiply(g[i], w);
        sum_to(sg, g[i]);
        dot_to(sn, g[i], n[i]);
      }
    }
    float s[2] = {sg[0] + sg[1], sn[0] + sn[1]};
    if (a.y) {
      group_sum<G>(s, red);
      const float mg = s[0] * inv, mgn = s[1] * inv;
      T *gx = (T *)a.y + row * a.cols;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * G + t) * V;
        if (c < a.cols) {
          // ((g - mg) - n mgn) rstd
          affine(n[i], -mgn, -mg);
          accumulate(g[i], n[i]);
          affine(g[i], rstd, 0.f);
          store_vec<T, V>(gx + c, g[i]);
        }
      }
    }
  }
  static_assert(G >= 32, "whole warps leave the loop together");
  if constexpr (kParams) {
    float *out = a.part + (long long)blockIdx.x * 2 * a.cols;
    if constexpr (RPB == 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * G + t) * V;
        if (c < a.cols)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            out[c + e] = gw[i][e];
            out[a.cols + c + e] = gb[i][e];
          }
      }
    } else {
      float *mine = cols_s + threadIdx.x / G * (2 * G * E);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          mine[(i * G + t) * V + e] = gw[i][e];
          mine[G * E + (i * G + t) * V + e] = gb[i][e];
        }
      __syncthreads();
      for (int c = threadIdx.x; c < a.cols; c += kThreads) {
        float sw = 0.f, sb = 0.f;
#pragma unroll
        for (int q = 0; q < RPB; ++q) {   // the groups in order
          sw += cols_s[q * 2 * G * E + c];
          sb += cols_s[q * 2 * G * E + G * E + c];
        }
        out[c] = sw;
        out[a.cols + c] = sb;
      }
    }
  }
}

// Rows beyond 8192 columns: a block of 1024 threads reads its row three times (twice from cache).
template <typename T>
__global__ void __launch_bounds__(1024) norm_forward_wide(const NormArgs a) {
  __shared__ float red[32 * 2];
  const long long row = blockIdx.x;
  pdl_wait();
  pdl_launch();
  const T *x = (const T *)a.x + row * a.ldx;
  float s[1] = {0.f};
  for (int c = threadIdx.x; c < a.cols; c += 1024) s[0] += ElemOf<T>::to(x[c]);
  group_sum<1024>(s, red);
  const float inv = 1.f / (float)a.cols, m = s[0] * inv;
  float q[2] = {0.f, 0.f};
  for (int c = threadIdx.x; c < a.cols; c += 1024) {
    const float d = ElemOf<T>::to(x[c]) - m;
    q[0] += d;
    q[1] = fmaf(d, d, q[1]);
  }
  group_sum<1024>(q, red);
  const float corr = q[0] * inv;
  const float rstd = 1.f / sqrtf(fmaxf(q[1] * inv - corr * corr, 0.f) + a.eps);
  T *y = (T *)a.y + row * a.cols;
  for (int c = threadIdx.x; c < a.cols; c += 1024) {
    float w[1], b[1];
    load_param<T, 1>(a.w, a.wf32, c, 1.f, w);
    load_param<T, 1>(a.b, a.wf32, c, 0.f, b);
    y[c] = ElemOf<T>::from(fmaf((ElemOf<T>::to(x[c]) - m - corr) * rstd, w[0], b[0]));
  }
  if (a.stats && threadIdx.x == 0) {
    a.stats[row] = m;
    a.stats[a.rows + row] = corr;
    a.stats[2 * a.rows + row] = rstd;
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) norm_backward_wide(const NormArgs a) {
  __shared__ float red[32 * 2];
  const long long row = blockIdx.x;
  pdl_wait();
  pdl_launch();
  const T *x = (const T *)a.x + row * a.ldx, *gy = (const T *)a.gy + row * a.ldgy;
  const float m = a.stats[row], corr = a.stats[a.rows + row], rstd = a.stats[2 * a.rows + row];
  float s[2] = {0.f, 0.f};
  for (int c = threadIdx.x; c < a.cols; c += 1024) {
    float w[1];
    load_param<T, 1>(a.w, a.wf32, c, 1.f, w);
    const float g = ElemOf<T>::to(gy[c]) * w[0];
    s[0] += g;
    s[1] = fmaf(g, (ElemOf<T>::to(x[c]) - m - corr) * rstd, s[1]);
  }
  group_sum<1024>(s, red);
  const float inv = 1.f / (float)a.cols, mg = s[0] * inv, mgn = s[1] * inv;
  T *gx = (T *)a.y + row * a.cols;
  for (int c = threadIdx.x; c < a.cols; c += 1024) {
    float w[1];
    load_param<T, 1>(a.w, a.wf32, c, 1.f, w);
    const float n = (ElemOf<T>::to(x[c]) - m - corr) * rstd;
    gx[c] = ElemOf<T>::from((ElemOf<T>::to(gy[c]) * w[0] - mg - n * mgn) * rstd);
  }
}

// ... and their gw and gb: a thread owns a column, blockIdx.y a slab of rows
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_columns_wide(const NormArgs a) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  pdl_wait();
  pdl_launch();
  if (c >= a.cols) return;
  float gw = 0.f, gb = 0.f;
  for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float g = ElemOf<T>::to(((const T *)a.gy)[row * a.ldgy + c]);
    const float n = (ElemOf<T>::to(((const T *)a.x)[row * a.ldx + c]) - a.stats[row] - a.stats[a.rows + row]) *
                    a.stats[2 * a.rows + row];
    gw = fmaf(g, n, gw);
    gb += g;
  }
  a.part[(long long)blockIdx.y * 2 * a.cols + c] = gw;
  a.part[((long long)blockIdx.y * 2 + 1) * a.cols + c] = gb;
}

// out[c] = sum over the partial rows; blockIdx.y: 0 gw, 1 gb
template <typename T, int C>
__global__ void __launch_bounds__(1024) norm_reduce(const float *__restrict__ part, int parts, int cols, T *gw, T *gb) {
  const int c = blockIdx.x * C + threadIdx.x % C;
  T *out = blockIdx.y ? gb : gw;
  pdl_wait();
  pdl_launch();
  if (!out) return;
  const float v = column_join<1024, C>(part + blockIdx.y * (long long)cols + c, parts, 2LL * cols, c < cols);
  if (threadIdx.x < C && c < cols) out[c] = ElemOf<T>::from(v);
}

template <typename T>
cudaError_t run_reduce(const NormArgs &a, int parts, void *gw, void *gb, cudaStream_t s) {
  const int c = join_columns(a.cols);
  const dim3 grid((unsigned)((a.cols + c - 1) / c), 2);
  if (c == 8) return launch_pdl(norm_reduce<T, 8>, grid, 1024, 0, s, 1, a.part, parts, a.cols, (T *)gw, (T *)gb);
  return launch_pdl(norm_reduce<T, 32>, grid, 1024, 0, s, 1, a.part, parts, a.cols, (T *)gw, (T *)gb);
}

template <typename T, int V, int E, int G>
cudaError_t run_forward(const NormArgs &a, cudaStream_t s) {
  constexpr int rpb = kThreads / G;
  return launch_pdl(norm_forward<T, V, E, G>, (unsigned)((a.rows + rpb - 1) / rpb), kThreads, 0, s, 1, a);
}
template <typename T, int V, int E, int G>
cudaError_t run_backward(const NormArgs &a, bool params, int *parts, cudaStream_t s) {
  constexpr int rpb = kThreads / G, most = 148 * kResident<V, E>;
  static_assert(most <= kMaxPartials, "the workspace");
  const long long blocks = (a.rows + rpb - 1) / rpb;
  *parts = (int)(blocks < most ? blocks : most);
  if (params) return launch_pdl(norm_backward<T, V, E, G, true>, *parts, kThreads, 0, s, 1, a);
  return launch_pdl(norm_backward<T, V, E, G, false>, *parts, kThreads, 0, s, 1, a);
}

// Elements to a thread and threads to a row.
//
// Forward: two loads of 16 bytes while that keeps a row within a warp (35642 x 64 bf16: 3.9 us against 11.3 us
// with a warp to each row; 35642 x 256 bf16, before the arithmetic went two elements at a time: 9.5 us, with one
// load 11.5, with four 10.6), 32 elements beyond
// (20000 x 768 bf16 16.8 us, with two loads 20.3; 5000 x 1536 10.0 us, with one load 13.8).  Keeping the
// parameters in registers over several rows, with the next row's loads ahead, was slower everywhere
// (35642 x 256 fp32 25 us against 11.6).  One element at a time: a warp's lanes side by side, for the sake of
// whole sectors.
//
// Backward: 8 elements and a fixed set of blocks, so that the sums for gw and gb leave room for several rows
// at once on an SM (20000 x 768 bf16 41 us, with 32 elements 78); the same without those sums, so that gx
// does not depend on what else is wanted.
template <typename T, int V>
cudaError_t run_rows(const NormArgs &a, bool backward, bool params, int *parts, cudaStream_t s) {
  const int cols = a.cols;
  if (backward) {
    if (cols <= 256) return run_backward<T, V, 8, 32>(a, params, parts, s);
    if (cols <= 512) return run_backward<T, V, 8, 64>(a, params, parts, s);
    if (cols <= 1024) return run_backward<T, V, 8, 128>(a, params, parts, s);
    if (cols <= 2048) return run_backward<T, V, 8, 256>(a, params, parts, s);
    if (cols <= 4096) return run_backward<T, V, 16, 256>(a, params, parts, s);
    return run_backward<T, V, 32, 256>(a, params, parts, s);
  }
  if constexpr (V > 1) {
    constexpr int E = 2 * V;
    if (cols <= 4 * E) return run_forward<T, V, E, 4>(a, s);
    if (cols <= 8 * E) return run_forward<T, V, E, 8>(a, s);
    if (cols <= 16 * E) return run_forward<T, V, E, 16>(a, s);
    if (cols <= 32 * E) return run_forward<T, V, E, 32>(a, s);
    if (cols <= 1024) return run_forward<T, V, 32, 32>(a, s);
    if (cols <= 2048) return run_forward<T, V, 32, 64>(a, s);
    if (cols <= 4096) return run_forward<T, V, 32, 128>(a, s);
  } else {
    if (cols <= 256) return run_forward<T, V, 8, 32>(a, s);
    if (cols <= 512) return run_forward<T, V, 16, 32>(a, s);
    if (cols <= 1024) return run_forward<T, V, 32, 32>(a, s);
    if (cols <= 2048) return run_forward<T, V, 8, 256>(a, s);
    if (cols <= 4096) return run_forward<T, V, 16, 256>(a, s);
  }
  return run_forward<T, V, 32, 256>(a, s);
}

template <typename T>
cudaError_t run(const NormArgs &a, bool backward, bool params, int *parts, cudaStream_t s) {
  if (a.cols > 8192) {
    if (!backward) return launch_pdl(norm_forward_wide<T>, (unsigned)a.rows, 1024, 0, s, 1, a);
    cudaError_t e = cudaSuccess;
    if (a.y) e = launch_pdl(norm_backward_wide<T>, (unsigned)a.rows, 1024, 0, s, 1, a);
    if (e == cudaSuccess && params) {
      *parts = (int)(a.rows < 64 ? a.rows : 64);
      e = launch_pdl(norm_columns_wide<T>, dim3((a.cols + kThreads - 1) / kThreads, *parts), kThreads, 0, s, 1, a);
    }
    return e;
  }
  // 16-byte accesses need every row of every tensor to start on 16 bytes; the dense output's does
  // when cols is a multiple of V
  constexpr int V = 16 / (int)sizeof(T);
  const bool vec = a.cols % V == 0 && a.ldx % V == 0 && (!backward || a.ldgy % V == 0) && aligned16(a.x) &&
                   aligned16(a.y) && aligned16(a.w) && aligned16(a.b) && (!backward || aligned16(a.gy));
  return vec ? run_rows<T, V>(a, backward, params, parts, s) : run_rows<T, 1>(a, backward, params, parts, s);
}

cudaError_t run_typed(const NormArgs &a, int dtype, bool backward, bool params, int *parts, cudaStream_t s) {
  if (dtype == DCN_DTYPE_F32) return run<float>(a, backward, params, parts, s);
  if (dtype == DCN_DTYPE_BF16) return run<__nv_bfloat16>(a, backward, params, parts, s);
  return run<__half>(a, backward, params, parts, s);
}

int check(int32_t dtype, int32_t wdtype, int64_t rows, int64_t cols) {
  if (dtype != DCN_DTYPE_F32 && dtype != DCN_DTYPE_BF16 && dtype != DCN_DTYPE_F16)
    return set_error(DCN_ERR_UNSUPPORTED, "layer norm: fp32, bf16 and fp16 tensors only");
  if (wdtype != dtype && wdtype != DCN_DTYPE_F32)
    return set_error(DCN_ERR_ARG, "layer norm: weight and bias must have x's type or fp32");
  if (rows < 0 || cols <= 0) return set_error(DCN_ERR_ARG, "layer norm: cols must be positive, rows must not be negative");
  if (rows > 2147483647LL || cols > (1 << 24))
    return set_error(DCN_ERR_UNSUPPORTED, "layer norm: at most 2^31 - 1 rows and 2^24 columns");
  return DCN_OK;
}

size_t workspace_of(int64_t rows, int64_t cols) {
  return (size_t)(rows < kMaxPartials ? rows : kMaxPartials) * 2 * (size_t)cols * sizeof(float);
}

}  // namespace
}  // namespace dcn

using namespace dcn;

extern "C" {

int dcn_layer_norm_forward(const void *x, int64_t ldx, const void *weight, const void *bias, void *y,
                           float *stats, int32_t dtype, int32_t wdtype, int64_t rows, int64_t cols, float eps,
                           int32_t device, void *stream) {
  int rc = check(dtype, wdtype, rows, cols);
  if (rc) return rc;
  if (rows == 0) return DCN_OK;
  if (!x || !y) return set_error(DCN_ERR_ARG, "layer norm: x and y must be non-NULL");
  if (ldx < cols) return set_error(DCN_ERR_ARG, "layer norm: the row stride is smaller than the row");
  LayerDeviceScope scope(device);
  if (scope.err != cudaSuccess) return set_error(DCN_ERR_CUDA, cudaGetErrorString(scope.err));
  NormArgs a = {};
  a.x = x; a.w = weight; a.b = bias; a.y = y; a.stats = stats;
  a.ldx = ldx; a.rows = rows; a.cols = (int)cols; a.wf32 = wdtype == DCN_DTYPE_F32; a.eps = eps;
  int parts = 0;
  const cudaError_t e = run_typed(a, dtype, false, false, &parts, (cudaStream_t)stream);
  return e == cudaSuccess ? DCN_OK : set_error(DCN_ERR_CUDA, cudaGetErrorString(e));
}

int dcn_layer_norm_workspace_bytes(int64_t rows, int64_t cols, size_t *bytes) {
  if (!bytes) return set_error(DCN_ERR_ARG, "layer norm: bytes is NULL");
  int rc = check(DCN_DTYPE_F32, DCN_DTYPE_F32, rows, cols);
  if (rc) return rc;
  *bytes = workspace_of(rows, cols);
  return DCN_OK;
}

int dcn_layer_norm_backward(const void *gy, int64_t ldgy, const void *x, int64_t ldx, const void *weight,
                            const float *stats, void *gx, void *gw, void *gb, int32_t dtype, int32_t wdtype,
                            int64_t rows, int64_t cols, int32_t device, void *workspace,
                            size_t workspace_bytes, void *stream) {
  int rc = check(dtype, wdtype, rows, cols);
  if (rc) return rc;
  LayerDeviceScope scope(device);
  if (scope.err != cudaSuccess) return set_error(DCN_ERR_CUDA, cudaGetErrorString(scope.err));
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e = cudaSuccess;
  if (rows == 0) {
    const size_t n = (size_t)cols * (wdtype == DCN_DTYPE_F32 ? 4 : 2);
    if (gw) e = cudaMemsetAsync(gw, 0, n, s);
    if (e == cudaSuccess && gb) e = cudaMemsetAsync(gb, 0, n, s);
    return e == cudaSuccess ? DCN_OK : set_error(DCN_ERR_CUDA, cudaGetErrorString(e));
  }
  if (!gx && !gw && !gb) return DCN_OK;
  if (!gy || !x || !stats) return set_error(DCN_ERR_ARG, "layer norm backward: gy, x and stats must be non-NULL");
  if (ldx < cols || ldgy < cols)
    return set_error(DCN_ERR_ARG, "layer norm backward: a row stride is smaller than the row");
  const bool params = gw || gb;
  if (params && (!workspace || workspace_bytes < workspace_of(rows, cols) || ((uintptr_t)workspace & 255)))
    return set_error(DCN_ERR_WORKSPACE, "layer norm backward: workspace missing, too small or misaligned");
  NormArgs a = {};
  a.x = x; a.gy = gy; a.w = weight; a.y = gx; a.stats = const_cast<float *>(stats); a.part = (float *)workspace;
  a.ldx = ldx; a.ldgy = ldgy; a.rows = rows; a.cols = (int)cols; a.wf32 = wdtype == DCN_DTYPE_F32;
  int parts = 0;
  e = run_typed(a, dtype, true, params, &parts, s);
  if (e == cudaSuccess && params) {
    if (wdtype == DCN_DTYPE_F32) e = run_reduce<float>(a, parts, gw, gb, s);
    else if (wdtype == DCN_DTYPE_BF16) e = run_reduce<__nv_bfloat16>(a, parts, gw, gb, s);
    else e = run_reduce<__half>(a, parts, gw, gb, s);
  }
  return e == cudaSuccess ? DCN_OK : set_error(DCN_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
