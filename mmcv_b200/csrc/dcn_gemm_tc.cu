// Around the tensor-core products (dcn_gemm_tc.cuh): how a product is cut up, its tensor maps, the
// element-wise pass that writes operand planes, and the ordered sums of split results.
#include <atomic>
#include <cstring>

#include <cuda.h>

#include "dcn_gemm.cuh"

namespace dcn {

namespace {

// out[i, j] = sum over the ranges of part [splits][m][ldp]: a thread has four columns and, in a block cut into
// `groups`, every groups-th range; the groups are joined in order.  Blocks from `blocks` on: a bias gradient's
// partial rows, eight columns each, which saves a launch.
template <typename T>
__global__ void __launch_bounds__(256) dcn_gemm_reduce(const float *__restrict__ part, int splits, long long m,
                                                       long long n, long long ldp, int groups, T *__restrict__ out,
                                                       unsigned blocks, const float *join_part, int join_parts,
                                                       T *join_out) {
  __shared__ float4 join[256];
  const int across = 256 / groups, group = threadIdx.x / across;
  const long long per_row = ldp / 4, idx = blockIdx.x * (long long)across + (threadIdx.x - group * across);
  const bool live = idx < m * per_row;
  pdl_wait();
  pdl_launch();
  if (blockIdx.x >= blocks) {
    const long long c = (blockIdx.x - blocks) * 8LL + (threadIdx.x & 7);
    const float v = column_join<256, 8>(join_part + c, join_parts, m, c < m);
    if (threadIdx.x < 8 && c < m) join_out[c] = ElemOf<T>::from(v);
    return;
  }
  const long long i = idx / per_row, j = (idx - i * per_row) * 4;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
    const float4 *p = reinterpret_cast<const float4 *>(part + i * ldp + j);
    const long long step = m * ldp / 4;
#pragma unroll 8
    for (int s = group; s < splits; s += groups) {
      const float4 a = p[s * step];
      v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
    }
  }
  join[threadIdx.x] = v;
  __syncthreads();
  if (group || !live) return;
  for (int k = 1; k < groups; ++k) {
    const float4 a = join[k * across + threadIdx.x];
    v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
  }
  T *o = out + i * n + j;
  if (j < n) o[0] = ElemOf<T>::from(v.x);
  if (j + 1 < n) o[1] = ElemOf<T>::from(v.y);
  if (j + 2 < n) o[2] = ElemOf<T>::from(v.z);
  if (j + 3 < n) o[3] = ElemOf<T>::from(v.w);
}

// out[c] = sum over the parts, in the order that dcn_gemm_reduce has: the same bits whichever does it
template <typename T>
__global__ void __launch_bounds__(256) dcn_column_reduce(const float *__restrict__ part, int parts, long long cols, T *out) {
  const long long c = blockIdx.x * 8LL + (threadIdx.x & 7);
  pdl_wait();
  pdl_launch();
  const float v = column_join<256, 8>(part + c, parts, cols, c < cols);
  if (threadIdx.x < 8 && c < cols) out[c] = ElemOf<T>::from(v);
}

// Two values as x = x1 + x2 + x3 of 8 bits each, exact, rounded to nearest one after another: |x2| <= 2^-8 |x|,
// |x3| <= 2^-17 |x|, of either sign.  Truncated planes are twice as large and all of x's sign, so that what the
// product leaves out would add up (7.8 times 2^-24 of |x||y| at worst).  w: a plane's pair, the second value on top.
// A finite x that would round to infinity is truncated; an infinity or NaN stays in x1, the others are 0.
// (A product within 2^-7 of fp32's largest value may come out infinite: both leading planes rounded up.)
__device__ __forceinline__ void split3(float x, float y, uint32_t (&w)[3]) {
  float rx = x, ry = y;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[k]) : "f"(ry), "f"(rx));
    uint32_t bx = w[k] << 16, by = w[k] & 0xffff0000u;
    if (k == 0) {
      const bool infx = (bx & 0x7fffffffu) == 0x7f800000u, infy = (by & 0x7fffffffu) == 0x7f800000u;
      if (infx) bx = __float_as_uint(x) & 0xffff0000u;
      if (infy) by = __float_as_uint(y) & 0xffff0000u;
      w[0] = (bx >> 16) | by;
      rx = (bx & 0x7f800000u) == 0x7f800000u ? 0.f : x - __uint_as_float(bx);
      ry = (by & 0x7f800000u) == 0x7f800000u ? 0.f : y - __uint_as_float(by);
    } else {
      rx -= __uint_as_float(bx);
      ry -= __uint_as_float(by);
    }
  }
}

constexpr int kStageResident = 3;   // blocks that share an SM: two rows a thread in flight take 80 registers

// The operands of a pass in one launch, a range of blocks each.  In a block, a power of two of threads of
// 8 columns each, the rest side by side on rows; a slab of blocks takes every gy-th group of rows.
template <typename T, int PL>
__global__ void __launch_bounds__(256, kStageResident) dcn_gemm_stage(const __grid_constant__ StageJobs jobs) {
  __shared__ float red[256 * 8];
  const int which = (int)blockIdx.x < jobs.job[1].first ? 0 : (int)blockIdx.x < jobs.job[2].first ? 1 : 2;
  const StageJob &a = jobs.job[which];
  const int block = (int)blockIdx.x - a.first, slab = block / a.gx, tx = threadIdx.x & ((1 << a.log_tx) - 1),
            ty = threadIdx.x >> a.log_tx, rows_at_once = 256 >> a.log_tx;
  const long long c = ((long long)((block - slab * a.gx) << a.log_tx) + tx) * 8;
  const long long words = (a.cols + 31) / 32;
  pdl_wait();
  pdl_launch();
  float sum[8] = {};
  constexpr int Q = (int)sizeof(T) / 2;   // 16-byte pieces of 8 elements, and of 8 kept derivatives
  struct Piece {
    uint4 v[Q], z[Q];
    uint32_t bits;
  };
  auto load = [&](long long r, Piece &p) {
    const T *src = (const T *)a.src + r * a.ld + c;
    if (a.vec_src && c + 8 <= a.cols) {
#pragma unroll
      for (int i = 0; i < Q; ++i) p.v[i] = reinterpret_cast<const uint4 *>(src)[i];
    } else {
      T *e = reinterpret_cast<T *>(p.v);
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = c + i < a.cols ? src[i] : ElemOf<T>::from(0.f);
    }
    if (a.act == DCN_ACT_RELU) {
      p.bits = c < a.cols ? ((const uint32_t *)a.saved)[r * words + (c >> 5)] >> (c & 31) : 0u;
    } else if (a.act == DCN_ACT_GELU) {
#pragma unroll
      for (int i = 0; i < Q; ++i) p.z[i] = reinterpret_cast<const uint4 *>((const uint8_t *)a.saved + (r * a.pitch + c) * sizeof(T))[i];
    }
  };
  auto finish = [&](long long r, const Piece &p) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = ElemOf<T>::to(reinterpret_cast<const T *>(p.v)[i]);
    if (a.act == DCN_ACT_RELU) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (p.bits >> i) & 1u ? v[i] : 0.f;
    } else if (a.act == DCN_ACT_GELU) {
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        float z[8 / Q];
        unpack_slopes<T>(p.z[i], z);
#pragma unroll
        for (int k = 0; k < 8 / Q; ++k) v[i * (8 / Q) + k] *= z[k];
      }
    }
    if constexpr (PL == 1) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        T lo = ElemOf<T>::from(v[2 * i]), hi = ElemOf<T>::from(v[2 * i + 1]);
        w[i] = (uint32_t)*reinterpret_cast<uint16_t *>(&lo) | ((uint32_t)*reinterpret_cast<uint16_t *>(&hi) << 16);
      }
      *reinterpret_cast<uint4 *>((T *)a.dst + r * a.pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      uint32_t w[3][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t pair[3];
        split3(v[2 * i], v[2 * i + 1], pair);
#pragma unroll
        for (int k = 0; k < 3; ++k) w[k][i] = pair[k];
      }
#pragma unroll
      for (int k = 0; k < 3; ++k)
        *reinterpret_cast<uint4 *>((uint16_t *)a.dst + (k * a.rows + r) * a.pitch + c) =
            make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += v[i];
  };
  if (c < a.pitch) {   // two rows in flight
    const long long step = (long long)a.gy * rows_at_once;
    for (long long r = (long long)slab * rows_at_once + ty; r < a.rows; r += 2 * step) {
      Piece p0, p1;
      load(r, p0);
      if (r + step < a.rows) load(r + step, p1);
      finish(r, p0);
      if (r + step < a.rows) finish(r + step, p1);
    }
  }
  if (!a.sums) return;
  // the block's rows in order, one row of threads after another
  for (int y = 0; y < rows_at_once; ++y) {
    if (ty == y)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float *s = red + tx * 8 + i;
        *s = y ? *s + sum[i] : sum[i];
      }
    __syncthreads();
  }
  if (ty == 0)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < a.cols) a.sums[(long long)slab * a.cols + c + i] = red[tx * 8 + i];
}

void stage_shape(long long rows, long long pitch, StageJob *j) {
  j->log_tx = 0;
  while (j->log_tx < 5 && (8LL << j->log_tx) < pitch) ++j->log_tx;
  const long long x = 1LL << j->log_tx, y = 256 / x;
  j->gx = (int)((pitch + x * 8 - 1) / (x * 8));
  const long long want = (rows + y - 1) / y;
  long long most = 148 * kStageResident / j->gx;
  if (most < 1) most = 1;
  j->gy = (int)(want < 1 ? 1 : want < most ? want : most);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static std::atomic<EncodeTiledFn> fn{nullptr};
  EncodeTiledFn f = fn.load(std::memory_order_acquire);
  if (f) return f;
  void *p = nullptr;
  cudaDriverEntryPointQueryResult qres;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qres) != cudaSuccess ||
      qres != cudaDriverEntryPointSuccess || !p) {
    cudaGetLastError();
    return nullptr;
  }
  f = (EncodeTiledFn)p;
  fn.store(f, std::memory_order_release);
  return f;
}

// [depth][rows][inner] with the given row stride (elements), boxes of box_inner (128 or 64 bytes, the
// swizzle's width) x box_rows x 1
bool encode3(CUtensorMap *map, CUtensorMapDataType type, int esize, const void *base, long long inner, long long rows,
             long long depth, long long ld, unsigned box_inner, unsigned box_rows) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)depth};
  const cuuint64_t strides[2] = {(cuuint64_t)(ld * esize), (cuuint64_t)(rows * ld * esize)};
  const cuuint32_t box[3] = {box_inner, box_rows, 1}, estr[3] = {1, 1, 1};
  return enc(map, type, 3, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             box_inner * (unsigned)esize == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
cudaError_t run_reduce(const float *part, const GemmPlan &plan, const GemmArgs &g, cudaStream_t s) {
  const long long n = g.m * (plan.ldp / 4);
  // as many groups as fill the SMs (74 parts of 256 x 256: 5 us, with one group 19)
  int groups = 1;
  while (groups < 8 && plan.splits >= 4 * groups && n * groups < 148LL * 4 * 256) groups *= 2;
  const int across = 256 / groups;
  const unsigned blocks = (unsigned)((n + across - 1) / across), more = g.join_out ? (unsigned)((g.m + 7) / 8) : 0u;
  return launch_pdl(dcn_gemm_reduce<T>, blocks + more, 256, 0, s, 1, part, plan.splits, g.m, g.n, plan.ldp, groups,
                    (T *)g.out, blocks, g.join_part, g.join_parts, (T *)g.join_out);
}

template <typename T>
cudaError_t run_columns(const float *part, int parts, long long cols, void *out, cudaStream_t s) {
  return launch_pdl(dcn_column_reduce<T>, (unsigned)((cols + 7) / 8), 256, 0, s, 1, part, parts, cols, (T *)out);
}

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace

GemmPlan plan_gemm(int planes, long long m, long long n, long long k, bool weight_gradient) {
  GemmPlan p = {};
  const int wide = planes == 1 ? 256 : 128;
  auto tiles = [&](int rows, int bn) { return (m + rows - 1) / rows * ((n + bn - 1) / bn); };
  p.kb_total = (int)((k + 63) / 64);
  p.splits = 1;
  p.cg = p.ks = 1;
  if (weight_gradient) {
    p.bn = n > wide / 2 ? wide : n > 64 ? 128 : 64;
    if (m > 128 && p.bn == wide) p.cg = 2;
    long long splits = 148 / p.cg / tiles(128 * p.cg, p.bn);
    if (splits > p.kb_total / 4) splits = p.kb_total / 4;
    if (splits < 1) splits = 1;
    p.kb_split = (int)((p.kb_total + splits - 1) / splits);
    p.splits = (p.kb_total + p.kb_split - 1) / p.kb_split;
  } else {
    // The shape of least time by what was measured, in clocks: a block takes operands in at 46 bytes a clock
    // (fp32: its six products are as slow), its epilogue works under the next tile's steps, and tiles come in
    // rounds of as many as there are blocks or pairs.  us, chosen / next best / 128 x 128 tiles:
    //   bf16 8192 x 4096 x 4096 173 / 214 / 352, 4096 x 2048 x 1024 18.4 / 19.5 / 27.0, 3000 x 2048 x 512 15.7 /
    //   16.6, 600 x 1024 x 256 8.7 / 9.0; fp32 3000 x 2048 x 512 50.0 / 54.1, 4096 x 1024 x 2048 83 / 94 / 120
    struct Shape {
      int bn, cg;
      long long step, epilogue;   // of 64 values of k; of a tile
    };
    const Shape shapes16[] = {{256, 2, 711, 7000}, {256, 1, 1050, 6000}, {128, 1, 711, 3000}, {64, 1, 520, 1600}};
    const Shape shapes32[] = {{128, 2, 1600, 4000}, {128, 1, 2140, 4000}, {64, 1, 1600, 2000}};
    const Shape *shapes = planes == 1 ? shapes16 : shapes32;
    long long best = 0;
    for (int i = 0; i < (planes == 1 ? 4 : 3); ++i) {
      const Shape &c = shapes[i];
      const long long rounds = (tiles(128 * c.cg, c.bn) * c.cg + 147) / 148, steps = p.kb_total * c.step;
      const long long time = rounds * (steps > c.epilogue ? steps : c.epilogue) + (steps > c.epilogue ? c.epilogue : steps);
      if (i == 0 || time < best) {
        best = time;
        p.bn = c.bn;
        p.cg = c.cg;
      }
    }
    // 16-bit tiles of few steps are bound by their stores and epilogues, which that does not tell apart: the
    // widest tile that fills the SMs, no pairs (35642 x 256 x 1024 27.6 us, in pairs 31.6, 128 wide 31.7;
    // 35642 x 256 x 256 10.1, 11.8, 11.2)
    if (planes == 1 && p.kb_total <= 6) {
      p.cg = 1;
      p.bn = n > 128 && tiles(128, 256) >= 148 ? 256 : n > 64 && tiles(128, 128) >= 148 ? 128 : 64;
    }
    if (p.bn == 64) {
      // Few tiles and a long sum: a block takes in 24 KB (fp32: 72 KB) a step at 46 bytes a cycle, so that
      // sharing the steps pays for the cluster's 2 us from some length on.  One block / two / four, us:
      // bf16 600 x 1024 x 256 8.4 / 8.7 / 9.2, 600 x 2048 x 64 12.9 / 10.8 / 9.4, 32 x 4096 x 4096 22.3 / 16.7;
      // fp32 (two at most: each has 32 KB of sums to send) 600 x 256 x 256 10.0 / 10.7, 600 x 512 x 256
      // 13.4 / 12.6, 600 x 1024 x 256 21.3 / 16.8, 32 x 4096 x 4096 97 / 68.
      const int most = planes == 1 ? 4 : 2;
      if (p.kb_total >= (planes == 1 ? 20 : 8))
        while (p.ks < most && tiles(128, 64) * p.ks * 2 <= 148) p.ks *= 2;
    }
    p.kb_split = (p.kb_total + p.ks - 1) / p.ks;
    while ((p.ks - 1) * p.kb_split >= p.kb_total) --p.ks;   // a range each
  }
  p.ldp = (n + 3) / 4 * 4;
  if (p.splits > 1) {
    p.part_bytes = up256((size_t)p.splits * m * p.ldp * 4);
    p.row_part_bytes = up256((size_t)p.splits * m * 4);
  }
  return p;
}

cudaError_t launch_gemm_tc(const GemmArgs &g, const GemmPlan &plan, int dtype, float *part, float *row_part,
                           cudaStream_t s) {
  GemmTc p;
  memset(&p, 0, sizeof(p));
  p.g = g;
  p.m = (int)g.m;
  p.n = (int)g.n;
  const int planes = dtype == DCN_DTYPE_F32 ? 3 : 1, esize = dtype == DCN_DTYPE_F32 ? 4 : 2;
  const bool parts = plan.splits > 1;
  const CUtensorMapDataType t16 = dtype == DCN_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapDataType tio = dtype == DCN_DTYPE_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : t16;
  p.tiles_m = (int)((g.m + 128 * plan.cg - 1) / (128 * plan.cg));
  p.tiles_n = (int)((g.n + plan.bn - 1) / plan.bn);
  p.splits = plan.splits;
  p.ks = plan.ks;
  p.kb_total = plan.kb_total;
  p.kb_split = plan.kb_split;
  p.row_part = row_part;
  p.wait_limit_ns = 2000000000ull;   // two seconds a wait
  p.bias16 = aligned16(g.bias);
  bool ok = g.a_mn ? encode3(&p.a, t16, 2, g.a, g.m, g.kk, planes, g.lda, 64, 64)
                   : encode3(&p.a, t16, 2, g.a, g.kk, g.m, planes, g.lda, 64, 128);
  ok = ok && (g.b_mn ? encode3(&p.b, t16, 2, g.b, g.n, g.kk, planes, g.ldb, 64, 64)
                     : encode3(&p.b, t16, 2, g.b, g.kk, g.n, planes, g.ldb, 64, plan.bn / plan.cg));
  const bool rows16 = g.n * esize % 16 == 0;
  const unsigned cw = esize == 4 || plan.bn < 256 || plan.cg == 2 ? 32 : 64;   // kChunkRow
  if (parts) {
    p.out_tma = 1;
    ok = ok && encode3(&p.out, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, part, g.n, g.m, plan.splits, plan.ldp, 32, 32);
  } else if (rows16 && aligned16(g.out)) {
    p.out_tma = 1;
    ok = ok && encode3(&p.out, tio, esize, g.out, g.n, g.m, 1, g.n, cw, 32);
  }
  if (g.res && aligned16(g.res) && g.ldr * esize % 16 == 0) {
    p.res_tma = 1;
    ok = ok && encode3(&p.res, tio, esize, g.res, g.n, g.m, 1, g.ldr, cw, 32);
  }
  const void *aux = g.slope_act == DCN_ACT_GELU ? g.slope : g.act == DCN_ACT_GELU ? g.saved : nullptr;
  p.ldz = (g.n + 7) / 8 * 8;
  if (aux) {
    ok = ok && encode3(&p.aux, tio, esize, aux, p.ldz, g.m, 1, p.ldz, cw, 32);
  }
  if (!ok) return cudaErrorInvalidValue;
  cudaError_t e;
  if (dtype == DCN_DTYPE_F32) e = run_gemm_f32(p, plan.bn, plan.cg, parts, s);
  else if (dtype == DCN_DTYPE_BF16) e = run_gemm_bf16(p, plan.bn, plan.cg, parts, s);
  else e = run_gemm_f16(p, plan.bn, plan.cg, parts, s);
  if (e != cudaSuccess || !parts) return e;
  GemmArgs r = g;
  if (g.row_sum) {
    r.join_part = row_part;
    r.join_parts = plan.splits;
    r.join_out = g.row_sum;
  }
  if (dtype == DCN_DTYPE_F32) return run_reduce<float>(part, plan, r, s);
  if (dtype == DCN_DTYPE_BF16) return run_reduce<__nv_bfloat16>(part, plan, r, s);
  return run_reduce<__half>(part, plan, r, s);
}

int stage_slabs(long long rows, long long cols) {
  StageJob j;
  stage_shape(rows, (cols + 7) / 8 * 8, &j);
  return j.gy;
}

void add_stage(StageJobs *jobs, const void *src, long long ld, const void *saved, int act, long long rows, long long cols,
               int dtype, void *planes, float *sums) {
  StageJob &j = jobs->job[jobs->count++];
  j.src = src; j.saved = saved; j.dst = planes; j.sums = sums;
  j.ld = ld; j.rows = rows; j.cols = cols; j.pitch = (cols + 7) / 8 * 8; j.act = act;
  j.vec_src = aligned16(src) && ld * (dtype == DCN_DTYPE_F32 ? 4 : 2) % 16 == 0;
  stage_shape(rows, j.pitch, &j);
  j.first = jobs->blocks;
  jobs->blocks += j.gx * j.gy;
}

cudaError_t launch_gemm_stage(StageJobs &jobs, int dtype, cudaStream_t s) {
  if (!jobs.count) return cudaSuccess;
  for (int i = jobs.count; i < 3; ++i) jobs.job[i].first = jobs.blocks;
  if (dtype == DCN_DTYPE_F32) return launch_pdl(dcn_gemm_stage<float, 3>, jobs.blocks, 256, 0, s, 1, jobs);
  if (dtype == DCN_DTYPE_BF16) return launch_pdl(dcn_gemm_stage<__nv_bfloat16, 1>, jobs.blocks, 256, 0, s, 1, jobs);
  return launch_pdl(dcn_gemm_stage<__half, 1>, jobs.blocks, 256, 0, s, 1, jobs);
}

cudaError_t launch_column_reduce(const float *part, int parts, long long cols, int dtype, void *out, cudaStream_t s) {
  if (dtype == DCN_DTYPE_F32) return run_columns<float>(part, parts, cols, out, s);
  if (dtype == DCN_DTYPE_BF16) return run_columns<__nv_bfloat16>(part, parts, cols, out, s);
  return run_columns<__half>(part, parts, cols, out, s);
}

cudaError_t read_gemm_status(cudaStream_t s, int *status) {
  *status = 0;
  for (auto read : {read_gemm_status_bf16, read_gemm_status_f16, read_gemm_status_f32}) {
    int one = 0;
    const cudaError_t e = read(s, &one);
    if (e != cudaSuccess) return e;
    if (!*status) *status = one;
  }
  return cudaSuccess;
}

}  // namespace dcn
