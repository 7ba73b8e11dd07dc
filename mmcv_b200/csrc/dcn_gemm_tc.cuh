// Matrix product with an epilogue on the tensor cores (sm_100a), instantiated for one tensor type per
// translation unit (dcn_gemm_bf16.cu, dcn_gemm_f16.cu, dcn_gemm_f32.cu):
//   out[i, j] = epilogue(sum_k A[i, k] * B[j, k])
// for the three products of a linear layer.  Forward reads both operands with k contiguous; the
// gradient of the input reads the weight, and the gradient of the weight both operands, with the
// output index contiguous.  Tensor maps and tcgen05 descriptors take either order, so nothing is
// transposed in memory.
//
// Two blocks of a cluster may work on one tile of 256 rows (CG = 2): each loads its own 128 rows of A and
// half of the rows of B, and one tcgen05.mma.cta_group::2 multiplies what lies in both.  A step of a
// 256-column tile then brings 32 KB into an SM instead of 48, and what bounds the long products is the rate
// at which tiles come in (46 bytes a clock and SM with five stages in flight, 40 with three).  plan_gemm
// chooses; where tiles are few and sums long, two to four blocks of a cluster share a tile's sum instead.
//
// One persistent block per SM: a loader lane fills a ring of stages (64 values of k of a 128-row A
// tile and a BN-row B tile, 128-byte swizzle) with cp.async.bulk.tensor; one warp issues tcgen05.mma
// into fp32 accumulators in tensor memory, double-buffered so that the epilogue of a tile runs under
// the main loop of the next; epilogue warps do the rest: tcgen05.ld, bias, activation, derivative,
// residual, one rounding, a 32-row chunk in shared memory, a tensor store.  The residual arrives by
// tensor load in the chunk that the result leaves from, as do the kept derivatives of gelu.
// Sixteen epilogue warps (eight with fp32 tensors) and not four: a warp's share of a tile is a chain of waits
// (tensor memory, loads, the store of its last chunk), and the products around an embedding of 256 have main
// loops of four steps only (35642 x 256 x 1024 bf16 with relu: 42 us with eight warps, 28 with sixteen).
// Every wait is bounded.
//
// Measured: 8192 x 4096 x 4096 bf16 171 us, 1.61 PFLOP/s, the tensor pipe 87 % busy; 35642 x 256 x 1024 28 us
// (its bytes 14 us at the copy rate), bound by the epilogue's chain.
//
// 16-bit tensors: one plane (PL = 1).  fp32 tensors: every operand is the exact sum of three bf16
// planes x = x1 + x2 + x3 of 8 bits each (dcn_gemm_stage writes them), and the product is
//   x1 y1 + (x1 y2 + x2 y1 + x2 y2 + x1 y3 + x3 y1);
// what is left out, x2 y3 + x3 y2 + x3 y3, is at most 2^-24 + 2^-34 of |x||y|, of either sign.
// A tensor core truncates where it adds to its accumulator, so long fp32 sums would drift by 2^-24 a step:
// the leading product and the five small ones have accumulators of their own, and every 256 values of k the
// epilogue warps take both out into registers, where the additions round to nearest.
//
// The weight gradient's sum over the rows is cut into `splits` ranges when its tiles alone do not
// fill the SMs; the fp32 parts are added in order by dcn_gemm_reduce.  With 16-bit tensors its bias gradient
// (row sums of A) costs one more instruction a step: a product with a tile of ones.
#pragma once

#include <atomic>
#include <type_traits>

#include <cuda.h>

#include "dcn_gemm.cuh"
#include "dcn_ptx.cuh"

namespace dcn {

namespace {

enum { kEpiPlain, kEpiRelu, kEpiGelu, kEpiSlopeRelu, kEpiSlopeGelu };

// Epilogue warps: four to each quarter of the accumulator's rows, two where three planes take the shared
// memory that their staging would need.  With them the MMA warp and the loader warp.
template <int PL>
constexpr int kEpi = PL == 3 ? 8 : 16;
template <int PL>
constexpr int kThreadsOf = (kEpi<PL> + 2) * 32;

// Bytes of a row of an epilogue warp's staging chunk (32 rows).  128 where a warp of a 256-column tile has 64
// columns of 16 bits: fewer, wider stores for tiles of few steps.  Pairs, which take the long sums, give the
// memory to a sixth stage instead (8192 x 4096 x 4096: 176 -> 171 us).
template <typename TO, int BN, int CG>
constexpr int kChunkRow = sizeof(TO) == 4 || (BN == 256 && CG == 1) ? 128 : 64;
constexpr int kUnitBlocks = 4;          // PL = 3: 64-value blocks between two drains of the accumulators

__device__ int g_gemm_status;           // the first wait that ran out (0: none), until it is read

__device__ __forceinline__ bool g_wait(uint32_t bar, uint32_t parity, volatile int *abort_s, int code,
                                       unsigned long long limit, unsigned backoff) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = globaltimer_ns();
  for (uint32_t it = 1;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if (backoff) __nanosleep(backoff);
    if ((it & 15u) == 0u) {
      if (*abort_s) return false;
      if (globaltimer_ns() - t0 > limit) {
        *abort_s = 1;
        atomicCAS(&g_gemm_status, 0, code);
        return false;
      }
    }
  }
}

// CG = 2: the barrier may be the other block's of the pair.
template <int CG = 1>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, int c0, int c1, int c2,
                                            uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
}
// One block (CG = 1) or the pair of blocks of a cluster (CG = 2) that works on one accumulator.
template <int CG>
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 1) {
    umma_bf16(d, a, b, idesc, accumulate);
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}
// Arrives on `bar` (of both blocks) when the products issued so far have been computed.
template <int CG>
__device__ __forceinline__ void pair_commit(uint32_t bar) {
  if constexpr (CG == 1)
    umma_commit(bar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        ::"r"(bar), "h"((uint16_t)3)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void pair_tmem_alloc(uint32_t slot, uint32_t cols) {
  if constexpr (CG == 1) {
    tmem_alloc(slot, cols);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t cols) {
  if constexpr (CG == 1)
    tmem_dealloc(taddr, cols);
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
__device__ __forceinline__ void cluster_sync(bool clustered) {
  if (clustered) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}
// To the first block of a cluster: where its copy of a shared address is, 16 bytes there, an arrival there.
__device__ __forceinline__ uint32_t first_block(uint32_t addr) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void cluster_store16(uint32_t addr, const float *v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3])
               : "memory");
}
__device__ __forceinline__ void cluster_arrive(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// The address of the first block's copy of a shared variable, and an arrival there.
template <int CG>
__device__ __forceinline__ uint32_t lead_addr(uint32_t addr) {
  return CG == 1 ? addr : first_block(addr);
}
template <int CG>
__device__ __forceinline__ void lead_arrive(uint32_t addr) {
  if constexpr (CG == 1)
    mbar_arrive(addr);
  else
    cluster_arrive(addr);
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap *map, uint32_t src, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];"
               ::"l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(src)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr) : "memory");
  return r;
}

// Shared-memory descriptor of a tile with the 128-byte swizzle whose rows of 128 bytes hold 64
// values of the row (or column) index, one row per k: 8 k are 1024 bytes, the next 64 rows of the
// tile 8192 bytes away.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t saddr) {
  uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)(8192 >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// The tiles that a block (or pair) works on, in the order (range, row tile, column tile): column tiles of
// one row tile are neighbours, so that A stays in L2.  The stride is added digit by digit: no divisions.
struct Walk {
  int tn, tm, sp;
  __device__ __forceinline__ Walk(uint32_t item, const GemmTc &p) {
    const uint32_t t = item / (uint32_t)p.tiles_n;
    tn = (int)(item - t * (uint32_t)p.tiles_n);
    sp = (int)(t / (uint32_t)p.tiles_m);
    tm = (int)(t - (uint32_t)sp * (uint32_t)p.tiles_m);
  }
  __device__ __forceinline__ void next(const GemmTc &p) {
    tn += p.step_n;
    tm += p.step_m;
    sp += p.step_s;
    if (tn >= p.tiles_n) { tn -= p.tiles_n; ++tm; }
    if (tm >= p.tiles_m) { tm -= p.tiles_m; ++sp; }
  }
};

// A staging chunk: 32 rows of RB bytes, 16-byte pieces permuted within a row as the tensor maps'
// swizzles of that width have them, so that the lanes of a warp, a row each, meet no bank conflicts.
template <int RB>
__device__ __forceinline__ int chunk_piece(int row, int q) {
  return row * RB + ((q ^ (RB == 128 ? row & 7 : (row >> 1) & 3)) << 4);
}
// 16 bytes of elements as floats, and back
template <typename TO>
__device__ __forceinline__ void unpack16(const uint4 &u, float *v) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(TO) == 4) {
      v[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same_v<TO, __nv_bfloat16>) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}
// two floats to a pair of 16-bit values; kRelu: negative ones become 0 (a NaN stays one)
template <typename TO, bool kRelu>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t w;
  if constexpr (std::is_same_v<TO, __nv_bfloat16>) {
    if constexpr (kRelu) asm("cvt.rn.relu.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  } else {
    if constexpr (kRelu) asm("cvt.rn.relu.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  }
  return w;
}
// 32 values to a lane's row, q0: the first 16-byte piece
template <typename TO, int RB, bool kRelu = false>
__device__ __forceinline__ void stage_store(uint8_t *chunk, int row, int q0, const float (&v)[32]) {
  constexpr int E = 16 / (int)sizeof(TO);
#pragma unroll
  for (int q = 0; q < 32 / E; ++q) {
    uint4 u;
    if constexpr (sizeof(TO) == 4) {
      u = make_uint4(__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]), __float_as_uint(v[4 * q + 2]),
                     __float_as_uint(v[4 * q + 3]));
    } else {
      u = make_uint4(pack2<TO, kRelu>(v[8 * q], v[8 * q + 1]), pack2<TO, kRelu>(v[8 * q + 2], v[8 * q + 3]),
                     pack2<TO, kRelu>(v[8 * q + 4], v[8 * q + 5]), pack2<TO, kRelu>(v[8 * q + 6], v[8 * q + 7]));
    }
    *reinterpret_cast<uint4 *>(chunk + chunk_piece<RB>(row, q0 + q)) = u;
  }
}

// the same of gelu's derivatives, as they are kept
template <typename TO, int RB>
__device__ __forceinline__ void stage_slopes(uint8_t *chunk, int row, int q0, const float (&v)[32]) {
  if constexpr (sizeof(TO) == 4) {
    stage_store<TO, RB>(chunk, row, q0, v);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<uint4 *>(chunk + chunk_piece<RB>(row, q0 + q)) =
          make_uint4(slope_codes(v[8 * q], v[8 * q + 1]), slope_codes(v[8 * q + 2], v[8 * q + 3]),
                     slope_codes(v[8 * q + 4], v[8 * q + 5]), slope_codes(v[8 * q + 6], v[8 * q + 7]));
  }
}

// v[0..31] += bias[j1 ..]; whole groups of a bias that starts on 16 bytes by 16-byte loads (the same
// address in every lane)
template <typename TO>
__device__ __forceinline__ void add_bias(const TO *bias, int j1, int n, bool vec, float (&v)[32]) {
  if (vec && j1 + 32 <= n) {
    constexpr int E = 16 / (int)sizeof(TO);
#pragma unroll
    for (int i = 0; i < 32 / E; ++i) {
      float b[E];
      unpack16<TO>(__ldg(reinterpret_cast<const uint4 *>(bias + j1) + i), b);
#pragma unroll
      for (int k = 0; k < E; k += 2) add2(v[E * i + k], v[E * i + k + 1], b[k], b[k + 1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] += j1 + j < n ? ElemOf<TO>::to(__ldg(bias + j1 + j)) : 0.f;
  }
}

// The element-by-element forms of the chunk's tensor load and store, for tensors whose rows do not
// start on 16 bytes: the warp walks the 32 rows, neighbouring lanes on neighbouring columns.
template <typename TO, int RB>
__device__ __forceinline__ TO *chunk_at(uint8_t *chunk, int r, int c) {
  const int at = c * (int)sizeof(TO);
  return reinterpret_cast<TO *>(chunk + chunk_piece<RB>(r, at >> 4) + (at & 15));
}
template <typename TO, int RB>
__device__ __forceinline__ void chunk_in(uint8_t *chunk, const TO *src, long long ld, int i0, int m, int j0, int n,
                                         int lane) {
  constexpr int P = RB / (int)sizeof(TO) / 32;
  const int rows = min(32, m - i0);
  src += i0 * ld + j0;
  for (int r0 = 0; r0 < rows; r0 += 8) {   // eight rows in flight
    TO v[8][P];
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int c = 0; c < P; ++c)
        if (r0 + r < rows && j0 + c * 32 + lane < n) v[r][c] = src[(r0 + r) * ld + c * 32 + lane];
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int c = 0; c < P; ++c)
        if (r0 + r < rows && j0 + c * 32 + lane < n) *chunk_at<TO, RB>(chunk, r0 + r, c * 32 + lane) = v[r][c];
  }
}
template <typename TO, int RB>
__device__ __forceinline__ void chunk_out(uint8_t *chunk, TO *dst, long long ld, int i0, int m, int j0, int n,
                                          int lane) {
  constexpr int P = RB / (int)sizeof(TO) / 32;
  const int rows = min(32, m - i0);
  dst += i0 * ld + j0;
#pragma unroll 8
  for (int r = 0; r < rows; ++r)
#pragma unroll
    for (int c = 0; c < P; ++c)
      if (j0 + c * 32 + lane < n) dst[r * ld + c * 32 + lane] = *chunk_at<TO, RB>(chunk, r, c * 32 + lane);
}
// The sum over the lanes of v[j], in lane j: 31 exchanges, each lane giving away the half that the other
// keeps.  v is used up.
__device__ __forceinline__ float column_sums(float (&v)[32], int lane) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const bool up = (lane & d) != 0;
#pragma unroll
    for (int j = 0; j < d; ++j) {
      const float give = up ? v[j] : v[j + d], keep = up ? v[j + d] : v[j];
      v[j] = keep + __shfl_xor_sync(0xffffffffu, give, d);
    }
  }
  return v[0];
}
// v[0..31] += a lane's own row of the residual, for the rare epilogue whose chunk is taken
template <typename TO>
__device__ __forceinline__ void add_row(const TO *src, int j1, int n, float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 32; ++j)
    if (j1 + j < n) v[j] += ElemOf<TO>::to(__ldg(src + j));
}

}  // namespace

// PL planes per operand; TI the 16-bit type of the planes, TO the output's (and residual's) type;
// AMN / BMN: the operand lies with its row index contiguous; CG blocks to a tile; EPI: what the epilogue
// does between bias and residual (a kernel of its own each: with all of them in one, its code ran out of
// the instruction cache and its registers).
template <typename TI, typename TO, int PL, int BN, bool AMN, bool BMN, int CG, int EPI>
__global__ void __launch_bounds__(kThreadsOf<PL>, 1) dcn_gemm_tc(const __grid_constant__ GemmTc p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr uint32_t kABytes = PL * 16384u, kBBytes = PL * (BN / CG) * 128u, kStage = kABytes + kBBytes;
  constexpr int kEpiWarps = kEpi<PL>, kGemmThreads = kThreadsOf<PL>, kGroups = kEpiWarps / 4;
  constexpr bool kRowSum = AMN && PL == 1;             // only the weight gradient asks for row sums
  constexpr int kBufs = (kRowSum && BN == 256) ? 1 : 2;   // accumulator buffers that fit beside the row sums
  constexpr int kOnes = 16 * CG;   // columns of the product with the tile of ones
  constexpr int kBufCols = PL == 3 ? 2 * BN : BN;
  constexpr int kCols = kBufs * kBufCols + (kRowSum ? kOnes * kBufs : 0);
  constexpr int kAlloc = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static_assert(kCols <= 512, "tensor memory");
  constexpr int RB = kChunkRow<TO, BN, CG>, kChunkBytes = 32 * RB;
  constexpr int CW = RB / (int)sizeof(TO);             // columns of a staging chunk
  constexpr int kWarpCols = BN / kGroups > CW ? BN / kGroups : CW;   // columns of an epilogue warp

  const GemmArgs &g = p.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ST = p.stages;
  const uint32_t bar0 = smem_u32(smem);
  const uint32_t full = bar0, empty = full + 8 * ST, tmem_full = empty + 8 * ST, tmem_empty = tmem_full + 16,
                 in_bar = tmem_empty + 16, part_bar = in_bar + 8 * kEpiWarps;   // one each per epilogue warp
  // p.ks blocks of a cluster each sum a range of k of one tile; the first adds the others' sums, in order, to
  // its own.  There are as many clusters as tiles then.
  constexpr bool kCanShare = CG == 1 && BN == 64 && !AMN;
  static_assert(!kCanShare || kWarpCols == 32, "a warp's part: 32 x 32");
  const int ks = kCanShare ? p.ks : 1, krank = kCanShare && ks > 1 ? (int)(blockIdx.x % (uint32_t)ks) : 0;
  uint32_t *tmem_slot = (uint32_t *)(smem + 896);
  volatile int *abort_s = (volatile int *)(smem + 904);
  uint8_t *ring = smem + 1024;
  uint8_t *staging = ring + (size_t)ST * kStage;
  uint8_t *ones = staging + (size_t)kEpiWarps * kChunkBytes;
  uint8_t *parts = ones;   // (nobody has both) [ks - 1][active epilogue warps][8][32 lanes] x 16 bytes
  const unsigned long long limit = p.wait_limit_ns;

  if (bar0 & 1023u) {   // the swizzles go by addresses; the declaration sees to this
    if (threadIdx.x == 0) atomicCAS(&g_gemm_status, 0, 10);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(tmem_full + 8 * i, 1);
      mbar_init(tmem_empty + 8 * i, CG * kEpiWarps);
    }
    for (int i = 0; i < kEpiWarps; ++i) {
      mbar_init(in_bar + 8 * i, 1);
      if (ks > 1) mbar_init(part_bar + 8 * i, ks - 1);
    }
    *abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (kRowSum && g.row_sum) {
    // 16 rows (of each block) x 64 values, all one: the same in every layout
    for (int i = threadIdx.x; i < 1024; i += kGemmThreads) ((TI *)ones)[i] = ElemOf<TI>::from(1.f);
    fence_proxy_async_smem();
  }
  if (warp == kEpiWarps) {
    pair_tmem_alloc<CG>(smem_u32(tmem_slot), kAlloc);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync(CG == 2 || ks > 1);
  tc_fence_after();
  pdl_wait();
  pdl_launch();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t items = (uint32_t)p.tiles_m * (uint32_t)p.tiles_n * (uint32_t)p.splits;
  const int rank = CG == 1 ? 0 : (int)(blockIdx.x & 1);   // a cluster is two neighbouring blocks
  const uint32_t first_item = ks > 1 ? blockIdx.x / (uint32_t)ks : blockIdx.x / CG,
                 item_step = ks > 1 ? items : gridDim.x / CG;
  const uint32_t lead_empty = lead_addr<CG>(tmem_empty), lead_full = lead_addr<CG>(full);

  if (warp < kEpiWarps) {
    // ------------------------------ epilogue ------------------------------
    const int q = warp & 3, cg = warp >> 2;
    const uint32_t lane_base = tmem_base + ((uint32_t)(q * 32) << 16);
    uint8_t *chunk = staging + (size_t)warp * kChunkBytes;
    const uint32_t chunk_u = smem_u32(chunk), ib = in_bar + 8 * warp;
    uint32_t iph = 0, unit = 0;
    const int m = p.m, n = p.n, words = (n + 31) / 32;
    constexpr bool aux_in = EPI == kEpiSlopeGelu;
    const bool aux_out = EPI == kEpiGelu && g.saved != nullptr;
    const bool res_staged = g.res && !aux_in && !aux_out;
    const bool load_in = aux_in || (res_staged && p.res_tma);
    bool ok = true;
    Walk walk(first_item, p);
    for (uint32_t item = first_item; item < items && ok; item += item_step, walk.next(p)) {
      const int i0 = (walk.tm * CG + rank) * 128 + q * 32, row = i0 + lane;
      const int jw = walk.tn * BN + cg * kWarpCols;   // this warp's first column
      const int kb0 = (ks > 1 ? krank : walk.sp) * p.kb_split, kb1 = min(p.kb_total, kb0 + p.kb_split);
      const int chunks = cg * kWarpCols < BN && jw < n ? (min(n - jw, kWarpCols) + CW - 1) / CW : 0;
      // the store that read the chunk last is done with it
      auto chunk_free = [&] {
        if (lane == 0) bulk_wait_read();
        __syncwarp();
      };
      // what a chunk takes in, to its own place: asked for as soon as that is free, the first chunk's under
      // the main loop
      auto fetch = [&](int j0) {
        chunk_free();
        if (load_in) {
          if (lane == 0) {
            fence_proxy_async_smem();
            mbar_arrive_expect_tx(ib, kChunkBytes);
            tma_load_3d(chunk_u, aux_in ? &p.aux : &p.res, j0, i0, 0, ib);
          }
        } else if (res_staged) {
          chunk_in<TO, RB>(chunk, (const TO *)g.res, g.ldr, i0, m, j0, n, lane);
          __syncwarp();   // written along columns, read a row to a lane
        }
      };
      const bool takes = load_in || res_staged;
      if (takes && chunks && krank == 0) fetch(jw);
      float facc[PL == 3 ? kWarpCols : 1];
      const int units = PL == 3 ? (kb1 - kb0 + kUnitBlocks - 1) / kUnitBlocks : 1;
      int buf = 0;
      for (int u = 0; u < units && ok; ++u, ++unit) {
        buf = kBufs == 2 ? (int)(unit & 1) : 0;
        const uint32_t ph = kBufs == 2 ? (unit >> 1) & 1u : unit & 1u;
        ok = __all_sync(0xffffffffu, g_wait(tmem_full + 8 * buf, ph, abort_s, 3, 2 * limit, 32));
        if (!ok) break;
        tc_fence_after();
        if constexpr (PL == 3) {
          if (chunks) {
            const uint32_t t = lane_base + (uint32_t)(buf * kBufCols + cg * kWarpCols);
#pragma unroll
            for (int c = 0; c < kWarpCols; c += 16) {
              uint32_t a[16], b[16];
              tmem_ld16(t + c, a);
              tmem_ld16(t + BN + c, b);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                // an infinite element has planes inf, 0, 0: the leading product is right, the small ones
                // may hold inf * 0
                const float lead = __uint_as_float(a[j]);
                const float v = isinf(lead) ? lead : lead + __uint_as_float(b[j]);
                facc[c + j] = u ? facc[c + j] + v : v;
              }
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) lead_arrive<CG>(lead_empty + 8 * buf);
        }
      }
      if (!ok) break;
      if (kRowSum && g.row_sum && walk.tn == 0 && cg == 0) {
        const float v = __uint_as_float(tmem_ld1(lane_base + (uint32_t)(kBufs * kBufCols + kOnes * buf)));
        tmem_ld_wait();
        if (row < m) {
          if (p.splits > 1) p.row_part[(long long)walk.sp * m + row] = v;
          else ((TI *)g.row_sum)[row] = ElemOf<TI>::from(v);
        }
      }
      if constexpr (kCanShare) {
        if (ks > 1) {
          const uint32_t mine = smem_u32(parts) + (uint32_t)warp * 4096u + (uint32_t)lane * 16u;
          constexpr uint32_t kPart = BN / 32 * 4 * 4096u;   // of a block
          if (krank) {
            if (chunks) {
              float v[32];
              if constexpr (PL == 3) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = facc[j];
              } else {
                uint32_t r[32];
                tmem_ld32(lane_base + (uint32_t)(cg * kWarpCols), r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
              }
              const uint32_t to = first_block(mine + (uint32_t)(krank - 1) * kPart);
#pragma unroll
              for (int j = 0; j < 8; ++j) cluster_store16(to + j * 512, v + 4 * j);
              __syncwarp();
              if (lane == 0) cluster_arrive(first_block(part_bar + 8 * warp));
            }
            break;   // the first block has the rest
          }
          if (chunks) {
            ok = __all_sync(0xffffffffu, g_wait(part_bar + 8 * warp, 0, abort_s, 9, 2 * limit, 0));
            if (!ok) break;
            asm volatile("fence.acq_rel.cluster;" ::: "memory");
          }
        }
      }
      // the 32 sums of a group of columns, with the bias
      auto sums = [&](int j1, int c, float (&v)[32]) {
        if constexpr (PL == 3) {
#pragma unroll
          for (int j = 0; j < 32; ++j) {   // c is a runtime index: pick without indexing registers by it
            v[j] = facc[j];
            if constexpr (kWarpCols > 32) v[j] = c ? facc[32 + j] : v[j];
          }
        } else {
          uint32_t r[32];
          tmem_ld32(lane_base + (uint32_t)(buf * kBufCols + cg * kWarpCols + c), r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
        }
        if constexpr (kCanShare) {
          for (int k = 1; k < ks; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 f = *reinterpret_cast<const float4 *>(
                  parts + (size_t)(k - 1) * (BN / 32 * 4 * 4096) + warp * 4096 + j * 512 + lane * 16);
              add2(v[4 * j], v[4 * j + 1], f.x, f.y);
              add2(v[4 * j + 2], v[4 * j + 3], f.z, f.w);
            }
        }
        if (g.bias) add_bias<TO>((const TO *)g.bias, j1, n, p.bias16 != 0, v);
      };
      static_assert(PL == 1 || kWarpCols <= 64, "two groups");
      // all read: the next tile may have the accumulator
      auto accumulator_free = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) lead_arrive<CG>(lead_empty + 8 * buf);
      };
      auto chunk_leaves = [&](int j0) {
        fence_proxy_async_smem();
        __syncwarp();
        if (!p.out_tma) {
          chunk_out<TO, RB>(chunk, (TO *)g.out, n, i0, m, j0, n, lane);
          __syncwarp();
        } else if (lane == 0) {
          tma_store_3d(&p.out, chunk_u, j0, i0, walk.sp);
          bulk_commit();
        }
      };
#pragma unroll 1
      for (int ch = 0; ch < chunks; ++ch) {
        const int j0 = jw + ch * CW;
        if (takes && ch) fetch(j0);
        if constexpr (EPI == kEpiGelu && PL == 1) {
          if (aux_out && !g.res) {   // derivatives and values at once; the values wait in registers
            uint32_t keep[CW / 32][16];
            chunk_free();
#pragma unroll
            for (int c1 = 0; c1 < CW; c1 += 32) {
              float v[32], slope[32];
              sums(j0 + c1, ch * CW + c1, v);
              if (ch == chunks - 1 && c1 == CW - 32) accumulator_free();
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                gelu_both<false>(v[j], v[j + 1], slope[j], slope[j + 1]);
                keep[c1 / 32][j / 2] = pack2<TO, false>(v[j], v[j + 1]);
              }
              stage_slopes<TO, RB>(chunk, lane, c1 * (int)sizeof(TO) / 16, slope);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(&p.aux, chunk_u, j0, i0, 0);
              bulk_commit();
            }
            chunk_free();
#pragma unroll
            for (int q = 0; q < CW / 8; ++q)
              *reinterpret_cast<uint4 *>(chunk + chunk_piece<RB>(lane, q)) =
                  make_uint4(keep[q / 4][q % 4 * 4], keep[q / 4][q % 4 * 4 + 1], keep[q / 4][q % 4 * 4 + 2],
                             keep[q / 4][q % 4 * 4 + 3]);
            chunk_leaves(j0);
            continue;
          }
        }
        if (aux_out) {   // the derivatives leave first, through the same chunk
          chunk_free();
#pragma unroll 1
          for (int c1 = 0; c1 < CW; c1 += 32) {
            float v[32];
            sums(j0 + c1, ch * CW + c1, v);
#pragma unroll
            for (int j = 0; j < 32; j += 2) gelu_slopes<PL == 3>(v[j], v[j + 1]);
            stage_slopes<TO, RB>(chunk, lane, c1 * (int)sizeof(TO) / 16, v);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(&p.aux, chunk_u, j0, i0, 0);
            bulk_commit();
          }
        }
        if (load_in) {
          ok = __all_sync(0xffffffffu, g_wait(ib, iph, abort_s, 8, 2 * limit, 0));
          iph ^= 1u;
          if (!ok) break;
        }
#pragma unroll 1
        for (int c1 = 0; c1 < CW; c1 += 32) {
          const int j1 = j0 + c1, q0 = c1 * (int)sizeof(TO) / 16;
          float v[32];
          sums(j1, ch * CW + c1, v);
          if constexpr (PL == 1) {
            if (ch == chunks - 1 && c1 == CW - 32) accumulator_free();
          }
          if (c1 == 0 && !takes) chunk_free();
          constexpr int E = 16 / (int)sizeof(TO);
          if constexpr (EPI == kEpiRelu) {
            if (g.saved) {
              uint32_t bits = 0;
#pragma unroll
              for (int j = 0; j < 32; ++j) bits |= relu_bit(v[j]) ? 1u << j : 0u;
              if (row < m && j1 < n) ((uint32_t *)g.saved)[(long long)row * words + (j1 >> 5)] = bits;
            }
            if (g.res || sizeof(TO) == 4) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = relu_value(v[j]);
            }
          } else if constexpr (EPI == kEpiGelu) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) gelu_values<PL == 3>(v[j], v[j + 1]);
          } else if constexpr (EPI == kEpiSlopeRelu) {
            const uint32_t bits =
                row < m && j1 < n ? __ldg((const uint32_t *)g.slope + (long long)row * words + (j1 >> 5)) : 0u;
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = (bits >> j) & 1u ? v[j] : 0.f;
          } else if constexpr (EPI == kEpiSlopeGelu) {
#pragma unroll
            for (int k = 0; k < 32 / E; ++k) {
              float z[E];
              unpack_slopes<TO>(*reinterpret_cast<const uint4 *>(chunk + chunk_piece<RB>(lane, q0 + k)), z);
#pragma unroll
              for (int j = 0; j < E; ++j) v[E * k + j] *= z[j];
            }
          }
          if (res_staged) {
#pragma unroll
            for (int k = 0; k < 32 / E; ++k) {
              float r[E];
              unpack16<TO>(*reinterpret_cast<const uint4 *>(chunk + chunk_piece<RB>(lane, q0 + k)), r);
#pragma unroll
              for (int j = 0; j < E; j += 2) add2(v[E * k + j], v[E * k + j + 1], r[j], r[j + 1]);
            }
          } else if (g.res && row < m) {
            add_row<TO>((const TO *)g.res + row * g.ldr + j1, j1, n, v);
          }
          if (EPI == kEpiRelu && sizeof(TO) == 2 && !g.res) stage_store<TO, RB, EPI == kEpiRelu>(chunk, lane, q0, v);
          else stage_store<TO, RB>(chunk, lane, q0, v);
          if constexpr (EPI == kEpiSlopeRelu || EPI == kEpiSlopeGelu) {
            if (g.col_part) {   // no residual then: v is the gradient itself
              if (row >= m) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = 0.f;
              }
              const float s = column_sums(v, lane);
              if (i0 < m && j1 + lane < n) g.col_part[(long long)(i0 >> 5) * n + j1 + lane] = s;
            }
          }
        }
        chunk_leaves(j0);
      }
      if constexpr (PL == 1) {
        if (!chunks) accumulator_free();
      }
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  } else if (warp == kEpiWarps) {
    // ------------------------------ MMA issuer ------------------------------
    constexpr uint32_t kFmt = std::is_same_v<TI, __nv_bfloat16> ? 1u : 0u;
    constexpr uint32_t kDesc = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((AMN ? 1u : 0u) << 15) | ((128u * CG >> 4) << 24);
    constexpr uint32_t idesc = kDesc | ((BMN ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17);
    constexpr uint32_t idesc_ones = kDesc | (((uint32_t)kOnes >> 3) << 17);
    constexpr uint32_t kAStep = AMN ? 2048 >> 4 : 32 >> 4, kBStep = BMN ? 2048 >> 4 : 32 >> 4;
    const uint64_t ones_desc = smem_desc_sw128(smem_u32(ones));
    uint32_t st = 0, ph = 0, unit = 0;
    bool ok = rank == 0;   // the first block of a pair issues for both
    Walk walk(first_item, p);
    for (uint32_t item = first_item; item < items && ok; item += item_step, walk.next(p)) {
      const int kb0 = (ks > 1 ? krank : walk.sp) * p.kb_split, kb1 = min(p.kb_total, kb0 + p.kb_split);
      const bool sums = kRowSum && g.row_sum && walk.tn == 0;
      uint32_t d = 0;
      int buf = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        const bool first = PL == 3 ? (kb - kb0) % kUnitBlocks == 0 : kb == kb0;
        const bool last = PL == 3 ? (kb - kb0) % kUnitBlocks == kUnitBlocks - 1 || kb == kb1 - 1 : kb == kb1 - 1;
        if (first) {
          buf = kBufs == 2 ? (int)(unit & 1) : 0;
          const uint32_t eph = (kBufs == 2 ? (unit >> 1) & 1u : unit & 1u) ^ 1u;
          ok = __all_sync(0xffffffffu, g_wait(tmem_empty + 8 * buf, eph, abort_s, 4, limit, 0));
          if (!ok) break;
          d = tmem_base + (uint32_t)(buf * kBufCols);
          ++unit;
        }
        ok = __all_sync(0xffffffffu, g_wait(full + 8 * st, ph, abort_s, 5, limit, 0));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t sa = smem_u32(ring) + st * kStage, sb = sa + kABytes;
          uint64_t ad[PL], bd[PL];
#pragma unroll
          for (int i = 0; i < PL; ++i) {
            ad[i] = AMN ? smem_desc_mn(sa + i * 16384u) : smem_desc_sw128(sa + i * 16384u);
            bd[i] = BMN ? smem_desc_mn(sb + i * (BN / CG) * 128u) : smem_desc_sw128(sb + i * (BN / CG) * 128u);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint64_t ka = (uint64_t)(k * kAStep), kb_ = (uint64_t)(k * kBStep);
            const uint32_t more = !first || k ? 1u : 0u;
            pair_mma<CG>(d, ad[0] + ka, bd[0] + kb_, idesc, more);
            if constexpr (PL == 3) {
              pair_mma<CG>(d + BN, ad[0] + ka, bd[2] + kb_, idesc, more);
              pair_mma<CG>(d + BN, ad[2] + ka, bd[0] + kb_, idesc, 1u);
              pair_mma<CG>(d + BN, ad[1] + ka, bd[1] + kb_, idesc, 1u);
              pair_mma<CG>(d + BN, ad[0] + ka, bd[1] + kb_, idesc, 1u);
              pair_mma<CG>(d + BN, ad[1] + ka, bd[0] + kb_, idesc, 1u);
            }
            if (kRowSum && sums)
              pair_mma<CG>(tmem_base + (uint32_t)(kBufs * kBufCols + kOnes * buf), ad[0] + ka, ones_desc, idesc_ones, more);
          }
          pair_commit<CG>(empty + 8 * st);
          if (last) pair_commit<CG>(tmem_full + 8 * buf);
        }
        __syncwarp();
        if (++st == (uint32_t)ST) { st = 0; ph ^= 1u; }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------ loader ------------------------------
    if (lane == 0) {
      uint32_t st = 0, ph = 0;
      bool ok = true;
      Walk walk(first_item, p);
      for (uint32_t item = first_item; item < items && ok; item += item_step, walk.next(p)) {
        const int kb0 = (ks > 1 ? krank : walk.sp) * p.kb_split, kb1 = min(p.kb_total, kb0 + p.kb_split);
        const int m0 = (walk.tm * CG + rank) * 128, nb = walk.tn * BN + rank * (BN / CG);
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = g_wait(empty + 8 * st, ph ^ 1u, abort_s, 7, 2 * limit, 32);
          if (!ok) break;
          // a pair's loads all count on the first block's barrier
          const uint32_t bar = lead_full + 8 * st, sa = smem_u32(ring) + st * kStage, sb = sa + kABytes;
          if (rank == 0) mbar_arrive_expect_tx(full + 8 * st, CG * kStage);
          const int k0 = kb * 64;
#pragma unroll
          for (int i = 0; i < PL; ++i) {
            if constexpr (AMN) {
#pragma unroll
              for (int j = 0; j < 2; ++j)
                tma_load_3d<CG>(sa + i * 16384u + j * 8192u, &p.a, m0 + 64 * j, k0, i, bar);
            } else {
              tma_load_3d<CG>(sa + i * 16384u, &p.a, k0, m0, i, bar);
            }
            if constexpr (BMN) {
#pragma unroll
              for (int j = 0; j < BN / CG / 64; ++j)
                tma_load_3d<CG>(sb + i * (BN / CG) * 128u + j * 8192u, &p.b, nb + 64 * j, k0, i, bar);
            } else {
              tma_load_3d<CG>(sb + i * (BN / CG) * 128u, &p.b, k0, nb, i, bar);
            }
          }
          if (++st == (uint32_t)ST) { st = 0; ph ^= 1u; }
        }
      }
    }
    __syncwarp();
  }

  if (*abort_s) {
    for (int i = 0; i < 20; ++i) __nanosleep(50000);   // copies and products in flight land
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync(CG == 2 || ks > 1);   // no block leaves while the other may still reach into it
  if (warp == kEpiWarps) {
    tc_fence_after();
    pair_tmem_dealloc<CG>(tmem_base, kAlloc);
  }
}

namespace {

template <typename TI, typename TO, int PL, int BN, bool AMN, bool BMN, int CG, int EPI>
cudaError_t run_tc(GemmTc &p, cudaStream_t s) {
  auto kern = dcn_gemm_tc<TI, TO, PL, BN, AMN, BMN, CG, EPI>;
  static std::atomic<unsigned long long> done_mask{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  constexpr size_t kMost = 232448;
  if (!(done_mask.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost);
    if (e != cudaSuccess) return e;
    done_mask.fetch_or(bit, std::memory_order_release);
  }
  constexpr size_t stage = (size_t)PL * (16384 + BN / CG * 128);
  constexpr size_t fixed = 1024 + (size_t)kEpi<PL> * 32 * kChunkRow<TO, BN, CG> + (AMN && PL == 1 ? 2048 : 0);
  const size_t parts = (size_t)(p.ks - 1) * (BN / 32 * 4 * 4096);
  const int fit = (int)((kMost - fixed - parts) / stage), stages = fit > 8 ? 8 : fit;
  static_assert((kMost - fixed) / stage >= 2, "a ring");
  if (stages < 2 || (p.ks > 1 && (CG == 2 || BN != 64 || AMN))) return cudaErrorInvalidValue;
  p.stages = stages;
  const long long items = (long long)p.tiles_m * p.tiles_n * p.splits;
  const int grid = p.ks > 1 ? (int)items * p.ks : CG * (int)(items < 148 / CG ? items : 148 / CG), step = grid / CG;
  p.step_n = step % p.tiles_n;
  p.step_m = step / p.tiles_n % p.tiles_m;
  p.step_s = step / p.tiles_n / p.tiles_m;
  return launch_pdl(kern, grid, kThreadsOf<PL>, fixed + parts + stages * stage, s, p.ks > 1 ? p.ks : CG, p);
}

template <typename TI, typename TO, int PL, bool AMN, bool BMN, int EPI>
cudaError_t run_bn(GemmTc &p, int bn, int cg, cudaStream_t s) {
  if constexpr (PL == 1) {
    if (cg == 2) return run_tc<TI, TO, PL, 256, AMN, BMN, 2, EPI>(p, s);
    if (bn == 256) return run_tc<TI, TO, PL, 256, AMN, BMN, 1, EPI>(p, s);
  } else {
    if (cg == 2) return run_tc<TI, TO, PL, 128, AMN, BMN, 2, EPI>(p, s);
  }
  if (bn == 128) return run_tc<TI, TO, PL, 128, AMN, BMN, 1, EPI>(p, s);
  return run_tc<TI, TO, PL, 64, AMN, BMN, 1, EPI>(p, s);
}

// The forward product (k contiguous in both) has the activations, the input gradient (weight by its rows)
// their derivatives, the weight gradient (both by their rows) neither.
template <typename TI, typename T, int PL>
cudaError_t run_order(GemmTc &p, int bn, int cg, bool parts, cudaStream_t s) {
  const GemmArgs &g = p.g;
  if (!g.a_mn && !g.b_mn) {
    if (g.act == DCN_ACT_RELU) return run_bn<TI, T, PL, false, false, kEpiRelu>(p, bn, cg, s);
    if (g.act == DCN_ACT_GELU) return run_bn<TI, T, PL, false, false, kEpiGelu>(p, bn, cg, s);
    return run_bn<TI, T, PL, false, false, kEpiPlain>(p, bn, cg, s);
  }
  if (!g.a_mn) {
    if (g.slope_act == DCN_ACT_RELU) return run_bn<TI, T, PL, false, true, kEpiSlopeRelu>(p, bn, cg, s);
    if (g.slope_act == DCN_ACT_GELU) return run_bn<TI, T, PL, false, true, kEpiSlopeGelu>(p, bn, cg, s);
    return run_bn<TI, T, PL, false, true, kEpiPlain>(p, bn, cg, s);
  }
  if (parts) return run_bn<TI, float, PL, true, true, kEpiPlain>(p, bn, cg, s);
  return run_bn<TI, T, PL, true, true, kEpiPlain>(p, bn, cg, s);
}

// Reads and clears this translation unit's status word on the current device, after the work on `s`.
cudaError_t read_status(cudaStream_t s, int *status) {
  const int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(status, g_gemm_status, sizeof(int), 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaMemcpyToSymbolAsync(g_gemm_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  return e;
}

}  // namespace

}  // namespace dcn
