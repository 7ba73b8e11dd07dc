// Matrix product with an epilogue on the tensor cores (sm_100a):
//   out[i, j] = epilogue(sum_k A[i, k] * B[j, k])
// for the three products of a linear layer.  Forward reads both operands with k contiguous; the
// gradient of the input reads the weight, and the gradient of the weight both operands, with the
// output index contiguous.  Tensor maps and tcgen05 descriptors take either order, so nothing is
// transposed in memory.
//
// Where there are enough tiles, two blocks of a cluster work on one tile of 256 rows (CG = 2): each loads
// its own 128 rows of A and half of the rows of B, and one tcgen05.mma.cta_group::2 multiplies what
// lies in both.  A step of a 256-column tile then brings 32 KB into an SM instead of 48: what bounds
// the products with few steps or few output columns is the rate at which tiles come in (about 35
// bytes a cycle and SM measured, from L2 or memory).
//
// One persistent block per SM: a loader lane fills a ring of stages (64 values of k of a 128-row A
// tile and a BN-row B tile, 128-byte swizzle) with cp.async.bulk.tensor; one warp issues tcgen05.mma
// into fp32 accumulators in tensor memory, double-buffered so that the epilogue of a tile runs under
// the main loop of the next; eight warps run the epilogue: tcgen05.ld, bias, activation, derivative,
// residual, one rounding, a 32-row chunk in shared memory, a tensor store.  The residual arrives by
// tensor load in the chunk that the result leaves from, as do the kept pre-activations of a derivative.
// Sixteen epilogue warps (eight with fp32 tensors) and not four: a warp's share of a tile is a chain of waits (tensor memory,
// loads, the store of its last chunk), and the products around an embedding of 256 have main loops of
// four steps only (35642 x 256 x 1024 bf16 with relu: 42 us with eight warps).  Every wait is bounded.
//
// 16-bit tensors: one plane (PL = 1).  fp32 tensors: every operand is the exact sum of three bf16
// planes x = x1 + x2 + x3 of 8 bits each (dcn_gemm_split writes them), and the product is
//   x1 y1 + (x1 y2 + x2 y1 + x2 y2 + x1 y3 + x3 y1);
// what is left out is below 2^-24 of |x||y|.  A tensor core truncates where it adds to its
// accumulator, so long fp32 sums would drift by 2^-24 a step: the leading product and the five small
// ones have accumulators of their own, and every 256 values of k the epilogue warps take both out
// into registers, where the additions round to nearest.
//
// The weight gradient's sum over the rows is cut into `splits` ranges when its tiles alone do not
// fill the SMs; the fp32 parts are added in order by dcn_gemm_reduce.  Its bias gradient (row sums
// of A) costs one more 128x16 instruction a step: a product with a tile of ones.
#include <atomic>
#include <cstring>
#include <type_traits>

#include <cuda.h>

#include "dcn_gemm.cuh"
#include "dcn_ptx.cuh"

namespace dcn {

namespace {

// Epilogue warps: four to each quarter of the accumulator's rows, two where three planes take the shared
// memory that their staging would need.  With them the MMA warp and the loader warp.
template <int PL>
constexpr int kEpi = PL == 3 ? 8 : 16;
template <int PL>
constexpr int kThreadsOf = (kEpi<PL> + 2) * 32;

// Bytes of a row of an epilogue warp's staging chunk (32 rows): with 16-bit results a warp has 64
// columns of a 256-column tile, else (at least) 32.
template <typename TO, int BN>
constexpr int kChunkRow = sizeof(TO) == 4 || BN == 256 ? 128 : 64;
constexpr int kUnitBlocks = 4;          // PL = 3: 64-value blocks between two drains of the accumulators

__device__ int g_gemm_status;           // the first wait that ran out (0: none), until it is read

struct alignas(64) GemmTc {
  CUtensorMap a, b, out, res, aux;
  GemmArgs g;
  int tiles_m, tiles_n, splits, kb_total, kb_split;
  int stages;
  int out_tma, res_tma;            // 0: element by element
  int bias16;                      // the bias starts on 16 bytes
  long long ldz;                   // row stride of kept pre-activations: a multiple of 8
  float *row_part;                 // [splits][m], with splits > 1
  unsigned long long wait_limit_ns;
};

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
template <int CG>
__device__ __forceinline__ void pair_sync() {
  if constexpr (CG == 2) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}
// The address of the first block's copy of a shared variable, and an arrival there.
template <int CG>
__device__ __forceinline__ uint32_t lead_addr(uint32_t addr) {
  if constexpr (CG == 1) return addr;
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
template <int CG>
__device__ __forceinline__ void lead_arrive(uint32_t addr) {
  if constexpr (CG == 1)
    mbar_arrive(addr);
  else
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
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

struct Item {
  int m0, n0, split, kb0, kb1;
};
// rank: which block of its pair this one is; a pair's tile is 256 rows
__device__ __forceinline__ Item decode(uint32_t item, const GemmTc &p, int BN, int CG, int rank) {
  const uint32_t tiles = (uint32_t)p.tiles_m * (uint32_t)p.tiles_n;
  Item it;
  it.split = (int)(item / tiles);
  const uint32_t t = item - (uint32_t)it.split * tiles;
  const uint32_t tm = t / (uint32_t)p.tiles_n;   // column tiles of one row tile are neighbours: A stays in L2
  it.m0 = ((int)tm * CG + rank) * 128;
  it.n0 = (int)(t - tm * (uint32_t)p.tiles_n) * BN;
  it.kb0 = it.split * p.kb_split;
  it.kb1 = min(p.kb_total, it.kb0 + p.kb_split);
  return it;
}

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
template <typename TO>
__device__ __forceinline__ uint4 pack16(const float *v) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(TO) == 4) {
      w[i] = __float_as_uint(v[i]);
    } else if constexpr (std::is_same_v<TO, __nv_bfloat16>) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    } else {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// 32 values from or to a lane's row, q0: the first 16-byte piece
template <typename TO, int RB>
__device__ __forceinline__ void stage_store(uint8_t *chunk, int row, int q0, const float (&v)[32]) {
  constexpr int E = 16 / (int)sizeof(TO);
#pragma unroll
  for (int q = 0; q < 32 / E; ++q)
    *reinterpret_cast<uint4 *>(chunk + chunk_piece<RB>(row, q0 + q)) = pack16<TO>(v + E * q);
}

// v[0..31] += bias[j1 ..]; whole groups of a bias that starts on 16 bytes by 16-byte loads (the same
// address in every lane)
template <typename TO>
__device__ __forceinline__ void add_bias(const TO *bias, long long j1, long long n, bool vec, float (&v)[32]) {
  if (vec && j1 + 32 <= n) {
    constexpr int E = 16 / (int)sizeof(TO);
#pragma unroll
    for (int i = 0; i < 32 / E; ++i) {
      float b[E];
      unpack16<TO>(__ldg(reinterpret_cast<const uint4 *>(bias + j1) + i), b);
#pragma unroll
      for (int k = 0; k < E; ++k) v[E * i + k] += b[k];
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
__device__ __forceinline__ void chunk_in(uint8_t *chunk, const TO *src, long long ld, long long i0, long long m,
                                         long long j0, long long n, int lane) {
  constexpr int P = RB / (int)sizeof(TO) / 32;
  const int rows = (int)min(32LL, m - i0);
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
__device__ __forceinline__ void chunk_out(uint8_t *chunk, TO *dst, long long ld, long long i0, long long m,
                                          long long j0, long long n, int lane) {
  constexpr int P = RB / (int)sizeof(TO) / 32;
  const int rows = (int)min(32LL, m - i0);
  dst += i0 * ld + j0;
#pragma unroll 8
  for (int r = 0; r < rows; ++r)
#pragma unroll
    for (int c = 0; c < P; ++c)
      if (j0 + c * 32 + lane < n) dst[r * ld + c * 32 + lane] = *chunk_at<TO, RB>(chunk, r, c * 32 + lane);
}
// v[0..31] += a lane's own row of the residual, for the rare epilogue whose chunk is taken
template <typename TO>
__device__ __forceinline__ void add_row(const TO *src, long long j1, long long n, float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 32; ++j)
    if (j1 + j < n) v[j] += ElemOf<TO>::to(__ldg(src + j));
}

}  // namespace

// PL planes per operand; TI the 16-bit type of the planes, TO the output's (and residual's) type;
// AMN / BMN: the operand lies with its row index contiguous; CG blocks to a tile.
template <typename TI, typename TO, int PL, int BN, bool AMN, bool BMN, int CG>
__global__ void __launch_bounds__(kThreadsOf<PL>, 1) dcn_gemm_tc(const __grid_constant__ GemmTc p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  constexpr uint32_t kABytes = PL * 16384u, kBBytes = PL * (BN / CG) * 128u, kStage = kABytes + kBBytes;
  constexpr int kEpiWarps = kEpi<PL>, kGemmThreads = kThreadsOf<PL>, kGroups = kEpiWarps / 4;
  constexpr bool kRowSum = AMN && PL == 1;             // only the weight gradient asks for row sums
  constexpr int kBufs = (kRowSum && BN == 256) ? 1 : 2;   // accumulator buffers that fit beside the row sums
  constexpr int kOnes = 16 * CG;   // columns of the product with the tile of ones
  constexpr int kBufCols = PL == 3 ? 2 * BN : BN;
  constexpr int kCols = kBufs * kBufCols + (kRowSum ? kOnes * kBufs : 0);
  constexpr int kAlloc = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static_assert(kCols <= 512, "tensor memory");
  constexpr int RB = kChunkRow<TO, BN>, kChunkBytes = 32 * RB;
  constexpr int CW = RB / (int)sizeof(TO);             // columns of a staging chunk
  constexpr int kWarpCols = BN / kGroups > CW ? BN / kGroups : CW;   // columns of an epilogue warp

  const GemmArgs &g = p.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ST = p.stages;
  const uint32_t bar0 = smem_u32(smem);
  const uint32_t full = bar0, empty = full + 8 * ST, tmem_full = empty + 8 * ST, tmem_empty = tmem_full + 16,
                 in_bar = tmem_empty + 16;             // one per epilogue warp
  uint32_t *tmem_slot = (uint32_t *)(smem + 896);
  volatile int *abort_s = (volatile int *)(smem + 904);
  uint8_t *ring = smem + 1024;
  uint8_t *staging = ring + (size_t)ST * kStage;
  uint8_t *ones = staging + (size_t)kEpiWarps * kChunkBytes;
  const unsigned long long limit = p.wait_limit_ns;

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(tmem_full + 8 * i, 1);
      mbar_init(tmem_empty + 8 * i, CG * kEpiWarps);
    }
    for (int i = 0; i < kEpiWarps; ++i) mbar_init(in_bar + 8 * i, 1);
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
  pair_sync<CG>();
  tc_fence_after();
  pdl_wait();
  pdl_launch();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t items = (uint32_t)p.tiles_m * (uint32_t)p.tiles_n * (uint32_t)p.splits;
  const int rank = CG == 1 ? 0 : (int)(blockIdx.x & 1);   // a cluster is two neighbouring blocks
  const uint32_t first_item = blockIdx.x / CG, item_step = gridDim.x / CG;
  const uint32_t lead_empty = lead_addr<CG>(tmem_empty), lead_full = lead_addr<CG>(full);

  if (warp < kEpiWarps) {
    // ------------------------------ epilogue ------------------------------
    const int q = warp & 3, cg = warp >> 2;
    const uint32_t lane_base = tmem_base + ((uint32_t)(q * 32) << 16);
    uint8_t *chunk = staging + (size_t)warp * kChunkBytes;
    const uint32_t chunk_u = smem_u32(chunk), ib = in_bar + 8 * warp;
    uint32_t iph = 0, unit = 0;
    const long long words = (g.n + 31) / 32;
    const bool aux_in = g.slope_act == DCN_ACT_GELU, aux_out = g.saved && g.act == DCN_ACT_GELU;
    const bool res_staged = g.res && !aux_in && !aux_out;
    const bool load_in = aux_in || (res_staged && p.res_tma);
    bool ok = true;
    for (uint32_t item = first_item; item < items && ok; item += item_step) {
      const Item it = decode(item, p, BN, CG, rank);
      const long long i0 = it.m0 + q * 32, row = i0 + lane;
      const long long jw = it.n0 + cg * kWarpCols;   // this warp's first column
      const int chunks =
          cg * kWarpCols < BN && jw < g.n ? (int)((min(g.n - jw, (long long)kWarpCols) + CW - 1) / CW) : 0;
      // what a chunk takes in, to its own place: asked for as soon as the store of the result that lay
      // there has been read, the first chunk's under the main loop
      auto fetch = [&](long long j0) {
        if (lane == 0) bulk_wait_read();
        __syncwarp();
        if (load_in) {
          if (lane == 0) {
            fence_proxy_async_smem();
            mbar_arrive_expect_tx(ib, kChunkBytes);
            tma_load_3d(chunk_u, aux_in ? &p.aux : &p.res, (int)j0, (int)i0, 0, ib);
          }
        } else if (res_staged) {
          chunk_in<TO, RB>(chunk, (const TO *)g.res, g.ldr, i0, g.m, j0, g.n, lane);
        }
      };
      if (chunks) fetch(jw);
      float facc[PL == 3 ? kWarpCols : 1];
      const int units = PL == 3 ? (it.kb1 - it.kb0 + kUnitBlocks - 1) / kUnitBlocks : 1;
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
                const float v = __uint_as_float(a[j]) + __uint_as_float(b[j]);
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
      if (kRowSum && g.row_sum && it.n0 == 0 && cg == 0) {
        const float v = __uint_as_float(tmem_ld1(lane_base + (uint32_t)(kBufs * kBufCols + kOnes * buf)));
        tmem_ld_wait();
        if (row < g.m) {
          if (p.splits > 1) p.row_part[(long long)it.split * g.m + row] = v;
          else ((TI *)g.row_sum)[row] = ElemOf<TI>::from(v);
        }
      }
      // the 32 sums of a group of columns, with the bias
      auto sums = [&](long long j1, int c, float (&v)[32]) {
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
        if (g.bias) add_bias<TO>((const TO *)g.bias, j1, g.n, p.bias16 != 0, v);
      };
      static_assert(PL == 1 || kWarpCols <= 64, "two groups");
#pragma unroll 1
      for (int ch = 0; ch < chunks; ++ch) {
        const long long j0 = jw + ch * CW;
        if (ch) fetch(j0);
        if (aux_out) {   // the pre-activations leave first, through the same chunk
#pragma unroll 1
          for (int c1 = 0; c1 < CW; c1 += 32) {
            float v[32];
            sums(j0 + c1, ch * CW + c1, v);
            stage_store<TO, RB>(chunk, lane, c1 * (int)sizeof(TO) / 16, v);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(&p.aux, chunk_u, (int)j0, (int)i0, 0);
            bulk_commit();
            bulk_wait_read();
          }
          __syncwarp();
        }
        if (load_in) {
          ok = __all_sync(0xffffffffu, g_wait(ib, iph, abort_s, 8, 2 * limit, 0));
          iph ^= 1u;
          if (!ok) break;
        }
#pragma unroll 1
        for (int c1 = 0; c1 < CW; c1 += 32) {
          const long long j1 = j0 + c1;
          const int q0 = c1 * (int)sizeof(TO) / 16;
          float v[32];
          sums(j1, ch * CW + c1, v);
          if constexpr (PL == 1) {
            if (ch == chunks - 1 && c1 == CW - 32) {   // all read: the next tile may have the accumulator
              tc_fence_before();
              __syncwarp();
              if (lane == 0) lead_arrive<CG>(lead_empty + 8 * buf);
            }
          }
          if (g.act == DCN_ACT_RELU) {
            if (g.saved) {
              uint32_t bits = 0;
#pragma unroll
              for (int j = 0; j < 32; ++j) bits |= relu_bit(v[j]) ? 1u << j : 0u;
              if (row < g.m && j1 < g.n) ((uint32_t *)g.saved)[row * words + (j1 >> 5)] = bits;
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = relu_value(v[j]);
          } else if (g.act == DCN_ACT_GELU) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = gelu_value<PL == 3>(v[j]);
          }
          constexpr int E = 16 / (int)sizeof(TO);
          if (g.slope_act == DCN_ACT_RELU) {
            const uint32_t bits = row < g.m && j1 < g.n ? __ldg((const uint32_t *)g.slope + row * words + (j1 >> 5)) : 0u;
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = (bits >> j) & 1u ? v[j] : 0.f;
          } else if (aux_in) {
#pragma unroll
            for (int k = 0; k < 32 / E; ++k) {
              float z[E];
              unpack16<TO>(*reinterpret_cast<const uint4 *>(chunk + chunk_piece<RB>(lane, q0 + k)), z);
#pragma unroll
              for (int j = 0; j < E; ++j) v[E * k + j] *= gelu_slope<PL == 3>(z[j]);
            }
          }
          if (res_staged) {
#pragma unroll
            for (int k = 0; k < 32 / E; ++k) {
              float r[E];
              unpack16<TO>(*reinterpret_cast<const uint4 *>(chunk + chunk_piece<RB>(lane, q0 + k)), r);
#pragma unroll
              for (int j = 0; j < E; ++j) v[E * k + j] += r[j];
            }
          } else if (g.res && row < g.m) {
            add_row<TO>((const TO *)g.res + row * g.ldr + j1, j1, g.n, v);
          }
          stage_store<TO, RB>(chunk, lane, q0, v);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (!p.out_tma) {
          chunk_out<TO, RB>(chunk, (TO *)g.out, g.n, i0, g.m, j0, g.n, lane);
        } else if (lane == 0) {
          tma_store_3d(&p.out, chunk_u, (int)j0, (int)i0, it.split);
          bulk_commit();
        }
        __syncwarp();
      }
      if constexpr (PL == 1) {
        if (!chunks) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) lead_arrive<CG>(lead_empty + 8 * buf);
        }
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
    for (uint32_t item = first_item; item < items && ok; item += item_step) {
      const Item it = decode(item, p, BN, CG, rank);
      const bool sums = kRowSum && g.row_sum && it.n0 == 0;
      uint32_t d = 0;
      int buf = 0;
      for (int kb = it.kb0; kb < it.kb1; ++kb) {
        const bool first = PL == 3 ? (kb - it.kb0) % kUnitBlocks == 0 : kb == it.kb0;
        const bool last = PL == 3 ? (kb - it.kb0) % kUnitBlocks == kUnitBlocks - 1 || kb == it.kb1 - 1 : kb == it.kb1 - 1;
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
      for (uint32_t item = first_item; item < items && ok; item += item_step) {
        const Item it = decode(item, p, BN, CG, rank);
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          ok = g_wait(empty + 8 * st, ph ^ 1u, abort_s, 7, 2 * limit, 32);
          if (!ok) break;
          // a pair's loads all count on the first block's barrier
          const uint32_t bar = lead_full + 8 * st, sa = smem_u32(ring) + st * kStage, sb = sa + kABytes;
          if (rank == 0) mbar_arrive_expect_tx(full + 8 * st, CG * kStage);
          const int k0 = kb * 64, nb = it.n0 + rank * (BN / CG);
#pragma unroll
          for (int i = 0; i < PL; ++i) {
            if constexpr (AMN) {
#pragma unroll
              for (int j = 0; j < 2; ++j)
                tma_load_3d<CG>(sa + i * 16384u + j * 8192u, &p.a, it.m0 + 64 * j, k0, i, bar);
            } else {
              tma_load_3d<CG>(sa + i * 16384u, &p.a, k0, it.m0, i, bar);
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
  pair_sync<CG>();   // no block leaves while the other may still reach into it
  if (warp == kEpiWarps) {
    tc_fence_after();
    pair_tmem_dealloc<CG>(tmem_base, kAlloc);
  }
}

namespace {

// out[i, j] = sum over the ranges of part [splits][m][ldp], in order; four columns a thread
template <typename T>
__global__ void __launch_bounds__(256) dcn_gemm_reduce(const float *__restrict__ part, int splits, long long m,
                                                       long long n, long long ldp, T *__restrict__ out) {
  const long long per_row = ldp / 4, idx = blockIdx.x * 256LL + threadIdx.x;
  pdl_wait();
  pdl_launch();
  if (idx >= m * per_row) return;
  const long long i = idx / per_row, j = (idx - i * per_row) * 4;
  const float4 *p = reinterpret_cast<const float4 *>(part + i * ldp + j);
  const long long step = m * ldp / 4;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int s = 0; s < splits; ++s) {
    const float4 a = p[s * step];
    v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
  }
  T *o = out + i * n + j;
  if (j < n) o[0] = ElemOf<T>::from(v.x);
  if (j + 1 < n) o[1] = ElemOf<T>::from(v.y);
  if (j + 2 < n) o[2] = ElemOf<T>::from(v.z);
  if (j + 3 < n) o[3] = ElemOf<T>::from(v.w);
}

// out[c] = sum over the parts, 32 of them side by side, joined in a tree
template <typename T>
__global__ void __launch_bounds__(1024) dcn_column_reduce(const float *__restrict__ part, int parts, long long cols, T *out) {
  __shared__ float sm[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long long c = blockIdx.x * 32LL + tx;
  float v = 0.f;
  pdl_wait();
  pdl_launch();
  if (c < cols)
    for (int p = ty; p < parts; p += 32) v += part[p * cols + c];
  sm[ty][tx] = v;
  __syncthreads();
  for (int d = 16; d > 0; d >>= 1) {
    if (ty < d) sm[ty][tx] += sm[ty + d][tx];
    __syncthreads();
  }
  if (ty == 0 && c < cols) out[c] = ElemOf<T>::from(sm[0][tx]);
}

// x = x1 + x2 + x3, 8 bits each (truncated, so that nothing overflows); an infinity or NaN stays in x1
__device__ __forceinline__ void split3(float x, uint32_t (&b)[3]) {
  b[0] = __float_as_uint(x) & 0xffff0000u;
  const float r1 = x - __uint_as_float(b[0]);
  const bool finite = (b[0] & 0x7f800000u) != 0x7f800000u;
  b[1] = finite ? __float_as_uint(r1) & 0xffff0000u : 0u;
  const float r2 = r1 - __uint_as_float(b[1]);
  b[2] = finite ? __float_as_uint(r2) & 0xffff0000u : 0u;
  // a NaN whose payload lies in the low bits must not turn into an infinity
  if (x != x) b[0] |= 0x00400000u;
}

struct StageArgs {
  const void *src, *saved;
  void *dst;
  float *sums;
  long long ld, rows, cols, pitch;
  int act;
  int vec_src;   // rows start on 16 bytes
};

// blockDim.x threads of 8 columns each, blockDim.y rows at a time; blockIdx.y: a slab of rows
template <typename T, int PL>
__global__ void __launch_bounds__(256) dcn_gemm_stage(const StageArgs a) {
  __shared__ float red[256 * 8];
  const long long c = (blockIdx.x * (long long)blockDim.x + threadIdx.x) * 8;
  const long long words = (a.cols + 31) / 32;
  pdl_wait();
  pdl_launch();
  float sum[8] = {};
  if (c < a.pitch) {
    for (long long r = blockIdx.y * (long long)blockDim.y + threadIdx.y; r < a.rows; r += (long long)gridDim.y * blockDim.y) {
      float v[8];
      const T *src = (const T *)a.src + r * a.ld + c;
      if (a.vec_src && c + 8 <= a.cols) {
        if constexpr (sizeof(T) == 4) {
          const float4 lo = *reinterpret_cast<const float4 *>(src), hi = *reinterpret_cast<const float4 *>(src + 4);
          v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
          v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
        } else {
          const uint4 u = *reinterpret_cast<const uint4 *>(src);
          const T *e = reinterpret_cast<const T *>(&u);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = ElemOf<T>::to(e[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < a.cols ? ElemOf<T>::to(src[i]) : 0.f;
      }
      if (a.act == DCN_ACT_RELU) {
        const uint32_t bits = c < a.cols ? ((const uint32_t *)a.saved)[r * words + (c >> 5)] >> (c & 31) : 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (bits >> i) & 1u ? v[i] : 0.f;
      } else if (a.act == DCN_ACT_GELU) {
        const T *z = (const T *)a.saved + r * a.pitch + c;   // kept with the same pitch
        uint4 u[sizeof(T) / 2];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = reinterpret_cast<const uint4 *>(z)[i];
        const T *e = reinterpret_cast<const T *>(u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= gelu_slope<PL == 3>(ElemOf<T>::to(e[i]));
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
          uint32_t lo[3], hi[3];
          split3(v[2 * i], lo);
          split3(v[2 * i + 1], hi);
#pragma unroll
          for (int k = 0; k < 3; ++k) w[k][i] = (lo[k] >> 16) | hi[k];
        }
#pragma unroll
        for (int k = 0; k < 3; ++k)
          *reinterpret_cast<uint4 *>((uint16_t *)a.dst + (k * a.rows + r) * a.pitch + c) =
              make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += v[i];
    }
  }
  if (!a.sums) return;
  // the block's rows in order, one row of threads after another
  for (int y = 0; y < (int)blockDim.y; ++y) {
    if ((int)threadIdx.y == y)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float *s = red + threadIdx.x * 8 + i;
        *s = y ? *s + sum[i] : sum[i];
      }
    __syncthreads();
  }
  if (threadIdx.y == 0)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < a.cols) a.sums[blockIdx.y * a.cols + c + i] = red[threadIdx.x * 8 + i];
}

void stage_shape(long long rows, long long pitch, int *tx, int *ty, int *gx, int *gy) {
  int x = 1;
  while (x < 32 && x * 8 < pitch) x *= 2;
  *tx = x;
  *ty = 256 / x;
  *gx = (int)((pitch + x * 8 - 1) / (x * 8));
  const long long want = (rows + *ty - 1) / *ty;
  long long most = 148 * 8 / *gx;
  if (most < 1) most = 1;
  *gy = (int)(want < 1 ? 1 : want < most ? want : most);
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

template <typename TI, typename TO, int PL, int BN, bool AMN, bool BMN, int CG>
cudaError_t run_tc(GemmTc &p, cudaStream_t s) {
  auto kern = dcn_gemm_tc<TI, TO, PL, BN, AMN, BMN, CG>;
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
  constexpr size_t fixed = 1024 + 1024 + (size_t)kEpi<PL> * 32 * kChunkRow<TO, BN> + (AMN && PL == 1 ? 2048 : 0);
  constexpr int stages = (kMost - fixed) / stage > 8 ? 8 : (int)((kMost - fixed) / stage);
  static_assert(stages >= 2, "a ring");
  p.stages = stages;
  const long long items = (long long)p.tiles_m * p.tiles_n * p.splits;
  const int grid = CG * (int)(items < 148 / CG ? items : 148 / CG);
  return launch_pdl(kern, grid, kThreadsOf<PL>, fixed + stages * stage, s, CG, p);
}

template <typename TI, typename TO, int PL, bool AMN, bool BMN>
cudaError_t run_bn(GemmTc &p, int bn, int cg, cudaStream_t s) {
  if constexpr (PL == 1) {
    if (cg == 2) return run_tc<TI, TO, PL, 256, AMN, BMN, 2>(p, s);
    if (bn == 256) return run_tc<TI, TO, PL, 256, AMN, BMN, 1>(p, s);
  } else {
    if (cg == 2) return run_tc<TI, TO, PL, 128, AMN, BMN, 2>(p, s);
  }
  if (bn == 128) return run_tc<TI, TO, PL, 128, AMN, BMN, 1>(p, s);
  return run_tc<TI, TO, PL, 64, AMN, BMN, 1>(p, s);
}

template <typename TI, typename T, int PL>
cudaError_t run_order(GemmTc &p, int bn, int cg, bool parts, cudaStream_t s) {
  const GemmArgs &g = p.g;
  if (!g.a_mn && !g.b_mn) return run_bn<TI, T, PL, false, false>(p, bn, cg, s);
  if (!g.a_mn) return run_bn<TI, T, PL, false, true>(p, bn, cg, s);
  if (parts) return run_bn<TI, float, PL, true, true>(p, bn, cg, s);
  return run_bn<TI, T, PL, true, true>(p, bn, cg, s);
}

template <typename T>
cudaError_t run_reduce(const float *part, const GemmPlan &plan, const GemmArgs &g, cudaStream_t s) {
  const long long n = g.m * (plan.ldp / 4);
  return launch_pdl(dcn_gemm_reduce<T>, (unsigned)((n + 255) / 256), 256, 0, s, 1, part, plan.splits, g.m, g.n, plan.ldp,
                    (T *)g.out);
}

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace

GemmPlan plan_gemm(int planes, long long m, long long n, long long k, bool weight_gradient) {
  GemmPlan p = {};
  const int wide = planes == 1 ? 256 : 128;
  auto tiles = [&](int rows, int bn) { return (m + rows - 1) / rows * ((n + bn - 1) / bn); };
  p.kb_total = (int)((k + 63) / 64);
  p.splits = 1;
  p.cg = 1;
  if (weight_gradient) {
    p.bn = n > wide / 2 ? wide : n > 64 ? 128 : 64;
    if (m > 128 && p.bn == wide) p.cg = 2;
    long long splits = 148 / p.cg / tiles(128 * p.cg, p.bn);
    if (splits > p.kb_total / 4) splits = p.kb_total / 4;
    if (splits < 1) splits = 1;
    p.kb_split = (int)((p.kb_total + splits - 1) / splits);
    p.splits = (p.kb_total + p.kb_split - 1) / p.kb_split;
  } else {
    if (n > wide / 2 && tiles(256, wide) >= 74) {
      p.bn = wide;
      p.cg = 2;
    } else {
      p.bn = n > wide / 2 && tiles(128, wide) >= 148 ? wide : n > 64 && tiles(128, 128) >= 148 ? 128 : 64;
    }
    p.kb_split = p.kb_total;
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
  const int planes = dtype == DCN_DTYPE_F32 ? 3 : 1, esize = dtype == DCN_DTYPE_F32 ? 4 : 2;
  const bool parts = plan.splits > 1;
  const CUtensorMapDataType t16 = dtype == DCN_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapDataType tio = dtype == DCN_DTYPE_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : t16;
  p.tiles_m = (int)((g.m + 128 * plan.cg - 1) / (128 * plan.cg));
  p.tiles_n = (int)((g.n + plan.bn - 1) / plan.bn);
  p.splits = plan.splits;
  p.kb_total = plan.kb_total;
  p.kb_split = plan.kb_split;
  p.row_part = row_part;
  p.wait_limit_ns = kWaitLimitNs;
  p.bias16 = aligned16(g.bias);
  bool ok = g.a_mn ? encode3(&p.a, t16, 2, g.a, g.m, g.kk, planes, g.lda, 64, 64)
                   : encode3(&p.a, t16, 2, g.a, g.kk, g.m, planes, g.lda, 64, 128);
  ok = ok && (g.b_mn ? encode3(&p.b, t16, 2, g.b, g.n, g.kk, planes, g.ldb, 64, 64)
                     : encode3(&p.b, t16, 2, g.b, g.kk, g.n, planes, g.ldb, 64, plan.bn / plan.cg));
  const bool rows16 = g.n * esize % 16 == 0;
  const unsigned cw = esize == 4 || plan.bn < 256 ? 32 : 64;   // kChunkRow
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
  if (dtype == DCN_DTYPE_F32) e = run_order<__nv_bfloat16, float, 3>(p, plan.bn, plan.cg, parts, s);
  else if (dtype == DCN_DTYPE_BF16) e = run_order<__nv_bfloat16, __nv_bfloat16, 1>(p, plan.bn, plan.cg, parts, s);
  else e = run_order<__half, __half, 1>(p, plan.bn, plan.cg, parts, s);
  if (e != cudaSuccess || !parts) return e;
  if (dtype == DCN_DTYPE_F32) e = run_reduce<float>(part, plan, g, s);
  else if (dtype == DCN_DTYPE_BF16) e = run_reduce<__nv_bfloat16>(part, plan, g, s);
  else e = run_reduce<__half>(part, plan, g, s);
  if (e == cudaSuccess && g.row_sum) e = launch_column_reduce(row_part, plan.splits, g.m, dtype, g.row_sum, s);
  return e;
}

int stage_slabs(long long rows, long long cols) {
  int tx, ty, gx, gy;
  stage_shape(rows, (cols + 7) / 8 * 8, &tx, &ty, &gx, &gy);
  return gy;
}

cudaError_t launch_gemm_stage(const void *src, long long ld, const void *saved, int act, long long rows,
                              long long cols, int dtype, void *planes, long long pitch, float *sums, int *slabs,
                              cudaStream_t s) {
  StageArgs a = {};
  a.src = src; a.saved = saved; a.dst = planes; a.sums = sums;
  a.ld = ld; a.rows = rows; a.cols = cols; a.pitch = pitch; a.act = act;
  const int esize = dtype == DCN_DTYPE_F32 ? 4 : 2;
  a.vec_src = aligned16(src) && ld * esize % 16 == 0;
  int tx, ty, gx, gy;
  stage_shape(rows, pitch, &tx, &ty, &gx, &gy);
  if (slabs) *slabs = gy;
  const dim3 grid(gx, gy), block(tx, ty);
  if (dtype == DCN_DTYPE_F32) return launch_pdl(dcn_gemm_stage<float, 3>, grid, block, 0, s, 1, a);
  if (dtype == DCN_DTYPE_BF16) return launch_pdl(dcn_gemm_stage<__nv_bfloat16, 1>, grid, block, 0, s, 1, a);
  return launch_pdl(dcn_gemm_stage<__half, 1>, grid, block, 0, s, 1, a);
}

cudaError_t launch_column_reduce(const float *part, int parts, long long cols, int dtype, void *out, cudaStream_t s) {
  const unsigned grid = (unsigned)((cols + 31) / 32);
  if (dtype == DCN_DTYPE_F32) return launch_pdl(dcn_column_reduce<float>, grid, 1024, 0, s, 1, part, parts, cols, (float *)out);
  if (dtype == DCN_DTYPE_BF16)
    return launch_pdl(dcn_column_reduce<__nv_bfloat16>, grid, 1024, 0, s, 1, part, parts, cols, (__nv_bfloat16 *)out);
  return launch_pdl(dcn_column_reduce<__half>, grid, 1024, 0, s, 1, part, parts, cols, (__half *)out);
}

// Reads and clears the status word of the current device, after the work on `s`.
cudaError_t read_gemm_status(cudaStream_t s, int *status) {
  int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(status, g_gemm_status, sizeof(int), 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaMemcpyToSymbolAsync(g_gemm_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  return e;
}

}  // namespace dcn
