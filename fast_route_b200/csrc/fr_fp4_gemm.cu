// c[m, n] = alpha * sum_k a[m, k] b[n, k] of two 4-bit block-scaled matrices (fr_fp4.cu) on the tensor cores:
// tcgen05.mma kind::mxf4nvf4 (E4M3 scales per 16) / kind::mxf4 (E8M0 scales per 32), fp32 accumulators in tensor memory.
//
// A CTA computes a tile of 128 "lane" rows by BN "column" rows.  For more than 128 tokens the tokens are the lane rows
// and BN = 256 weight rows; up to 128 tokens the weights are the lane rows and the tokens fill BN = 32 or 128 columns,
// so that the tensor core does not multiply padding and the stages hold weights.
//
//   warp 0       TMA producer: 128 bytes (256 codes) of every row per stage, 128-byte swizzle
//   warp 1       MMA issuer: copies the stage's scales from shared to tensor memory (tcgen05.cp), four MMAs of K = 64
//   warps 2-5    scale loaders: the scales lie row by row in global memory; cp.async puts each 4-byte group where the
//                hardware wants it (32 rows x 4 row groups x 4 bytes = one 512-byte block per 128 rows)
//   warps 6-13   epilogue: each takes 32 lanes and half the columns
//
// Every stage has its own columns in tensor memory for its scales, so a copy never overwrites scales that an MMA in
// flight may still read: the stage is refilled only after its MMAs have completed.
// Few tiles (small m * n): a cluster of up to eight CTAs splits K, the fp32 partial tiles meet in distributed shared
// memory and are added in rank order, so the result does not depend on timing.
#include <cooperative_groups.h>

#include "fr_common.cuh"

namespace fr {

constexpr int FG_THREADS = 14 * 32;
constexpr int FG_LANES = 128;
constexpr int FG_KSTAGE = 256;          // codes of K per stage: 128 bytes of a row

template <int BN, int BLOCK>
struct FgCfg {
  static constexpr int STAGES = BN == 256 ? 4 : (BN == 128 ? 6 : 8);
  static constexpr int A_BYTES = FG_LANES * 128;
  static constexpr int B_BYTES = BN * 128;
  static constexpr int SBLK = 512 * (BLOCK == 16 ? 4 : 2);             // scale bytes of 128 rows per stage
  static constexpr int BGRP = (BN + 127) / 128;                        // 128-row groups of the column side
  static constexpr int SF_BYTES = SBLK * (1 + BGRP);
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SF_BYTES;
  static constexpr int PIPE_BYTES = STAGES * STAGE_BYTES;
  static constexpr int SMEM = PIPE_BYTES + 1024 /* alignment */ + 512 /* barriers */;
  // tensor memory: the accumulator, then per stage 4 columns per scale block of the lane side and of each column group
  static constexpr int SFA_COLS = SBLK / 128;                          // 16 or 8
  static constexpr int SF_COLS = SFA_COLS * (1 + BGRP);
  static constexpr int TMEM_COLS = 512;
  static_assert(BN + STAGES * SF_COLS <= TMEM_COLS, "tensor memory");
  static_assert(SMEM <= 227 * 1024, "shared memory");
  static_assert(STAGE_BYTES % 1024 == 0, "swizzled tiles start on 1024-byte boundaries");
};

struct FgParams {
  int64_t rows_a, rows_b;        // lane rows, column rows
  const uint8_t *sa, *sb;        // scales, row pitch `spitch` bytes
  int spitch;
  int kstages;                   // stages along K
  int split;                     // CTAs of a cluster that share a tile (1 = persistent CTAs, no cluster)
  int tiles_a, tiles_b;
  const float *ga, *gb;          // global scales or null
  uint16_t* c;
  int64_t ldc;
  int swapped;                   // lane rows are weights: c[column row][lane row]
  int vec;                       // 16-byte stores are possible (not swapped)
};

// tcgen05.mma with block scales; the scale vectors are read from tensor memory
template <int BLOCK>
__device__ __forceinline__ void tc_mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                           uint32_t accumulate) {
  if constexpr (BLOCK == 16)
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n"
        "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n"
        "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
// 32 rows x 16 bytes from shared memory to 4 columns of tensor memory, repeated in the four lane quarters
__device__ __forceinline__ void tc_cp_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// descriptor of such a 512-byte block: no swizzle, groups of 8 rows (128 bytes) adjacent
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(128 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  return d;
}
// Instruction descriptor of the block-scaled kinds: A and B E2M1 (format 1), both K-major, dense, K = 64; scale type
// E4M3 (0) or E8M0 (1); which of the four scale bytes of a column a 2X instruction starts at (0 or 2), for A and B.
template <int BLOCK>
__device__ __forceinline__ uint32_t fp4_idesc(int n, uint32_t sf_id) {
  return (sf_id << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         ((BLOCK == 32 ? 1u : 0u) << 23) | (static_cast<uint32_t>(FG_LANES >> 7) << 27) | (sf_id << 29);
}

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t size) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
}

template <int BN, int BLOCK, bool BF16>
__global__ void __launch_bounds__(FG_THREADS, 1)
fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const FgParams p) {
  using C = FgCfg<BN, BLOCK>;
  constexpr int S = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::PIPE_BYTES);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1 + 4);         // the TMA producer and the four loader warps
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
    mbar_init(tempty, 8);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // tiles of this CTA (or of its cluster) and its share of K
  const int rank = p.split > 1 ? static_cast<int>(blockIdx.x % p.split) : 0;
  const int first = static_cast<int>(blockIdx.x) / p.split, stride = static_cast<int>(gridDim.x) / p.split;
  const int tiles = p.tiles_a * p.tiles_b;
  const int k0 = static_cast<int>(static_cast<int64_t>(p.kstages) * rank / p.split);
  const int k1 = static_cast<int>(static_cast<int64_t>(p.kstages) * (rank + 1) / p.split);

  if (warp == 0) {
    // ------------------------------ TMA producer ------------------------------
    if (lane == 0) {
      PipeState ps;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += stride) {
        const int ra = (tile % p.tiles_a) * FG_LANES, rbb = (tile / p.tiles_a) * BN;
        for (int k = k0; k < k1; ++k) {
          if (!wait_or_abort(&empty[ps.stage], ps.phase ^ 1, abort_flag, 0x700)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + ps.stage * C::STAGE_BYTES;
          mbar_expect_tx(&full[ps.stage], C::A_BYTES + C::B_BYTES);
          tma_load_2d(st, &tmA, &full[ps.stage], k * 128, ra);
          tma_load_2d(st + C::A_BYTES, &tmB, &full[ps.stage], k * 128, rbb);
          ps.advance_rt(S);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------ MMA issuer --------------------------------
    if (lane == 0) {
      PipeState ps;
      uint32_t it = 0;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += stride, ++it) {
        if (!wait_or_abort(tempty, (it & 1u) ^ 1, abort_flag, 0x701)) break;
        tc_fence_after();
        for (int k = k0; k < k1; ++k) {
          if (!wait_or_abort(&full[ps.stage], ps.phase, abort_flag, 0x702)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t st = smem_u32(smem + ps.stage * C::STAGE_BYTES);
          const uint32_t sf = st + C::A_BYTES + C::B_BYTES;
          const uint32_t tsf = tmem + BN + ps.stage * C::SF_COLS;
          constexpr int NB = C::SBLK / 512;      // 512-byte scale blocks per 128 rows: 4 (block 16) or 2 (block 32)
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            tc_cp_scales(tsf + 4 * j, scale_desc(sf + j * 512));
#pragma unroll
            for (int h = 0; h < C::BGRP; ++h)    // the column side's groups of one K step lie side by side
              tc_cp_scales(tsf + C::SFA_COLS + 4 * (j * C::BGRP + h), scale_desc(sf + C::SBLK * (1 + h) + j * 512));
          }
          const uint64_t ad = umma_desc_sw128(st), bd = umma_desc_sw128(st + C::A_BYTES);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int blk = BLOCK == 16 ? j : j >> 1;
            const uint32_t id = BLOCK == 16 ? 0u : static_cast<uint32_t>(j & 1) * 2u;
            tc_mma_fp4<BLOCK>(tmem, ad + 2 * j, bd + 2 * j, fp4_idesc<BLOCK>(BN, id), tsf + 4 * blk,
                              tsf + C::SFA_COLS + 4 * blk * C::BGRP, (k > k0 || j > 0) ? 1u : 0u);
          }
          tc_commit(&empty[ps.stage]);
          ps.advance_rt(S);
        }
        if (ok) tc_commit(tfull);
      }
    }
  } else if (warp < 6) {
    // ------------------------------ scale loaders -----------------------------
    // Thread r copies the scales of lane row r and of column rows r (and 128 + r).  The copies of two stages are in
    // flight behind the one being handed over.
    constexpr int LOOK = 2, SB = FG_KSTAGE / BLOCK, W = SB / 4;
    const int r = (warp - 2) * 32 + lane;
    const bool aligned = (p.spitch & 3) == 0 && ((reinterpret_cast<uintptr_t>(p.sa) | reinterpret_cast<uintptr_t>(p.sb)) & 3) == 0;
    const uint32_t spot = (r & 31) * 16 + (r >> 5) * 4;
    PipeState ps, done;
    int pending = 0;
    bool ok = true;
    auto hand_over = [&]() {       // the oldest pending stage has arrived: make it visible to the tensor core
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[done.stage]);
      done.advance_rt(S);
      --pending;
    };
    auto copy_row = [&](uint32_t dst, const uint8_t* base, int64_t row, int64_t rows, int kb) {
      const int left = p.spitch - kb;        // bytes of the row from kb on; past the end and past the rows: zeros
      const uint8_t* src = base + (row < rows ? row : 0) * p.spitch;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int n = row < rows ? min(max(left - 4 * w, 0), 4) : 0;
        if (aligned) {
          cp_async4(dst + w * 512, n > 0 ? src + kb + 4 * w : base, static_cast<uint32_t>(n));
        } else {
          uint32_t v = 0;
          for (int i = 0; i < n; ++i) v |= static_cast<uint32_t>(__ldg(src + kb + 4 * w + i)) << (8 * i);
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst + w * 512), "r"(v) : "memory");
        }
      }
    };
    for (int tile = first; tile < tiles && ok; tile += stride) {
      const int64_t ra = static_cast<int64_t>(tile % p.tiles_a) * FG_LANES + r;
      const int64_t rbb = static_cast<int64_t>(tile / p.tiles_a) * BN + r;
      for (int k = k0; k < k1; ++k) {
        if (!wait_or_abort(&empty[ps.stage], ps.phase ^ 1, abort_flag, 0x703)) {
          ok = false;
          break;
        }
        const uint32_t sf = smem_u32(smem + ps.stage * C::STAGE_BYTES) + C::A_BYTES + C::B_BYTES + spot;
        copy_row(sf, p.sa, ra, p.rows_a, k * SB);
#pragma unroll
        for (int h = 0; h < C::BGRP; ++h)
          if (BN >= 128 || r < BN) copy_row(sf + C::SBLK * (1 + h), p.sb, rbb + 128 * h, p.rows_b, k * SB);
        cp_async_commit();
        ps.advance_rt(S);
        if (++pending > LOOK) {
          cp_async_wait<LOOK>();
          hand_over();
        }
      }
    }
    cp_async_wait<0>();
    while (pending > 0) hand_over();
  } else {
    // ------------------------------ epilogue ----------------------------------
    const int q = warp & 3, half = (warp - 6) >> 2;       // lanes 32q .. 32q+31, columns of this half
    constexpr int HC = BN / 2 < 16 ? 16 : BN / 2;
    const float alpha = (p.ga ? __ldg(p.ga) : 1.0f) * (p.gb ? __ldg(p.gb) : 1.0f);
    uint32_t it = 0;
    for (int tile = first; tile < tiles; tile += stride, ++it) {
      const int64_t ra = static_cast<int64_t>(tile % p.tiles_a) * FG_LANES + q * 32 + lane;
      const int64_t rbb = static_cast<int64_t>(tile / p.tiles_a) * BN + half * HC;
      const bool got = wait_or_abort(tfull, it & 1u, abort_flag, 0x704);
      __syncwarp();
      if (!__all_sync(0xffffffffu, got)) break;
      tc_fence_after();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + half * HC;
      if (p.split > 1) {
        // park the partial tile, columns outermost, in the pipeline's memory: every MMA of this CTA has completed
        float* part = reinterpret_cast<float*>(smem);
#pragma unroll 1
        for (int c0 = 0; c0 < HC; c0 += 16) {
          uint32_t v[16];
          tmem_ld16(taddr + c0, v);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) part[(half * HC + c0 + i) * FG_LANES + q * 32 + lane] = __uint_as_float(v[i]);
        }
        break;                                             // one tile per cluster
      }
      // the accumulator goes to registers as 16-bit pairs first, so the next tile's MMAs wait for the reads only
      uint32_t pk[HC / 2];
#pragma unroll
      for (int c0 = 0; c0 < HC; c0 += 16) {
        uint32_t v[16];
        tmem_ld16(taddr + c0, v);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          pk[c0 / 2 + i] = pack2<BF16>(__uint_as_float(v[2 * i]) * alpha, __uint_as_float(v[2 * i + 1]) * alpha);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty);
      if (ra < p.rows_a) {
        if (p.swapped) {
          uint16_t* o = p.c + rbb * p.ldc + ra;
#pragma unroll
          for (int i = 0; i < HC; ++i)
            if (rbb + i < p.rows_b) o[static_cast<int64_t>(i) * p.ldc] = static_cast<uint16_t>(pk[i / 2] >> (16 * (i & 1)));
        } else {
          uint16_t* o = p.c + ra * p.ldc + rbb;
#pragma unroll
          for (int i = 0; i < HC; i += 8) {
            if (p.vec && rbb + i + 8 <= p.rows_b) {
              *reinterpret_cast<uint4*>(o + i) = make_uint4(pk[i / 2], pk[i / 2 + 1], pk[i / 2 + 2], pk[i / 2 + 3]);
            } else {
#pragma unroll
              for (int u = 0; u < 8; ++u)
                if (rbb + i + u < p.rows_b) o[i + u] = static_cast<uint16_t>(pk[(i + u) / 2] >> (16 * (u & 1)));
            }
          }
        }
      }
    }
  }

  if (p.split > 1) {
    // every CTA of the cluster adds a slice of the tile's columns over all ranks, in rank order
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    __syncwarp();
    cluster.sync();
    const bool ok = *abort_flag == 0;
    const float alpha = (p.ga ? __ldg(p.ga) : 1.0f) * (p.gb ? __ldg(p.gb) : 1.0f);
    const int c_lo = BN * rank / p.split, c_hi = BN * (rank + 1) / p.split;
    const int64_t ra0 = static_cast<int64_t>(first % p.tiles_a) * FG_LANES;
    const int64_t rb0 = static_cast<int64_t>(first / p.tiles_a) * BN;
    const float* parts[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) parts[s] = cluster.map_shared_rank(reinterpret_cast<float*>(smem), s < p.split ? s : 0);
    for (int i = threadIdx.x; ok && i < (c_hi - c_lo) * FG_LANES; i += FG_THREADS) {
      int cc, rr;
      if (p.swapped) cc = c_lo + i / FG_LANES, rr = i % FG_LANES;          // stores run along the lane rows
      else rr = i / (c_hi - c_lo), cc = c_lo + i % (c_hi - c_lo);          // stores run along the columns
      if (ra0 + rr >= p.rows_a || rb0 + cc >= p.rows_b) continue;
      float v = 0.0f;
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (s < p.split) v += parts[s][cc * FG_LANES + rr];
      const uint16_t r16 = static_cast<uint16_t>(pack2<BF16>(v * alpha, 0.0f));
      if (p.swapped) p.c[(rb0 + cc) * p.ldc + ra0 + rr] = r16;
      else p.c[(ra0 + rr) * p.ldc + rb0 + cc] = r16;
    }
    cluster.sync();                                          // nobody leaves while its memory is being read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

template <int BN, int BLOCK, bool BF16>
static int launch_fp4_gemm(const CUtensorMap& a, const CUtensorMap& b, const FgParams& p, int grid, cudaStream_t st) {
  auto kern = fp4_gemm_kernel<BN, BLOCK, BF16>;
  constexpr int smem = FgCfg<BN, BLOCK>::SMEM;
  FR_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(FG_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.split > 1 ? 1 : 0;
  FR_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, a, b, p));
  return FR_OK;
}

template <int BN>
static int launch_fp4_bn(const CUtensorMap& a, const CUtensorMap& b, const FgParams& p, int block, bool bf, int grid,
                         cudaStream_t st) {
  if (block == 16)
    return bf ? launch_fp4_gemm<BN, 16, true>(a, b, p, grid, st) : launch_fp4_gemm<BN, 16, false>(a, b, p, grid, st);
  return bf ? launch_fp4_gemm<BN, 32, true>(a, b, p, grid, st) : launch_fp4_gemm<BN, 32, false>(a, b, p, grid, st);
}

int fp4_gemm_dispatch(const void* a_q, const void* a_scale, const float* a_global, const void* b_q, const void* b_scale,
                      const float* b_global, int block, int64_t m, int64_t n, int64_t k, int dtype, void* c, int64_t ldc,
                      cudaStream_t st) {
  if (m < 0 || n < 0 || k <= 0 || (block != 16 && block != 32) || ldc < n) return FR_ERR_ARG;
  if (dtype != FR_F16 && dtype != FR_BF16) return FR_ERR_UNSUPPORTED;
  if (k % 32 || k > (int64_t(1) << 28) || m > (int64_t(1) << 31) - 256 || n > (int64_t(1) << 31) - 256)
    return FR_ERR_UNSUPPORTED;
  if (m == 0 || n == 0) return FR_OK;
  if (!a_q || !a_scale || !b_q || !b_scale || !c) return FR_ERR_ARG;
  if (((reinterpret_cast<uintptr_t>(a_q) | reinterpret_cast<uintptr_t>(b_q)) & 15) || (reinterpret_cast<uintptr_t>(c) & 1))
    return FR_ERR_ALIGN;
  // tokens (m) on the column side while they fit into one tile of at most 128 columns
  const bool swapped = m <= 128;
  const int bn = swapped ? (m <= 32 ? 32 : 128) : 256;
  FgParams p;
  p.rows_a = swapped ? n : m;
  p.rows_b = swapped ? m : n;
  p.sa = static_cast<const uint8_t*>(swapped ? b_scale : a_scale);
  p.sb = static_cast<const uint8_t*>(swapped ? a_scale : b_scale);
  p.spitch = static_cast<int>(k / block);
  p.kstages = static_cast<int>((k + FG_KSTAGE - 1) / FG_KSTAGE);
  const int64_t ta = (p.rows_a + FG_LANES - 1) / FG_LANES, tb = (p.rows_b + bn - 1) / bn;
  if (ta * tb > (int64_t(1) << 30)) return FR_ERR_UNSUPPORTED;
  p.tiles_a = static_cast<int>(ta);
  p.tiles_b = static_cast<int>(tb);
  p.ga = a_global;
  p.gb = b_global;
  p.c = static_cast<uint16_t*>(c);
  p.ldc = ldc;
  p.swapped = swapped;
  p.vec = !swapped && ldc % 8 == 0 && !(reinterpret_cast<uintptr_t>(c) & 15);
  // split K while the tiles leave at least half of the SMs idle and every CTA keeps a stage
  const DeviceInfo& di = device_info();
  const int64_t tiles = ta * tb;
  int split = 1;
  while (split < 8 && tiles * split * 2 <= di.sm_count && split * 2 <= p.kstages) split *= 2;
  p.split = split;
  const int grid = split > 1 ? static_cast<int>(tiles * split) : static_cast<int>(tiles < di.sm_count ? tiles : di.sm_count);
  CUtensorMap ma, mb;
  const uint64_t kb = static_cast<uint64_t>(k / 2);
  int rc = make_tmap_2d(&ma, swapped ? b_q : a_q, p.rows_a, kb, kb, FG_LANES, 128, true, 1);
  if (rc) return rc;
  rc = make_tmap_2d(&mb, swapped ? a_q : b_q, p.rows_b, kb, kb, bn, 128, true, 1);
  if (rc) return rc;
  const bool bf = dtype == FR_BF16;
  switch (bn) {
    case 32: return launch_fp4_bn<32>(ma, mb, p, block, bf, grid, st);
    case 128: return launch_fp4_bn<128>(ma, mb, p, block, bf, grid, st);
    default: return launch_fp4_bn<256>(ma, mb, p, block, bf, grid, st);
  }
}

}  // namespace fr
