// c[m, n] = alpha * sum_k a[m, k] b[n, k] of two 4-bit block-scaled matrices (fr_fp4.cu) on the tensor cores:
// tcgen05.mma kind::mxf4nvf4 (E4M3 scales per 16) / kind::mxf4 (E8M0 scales per 32), fp32 accumulators in tensor memory.
//
// A CTA computes a tile of 128 "lane" rows by BN "column" rows.  For more than 128 tokens the tokens are the lane rows
// and BN = 256 weight rows; up to 128 tokens the weights are the lane rows and the tokens fill BN = 32 or 128 columns,
// so that the tensor core does not multiply padding and the stages hold weights.
//
//   warp 0       TMA producer: 128 bytes (256 codes) of every row per stage, 128-byte swizzle
//   warp 1       MMA issuer: copies the stage's scales from shared to tensor memory (tcgen05.cp), four MMAs of K = 64
//   epilogue     eight warps, each takes 32 lanes and half the columns
//
// The scales lie row by row in global memory; the hardware wants, for 128 rows, 512-byte blocks of 32 rows x 4 row
// groups x 4 bytes.  For more than 128 tokens a small kernel lays them out that way in the workspace first (6 MB for
// 8192 x 14336 x 4096) and the producer fetches 2 KB blocks: loading them row by row inside the product asks for 4 bytes
// of 32 different lines per instruction (684 us instead of 300).  Up to 128 tokens four loader warps do just that with
// cp.async: the second launch costs as much as it saves (128 x 14336 x 4096: 25 us either way, 17 of them the product
// when the scales are laid out; 100 x 4096 x 4096: 13.6 against 16.8).
//
// Every stage has its own columns in tensor memory for its scales, so a copy never overwrites scales that an MMA in
// flight may still read: the stage is refilled only after its MMAs have completed.
// Few tiles (small m * n): a cluster of up to eight CTAs splits K, the fp32 partial tiles meet in distributed shared
// memory and are added in rank order, so the result does not depend on timing.
#include <cooperative_groups.h>

#include "fr_common.cuh"

namespace fr {

constexpr int FG_LANES = 128;
constexpr int FG_KSTAGE = 256;          // codes of K per stage: 128 bytes of a row

template <int BN, int BLOCK>
struct FgCfg {
  static constexpr bool LAID = BN == 256;                              // scales come laid out from the workspace
  static constexpr int LOADERS = LAID ? 0 : 4;                         // warps that load scales
  // threads that issue MMAs, each for its own share of the columns; with two, a third one issues the scale copies
  static constexpr int ISSUERS = BN == 256 ? 2 : 1;
  static constexpr int EPI0 = 1 + ISSUERS + (ISSUERS > 1 ? 1 : 0) + LOADERS;   // first epilogue warp
  static constexpr int THREADS = 32 * (EPI0 + 8);
  static constexpr int STAGES = BN == 256 ? 4 : (BN == 128 ? 6 : 8);
  static constexpr int A_BYTES = FG_LANES * 128;
  static constexpr int B_BYTES = BN * 128;
  static constexpr int SBLK = 512 * (BLOCK == 16 ? 4 : 2);             // scale bytes of 128 rows per stage
  static constexpr int BGRP = (BN + 127) / 128;                        // 128-row groups of the column side
  static constexpr int SF_BYTES = SBLK * (1 + BGRP);
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SF_BYTES;
  static constexpr int PIPE_BYTES = STAGES * STAGE_BYTES;
  static constexpr int TURN = 32 * 9;                                  // words per epilogue warp: 32 rows x 16 columns
  static constexpr int SMEM = PIPE_BYTES + 1024 /* alignment */ + 512 /* barriers */;
  static constexpr int SMEM_ANY = SMEM + 8 * TURN * 4;
  // tensor memory: the accumulator, then per stage 4 columns per scale block of the lane side and of each column group
  static constexpr int SFA_COLS = SBLK / 128;                          // 16 or 8
  static constexpr int SF_COLS = SFA_COLS * (1 + BGRP);
  static constexpr int TMEM_COLS = 512;
  static_assert(BN + STAGES * SF_COLS <= TMEM_COLS, "tensor memory");
  static_assert((BN < 256 ? SMEM : SMEM_ANY) <= 227 * 1024 && FG_LANES * (BN + 4) * 4 <= PIPE_BYTES, "shared memory");
  static_assert(STAGE_BYTES % 1024 == 0, "swizzled tiles start on 1024-byte boundaries");
};

struct FgParams {
  int64_t rows_a, rows_b;        // lane rows, column rows
  const uint8_t *sa, *sb;        // scales: rows of pitch `spitch` bytes, or laid out [128-row group][stage][block]
  int spitch;
  int kstages;                   // stages along K
  int split;                     // CTAs of a cluster that share a tile (1 = persistent CTAs, no cluster)
  int tiles_a, tiles_b;
  const float *ga, *gb;          // global scales or null
  uint16_t* c;
  int64_t ldc;
  int swapped;                   // lane rows are weights: c[column row][lane row]
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

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t size) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
}

// a stage's scale blocks to tensor memory: NB K steps of 4 columns for the lane side, then for the column side, whose
// 128-row groups lie side by side within a step
template <int BN, int BLOCK>
__device__ __forceinline__ void fg_copy_scales(uint32_t tsf, uint32_t sf) {
  using C = FgCfg<BN, BLOCK>;
  constexpr int NB = C::SBLK / 512;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    tc_cp_scales(tsf + 4 * j, scale_desc(sf + j * 512));
#pragma unroll
    for (int h = 0; h < C::BGRP; ++h)
      tc_cp_scales(tsf + C::SFA_COLS + 4 * (j * C::BGRP + h), scale_desc(sf + C::SBLK * (1 + h) + j * 512));
  }
}

// Where a partial sum waits: the index that runs along a row of c is innermost, so that four of them are read at once.
// (Not swapped: the pitch of BN + 4 floats gives the 16-byte stores of eight lanes, one row each, all 32 banks.)
template <int BN>
__device__ __forceinline__ int fg_park(int swapped, int row, int col) {
  return swapped ? col * FG_LANES + row : row * (BN + 4) + col;
}

// The sums' factor ga * gb.  Where the product of the two leaves fp32's normal range (results need not: two matrices of
// magnitude 1e-18), the second number holds half of its power of two: the first multiplication is then exact to fp32's
// precision, and the second scales.
struct FgAlpha {
  float a, b;
};
__device__ __forceinline__ FgAlpha fg_alpha(const float* ga, const float* gb) {
  const float x = ga ? __ldg(ga) : 1.0f, y = gb ? __ldg(gb) : 1.0f, xy = x * y;
  if (fabsf(xy) >= 1.17549435e-38f && fabsf(xy) <= 3.40282347e38f) return {xy, 1.0f};
  int ex, ey;
  const float m = frexpf(x, &ex) * frexpf(y, &ey);
  // (at most 2^127 in the second: sums are zero or at least 2^-20, so nothing else than zero is finite from 2^255 on)
  const int e = ex + ey, half = e / 2;
  return {ldexpf(m, half), ldexpf(1.0f, min(e - half, 127))};
}

// After a wait that ran out: copies and MMAs that are still in flight end before their memory is given back, each stage's
// last fill and what every issuing thread has issued.  Bounded again, by some milliseconds for what takes microseconds.
// (A stage whose scale loaders gave up never becomes full.)  Not inlined: its registers are none of the kernel's.
static __device__ __noinline__ void fg_drain(uint64_t* full, uint64_t* drained, uint32_t produced, int stages, int issuers) {
  auto wait = [](uint64_t* bar, uint32_t parity) {
    for (uint32_t it = 0; it < (1u << 14); ++it)
      if (mbar_try_wait(bar, parity)) return;
  };
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    const int stage = static_cast<int>(produced & 0xFFu);
    for (int s = 0; s < stages; ++s) wait(full + s, (produced >> 8) ^ (s < stage ? 0u : 1u));
  } else if ((threadIdx.x & 31) == 0 && warp >= 1 && warp <= issuers) {
    tc_commit(drained + warp - 1);
    wait(drained + warp - 1, 0);
  }
  __syncthreads();
}

// ANY: rows of c may start anywhere (not swapped, one CTA per tile); a kernel of its own, for as a branch it costs the
// other case 3 % (registers).
template <int BN, int BLOCK, bool BF16, bool ANY>
__global__ void __launch_bounds__((FgCfg<BN, BLOCK>::THREADS), 1)
fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const FgParams p) {
  using C = FgCfg<BN, BLOCK>;
  constexpr int S = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::PIPE_BYTES);
  uint64_t* empty = full + S;
  uint64_t* sfull = empty + S;            // scales of the stage are in tensor memory (two issuers)
  uint64_t* tfull = sfull + S;
  uint64_t* tempty = tfull + 1;
  uint64_t* drained = tempty + 1;         // of the issuing threads, used after a wait that ran out
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 3);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* produced = tmem_slot + 2;   // where the producer stopped: stage, and its phase in bit 8
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1 + C::LOADERS);   // the TMA producer and the loader warps
      mbar_init(&empty[s], C::ISSUERS);
      mbar_init(&sfull[s], 1);
    }
    mbar_init(tfull, C::ISSUERS);
    mbar_init(tempty, 8);
    for (int w = 0; w < 3; ++w) mbar_init(&drained[w], 1);
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
          mbar_expect_tx(&full[ps.stage], C::A_BYTES + C::B_BYTES + (C::LAID ? C::SF_BYTES : 0));
          tma_load_2d(st, &tmA, &full[ps.stage], k * 128, ra);
          tma_load_2d(st + C::A_BYTES, &tmB, &full[ps.stage], k * 128, rbb);
          if constexpr (C::LAID) {
            uint8_t* sf = st + C::A_BYTES + C::B_BYTES;
            const int64_t ga = static_cast<int64_t>(tile % p.tiles_a) * p.kstages + k;
            bulk_load(sf, p.sa + ga * C::SBLK, C::SBLK, &full[ps.stage]);
#pragma unroll
            for (int h = 0; h < C::BGRP; ++h) {
              const int64_t gb = (static_cast<int64_t>(tile / p.tiles_a) * C::BGRP + h) * p.kstages + k;
              bulk_load(sf + C::SBLK * (1 + h), p.sb + gb * C::SBLK, C::SBLK, &full[ps.stage]);
            }
          }
          ps.advance_rt(S);
        }
      }
      *produced = ps.stage | (ps.phase << 8);
    }
  } else if (warp <= C::ISSUERS) {
    // ------------------------------ MMA issuers -------------------------------
    if (lane == 0) {
      constexpr int NI = BN / C::ISSUERS;        // columns of this issuer: its own accumulators
      const int part = warp - 1;
      PipeState ps;
      uint32_t it = 0;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += stride, ++it) {
        if (!wait_or_abort(tempty, (it & 1u) ^ 1, abort_flag, 0x701)) break;
        tc_fence_after();
        for (int k = k0; k < k1; ++k) {
          if (!wait_or_abort(&full[ps.stage], ps.phase, abort_flag, 0x702) ||
              (C::ISSUERS > 1 && !wait_or_abort(&sfull[ps.stage], ps.phase, abort_flag, 0x705))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t st = smem_u32(smem + ps.stage * C::STAGE_BYTES);
          const uint32_t tsf = tmem + BN + ps.stage * C::SF_COLS;
          if constexpr (C::ISSUERS == 1) fg_copy_scales<BN, BLOCK>(tsf, st + C::A_BYTES + C::B_BYTES);
          const uint64_t ad = umma_desc_sw128(st), bd = umma_desc_sw128(st + C::A_BYTES + part * NI * 128);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int blk = BLOCK == 16 ? j : j >> 1;
            const uint32_t id = BLOCK == 16 ? 0u : static_cast<uint32_t>(j & 1) * 2u;
            tc_mma_fp4<BLOCK>(tmem + part * NI, ad + 2 * j, bd + 2 * j, fp4_idesc<BLOCK>(NI, id), tsf + 4 * blk,
                              tsf + C::SFA_COLS + 4 * (blk * C::BGRP + part), (k > k0 || j > 0) ? 1u : 0u);
          }
          tc_commit(&empty[ps.stage]);
          ps.advance_rt(S);
        }
        if (ok) tc_commit(tfull);
      }
    }
  } else if (C::ISSUERS > 1 && warp == C::ISSUERS + 1) {
    // ------------------------------ scale copies ------------------------------
    if (lane == 0) {
      PipeState ps;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += stride) {
        for (int k = k0; k < k1; ++k) {
          if (!wait_or_abort(&full[ps.stage], ps.phase, abort_flag, 0x706)) {
            ok = false;
            break;
          }
          tc_fence_after();
          fg_copy_scales<BN, BLOCK>(tmem + BN + ps.stage * C::SF_COLS,
                                    smem_u32(smem + ps.stage * C::STAGE_BYTES) + C::A_BYTES + C::B_BYTES);
          tc_commit(&sfull[ps.stage]);
          ps.advance_rt(S);
        }
      }
    }
  } else if (warp < C::EPI0) {
    if constexpr (!C::LAID) {
    // ------------------------------ scale loaders -----------------------------
    // Thread r copies the scales of lane row r and of column row r.  The copies of two stages are in flight behind
    // the one being handed over.
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
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < n) v |= static_cast<uint32_t>(__ldg(src + kb + 4 * w + i)) << (8 * i);
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
    }
  } else {
    // ------------------------------ epilogue ----------------------------------
    const int q = warp & 3, half = (warp - C::EPI0) >> 2;       // lanes 32q .. 32q+31, columns of this half
    constexpr int HC = BN / 2 < 16 ? 16 : BN / 2;
    const FgAlpha alpha = fg_alpha(p.ga, p.gb);
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
        // park the partial tile in the pipeline's memory: every MMA of this CTA has completed
        float* part = reinterpret_cast<float*>(smem);
#pragma unroll 1
        for (int c0 = 0; c0 < HC; c0 += 16) {
          uint32_t v[16];
          tmem_ld16(taddr + c0, v);
          tc_wait_ld();
          if (p.swapped) {
#pragma unroll
            for (int i = 0; i < 16; ++i) part[fg_park<BN>(1, q * 32 + lane, half * HC + c0 + i)] = __uint_as_float(v[i]);
          } else {
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<uint4*>(part + fg_park<BN>(0, q * 32 + lane, half * HC + c0 + i)) =
                  make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          }
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
          pk[c0 / 2 + i] = pack2<BF16>(__uint_as_float(v[2 * i]) * alpha.a * alpha.b, __uint_as_float(v[2 * i + 1]) * alpha.a * alpha.b);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty);
      if constexpr (ANY) {
        // Sixteen columns at a time through shared memory (pitch of nine words: no bank conflicts), so that a store
        // instruction writes 32 bytes of two rows, not two bytes of 32 rows (8192 x 14335 x 256: 188 us, not 1100).
        uint32_t* turn = reinterpret_cast<uint32_t*>(smem + C::PIPE_BYTES + 512) + (warp - C::EPI0) * C::TURN;
        const uint16_t* from = reinterpret_cast<const uint16_t*>(turn) + (lane >> 4) * 18 + (lane & 15);
        const int64_t row = ra - lane + (lane >> 4), col = rbb + (lane & 15);
        uint16_t* o = p.c + row * p.ldc + col;
#pragma unroll
        for (int i = 0; i < HC; i += 16) {
#pragma unroll
          for (int u = 0; u < 8; ++u) turn[lane * 9 + u] = pk[i / 2 + u];
          __syncwarp();
#pragma unroll 4
          for (int r = 0; r < 32; r += 2)
            if (row + r < p.rows_a && col + i < p.rows_b) o[r * p.ldc + i] = from[r * 18];
          __syncwarp();
        }
      } else if (ra < p.rows_a) {
        if (p.swapped) {
          uint16_t* o = p.c + rbb * p.ldc + ra;
#pragma unroll
          for (int i = 0; i < HC; ++i)
            if (rbb + i < p.rows_b) o[static_cast<int64_t>(i) * p.ldc] = static_cast<uint16_t>(pk[i / 2] >> (16 * (i & 1)));
        } else {
          uint16_t* o = p.c + ra * p.ldc + rbb;
#pragma unroll
          for (int i = 0; i < HC; i += 8) {
            if (rbb + i + 8 <= p.rows_b) {
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
    const FgAlpha alpha = fg_alpha(p.ga, p.gb);
    // slices of the tile's columns; BN / split is a multiple of 4
    const int cols = BN / p.split, c_lo = cols * rank;
    const int64_t ra0 = static_cast<int64_t>(first % p.tiles_a) * FG_LANES;
    const int64_t rb0 = static_cast<int64_t>(first / p.tiles_a) * BN;
    const float* parts[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) parts[s] = cluster.map_shared_rank(reinterpret_cast<float*>(smem), s < p.split ? s : 0);
    const bool pairs4 = p.ldc % 4 == 0 && !(reinterpret_cast<uintptr_t>(p.c) & 7);
#pragma unroll 2
    for (int i = threadIdx.x; ok && i < cols * FG_LANES / 4; i += C::THREADS) {
      int cc, rr;                                     // four neighbours along a row of c start here
      if (p.swapped) cc = c_lo + i / (FG_LANES / 4), rr = i % (FG_LANES / 4) * 4;
      else rr = i / (cols / 4), cc = c_lo + i % (cols / 4) * 4;
      const int64_t row = p.swapped ? rb0 + cc : ra0 + rr, col = p.swapped ? ra0 + rr : rb0 + cc;
      const int64_t rows = p.swapped ? p.rows_b : p.rows_a, width = p.swapped ? p.rows_a : p.rows_b;
      if (row >= rows || col >= width) continue;
      const int at = fg_park<BN>(p.swapped, rr, cc);
      float4 f[8];
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (s < p.split) f[s] = *reinterpret_cast<const float4*>(parts[s] + at);
      float4 v = f[0];
#pragma unroll
      for (int s = 1; s < 8; ++s)
        if (s < p.split) v.x += f[s].x, v.y += f[s].y, v.z += f[s].z, v.w += f[s].w;
      const uint32_t lo = pack2<BF16>(v.x * alpha.a * alpha.b, v.y * alpha.a * alpha.b);
      const uint32_t hi = pack2<BF16>(v.z * alpha.a * alpha.b, v.w * alpha.a * alpha.b);
      uint16_t* o = p.c + row * p.ldc + col;
      if (pairs4 && col + 4 <= width) {
        *reinterpret_cast<uint2*>(o) = make_uint2(lo, hi);
      } else {
        const uint16_t e[4] = {static_cast<uint16_t>(lo), static_cast<uint16_t>(lo >> 16), static_cast<uint16_t>(hi),
                               static_cast<uint16_t>(hi >> 16)};
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (col + u < width) o[u] = e[u];
      }
    }
    cluster.sync();                                          // nobody leaves while its memory is being read
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) fg_drain(full, drained, *produced, S, C::ISSUERS + (C::ISSUERS > 1 ? 1 : 0));
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// Scales [rows][spitch] -> [128-row group][stage][block of 512 bytes], zeros past the rows and past K.  One CTA: 128 rows
// and up to four stages (64 or 32 contiguous bytes of a row), turned in shared memory and written out whole.
struct FgLayout {
  const uint8_t *sa, *sb;
  uint8_t *da, *db;
  int64_t rows_a, rows_b;
  int groups_a;          // blockIdx.x below this: the lane side
  int spitch, kstages;
};
template <int BLOCK>
__global__ void __launch_bounds__(128) fp4_scale_layout_kernel(const FgLayout p) {
  constexpr int SB = FG_KSTAGE / BLOCK, W = SB / 4, NS = 4;
  __shared__ uint32_t sm[NS][W * 128];
  const bool lane_side = static_cast<int>(blockIdx.x) < p.groups_a;
  const int group = lane_side ? blockIdx.x : blockIdx.x - p.groups_a;
  const uint8_t* s = lane_side ? p.sa : p.sb;
  const int64_t rows = lane_side ? p.rows_a : p.rows_b, row = static_cast<int64_t>(group) * 128 + threadIdx.x;
  const int k0 = blockIdx.y * NS, ns = min(NS, p.kstages - k0);
  const uint8_t* src = s + row * p.spitch + static_cast<int64_t>(k0) * SB;
  const int left = row < rows ? min(ns * SB, p.spitch - k0 * SB) : 0;
  const bool word = ((p.spitch | static_cast<int>(reinterpret_cast<uintptr_t>(s))) & 3) == 0;
  uint32_t v[NS * W];
#pragma unroll
  for (int i = 0; i < NS * W; ++i) {
    v[i] = 0;
    if (word) {
      if (4 * i < left) v[i] = __ldg(reinterpret_cast<const uint32_t*>(src) + i);
    } else {
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (4 * i + b < left) v[i] |= static_cast<uint32_t>(__ldg(src + 4 * i + b)) << (8 * b);
    }
  }
  const int spot = (threadIdx.x & 31) * 4 + (threadIdx.x >> 5);
#pragma unroll
  for (int i = 0; i < NS * W; ++i) sm[i / W][(i % W) * 128 + spot] = v[i];
  __syncthreads();
  uint4* dst = reinterpret_cast<uint4*>((lane_side ? p.da : p.db) +
                                        (static_cast<int64_t>(group) * p.kstages + k0) * (W * 512));
  const uint4* from = reinterpret_cast<const uint4*>(&sm[0][0]);
  for (int i = threadIdx.x; i < ns * W * 32; i += 128) dst[i] = from[i];
}

template <int BN, int BLOCK, bool BF16, bool ANY>
static int launch_fp4_gemm(const CUtensorMap& a, const CUtensorMap& b, const FgParams& p, int grid, cudaStream_t st) {
  auto kern = fp4_gemm_kernel<BN, BLOCK, BF16, ANY>;
  constexpr int smem = ANY ? FgCfg<BN, BLOCK>::SMEM_ANY : FgCfg<BN, BLOCK>::SMEM;
  FR_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(FgCfg<BN, BLOCK>::THREADS);
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

template <int BN, bool ANY = false>
static int launch_fp4_bn(const CUtensorMap& a, const CUtensorMap& b, const FgParams& p, int block, bool bf, int grid,
                         cudaStream_t st) {
  if (block == 16)
    return bf ? launch_fp4_gemm<BN, 16, true, ANY>(a, b, p, grid, st) : launch_fp4_gemm<BN, 16, false, ANY>(a, b, p, grid, st);
  return bf ? launch_fp4_gemm<BN, 32, true, ANY>(a, b, p, grid, st) : launch_fp4_gemm<BN, 32, false, ANY>(a, b, p, grid, st);
}

// how a product is cut: tokens (m) on the column side while they fit into one tile of at most 128 columns
struct FgPlan {
  bool swapped;
  int bn, kstages, groups_a, groups_b, tiles_a, tiles_b;
  size_t sblk, ws_a, ws_total;
};
static FgPlan fp4_plan(int64_t m, int64_t n, int64_t k, int block) {
  FgPlan q;
  q.swapped = m <= 128;
  q.bn = q.swapped ? (m <= 32 ? 32 : 128) : 256;
  const int64_t ra = q.swapped ? n : m, rb = q.swapped ? m : n;
  q.kstages = static_cast<int>((k + FG_KSTAGE - 1) / FG_KSTAGE);
  q.tiles_a = static_cast<int>((ra + FG_LANES - 1) / FG_LANES);
  q.tiles_b = static_cast<int>((rb + q.bn - 1) / q.bn);
  q.groups_a = q.tiles_a;
  q.groups_b = q.bn < 256 ? 0 : q.tiles_b * (q.bn / 128);       // 0: no layout pass
  q.sblk = block == 16 ? 2048 : 1024;
  q.ws_a = static_cast<size_t>(q.groups_a) * q.kstages * q.sblk;
  q.ws_total = q.groups_b ? q.ws_a + static_cast<size_t>(q.groups_b) * q.kstages * q.sblk : 0;
  return q;
}
static bool fp4_gemm_sizes_ok(int64_t m, int64_t n, int64_t k) {
  constexpr int64_t kMax = int64_t(1) << 30;
  return k % 32 == 0 && k <= (int64_t(1) << 28) && m <= kMax && n <= kMax &&
         ((m + 127) / 128) * ((n + 127) / 128) <= kMax;
}

size_t fp4_gemm_workspace(int64_t m, int64_t n, int64_t k, int block) {
  if (m <= 0 || n <= 0 || k <= 0 || (block != 16 && block != 32) || !fp4_gemm_sizes_ok(m, n, k)) return 0;
  return fp4_plan(m, n, k, block).ws_total;
}

int fp4_gemm_dispatch(const void* a_q, const void* a_scale, const float* a_global, const void* b_q, const void* b_scale,
                      const float* b_global, int block, int64_t m, int64_t n, int64_t k, int dtype, void* c, int64_t ldc,
                      void* workspace, size_t workspace_bytes, cudaStream_t st) {
  if (m < 0 || n < 0 || k <= 0 || (block != 16 && block != 32) || ldc < n) return FR_ERR_ARG;
  if (dtype != FR_F16 && dtype != FR_BF16) return FR_ERR_UNSUPPORTED;
  if (!fp4_gemm_sizes_ok(m, n, k)) return FR_ERR_UNSUPPORTED;
  if (m == 0 || n == 0) return FR_OK;
  if (!a_q || !a_scale || !b_q || !b_scale || !c) return FR_ERR_ARG;
  if (((reinterpret_cast<uintptr_t>(a_q) | reinterpret_cast<uintptr_t>(b_q)) & 15) || (reinterpret_cast<uintptr_t>(c) & 1))
    return FR_ERR_ALIGN;
  const FgPlan q = fp4_plan(m, n, k, block);
  if (q.ws_total && (!workspace || workspace_bytes < q.ws_total)) return FR_ERR_WORKSPACE;
  if (q.ws_total && (reinterpret_cast<uintptr_t>(workspace) & 15)) return FR_ERR_ALIGN;
  FgParams p;
  p.rows_a = q.swapped ? n : m;
  p.rows_b = q.swapped ? m : n;
  p.sa = static_cast<const uint8_t*>(q.swapped ? b_scale : a_scale);
  p.sb = static_cast<const uint8_t*>(q.swapped ? a_scale : b_scale);
  p.spitch = static_cast<int>(k / block);
  p.kstages = q.kstages;
  p.tiles_a = q.tiles_a;
  p.tiles_b = q.tiles_b;
  p.ga = a_global;
  p.gb = b_global;
  p.c = static_cast<uint16_t*>(c);
  p.ldc = ldc;
  p.swapped = q.swapped;
  CUtensorMap ma, mb;
  const uint64_t kb = static_cast<uint64_t>(k / 2);
  int rc = make_tmap_2d(&ma, q.swapped ? b_q : a_q, p.rows_a, kb, kb, FG_LANES, 128, true, 1);
  if (rc) return rc;
  rc = make_tmap_2d(&mb, q.swapped ? a_q : b_q, p.rows_b, kb, kb, q.bn, 128, true, 1);
  if (rc) return rc;
  if (q.groups_b) {
    FgLayout l;
    l.sa = p.sa;
    l.sb = p.sb;
    l.da = static_cast<uint8_t*>(workspace);
    l.db = l.da + q.ws_a;
    l.rows_a = p.rows_a;
    l.rows_b = p.rows_b;
    l.groups_a = q.groups_a;
    l.spitch = p.spitch;
    l.kstages = q.kstages;
    // (at most 65535 x 4 stages of 256: k below 2^26)
    if ((q.kstages + 3) / 4 > 65535) return FR_ERR_UNSUPPORTED;
    const dim3 grid(static_cast<unsigned>(q.groups_a + q.groups_b), static_cast<unsigned>((q.kstages + 3) / 4));
    if (block == 16) fp4_scale_layout_kernel<16><<<grid, 128, 0, st>>>(l);
    else fp4_scale_layout_kernel<32><<<grid, 128, 0, st>>>(l);
    FR_CUDA_OK(cudaGetLastError());
    p.sa = l.da;
    p.sb = l.db;
  }
  // Split K while the tiles leave at least half of the SMs idle, every CTA keeps a stage, and all clusters run at once: a
  // cluster sits in one GPC, so eight CTAs of a whole SM each fit 16 times at most, four 32 times (333 x 1399 x 2080,
  // 18 tiles: 24.8 us with eight, in two waves).
  const DeviceInfo& di = device_info();
  const int64_t tiles = static_cast<int64_t>(q.tiles_a) * q.tiles_b;
  int split = 1;
  while (split < 8 && tiles * split * 2 <= di.sm_count && split * 2 <= p.kstages && tiles * split * 2 <= 128) split *= 2;
  p.split = split;
  const int grid = split > 1 ? static_cast<int>(tiles * split) : static_cast<int>(tiles < di.sm_count ? tiles : di.sm_count);
  const bool bf = dtype == FR_BF16;
  switch (q.bn) {
    case 32: return launch_fp4_bn<32>(ma, mb, p, block, bf, grid, st);
    case 128: return launch_fp4_bn<128>(ma, mb, p, block, bf, grid, st);
    default:     // (a cluster's tile is written by other code)
      return split > 1 || (ldc % 8 == 0 && !(reinterpret_cast<uintptr_t>(c) & 15))
                 ? launch_fp4_bn<256>(ma, mb, p, block, bf, grid, st)
                 : launch_fp4_bn<256, true>(ma, mb, p, block, bf, grid, st);
  }
}

}  // namespace fr
