// The whole MoE layer for at most 16 tokens in ONE cooperative launch: router, top-k, GEMM1 + SiLU * u, GEMM2,
// weighted sum.  A batch this small reads every active expert's weights once and does almost no arithmetic per byte,
// so the kernel is built around that stream:
//
//   logits -> grid barrier -> every CTA ranks all tokens (<= 16 KB of logits from L2) -> h = w1 x, act = silu(h_g) h_u
//          -> grid barrier -> out = sum_e weight * (w2 act)
//
// * Work is split by weight ROWS, not by tiles: the (active experts * I) row pairs of w1 and the H rows of w2 are cut
//   into equal contiguous ranges, so every CTA streams the same number of bytes whatever the sizes (16-row tiles left
//   up to a quarter of the CTAs without a last tile).
// * Each lane owns a FIFO in shared memory that it alone fills (16-byte cp.async) and drains, so the stream needs no
//   barriers and runs on across row tiles, across experts and across the grid barrier: the first weights of w2 are in
//   flight while the last activations are still being written.
// * The products are mma.sync m16n8k16 with the TOKENS on the 16-row side: 8 weight rows by 16 tokens per instruction
//   (a tcgen05 tile would be 128 weight rows, too coarse to split a layer of a few thousand rows over 296 CTAs, and
//   its operand has to pass through shared memory and a barrier).  A lane's 16 bytes are 8 consecutive k of one row;
//   the dot product does not care about the order of k, so both operands use the same permutation of k and no data is
//   moved between lanes.
// * 4-bit experts are expanded in registers: shifting a code's exponent and fraction into place gives the value times
//   a power of two, one multiplication by the block scale gives the exact 16-bit weight (E2M1 * E4M3 has at most six
//   significant bits), so the arithmetic is that of 16-bit weights.
//
// The eight warps of a CTA split K; their partial sums meet in shared memory in warp order, so results do not depend
// on timing.  fp32 accumulation throughout; the activations between the two products are rounded to the 16-bit type.
#include <atomic>

#include "fr_common.cuh"

namespace fr {

constexpr int kDecTokens = FR_DECODE_MAX_TOKENS;   // 16: the row side of the MMA
constexpr int kDecMaxExperts = 256;
constexpr int kDecWarps = 8;
constexpr int kDecThreads = 32 * kDecWarps;
constexpr int kDecStages = 4;
constexpr int kDecStageBytes = 2048;               // per warp: four 16-byte chunks per lane
constexpr int kDecPartStride = 20;                 // floats per weight row of a partial tile: conflict-free stores

enum { WF_16BIT = 0, WF_NV4 = 1, WF_MX4 = 2 };

struct DecodeParams {
  const uint16_t* x;
  const uint16_t* gate;
  int64_t gsh, gse;
  int gate_vec;                  // gate rows are contiguous and 16-byte aligned
  const uint8_t *w1, *w2;        // 16-bit weights or packed codes
  const uint8_t *s1, *s2;        // block scales
  const float *g1, *g2;          // one fp32 scale per expert, or null
  int M, H, I, E, topk, renormalize;
  int tokens_per_unit;           // router: tokens one CTA takes for one expert
  uint16_t* out;
  float* tw;
  int32_t* ti;
  unsigned int* barrier;
  float* logits;                 // [M, E]
  uint16_t* act;                 // [active expert][M][I]
};

struct DecodeSmem {
  uint8_t ring[kDecWarps][kDecStages][kDecStageBytes];
  float part[kDecWarps][32 * kDecPartStride];
  float weight[kDecMaxExperts][kDecTokens];   // routing weight by slot (position in `list`) and token
  uint32_t mask[kDecMaxExperts];              // by expert: bit t = token t goes there
  uint16_t list[kDecMaxExperts];              // active experts in ascending order
  uint32_t scan[kDecWarps];
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Expansion of packed codes.  expand(): the pairs (j, j + 4), j = 0..3, of a word's eight codes as 16-bit numbers
// times kUnit^-1; mult(): the factor for a block.  The fields of E2M1 (bias 1) placed in the low exponent bits and the
// top fraction bit of the 16-bit format are the value times 2^(1 - bias), subnormal 0.5 included.
template <bool BF16, int WF>
struct Fp4Expand {
  // what is left to multiply the sums with: the factors below keep every intermediate inside the 16-bit format
  static constexpr float kUnit = WF == WF_MX4 ? 4294967296.0f /* 2^32 */ : (BF16 ? 65536.0f : 128.0f);
  static __device__ __forceinline__ uint32_t mult(uint32_t byte) {
    if constexpr (WF == WF_MX4) {
      // bf16 only: 2^(byte - 127) * 2^94.  Scales above 2^33 overflow to infinity; far below 2^-60 the products with
      // small activations leave the fp32 range.
      const uint32_t e = byte + 94;
      const uint32_t b = byte == 0xFFu ? 0x7FC0u : (e < 255u ? e << 7 : 0x7F80u);
      return b | (b << 16);
    } else {
      const float s = __fmul_rn(e4m3_f32(byte), BF16 ? 1.298074214633706907e33f /* 2^110 */ : 128.0f);
      return pack2<BF16>(s, s);     // exact: four significant bits
    }
  }
  static __device__ __forceinline__ uint32_t mul(uint32_t a, uint32_t m) {
    uint32_t r;
    if constexpr (BF16) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(m));
    else asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(m));
    return r;
  }
  static __device__ __forceinline__ void expand(uint32_t w, uint32_t m, uint32_t (&o)[4]) {
    constexpr uint32_t S = 0x80008000u;
    constexpr uint32_t F = BF16 ? 0x01C001C0u : 0x0E000E00u;
    if constexpr (BF16) {
      o[0] = ((w << 12) & S) | ((w << 6) & F);
      o[1] = ((w << 8) & S) | ((w << 2) & F);
      o[2] = ((w << 4) & S) | ((w >> 2) & F);
      o[3] = (w & S) | ((w >> 6) & F);
    } else {
      o[0] = ((w << 12) & S) | ((w << 9) & F);
      o[1] = ((w << 8) & S) | ((w << 5) & F);
      o[2] = ((w << 4) & S) | ((w << 1) & F);
      o[3] = (w & S) | ((w >> 3) & F);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = mul(o[j], m);
  }
};

// One token row's operand for the 64 bytes of weights a quad holds: `p` points at the lane's first element.
// 16-bit weights: 8 elements; 4-bit: 32 elements, reordered to the pairs (j, j + 4) that Fp4Expand makes.
template <int WF>
__device__ __forceinline__ void load_tokens(const uint16_t* p, bool valid, bool coherent, uint32_t (&r)[WF == WF_16BIT ? 4 : 16]) {
  constexpr int NV = WF == WF_16BIT ? 1 : 4;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (valid) u = coherent ? __ldcg(reinterpret_cast<const uint4*>(p) + v) : __ldg(reinterpret_cast<const uint4*>(p) + v);
    if constexpr (WF == WF_16BIT) {
      r[0] = u.x, r[1] = u.y, r[2] = u.z, r[3] = u.w;
    } else {
      r[4 * v] = __byte_perm(u.x, u.z, 0x5410);
      r[4 * v + 1] = __byte_perm(u.x, u.z, 0x7632);
      r[4 * v + 2] = __byte_perm(u.y, u.w, 0x5410);
      r[4 * v + 3] = __byte_perm(u.y, u.w, 0x7632);
    }
  }
}

// acc += tokens * weights for one 16-byte chunk per lane
template <bool BF16, int WF>
__device__ __forceinline__ void chunk_mma(float (&acc)[4], const uint4& w, uint32_t scales,
                                          const uint32_t (&lo)[WF == WF_16BIT ? 4 : 16],
                                          const uint32_t (&hi)[WF == WF_16BIT ? 4 : 16]) {
  if constexpr (WF == WF_16BIT) {
    const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
    mma_16816<BF16>(acc, a0, w.x, w.y);
    mma_16816<BF16>(acc, a1, w.z, w.w);
  } else {
    using X = Fp4Expand<BF16, WF>;
    const uint32_t m0 = X::mult(scales & 0xFFu);
    const uint32_t m1 = WF == WF_NV4 ? X::mult(scales >> 8) : m0;   // a lane's 32 codes: two blocks of 16 or one of 32
    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t o[4];
      X::expand(ww[i], i < 2 ? m0 : m1, o);
      const uint32_t a0[4] = {lo[4 * i], hi[4 * i], lo[4 * i + 1], hi[4 * i + 1]};
      const uint32_t a1[4] = {lo[4 * i + 2], hi[4 * i + 2], lo[4 * i + 3], hi[4 * i + 3]};
      mma_16816<BF16>(acc, a0, o[0], o[1]);
      mma_16816<BF16>(acc, a1, o[2], o[3]);
    }
  }
}

// the scale bytes of the 16 bytes of codes at byte offset kb of a row
template <int WF>
__device__ __forceinline__ uint32_t load_scales(const uint8_t* row, int kb, bool valid) {
  if constexpr (WF == WF_16BIT) return 0;
  if (!valid) return 0;
  if constexpr (WF == WF_NV4) return __ldg(reinterpret_cast<const uint16_t*>(row + (kb >> 3)));
  return __ldg(row + (kb >> 4));
}

// ---- router: logits of all (token, expert) pairs, spread over the grid --------------------------------------
template <bool BF16>
__device__ __forceinline__ void decode_logits(const DecodeParams& p, float* red /* [kDecWarps][kDecTokens] */) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tpu = p.tokens_per_unit, groups = (p.M + tpu - 1) / tpu;
  for (int u = blockIdx.x; u < p.E * groups; u += gridDim.x) {
    const int e = u / groups, t0 = (u - e * groups) * tpu;
    const int nt = min(tpu, p.M - t0);
    float acc[kDecTokens];
#pragma unroll
    for (int i = 0; i < kDecTokens; ++i) acc[i] = 0.0f;
    const uint16_t* g = p.gate + static_cast<int64_t>(e) * p.gse;
    for (int h = threadIdx.x * 8; h < p.H; h += kDecThreads * 8) {
      uint32_t gw[4];
      if (p.gate_vec) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(g + h));
        gw[0] = v.x, gw[1] = v.y, gw[2] = v.z, gw[3] = v.w;
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          gw[q] = static_cast<uint32_t>(__ldg(g + (h + 2 * q) * p.gsh)) |
                  (static_cast<uint32_t>(__ldg(g + (h + 2 * q + 1) * p.gsh)) << 16);
      }
#pragma unroll
      for (int i = 0; i < kDecTokens; ++i) {
        if (i < nt) {
          const uint4 v = *reinterpret_cast<const uint4*>(p.x + static_cast<int64_t>(t0 + i) * p.H + h);
          const uint32_t xw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float2 a = unpack2<BF16>(xw[q]), b = unpack2<BF16>(gw[q]);
            acc[i] = fmaf(a.x, b.x, acc[i]);
            acc[i] = fmaf(a.y, b.y, acc[i]);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kDecTokens; ++i) {
      if (i < nt) {
        float v = acc[i];
        for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
        if (lane == 0) red[warp * kDecTokens + i] = v;
      }
    }
    __syncthreads();
    if (threadIdx.x < nt) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) v += red[w * kDecTokens + threadIdx.x];
      if (v != v) v = -INFINITY;       // NaN ranks last, as in the other routers
      p.logits[static_cast<int64_t>(t0 + threadIdx.x) * p.E + e] = v;
    }
    __syncthreads();
  }
}

__device__ __forceinline__ uint32_t order_key(float v) {   // larger value, larger key; -0 and +0 alike; never 0
  const uint32_t u = __float_as_uint(v == 0.0f ? 0.0f : v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Every CTA ranks all tokens: one warp per token, k rounds of arg-max (equal logits: lower expert id), softmax by the
// fixed fp32 recipe of the routers.  `sel` / `val`: [kDecTokens][E] scratch.
__device__ __forceinline__ void decode_rank(const DecodeParams& p, DecodeSmem& sm, uint16_t* sel, float* val) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < p.E; e += kDecThreads) sm.mask[e] = 0;
  __syncthreads();
  for (int t = warp; t < p.M; t += kDecWarps) {
    const float* l = p.logits + static_cast<int64_t>(t) * p.E;
    uint16_t* my_sel = sel + t * p.E;
    float* my_val = val + t * p.E;
    float v[kDecMaxExperts / 32];
    uint32_t key[kDecMaxExperts / 32];
#pragma unroll
    for (int i = 0; i < kDecMaxExperts / 32; ++i) {
      const int c = i * 32 + lane;
      v[i] = c < p.E ? __ldcg(l + c) : 0.0f;
      key[i] = c < p.E ? order_key(v[i]) : 0u;
    }
    for (int j = 0; j < p.topk; ++j) {
      uint32_t best = 0;
      int at = 0;
      float bv = 0.0f;
#pragma unroll
      for (int i = 0; i < kDecMaxExperts / 32; ++i)
        if (key[i] > best) best = key[i], at = i, bv = v[i];
      const uint32_t top = __reduce_max_sync(0xffffffffu, best);
      const uint32_t col = __reduce_min_sync(0xffffffffu, best == top ? static_cast<uint32_t>(at * 32 + lane) : 0xFFFFu);
      if (col == static_cast<uint32_t>(at * 32 + lane)) {
        my_sel[j] = static_cast<uint16_t>(col);
        my_val[j] = bv;
        atomicOr(&sm.mask[col], 1u << t);
#pragma unroll
        for (int i = 0; i < kDecMaxExperts / 32; ++i)
          if (i == at) key[i] = 0;
      }
      __syncwarp();
    }
    const float top = my_val[0];
    float s = 0.0f;
    if (p.renormalize) {
      for (int j = 0; j < p.topk; ++j) {
        const float ej = exp_recipe(__fsub_rn(my_val[j], top));
        s = (j == 0) ? ej : __fadd_rn(s, ej);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kDecMaxExperts / 32; ++i)
        if (i * 32 + lane < p.E) s += exp_recipe(__fsub_rn(v[i], top));
      for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    }
    __syncwarp();
    for (int j = lane; j < p.topk; j += 32) {
      const float w = __fdiv_rn(exp_recipe(__fsub_rn(my_val[j], top)), s);
      my_val[j] = w;
      if (blockIdx.x == 0 && p.tw) {
        p.tw[static_cast<int64_t>(t) * p.topk + j] = w;
        p.ti[static_cast<int64_t>(t) * p.topk + j] = my_sel[j];
      }
    }
  }
  __syncthreads();
  // active experts in ascending order; `scan` holds the warps' counts
  const bool active = threadIdx.x < p.E && sm.mask[threadIdx.x] != 0;
  const uint32_t vote = __ballot_sync(0xffffffffu, active);
  if (lane == 0) sm.scan[warp] = __popc(vote);
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < warp; ++w) before += sm.scan[w];
  const uint32_t slot = before + __popc(vote & ((1u << lane) - 1u));
  // the slot of an expert, in the upper half of its mask word
  if (active) {
    sm.list[slot] = static_cast<uint16_t>(threadIdx.x);
    sm.mask[threadIdx.x] |= slot << 16;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.M * p.topk; i += kDecThreads) {
    const int t = i / p.topk, j = i - t * p.topk;
    sm.weight[sm.mask[sel[t * p.E + j]] >> 16][t] = val[t * p.E + j];
  }
  __syncthreads();
}

template <bool BF16, int WF>
__global__ void __launch_bounds__(kDecThreads, 2) moe_decode_kernel(const DecodeParams p) {
  extern __shared__ __align__(16) uint8_t dec_smem[];
  DecodeSmem& sm = *reinterpret_cast<DecodeSmem*>(dec_smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const unsigned int G = gridDim.x;

  decode_logits<BF16>(p, &sm.part[0][0]);
  if (!grid_barrier(p.barrier, G)) return;
  decode_rank(p, sm, reinterpret_cast<uint16_t*>(&sm.part[0][0]), reinterpret_cast<float*>(&sm.ring[0][0][0]));
  int n_active = 0;
  for (int w = 0; w < kDecWarps; ++w) n_active += sm.scan[w];

  const int rb1 = WF == WF_16BIT ? p.H * 2 : p.H / 2;   // bytes of a row of w1 / w2
  const int rb2 = WF == WF_16BIT ? p.I * 2 : p.I / 2;
  constexpr int ELT = WF == WF_16BIT ? 8 : 32;     // elements in a lane's 16 bytes
  const int sb1 = WF == WF_NV4 ? p.H / 16 : p.H / 32;   // scale bytes of a row
  const int sb2 = WF == WF_NV4 ? p.I / 16 : p.I / 32;

  // this CTA's share: row pairs [pair0, pair1) of the active experts' w1, rows [row0, row1) of every active w2
  const int64_t pairs = static_cast<int64_t>(n_active) * p.I;
  const int64_t pair0 = pairs * blockIdx.x / G, pair1 = pairs * (blockIdx.x + 1) / G;
  const int row0 = static_cast<int>(static_cast<int64_t>(p.H) * blockIdx.x / G);
  const int row1 = static_cast<int>(static_cast<int64_t>(p.H) * (blockIdx.x + 1) / G);

  // GEMM1: tiles of 16 pairs = four sub-tiles of 4 SiLU + 4 linear rows, 64 bytes of K per step, warp w takes steps
  // w, w + 8, ...; GEMM2: tiles of 16 rows = two sub-tiles of 8 rows, 128 bytes of K per step, the steps of all active
  // experts in one sequence dealt to the warps in turn.
  const int nb1 = (rb1 + 63) / 64, nb2 = (rb2 + 127) / 128;

  // ---- the loading end of the stream ----
  int64_t ld_left = pair1 - pair0;     // pairs not yet fully requested
  int ld_a = static_cast<int>(pair0 / p.I), ld_j = static_cast<int>(pair0 - static_cast<int64_t>(ld_a) * p.I);
  int ld_b = warp;
  bool ld_first = warp < nb1 && ld_left > 0;
  int ld_row = row0, ld_slot = 0;
  auto settle2 = [&](int& slot, int& b) {
    while (slot < n_active && b >= nb2) b -= nb2, ++slot;
  };
  int ld_b2 = warp;
  settle2(ld_slot, ld_b2);
  int ld_stage = 0;
  const uint32_t ring = smem_u32(&sm.ring[warp][0][0]) + lane * 16;
  auto issue = [&]() {
    const uint32_t dst = ring + ld_stage * kDecStageBytes;
    if (ld_first) {
      const int cnt = static_cast<int>(min(static_cast<int64_t>(min(16, p.I - ld_j)), ld_left));
      const int kb = ld_b * 64 + t4 * 16;
      const int64_t row = static_cast<int64_t>(sm.list[ld_a]) * 2 * p.I + (g < 4 ? 0 : p.I) + ld_j + (g & 3);
      const uint8_t* src = p.w1 + row * rb1 + kb;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const bool ok = 4 * s + (g & 3) < cnt && kb < rb1;
        cp_async16(dst + s * 512, ok ? src + static_cast<int64_t>(4 * s) * rb1 : p.w1, ok);
      }
      ld_b += kDecWarps;
      if (ld_b >= nb1) {
        ld_b = warp;
        ld_left -= cnt;
        ld_j += cnt;
        if (ld_j == p.I) ld_j = 0, ++ld_a;
        ld_first = ld_left > 0;
      }
    } else if (ld_row < row1 && ld_slot < n_active) {
      const int64_t row = static_cast<int64_t>(sm.list[ld_slot]) * p.H + ld_row + g;
      const uint8_t* src = p.w2 + row * rb2;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const int kb = ld_b2 * 128 + st * 64 + t4 * 16;
          const bool ok = ld_row + 8 * s + g < row1 && kb < rb2;
          cp_async16(dst + (s * 2 + st) * 512, ok ? src + static_cast<int64_t>(8 * s) * rb2 + kb : p.w2, ok);
        }
      }
      ld_b2 += kDecWarps;
      settle2(ld_slot, ld_b2);
      if (ld_slot >= n_active) {
        ld_row += 16;
        ld_slot = 0;
        ld_b2 = warp;
        settle2(ld_slot, ld_b2);
      }
    }
    cp_async_commit();
    ld_stage = ld_stage + 1 == kDecStages ? 0 : ld_stage + 1;
  };
  int stage = 0;
  auto next_stage = [&]() {   // request one more, then wait for the oldest
    issue();
    cp_async_wait<kDecStages - 1>();
    const uint8_t* at = &sm.ring[warp][stage][lane * 16];
    stage = stage + 1 == kDecStages ? 0 : stage + 1;
    return at;
  };
#pragma unroll
  for (int s = 0; s < kDecStages - 1; ++s) issue();

  constexpr int TR = WF == WF_16BIT ? 4 : 16;
  // ---- GEMM1 + SiLU ----
  {
    int64_t left = pair1 - pair0;
    int a = static_cast<int>(pair0 / p.I), j0 = static_cast<int>(pair0 - static_cast<int64_t>(a) * p.I);
    while (left > 0) {
      const int cnt = static_cast<int>(min(static_cast<int64_t>(min(16, p.I - j0)), left));
      const int e = sm.list[a];
      const uint32_t mask = sm.mask[e];
      const bool use_lo = (mask >> g) & 1u, use_hi = (mask >> (g + 8)) & 1u;
      float acc[4][4];
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[s][i] = 0.0f;
      const uint16_t* x_lo = p.x + static_cast<int64_t>(g) * p.H;
      const uint8_t* srow = p.s1 + (static_cast<int64_t>(e) * 2 * p.I + (g < 4 ? 0 : p.I) + j0 + (g & 3)) * sb1;
      for (int b = warp; b < nb1; b += kDecWarps) {
        const int kb = b * 64 + t4 * 16, k = (b * 4 + t4) * ELT;
        uint32_t lo[TR], hi[TR];
        load_tokens<WF>(x_lo + k, use_lo && kb < rb1, false, lo);
        load_tokens<WF>(x_lo + static_cast<int64_t>(8) * p.H + k, use_hi && kb < rb1, false, hi);
        uint32_t sc[4];
#pragma unroll
        for (int s = 0; s < 4; ++s)
          sc[s] = load_scales<WF>(srow + static_cast<int64_t>(4 * s) * sb1, kb, 4 * s + (g & 3) < cnt && kb < rb1);
        const uint8_t* at = next_stage();
#pragma unroll
        for (int s = 0; s < 4; ++s)
          chunk_mma<BF16, WF>(acc[s], *reinterpret_cast<const uint4*>(at + s * 512), sc[s], lo, hi);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        float* o = sm.part[warp] + (8 * s + 2 * t4) * kDecPartStride + g;
        o[0] = acc[s][0];
        o[kDecPartStride] = acc[s][1];
        o[8] = acc[s][2];
        o[kDecPartStride + 8] = acc[s][3];
      }
      __syncthreads();
      {
        const int j = threadIdx.x & 15, t = threadIdx.x >> 4;
        if (j < cnt && ((mask >> t) & 1u)) {
          const int r = (8 * (j >> 2) + (j & 3)) * kDecPartStride + t;
          float hg = 0.0f, hu = 0.0f;
#pragma unroll
          for (int w = 0; w < kDecWarps; ++w) {
            hg += sm.part[w][r];
            hu += sm.part[w][r + 4 * kDecPartStride];
          }
          if constexpr (WF != WF_16BIT) {
            const float f = (p.g1 ? __ldg(p.g1 + e) : 1.0f) * Fp4Expand<BF16, WF>::kUnit;
            hg *= f;
            hu *= f;
          }
          const uint32_t v = pack2<BF16>(silu_f(hg) * hu, 0.0f);
          p.act[(static_cast<int64_t>(a) * p.M + t) * p.I + j0 + j] = static_cast<uint16_t>(v);
        }
      }
      __syncthreads();
      left -= cnt;
      j0 += cnt;
      if (j0 == p.I) j0 = 0, ++a;
    }
  }
  if (!grid_barrier(p.barrier, G)) {
    cp_async_wait<0>();
    return;
  }
  // ---- GEMM2 + weighted sum over the experts ----
  for (int r0 = row0; r0 < row1; r0 += 16) {
    float tot[2][4], acc[2][4];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) tot[s][i] = acc[s][i] = 0.0f;
    int slot = 0, b = warp;
    settle2(slot, b);
    // An expert's sum enters a token's total only where the token is routed to it: an infinity or NaN in its weights
    // must not reach the other tokens through a product with zero.
    auto fold = [&](int from) {
      const int e = sm.list[from];
      const uint32_t mask = sm.mask[e];
      float f = 1.0f;
      if constexpr (WF != WF_16BIT) f = (p.g2 ? __ldg(p.g2 + e) : 1.0f) * Fp4Expand<BF16, WF>::kUnit;
      const float w_lo = sm.weight[from][g] * f, w_hi = sm.weight[from][g + 8] * f;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if ((mask >> (i < 2 ? g : g + 8)) & 1u) tot[s][i] = fmaf(i < 2 ? w_lo : w_hi, acc[s][i], tot[s][i]);
          acc[s][i] = 0.0f;
        }
      }
    };
    while (slot < n_active) {
      const int e = sm.list[slot];
      const uint32_t mask = sm.mask[e];
      const bool use_lo = (mask >> g) & 1u, use_hi = (mask >> (g + 8)) & 1u;
      const uint16_t* a_lo = p.act + (static_cast<int64_t>(slot) * p.M + g) * p.I;
      const uint8_t* srow = p.s2 + (static_cast<int64_t>(e) * p.H + r0 + g) * sb2;
      uint32_t lo[2][TR], hi[2][TR], sc[2][2];
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const int kb = b * 128 + st * 64 + t4 * 16, k = (b * 8 + st * 4 + t4) * ELT;
        load_tokens<WF>(a_lo + k, use_lo && kb < rb2, true, lo[st]);
        load_tokens<WF>(a_lo + static_cast<int64_t>(8) * p.I + k, use_hi && kb < rb2, true, hi[st]);
#pragma unroll
        for (int s = 0; s < 2; ++s)
          sc[s][st] = load_scales<WF>(srow + static_cast<int64_t>(8 * s) * sb2, kb, r0 + 8 * s + g < row1 && kb < rb2);
      }
      const uint8_t* at = next_stage();
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int st = 0; st < 2; ++st)
          chunk_mma<BF16, WF>(acc[s], *reinterpret_cast<const uint4*>(at + (s * 2 + st) * 512), sc[s][st], lo[st], hi[st]);
      const int was = slot;
      b += kDecWarps;
      settle2(slot, b);
      if (slot != was) fold(was);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float* o = sm.part[warp] + (8 * s + 2 * t4) * kDecPartStride + g;
      o[0] = tot[s][0];
      o[kDecPartStride] = tot[s][1];
      o[8] = tot[s][2];
      o[kDecPartStride + 8] = tot[s][3];
    }
    __syncthreads();
    {
      const int r = threadIdx.x & 15, t = threadIdx.x >> 4;
      if (t < p.M && r0 + r < row1) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) v += sm.part[w][r * kDecPartStride + t];
        p.out[static_cast<int64_t>(t) * p.H + r0 + r] = static_cast<uint16_t>(pack2<BF16>(v, 0.0f));
      }
    }
    __syncthreads();
  }
  cp_async_wait<0>();
}

// ---- host ----------------------------------------------------------------------------------------------------
struct DecodeWs {
  size_t logits, act, total;
};
static DecodeWs decode_ws(int64_t M, int I, int E, int topk) {
  auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
  DecodeWs w;
  const int64_t active = M * topk < E ? M * topk : E;
  w.logits = 256;                                                    // grid-barrier words first
  w.act = w.logits + up(static_cast<size_t>(M) * E * sizeof(float));
  w.total = w.act + up(static_cast<size_t>(active) * M * I * 2);
  return w;
}

size_t moe_decode_workspace(int64_t M, int I, int E, int topk) {
  if (M <= 0 || M > kDecTokens || I <= 0 || E <= 0 || topk <= 0 || topk > E) return 0;
  return decode_ws(M, I, E, topk).total;
}

template <bool BF16, int WF>
static int launch_decode(const DecodeParams& p, cudaStream_t st) {
  auto kern = moe_decode_kernel<BF16, WF>;
  constexpr int smem = sizeof(DecodeSmem);
  // resident CTAs of the device, looked up once (0 = not yet)
  constexpr int kMaxDevices = 64;
  static std::atomic<int> grids[kMaxDevices];
  const DeviceInfo& di = device_info();
  if (di.device < 0 || di.device >= kMaxDevices) return FR_ERR_UNSUPPORTED;
  int grid = grids[di.device].load(std::memory_order_acquire);
  if (!grid) {
    FR_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    int per_sm = 0;
    FR_CUDA_OK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, kDecThreads, smem));
    if (per_sm < 1) return FR_ERR_UNSUPPORTED;
    grid = (per_sm > 2 ? 2 : per_sm) * di.sm_count;
    grids[di.device].store(grid, std::memory_order_release);
  }
  DecodeParams q = p;
  // one (expert, group of tokens) per CTA where the grid is large enough
  q.tokens_per_unit = static_cast<int>((static_cast<int64_t>(p.M) * p.E + grid - 1) / grid);
  if (q.tokens_per_unit > p.M) q.tokens_per_unit = p.M;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kDecThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  FR_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, q));
  return FR_OK;
}

int moe_decode_dispatch(const void* x, const void* gate, int64_t gsh, int64_t gse, const void* w1, const void* s1,
                        const float* g1, const void* w2, const void* s2, const float* g2, int dtype, int block,
                        int64_t M, int H, int I, int E, int topk, int renormalize, void* out, float* tw, int32_t* ti,
                        void* workspace, size_t workspace_bytes, cudaStream_t st) {
  if (M < 0 || H <= 0 || I <= 0 || E <= 0 || topk <= 0 || topk > E) return FR_ERR_ARG;
  if (block != 0 && block != 16 && block != 32) return FR_ERR_ARG;
  if ((tw == nullptr) != (ti == nullptr)) return FR_ERR_ARG;
  if (dtype != FR_F16 && dtype != FR_BF16) return FR_ERR_UNSUPPORTED;
  if (M > kDecTokens || E > kDecMaxExperts) return FR_ERR_UNSUPPORTED;
  if (block == 32 && dtype != FR_BF16) return FR_ERR_UNSUPPORTED;     // E8M0 scales reach beyond fp16
  const int unit = block ? 32 : 8;                                    // 16 bytes of a weight row
  if (H % unit || I % unit) return FR_ERR_ALIGN;
  if (M == 0) return FR_OK;
  if (!x || !gate || !w1 || !w2 || !out || (block && (!s1 || !s2))) return FR_ERR_ARG;
  for (const void* q : {x, w1, w2})
    if (reinterpret_cast<uintptr_t>(q) & 15) return FR_ERR_ALIGN;
  if (block == 16 && ((reinterpret_cast<uintptr_t>(s1) | reinterpret_cast<uintptr_t>(s2)) & 1)) return FR_ERR_ALIGN;
  const DecodeWs ws = decode_ws(M, I, E, topk);
  if (!workspace || workspace_bytes < ws.total) return FR_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 255) return FR_ERR_ALIGN;
  uint8_t* base = static_cast<uint8_t*>(workspace);
  DecodeParams p;
  p.x = static_cast<const uint16_t*>(x);
  p.gate = static_cast<const uint16_t*>(gate);
  p.gsh = gsh;
  p.gse = gse;
  p.gate_vec = gsh == 1 && gse % 8 == 0 && !(reinterpret_cast<uintptr_t>(gate) & 15);
  p.w1 = static_cast<const uint8_t*>(w1);
  p.w2 = static_cast<const uint8_t*>(w2);
  p.s1 = static_cast<const uint8_t*>(s1);
  p.s2 = static_cast<const uint8_t*>(s2);
  p.g1 = block == 16 ? g1 : nullptr;
  p.g2 = block == 16 ? g2 : nullptr;
  p.M = static_cast<int>(M);
  p.H = H;
  p.I = I;
  p.E = E;
  p.topk = topk;
  p.renormalize = renormalize;
  p.tokens_per_unit = 1;
  p.out = static_cast<uint16_t*>(out);
  p.tw = tw;
  p.ti = ti;
  p.barrier = reinterpret_cast<unsigned int*>(base);
  p.logits = reinterpret_cast<float*>(base + ws.logits);
  p.act = reinterpret_cast<uint16_t*>(base + ws.act);
  const bool bf = dtype == FR_BF16;
  if (block == 0) return bf ? launch_decode<true, WF_16BIT>(p, st) : launch_decode<false, WF_16BIT>(p, st);
  if (block == 16) return bf ? launch_decode<true, WF_NV4>(p, st) : launch_decode<false, WF_NV4>(p, st);
  return launch_decode<true, WF_MX4>(p, st);
}

}  // namespace fr
