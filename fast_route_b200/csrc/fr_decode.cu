// The whole MoE layer for at most 16 tokens in ONE cooperative launch: router, top-k, GEMM1 + SiLU * u, GEMM2,
// weighted sum.  A batch this small reads every active expert's weights once and does almost no arithmetic per byte,
// so the kernel is built around that stream:
//
//   logits, tagged with the call -> every CTA waits for all of them and ranks all tokens -> h = w1 x, act = silu(h_g) h_u
//          -> grid barrier -> out = sum_e weight * (w2 act)
//
// * Work is split by weight ROWS, not by tiles: the (active experts * I) row pairs of w1 and the H rows of w2 are cut
//   into equal contiguous ranges, so every CTA streams the same number of bytes whatever the sizes (16-row tiles would
//   leave up to a quarter of the CTAs without a last tile).
// * Each warp owns a FIFO in shared memory that it alone fills (cp.async, full 128-byte lines) and drains, so the
//   stream needs no block barriers and runs on across row tiles, across experts and across the grid barrier: the first
//   weights of w2 are in flight while the last activations are still being written.
// * The products are mma.sync m16n8k16 with the TOKENS on the 16-row side: 8 weight rows by 16 tokens per instruction
//   (a tcgen05 tile is 128 weight rows: too coarse to split a layer of a few thousand rows over 296 CTAs; a large layer
//   has rows enough, but its memory stream is the limit with 16-bit weights, and 4-bit weights would have to be expanded
//   into shared or tensor memory behind a barrier, or multiplied as they are with tokens in 4-bit terms).
//   A lane's 16 bytes are 8 consecutive k of one row; the dot product does not care about the order of k, so both
//   operands use the same permutation of k and no data is moved between lanes.
// * 4-bit experts are expanded in registers to the exact 16-bit weight (E2M1 * E4M3 has at most six significant bits),
//   so the arithmetic is that of 16-bit weights.  No single pipe limits them (1 token of 8 experts: integer pipe active for
//   41 % of the cycles, FMA 23, tensor 21): 37 instructions per word of eight codes on two warps per scheduler leave
//   latencies and instruction fetches in the open.
//
// The eight warps of a CTA split K; their partial sums meet in shared memory in warp order, so results do not depend
// on timing.  fp32 accumulation throughout; the activations between the two products are rounded to the 16-bit type.
#include <algorithm>
#include <atomic>

#include "fr_common.cuh"

namespace fr {

constexpr int kDecTokens = FR_DECODE_MAX_TOKENS;   // 16: the row side of the MMA
constexpr int kDecMaxExperts = 256;
constexpr int kDecWarps = 8;
constexpr int kDecThreads = 32 * kDecWarps;
constexpr int kDecCodeBytes = 4096;                // of a stage, per warp: 32 chunks of 128 bytes of a weight row
constexpr int kDecScaleBytes = 512;                // and, for 4-bit weights, 32 chunks' block scales

// Control words of a workspace: zero before the first call, kept up by every call (the CTA that finishes last adds what
// the call used, so nothing has to be cleared in between).
enum { DC_COUNT = 0, DC_BASE = 1, DC_FINISHED = 2, DC_BUDGET = 3, DC_EPOCH = 4, DC_GROUP = 64 /* one per row range */ };
constexpr int kDecMaxGroups = 512;
constexpr uint32_t kDecPolls = 1u << 22;           // a second or a few, unless DC_BUDGET holds another limit

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
  int scale_copy1, scale_copy2;  // bytes per cp.async of w1's / w2's scales: 16, 8 or 4; 0: rows start anywhere
  int ksplit, groups;            // GEMM2: `groups` row ranges, each shared by `ksplit` CTAs that split K
  float* partial;                // [ksplit][M][H], with ksplit > 1
  int tokens_per_unit;           // router: tokens one CTA takes for one expert
  uint16_t* out;
  float* tw;
  int32_t* ti;
  unsigned int* control;         // DC_* above
  unsigned long long* logits;    // [M, E]: fp32 bits below, the call's tag above
  uint16_t* act;                 // [active expert][M][I]
};

// 16-bit weights: two CTAs per SM with 128 registers a thread; 4-bit weights: one with 255, the expansion needs them (two
// CTAs of it, with spills: 109 instead of 94 us for 1 token of 8 experts).  HI: more than 8 tokens.
template <int WF, bool HI>
struct DecodeCfg {
  static constexpr bool TWO = WF == WF_16BIT;
  static constexpr int STAGES = 2;                  // FIFO depth (4-bit: four are 6 to 8 % slower; 16-bit: no room)
  static constexpr int STAGE = TWO ? kDecCodeBytes : kDecCodeBytes + kDecScaleBytes;
  static constexpr int NS2 = 2, LN2 = 2;            // GEMM2: sub-tiles of 8 rows, and 128-byte lines of a row per stage
  static constexpr int TOKENS = HI ? 16 : 8;
  static constexpr int STRIDE = HI ? 20 : 12;       // floats per weight row of a partial tile: conflict-free stores
  static constexpr int PBUFS = TWO && HI ? 1 : 2;   // buffers of partial sums in turn: one barrier per tile instead of two
};
template <int WF, bool HI>
struct DecodeSmem {
  using C = DecodeCfg<WF, HI>;
  uint8_t ring[kDecWarps][C::STAGES][C::STAGE];
  float part[C::PBUFS][kDecWarps][32 * C::STRIDE];
  float weight[kDecMaxExperts][C::TOKENS];    // routing weight by expert and token
  uint32_t mask[kDecMaxExperts];              // by expert: bit t = token t goes there
  uint16_t list[kDecMaxExperts];              // active experts in ascending order
  uint32_t scan[kDecWarps];
  uint32_t base, epoch;                       // of the control words, read once
  int ok, last;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t size) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// the scales of 128 bytes of codes of one row (16 bytes, or 8 for blocks of 32), `left` bytes of the row remaining;
// what lies past the row's end becomes zero
template <int BYTES>
__device__ __forceinline__ void cp_async_scales(uint32_t dst, const uint8_t* src, int left, int unit) {
  if (unit == 0) {                 // rows that start anywhere: byte by byte, at once
#pragma unroll
    for (int i = 0; i < BYTES; i += 4) {
      uint32_t v = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (i + b < left) v |= static_cast<uint32_t>(__ldg(src + i + b)) << (8 * b);
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst + i), "r"(v) : "memory");
    }
  } else if (BYTES == 16 && unit == 16) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(min(max(left, 0), 16)) : "memory");
  } else if (unit >= 8) {
#pragma unroll
    for (int i = 0; i < BYTES; i += 8)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst + i), "l"(left > i ? src + i : src),
                   "r"(min(max(left - i, 0), 8))
                   : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < BYTES; i += 4)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + i), "l"(left > i ? src + i : src),
                   "r"(min(max(left - i, 0), 4))
                   : "memory");
  }
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Expansion of a word of eight packed codes to 16-bit numbers: value * block scale / kUnit, exact.  fp16 has a conversion
// instruction (half the issue slots of the shifts: 4-bit experts of a 1-token layer 94 us in bf16, 76 in fp16); bf16 has none.
template <bool BF16, int WF>
struct Fp4Expand {
  // what is left to multiply the sums with: the factors below keep every intermediate inside the 16-bit format
  static constexpr uint32_t kMx4Top = 133;
  static constexpr float kUnit = WF == WF_MX4 ? 32.0f : (BF16 ? 65536.0f : 1.0f);
  // the factors of a lane's 32 codes: two blocks of 16 (m[0], m[1]) or one of 32
  static __device__ __forceinline__ void mult(uint32_t scales, uint32_t (&m)[2]) {
    if constexpr (WF == WF_MX4) {
      // bf16 only: 2^(byte - 127) * 2^121.  That reaches from the smallest scale, whose 0.5 is a subnormal bf16 number, to
      // 2^6 (byte 133); what comes of larger scales and of NaN is not used: fp4_dot sums their tiles.
      const uint32_t b = (scales + 121u) << 7;
      m[0] = m[1] = b | (b << 16);
    } else {
      uint32_t h;   // both scales in fp16, exact, NaN included
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(scales)));
      if constexpr (BF16) {
        const float2 f = unpack2<false>(h);
        const float a = __fmul_rn(f.x, 1.298074214633706907e33f /* 2^110 */), b = __fmul_rn(f.y, 1.298074214633706907e33f);
        m[0] = pack2<true>(a, a);     // exact: four significant bits
        m[1] = pack2<true>(b, b);
      } else {
        m[0] = __byte_perm(h, h, 0x1010);
        m[1] = __byte_perm(h, h, 0x3232);
      }
    }
  }
  static __device__ __forceinline__ void order(const uint4& u, uint32_t (&r)[4]) {
    if constexpr (BF16) {            // pairs (j, j + 4)
      r[0] = __byte_perm(u.x, u.z, 0x5410);
      r[1] = __byte_perm(u.x, u.z, 0x7632);
      r[2] = __byte_perm(u.y, u.w, 0x5410);
      r[3] = __byte_perm(u.y, u.w, 0x7632);
    } else {
      r[0] = u.x, r[1] = u.y, r[2] = u.z, r[3] = u.w;
    }
  }
  static __device__ __forceinline__ uint32_t mul(uint32_t a, uint32_t m) {
    uint32_t r;
    if constexpr (BF16) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(m));
    else asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(m));
    return r;
  }
  static __device__ __forceinline__ void expand(uint32_t w, uint32_t m, uint32_t (&o)[4]) {
    if constexpr (BF16) {
      // pairs (j, j + 4), as the fields of E2M1 (bias 1) in the low exponent bits and the top fraction bit of bf16:
      // the value times 2^-126, subnormal 0.5 included
      constexpr uint32_t S = 0x80008000u, F = 0x01C001C0u;
      o[0] = ((w << 12) & S) | ((w << 6) & F);
      o[1] = ((w << 8) & S) | ((w << 2) & F);
      o[2] = ((w << 4) & S) | ((w >> 2) & F);
      o[3] = (w & S) | ((w >> 6) & F);
    } else {
      cvt8_f16(w, o);                 // pairs (2j, 2j + 1)
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = mul(o[j], m);
  }
};

static __device__ __noinline__ bool mx4_beyond(const uint8_t* scales, int n) {
  for (int i = 0; i < n; ++i)
    if (__ldg(scales + i) > Fp4Expand<true, WF_MX4>::kMx4Top) return true;
  return false;
}

// sum of n (a multiple of 32) products of E8M0-scaled codes and 16-bit numbers in fp32: for the tiles with scales beyond 2^6
// (weights of 512 and more), which no trained layer is known to have, so it is short rather than fast (all of a layer in
// such scales: 1690 us instead of 93 for 1 token of 8 experts, 1910 instead of 157 for 16 tokens of 64; a second factor in
// the expansion costs everybody 11 to 14 %, behind a branch 4 to 8).  It replaces the sums of (row, token) pairs with such a
// scale only: the others keep their bits whatever the tile's other rows, or the FIFO's places past its end, hold.
static __device__ __noinline__ float fp4_dot(const uint8_t* codes, const uint8_t* scales, const uint16_t* x, int n) {
  float sum = 0.0f;
  for (int k = 0; k < n; k += 32) {
    const float unit = e8m0_f32(__ldg(scales + k / 32));
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(codes + k / 2));
    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(x + k + 8 * i);
      const uint32_t pair[4] = {v.x, v.y, v.z, v.w};
      uint32_t h[4];
      cvt8_f16(word[i], h);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 c = unpack2<false>(h[j]), t = unpack2<true>(pair[j]);
        sum = fmaf(__fmul_rn(c.x, unit), t.x, sum);
        sum = fmaf(__fmul_rn(c.y, unit), t.y, sum);
      }
    }
  }
  return sum;
}

// Sums of 4-bit weights are multiplied with global * kUnit.  That leaves fp32's range for global scales from 2^112 on (bf16,
// blocks of 16: the only case with both), while results need not: a matrix of magnitude 1e37 has such a scale, but rows of
// zeros stay zero and small tokens give ordinary results.  Then the two are applied one after the other.  (Decided for the
// whole warp by the expert's scale: a factor of two parts for everybody costs 2 %.)
template <bool BF16, int WF>
__device__ __forceinline__ bool fp4_wide_global(float global) {
  return BF16 && WF == WF_NV4 && fabsf(global) > 3.40282347e38f / Fp4Expand<BF16, WF>::kUnit;
}

// One token row's operand for the 64 bytes of weights a quad holds (16-bit weights: the lane's 8 elements, 4-bit: 32);
// `p` points at the lane's first element.  For a token that the expert does not get (`use` false) the registers keep what
// they held: its sums are not used.  Past the end of the row (`in` false) the weights are zero; where row lengths end
// inside a step (RAGGED) the tokens' registers become zero as well, for an earlier infinity left in them would make a NaN
// of that.  (A kernel of its own, since the test alone costs 1 to 6 % of the others; zeros first: written after the load
// they would have to wait for it.)
template <int WF, bool RAGGED>
__device__ __forceinline__ void load_tokens(const uint16_t* p, bool use, bool in, uint4 (&r)[WF == WF_16BIT ? 1 : 4]) {
  constexpr int NV = WF == WF_16BIT ? 1 : 4;
  if (RAGGED && !in) {
#pragma unroll
    for (int v = 0; v < NV; ++v) r[v] = make_uint4(0, 0, 0, 0);
  }
  if (use && in) {
#pragma unroll
    for (int v = 0; v < NV; ++v) r[v] = *(reinterpret_cast<const uint4*>(p) + v);
  }
}

// acc += tokens * weights for one 16-byte chunk per lane of 16-bit weights
template <bool BF16>
__device__ __forceinline__ void chunk_mma(float (&acc)[4], const uint4& w, const uint4& lo, const uint4& hi) {
  const uint32_t a0[4] = {lo.x, hi.x, lo.y, hi.y}, a1[4] = {lo.z, hi.z, lo.w, hi.w};
  mma_16816<BF16>(acc, a0, w.x, w.y);
  mma_16816<BF16>(acc, a1, w.z, w.w);
}

// the same for NS sub-tiles of 4-bit weights: word by word, so that the sub-tiles' products are independent
template <bool BF16, int WF, int NS>
__device__ __forceinline__ void chunk_mma4(float (&acc)[NS][4], const uint4 (&w)[NS], const uint32_t (&scales)[NS],
                                           const uint4 (&lo)[4], const uint4 (&hi)[4]) {
  using X = Fp4Expand<BF16, WF>;
  uint32_t m[NS][2];
#pragma unroll
  for (int s = 0; s < NS; ++s) X::mult(scales[s], m[s]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // a word's eight elements as four registers, in the order Fp4Expand gives the codes
    uint32_t l[4], h[4];
    X::order(lo[i], l);
    X::order(hi[i], h);
    const uint32_t a0[4] = {l[0], h[0], l[1], h[1]}, a1[4] = {l[2], h[2], l[3], h[3]};
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const uint32_t word = i == 0 ? w[s].x : i == 1 ? w[s].y : i == 2 ? w[s].z : w[s].w;
      uint32_t o[4];
      X::expand(word, m[s][i >> 1], o);
      mma_16816<BF16>(acc[s], a0, o[0], o[1]);
      mma_16816<BF16>(acc[s], a1, o[2], o[3]);
    }
  }
}

// One stage (LN lines of 128 bytes of every row of NS sub-tiles) of 4-bit weights, in half lines with two operand buffers
// in turn: `fetch(st)` requests the operand of the half line after st into the buffer that st does not use, `stage` waits
// for the weights and says where the lane's first chunk and scales are.  `top_scale`: the largest E8M0 scale so far.
template <bool BF16, int WF, int NS, int LN, class Fetch, class Stage>
__device__ __forceinline__ void full_step4(float (&acc)[NS][4], const uint4 (&lo)[2][4], const uint4 (&hi)[2][4],
                                           Fetch fetch, Stage stage, uint32_t& top_scale) {
  constexpr int SCB = WF == WF_NV4 ? 16 : 8;
  const uint8_t* at = nullptr;
  const uint8_t* sc_at = nullptr;
#pragma unroll
  for (int st = 0; st < 2 * LN; ++st) {
    fetch(st);
    if (st == 0) stage(at, sc_at);
    const uint8_t* half = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(at) ^ ((st & 1) << 6)) + (st >> 1) * NS * 1024;
    uint4 w[NS];
    uint32_t sc[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      w[s] = *reinterpret_cast<const uint4*>(half + s * 1024);
      const uint8_t* q = sc_at + (s + (st >> 1) * NS) * 8 * SCB + (st & 1) * (SCB / 2);
      sc[s] = WF == WF_NV4 ? *reinterpret_cast<const uint16_t*>(q) : *q;
      if constexpr (WF == WF_MX4) top_scale = max(top_scale, sc[s]);
    }
    chunk_mma4<BF16, WF, NS>(acc, w, sc, lo[st & 1], hi[st & 1]);
  }
}

struct DecodeStep {     // GEMM2: a double step of one active expert
  int slot, b;
};

// ---- router: logits of all (token, expert) pairs, spread over the grid --------------------------------------
template <bool BF16>
__device__ __forceinline__ void decode_logits(const DecodeParams& p, uint32_t tag, float* red /* [kDecWarps][kDecTokens] */) {
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
      // value and tag in one 8-byte store: a reader that sees the tag has the value, no fence or barrier in between
      p.logits[static_cast<int64_t>(t0 + threadIdx.x) * p.E + e] =
          (static_cast<unsigned long long>(tag) << 32) | __float_as_uint(v);
    }
    __syncthreads();
  }
}

__device__ __forceinline__ uint32_t order_key(float v) {   // larger value, larger key; -0 and +0 alike; never 0
  const uint32_t u = __float_as_uint(v == 0.0f ? 0.0f : v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Every CTA ranks all tokens: a warp polls the logits of its (up to two) tokens until all carry this call's tag
// (bounded), then k rounds of arg-max (equal logits: lower expert id), softmax by the fixed fp32 recipe of the routers.
// `sel` / `val`: [kDecTokens][E] scratch.  False: the logits did not arrive in time.
// NE: logits per lane, NT: tokens per warp.
template <int NE, int NT, class Smem>
__device__ __forceinline__ bool decode_rank(const DecodeParams& p, Smem& sm, uint32_t tag, uint16_t* sel, float* val) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < p.E; e += kDecThreads) sm.mask[e] = 0;
  __syncthreads();
  if (warp < p.M) {
    float v[NT][NE];
    uint32_t key[NT][NE];
    bool all = false;
    const uint32_t asked = __ldcg(p.control + DC_BUDGET), budget = asked ? asked : kDecPolls;
    for (uint32_t poll = 0; poll <= budget && !all; ++poll) {
      unsigned long long u[NT][NE];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < NE; ++i) {
          const int t = warp + n * kDecWarps, c = i * 32 + lane;
          u[n][i] = static_cast<unsigned long long>(tag) << 32;
          if (t < p.M && c < p.E)
            asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(u[n][i]) : "l"(p.logits + static_cast<int64_t>(t) * p.E + c));
        }
      bool mine = true;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < NE; ++i) {
          mine &= static_cast<uint32_t>(u[n][i] >> 32) == tag;
          v[n][i] = __uint_as_float(static_cast<uint32_t>(u[n][i]));
          key[n][i] = i * 32 + lane < p.E ? order_key(v[n][i]) : 0u;
        }
      all = __all_sync(0xffffffffu, mine);
      if (!all) __nanosleep(300);      // every CTA polls the same lines: without a pause the stores wait for the polls
    }
    if (!all && lane == 0) {
      report(ST_WAIT_TIMEOUT, 0x800);
      sm.ok = 0;
    }
    for (int j = 0; j < p.topk && all; ++j) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int t = warp + n * kDecWarps;
        uint32_t best = 0;
        int at = 0;
        float bv = 0.0f;
#pragma unroll
        for (int i = 0; i < NE; ++i)
          if (key[n][i] > best) best = key[n][i], at = i, bv = v[n][i];
        const uint32_t top = __reduce_max_sync(0xffffffffu, best);
        const uint32_t col = __reduce_min_sync(0xffffffffu, best == top ? static_cast<uint32_t>(at * 32 + lane) : 0xFFFFu);
        if (t < p.M && col == static_cast<uint32_t>(at * 32 + lane)) {
          sel[t * p.E + j] = static_cast<uint16_t>(col);
          val[t * p.E + j] = bv;
          atomicOr(&sm.mask[col], 1u << t);
#pragma unroll
          for (int i = 0; i < NE; ++i)
            if (i == at) key[n][i] = 0;
        }
      }
    }
    __syncwarp();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int t = warp + n * kDecWarps;
      if (t >= p.M || !all) break;
      float* my_val = val + t * p.E;
      const float top = my_val[0];
      float s = 0.0f;
      if (!p.renormalize) {
#pragma unroll
        for (int i = 0; i < NE; ++i)
          if (i * 32 + lane < p.E) s += exp_recipe(__fsub_rn(v[n][i], top));
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      }
      __syncwarp();
      for (int j = lane; j < p.topk; j += 32) my_val[j] = exp_recipe(__fsub_rn(my_val[j], top));
      __syncwarp();
      if (p.renormalize) {                 // in the order of the ranks
        s = my_val[0];
        for (int j = 1; j < p.topk; ++j) s = __fadd_rn(s, my_val[j]);
      }
      __syncwarp();
      for (int j = lane; j < p.topk; j += 32) {
        const float w = __fdiv_rn(my_val[j], s);
        sm.weight[sel[t * p.E + j]][t] = w;
        if (blockIdx.x == 0 && p.tw) {
          p.tw[static_cast<int64_t>(t) * p.topk + j] = w;
          p.ti[static_cast<int64_t>(t) * p.topk + j] = sel[t * p.E + j];
        }
      }
    }
  }
  __syncthreads();
  if (!sm.ok) return false;
  // active experts in ascending order; `scan` holds the warps' counts
  const bool active = threadIdx.x < p.E && sm.mask[threadIdx.x] != 0;
  const uint32_t vote = __ballot_sync(0xffffffffu, active);
  if (lane == 0) sm.scan[warp] = __popc(vote);
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < warp; ++w) before += sm.scan[w];
  if (active) sm.list[before + __popc(vote & ((1u << lane) - 1u))] = static_cast<uint16_t>(threadIdx.x);
  __syncthreads();
  return true;
}

// The CTA's last act: whoever is last of the grid moves the control words on for the next call.
__device__ __forceinline__ void decode_finish(const DecodeParams& p, uint32_t base, uint32_t epoch) {
  if (threadIdx.x != 0) return;
  __threadfence();
  if (atomicAdd(p.control + DC_FINISHED, 1u) == gridDim.x - 1) {
    p.control[DC_FINISHED] = 0;
    p.control[DC_BASE] = base + gridDim.x;
    p.control[DC_EPOCH] = epoch + 1;
  }
}

// The last act of a CTA whose wait ran out: it still arrives at its row range's counter, without which the range's next
// calls would take a wrong CTA for the last one.
__device__ __forceinline__ void decode_give_up(const DecodeParams& p, uint32_t base, uint32_t epoch) {
  const int ks = static_cast<int>(blockIdx.x) / p.groups, group = static_cast<int>(blockIdx.x) - ks * p.groups;
  if (threadIdx.x == 0 && p.ksplit > 1 && ks < p.ksplit &&
      atomicAdd(p.control + DC_GROUP + group, 1u) == static_cast<unsigned int>(p.ksplit) - 1u)
    p.control[DC_GROUP + group] = 0;
  decode_finish(p, base, epoch);
}

// RAGGED: rows of w1 or w2 end inside a step (of 128 or 256 bytes).
template <bool BF16, int WF, bool HI, bool RAGGED>
__global__ void __launch_bounds__(kDecThreads, (DecodeCfg<WF, HI>::TWO ? 2 : 1)) moe_decode_kernel(const DecodeParams p) {
  extern __shared__ __align__(128) uint8_t dec_smem[];
  using C = DecodeCfg<WF, HI>;
  using Smem = DecodeSmem<WF, HI>;
  Smem& sm = *reinterpret_cast<Smem*>(dec_smem);
  constexpr int PS = C::STRIDE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const unsigned int G = gridDim.x;

  if (threadIdx.x == 0) {
    sm.base = __ldcg(p.control + DC_BASE);
    sm.epoch = __ldcg(p.control + DC_EPOCH);
    sm.ok = 1;
  }
  __syncthreads();
  const uint32_t base = sm.base, epoch = sm.epoch;
  decode_logits<BF16>(p, epoch + 1, &sm.part[0][0][0]);
  uint16_t* sel = reinterpret_cast<uint16_t*>(&sm.part[0][0][0]);
  float* val = reinterpret_cast<float*>(&sm.ring[0][0][0]);
  constexpr int NT = HI ? 2 : 1;
  if (!(p.E <= 64 ? decode_rank<2, NT>(p, sm, epoch + 1, sel, val)
                  : decode_rank<kDecMaxExperts / 32, NT>(p, sm, epoch + 1, sel, val))) {
    if (threadIdx.x == 0) atomicAdd(p.control + DC_COUNT, 1u);      // the others' barrier counts every CTA
    decode_give_up(p, base, epoch);
    return;
  }
  int n_active = 0;
  for (int w = 0; w < kDecWarps; ++w) n_active += sm.scan[w];

  const int rb1 = WF == WF_16BIT ? p.H * 2 : p.H / 2;   // bytes of a row of w1 / w2
  const int rb2 = WF == WF_16BIT ? p.I * 2 : p.I / 2;
  constexpr int ELT = WF == WF_16BIT ? 8 : 32;     // elements in a lane's 16 bytes
  const int sb1 = WF == WF_NV4 ? p.H / 16 : p.H / 32;   // scale bytes of a row
  const int sb2 = WF == WF_NV4 ? p.I / 16 : p.I / 32;

  // this CTA's share: row pairs [pair0, pair1) of the active experts' w1, rows [row0, row1) of every active w2, of which
  // it takes every ksplit-th part of K
  const int64_t pairs = static_cast<int64_t>(n_active) * p.I;
  const int64_t pair0 = pairs * blockIdx.x / G, pair1 = pairs * (blockIdx.x + 1) / G;
  const int ks = static_cast<int>(blockIdx.x) / p.groups, group = static_cast<int>(blockIdx.x) - ks * p.groups;
  const bool second = ks < p.ksplit;                   // the last few CTAs may have no part in GEMM2
  const int row0 = second ? static_cast<int>(static_cast<int64_t>(p.H) * group / p.groups) : 0;
  const int row1 = second ? static_cast<int>(static_cast<int64_t>(p.H) * (group + 1) / p.groups) : 0;
  const int w2nd = ks * kDecWarps + warp, n2nd = p.ksplit * kDecWarps;     // this warp among those of its rows

  // A step is 128 bytes (a full line) of every row of a tile.  GEMM1: tiles of 16 pairs = four sub-tiles of 4 SiLU + 4
  // linear rows, warp w takes steps w, w + 8, ...; GEMM2: tiles of 16 rows = two sub-tiles of 8, two steps at a time,
  // the double steps of all active experts in one sequence dealt to the warps in turn.
  constexpr int NS2 = C::NS2, LN2 = C::LN2;
  const int nb1 = (rb1 + 127) / 128, nb2 = (rb2 + 128 * LN2 - 1) / (128 * LN2);

  // ---- the loading end of the stream: one segment = one row tile of GEMM1, or one (row tile, expert) of GEMM2 ----
  // Warp w's steps of a segment are b0, b0 + 8, ...; ld_rem counts those still to be requested.  Eight lanes copy one
  // row's 128 bytes, four rows per instruction.  Rows past the tile are not copied (what the FIFO holds there ends up
  // in sums nobody reads); k past the row's end is filled with zeros.
  const int cr = lane >> 3, cc = lane & 7;
  int64_t ld_left = pair1 - pair0;     // GEMM1 pairs from the next segment on
  int ld_a = static_cast<int>(pair0 / p.I), ld_j = static_cast<int>(pair0 - static_cast<int64_t>(ld_a) * p.I);
  int ld_row = row0, ld_slot = 0, ld_b2 = w2nd;
  int ld_rem = 0, ld_k = 0, ld_rows = 0;
  bool ld_second = false;
  const uint8_t* ld_src = p.w1;
  // chunk c of row r sits at position c ^ 4 * (r & 1) of the row: the reads below then touch every bank once
  const uint32_t ring = smem_u32(&sm.ring[warp][0][0]) + cr * 128 + ((cc ^ ((cr & 1) << 2)) << 4);
  uint32_t ld_at = 0, at_off = 0;
  constexpr uint32_t STAGE = C::STAGE;
  constexpr int kDecStages = C::STAGES;
  // 4-bit weights: lane r copies the scales of chunk r of the stage (row r, or row r & 15 of line r >> 4)
  constexpr int SCB = WF == WF_NV4 ? 16 : 8;
  const uint8_t* ld_sc = nullptr;
  int ld_sc_left = 0;
  bool ld_sc_ok = false;
  const uint32_t sc_ring = smem_u32(&sm.ring[warp][0][0]) + kDecCodeBytes + lane * SCB;
  const int64_t lin1 = static_cast<int64_t>(p.I) * rb1;     // from a SiLU row to its linear row
  auto issue = [&]() {
    while (ld_rem == 0) {              // next segment; the loop is for segments that have no step for this warp
      if (ld_left > 0) {
        const int cnt = static_cast<int>(min(static_cast<int64_t>(min(16, p.I - ld_j)), ld_left));
        const int64_t row = static_cast<int64_t>(sm.list[ld_a]) * 2 * p.I + ld_j + cr;
        ld_k = warp * 128 + cc * 16;
        ld_src = p.w1 + row * rb1 + ld_k;
        ld_rows = cnt - cr;
        ld_rem = warp < nb1 ? (nb1 - warp + kDecWarps - 1) / kDecWarps : 0;
        if constexpr (WF != WF_16BIT) {
          const int pair = 4 * (lane >> 3) + (lane & 3);
          ld_sc_ok = pair < cnt;
          ld_sc_left = sb1 - warp * SCB;
          ld_sc = p.s1 + (static_cast<int64_t>(sm.list[ld_a]) * 2 * p.I + ld_j + pair + ((lane & 4) ? p.I : 0)) * sb1 + warp * SCB;
        }
        ld_left -= cnt;
        ld_j += cnt;
        if (ld_j == p.I) ld_j = 0, ++ld_a;
      } else if (ld_row < row1) {
        ld_second = true;
        const int64_t row = static_cast<int64_t>(sm.list[ld_slot]) * p.H + ld_row + cr;
        ld_k = ld_b2 * (128 * LN2) + cc * 16;
        ld_src = p.w2 + row * rb2 + ld_k;
        ld_rows = row1 - ld_row - cr;
        if (ld_b2 < nb2) ld_rem = (nb2 - ld_b2 + n2nd - 1) / n2nd;
        if constexpr (WF != WF_16BIT) {
          const int off = (ld_b2 * 2 + (lane >> 4)) * SCB;
          ld_sc_ok = ld_row + (lane & 15) < row1;
          ld_sc_left = sb2 - off;
          ld_sc = p.s2 + (static_cast<int64_t>(sm.list[ld_slot]) * p.H + ld_row + (lane & 15)) * sb2 + off;
        }
        ld_b2 += ld_rem * n2nd - nb2;
        if (++ld_slot == n_active) {
          ld_slot = 0;
          ld_b2 = w2nd;
          ld_row += 8 * NS2;
        }
      } else {
        cp_async_commit();
        return;
      }
    }
    const uint32_t dst = ring + ld_at;
    if (!ld_second) {
      const uint32_t size = ld_k < rb1 ? 16u : 0u;
      const uint8_t* src = ld_src;
      const int64_t step = static_cast<int64_t>(4) * rb1;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (4 * s < ld_rows) {
          cp_async16(dst + s * 1024, src, size);
          cp_async16(dst + s * 1024 + 512, src + lin1, size);
        }
        src += step;
      }
      ld_k += kDecWarps * 128;
      ld_src += kDecWarps * 128;
      if constexpr (WF != WF_16BIT) {
        if (ld_sc_ok) cp_async_scales<SCB>(sc_ring + ld_at, ld_sc_left > 0 ? ld_sc : p.s1, ld_sc_left, p.scale_copy1);
        ld_sc += kDecWarps * SCB;
        ld_sc_left -= kDecWarps * SCB;
      }
    } else {
      const uint8_t* src = ld_src;
      const int64_t step = static_cast<int64_t>(4) * rb2;
#pragma unroll
      for (int s = 0; s < 2 * NS2; ++s) {  // half a sub-tile: 4 rows
        if (4 * s < ld_rows) {
#pragma unroll
          for (int l = 0; l < LN2; ++l)
            cp_async16(dst + s * 512 + l * 2048, src + l * 128, ld_k + l * 128 < rb2 ? 16u : 0u);
        }
        src += step;
      }
      ld_k += n2nd * 128 * LN2;
      ld_src += n2nd * 128 * LN2;
      if constexpr (WF != WF_16BIT) {
        if (ld_sc_ok) cp_async_scales<SCB>(sc_ring + ld_at, ld_sc_left > 0 ? ld_sc : p.s2, ld_sc_left, p.scale_copy2);
        ld_sc += n2nd * 2 * SCB;
        ld_sc_left -= n2nd * 2 * SCB;
      }
    }
    --ld_rem;
    cp_async_commit();
    ld_at = ld_at == (kDecStages - 1) * STAGE ? 0 : ld_at + STAGE;
  };
  // E8M0: the largest scale of a tile is that of all slots, also of those past its rows, which hold nothing yet
  uint32_t top_scale = 0;
  if constexpr (WF == WF_MX4) {
    for (int s = 0; s < kDecStages; ++s)
      *reinterpret_cast<uint2*>(&sm.ring[warp][s][kDecCodeBytes + lane * SCB]) = make_uint2(0, 0);
    __syncwarp();
  }
  // the reading end: lane (g, t4) takes chunk t4 + 4 * st of row g of a sub-tile
  const uint8_t* fifo = &sm.ring[warp][0][0] + g * 128 + ((t4 ^ ((g & 1) << 2)) << 4);
  auto next_stage = [&](const uint8_t*& at, const uint8_t*& sc_at) {
    cp_async_wait<kDecStages - 1>();
    __syncwarp();
    at = fifo + at_off;
    sc_at = &sm.ring[warp][0][0] + at_off + kDecCodeBytes + g * SCB + t4 * (SCB / 8);
    at_off = at_off == (kDecStages - 1) * STAGE ? 0 : at_off + STAGE;
  };
  // the barrier behind a tile; true: the tile has scales that need fp4_dot
  auto tile_done = [&]() {
    if constexpr (WF == WF_MX4) {
      const bool any = __syncthreads_or(top_scale > Fp4Expand<BF16, WF>::kMx4Top) != 0;
      top_scale = 0;
      return any;
    } else {
      __syncthreads();
      return false;
    }
  };
  auto chunk = [&](const uint8_t* at, int st) {   // st: 0 or 1; the other half of a row is at ^ 64
    return *reinterpret_cast<const uint4*>(st ? reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(at) ^ 64) : at);
  };
#pragma unroll
  for (int s = 0; s < kDecStages; ++s) issue();

  constexpr int NV = WF == WF_16BIT ? 1 : 4;
  // ---- GEMM1 + SiLU ----
  {
    uint4 lo[2][NV] = {}, hi[2][NV] = {};     // of the two halves of a step
    int buf = 0;
    int64_t left = pair1 - pair0;
    int a = static_cast<int>(pair0 / p.I), j0 = static_cast<int>(pair0 - static_cast<int64_t>(a) * p.I);
    const uint16_t* const x0 = p.x + static_cast<int64_t>(g) * p.H + (warp * 8 + t4) * ELT;
    const int64_t x_hi = static_cast<int64_t>(8) * p.H;
    constexpr int XS = kDecWarps * 8 * ELT;             // elements from a warp's step to its next
    const int kb0 = warp * 128 + t4 * 16;
    if constexpr (WF != WF_16BIT) {
      if (left > 0 && warp < nb1) {
        const uint32_t mask = sm.mask[sm.list[a]];
        load_tokens<WF, RAGGED>(x0, (mask >> g) & 1u, kb0 < rb1, lo[0]);
        if constexpr (HI) load_tokens<WF, RAGGED>(x0 + x_hi, (mask >> (g + 8)) & 1u, kb0 < rb1, hi[0]);
      }
    }
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
      int kb = kb0;
      const uint16_t* xp = x0;
      for (int b = warp; b < nb1; b += kDecWarps) {
        if constexpr (WF == WF_16BIT) {
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            const bool in = kb + st * 64 < rb1;
            load_tokens<WF, RAGGED>(xp + st * 4 * ELT, use_lo, in, lo[st]);
            if constexpr (HI) load_tokens<WF, RAGGED>(xp + st * 4 * ELT + x_hi, use_hi, in, hi[st]);
          }
          const uint8_t *at, *no_scales;
          next_stage(at, no_scales);
#pragma unroll
          for (int st = 0; st < 2; ++st)
#pragma unroll
            for (int s = 0; s < 4; ++s) chunk_mma<BF16>(acc[s], chunk(at + s * 1024, st), lo[st][0], hi[st][0]);
        } else {
          auto fetch = [&](int st) {
            const uint16_t* np = xp + 4 * ELT;
            bool in = kb + 64 < rb1, nl = use_lo, nh = use_hi;
            if (st == 1) {
              if (b + kDecWarps < nb1) {
                np = xp + XS;
                in = kb + kDecWarps * 128 < rb1;
              } else {                       // the next tile's first step
                np = x0;
                in = kb0 < rb1 && left > cnt;
                if (in && j0 + cnt == p.I) {
                  const uint32_t m2 = sm.mask[sm.list[a + 1]];
                  nl = (m2 >> g) & 1u;
                  nh = (m2 >> (g + 8)) & 1u;
                }
              }
            }
            load_tokens<WF, RAGGED>(np, nl, in, lo[st ^ 1]);
            if constexpr (HI) load_tokens<WF, RAGGED>(np + x_hi, nh, in, hi[st ^ 1]);
          };
          full_step4<BF16, WF, 4, 1>(acc, lo, hi, fetch, next_stage, top_scale);
        }
        __syncwarp();
        issue();
        kb += kDecWarps * 128;
        xp += XS;
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        float* o = sm.part[buf][warp] + (8 * s + 2 * t4) * PS + g;
        o[0] = acc[s][0];
        o[PS] = acc[s][1];
        if constexpr (HI) {
          o[8] = acc[s][2];
          o[PS + 8] = acc[s][3];
        }
      }
      const bool dots = tile_done();
      {
        const int j = threadIdx.x & 15, t = threadIdx.x >> 4;   // t >= M: the mask has no such bit
        if (j < cnt && ((mask >> t) & 1u)) {
          const int r = (8 * (j >> 2) + (j & 3)) * PS + t;
          float hg = 0.0f, hu = 0.0f;
#pragma unroll
          for (int w = 0; w < kDecWarps; ++w) {
            hg += sm.part[buf][w][r];
            hu += sm.part[buf][w][r + 4 * PS];
          }
          if constexpr (WF != WF_16BIT) {
            const float gl = p.g1 ? __ldg(p.g1 + e) : 1.0f;
            constexpr float U = Fp4Expand<BF16, WF>::kUnit;
            if (fp4_wide_global<BF16, WF>(gl)) hg = hg * gl * U, hu = hu * gl * U;
            else hg *= gl * U, hu *= gl * U;
          }
          if (dots) {
            const int64_t row = static_cast<int64_t>(e) * 2 * p.I + j0 + j;
            const uint16_t* xr = p.x + static_cast<int64_t>(t) * p.H;
            if (mx4_beyond(p.s1 + row * sb1, sb1) || mx4_beyond(p.s1 + (row + p.I) * sb1, sb1)) {
              hg = fp4_dot(p.w1 + row * rb1, p.s1 + row * sb1, xr, p.H);
              hu = fp4_dot(p.w1 + (row + p.I) * rb1, p.s1 + (row + p.I) * sb1, xr, p.H);
            }
          }
          const uint32_t v = pack2<BF16>(silu_f(hg) * hu, 0.0f);
          p.act[(static_cast<int64_t>(a) * p.M + t) * p.I + j0 + j] = static_cast<uint16_t>(v);
        }
      }
      if constexpr (C::PBUFS == 2) buf ^= 1;
      else __syncthreads();
      left -= cnt;
      j0 += cnt;
      if (j0 == p.I) j0 = 0, ++a;
    }
  }
  // ---- every activation is written and visible ----
  __syncthreads();
  if (threadIdx.x == 0) {
    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p.control + DC_COUNT) : "memory");
    const uint32_t asked = __ldcg(p.control + DC_BUDGET), budget = asked ? asked : kDecPolls;
    uint32_t poll = 0, seen;
    while (true) {
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(p.control + DC_COUNT) : "memory");
      if (seen - base >= G) break;
      if (++poll > budget) {
        report(ST_WAIT_TIMEOUT, 0x802);
        sm.ok = 0;
        break;
      }
    }
  }
  __syncthreads();
  if (!sm.ok) {
    cp_async_wait<0>();
    decode_give_up(p, base, epoch);
    return;
  }
  // ---- GEMM2 + weighted sum over the experts ----
  for (int r0 = row0; r0 < row1; r0 += 8 * NS2) {
    constexpr int NT = WF == WF_16BIT ? 4 : 2;
    uint4 lo[NT][NV] = {}, hi[NT][NV] = {};
    float tot[NS2][4], acc[NS2][4];
#pragma unroll
    for (int s = 0; s < NS2; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) tot[s][i] = acc[s][i] = 0.0f;
    // An expert's sum enters a token's total only where the token is routed to it: an infinity or NaN in its weights
    // must not reach the other tokens through a product with zero.
    auto fold = [&](int from) {
      const int e = sm.list[from];
      const uint32_t mask = sm.mask[e];
      float f = 1.0f, last = 1.0f;
      bool wide = false;
      if constexpr (WF != WF_16BIT) {
        last = Fp4Expand<BF16, WF>::kUnit;
        const float gl = p.g2 ? __ldg(p.g2 + e) : 1.0f;
        wide = fp4_wide_global<BF16, WF>(gl);
        f = wide ? gl : gl * last;
      }
      float w_lo = sm.weight[e][g] * f, w_hi = HI ? sm.weight[e][(g + 8) % C::TOKENS] * f : 0.0f;
      if (wide) {
#pragma unroll
        for (int s = 0; s < NS2; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[s][i] *= i < 2 ? w_lo : w_hi;
        w_lo = w_hi = last;
      }
#pragma unroll
      for (int s = 0; s < NS2; ++s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if ((mask >> (i < 2 ? g : g + 8)) & 1u) tot[s][i] = fmaf(i < 2 ? w_lo : w_hi, acc[s][i], tot[s][i]);
          acc[s][i] = 0.0f;
        }
      }
    };
    // the warp's steps in order: (slot, b), then every n2nd-th, on into the next slots
    auto settle = [&](DecodeStep& s) {
      while (s.b >= nb2 && s.slot < n_active) s.b -= nb2, ++s.slot;
    };
    auto operand = [&](const DecodeStep& s) {
      return p.act + (static_cast<int64_t>(s.slot) * p.M + g) * p.I + (s.b * 8 * LN2 + t4) * ELT;
    };
    auto routed = [&](const DecodeStep& s, int row) { return ((sm.mask[sm.list[s.slot]] >> row) & 1u) != 0; };
    const int64_t a_hi = static_cast<int64_t>(8) * p.I;
    // The activations come from L2: those of the next step (4-bit: half step), whichever expert it belongs to, are
    // requested before this one's are used.  (16-bit weights and more than 8 tokens: no registers left for that.)
    constexpr bool AHEAD = WF != WF_16BIT || !HI;
    DecodeStep cur{0, w2nd};
    settle(cur);
    if (AHEAD && cur.slot < n_active) {
      const int kb = cur.b * (128 * LN2) + t4 * 16;
#pragma unroll
      for (int st = 0; st < (WF == WF_16BIT ? 4 : 1); ++st) {
        load_tokens<WF, RAGGED>(operand(cur) + st * 4 * ELT, routed(cur, g), kb + st * 64 < rb2, lo[st]);
        if constexpr (HI) load_tokens<WF, RAGGED>(operand(cur) + a_hi + st * 4 * ELT, routed(cur, g + 8), kb + st * 64 < rb2, hi[st]);
      }
    }
    while (cur.slot < n_active) {
      DecodeStep nxt{cur.slot, cur.b + n2nd};
      settle(nxt);
      const bool more = nxt.slot < n_active;
      const int kb = cur.b * (128 * LN2) + t4 * 16, nkb = nxt.b * (128 * LN2) + t4 * 16;
      if constexpr (WF == WF_16BIT) {
        uint4 nlo[AHEAD ? 4 : 1][NV];
        if constexpr (AHEAD) {
          const uint16_t* np = more ? operand(nxt) : nullptr;
          const bool use = more && routed(nxt, g);
#pragma unroll
          for (int st = 0; st < 4; ++st) {
            nlo[st][0] = lo[st][0];
            load_tokens<WF, RAGGED>(np + st * 4 * ELT, use, more && nkb + st * 64 < rb2, nlo[st]);
          }
        } else {
          const uint16_t* ap = operand(cur);
          const bool use_lo = routed(cur, g), use_hi = routed(cur, g + 8);
#pragma unroll
          for (int st = 0; st < 4; ++st) {
            load_tokens<WF, RAGGED>(ap + st * 4 * ELT, use_lo, kb + st * 64 < rb2, lo[st]);
            load_tokens<WF, RAGGED>(ap + st * 4 * ELT + a_hi, use_hi, kb + st * 64 < rb2, hi[st]);
          }
        }
        const uint8_t *at, *no_scales;
        next_stage(at, no_scales);
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
          for (int s = 0; s < NS2; ++s)
            if (r0 + 8 * s < row1)
              chunk_mma<BF16>(acc[s], chunk(at + s * 1024 + (st >> 1) * 2048, st & 1), lo[st][0], hi[st][0]);
        if constexpr (AHEAD) {
#pragma unroll
          for (int st = 0; st < 4; ++st) lo[st][0] = nlo[st][0];
        }
      } else {
        const uint16_t *ap = operand(cur), *nap = more ? operand(nxt) : ap;
        const bool use_lo = routed(cur, g), use_hi = routed(cur, g + 8);
        const bool nuse_lo = more && routed(nxt, g), nuse_hi = more && routed(nxt, g + 8);
        auto fetch = [&](int st) {
          constexpr int LAST = 2 * LN2 - 1;
          const bool in = st < LAST ? kb + (st + 1) * 64 < rb2 : more && nkb < rb2;
          const uint16_t* np = st < LAST ? ap + (st + 1) * 4 * ELT : nap;
          load_tokens<WF, RAGGED>(np, st < LAST ? use_lo : nuse_lo, in, lo[(st & 1) ^ 1]);
          if constexpr (HI) load_tokens<WF, RAGGED>(np + a_hi, st < LAST ? use_hi : nuse_hi, in, hi[(st & 1) ^ 1]);
        };
        full_step4<BF16, WF, NS2, LN2>(acc, lo, hi, fetch, next_stage, top_scale);
      }
      __syncwarp();
      issue();
      if (nxt.slot != cur.slot) fold(cur.slot);
      cur = nxt;
    }
#pragma unroll
    for (int s = 0; s < NS2; ++s) {
      float* o = sm.part[0][warp] + (8 * s + 2 * t4) * PS + g;
      o[0] = tot[s][0];
      o[PS] = tot[s][1];
      if constexpr (HI) {
        o[8] = tot[s][2];
        o[PS + 8] = tot[s][3];
      }
    }
    const bool dots = tile_done();
    for (int i = threadIdx.x; i < 8 * NS2 * p.M; i += kDecThreads) {
      const int r = i % (8 * NS2), t = i / (8 * NS2);
      if (r0 + r < row1) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) v += sm.part[0][w][r * PS + t];
        if (dots) {                // this CTA's double steps of every expert that has the token
          constexpr int KS = 128 * LN2 * 2;
          bool beyond = false;
          float sum = 0.0f;
          for (int pass = 0; pass < 1 + beyond; ++pass) {       // looks first, adds then
            for (int q = ks * kDecWarps; q < n_active * nb2; q = (q + 1) % kDecWarps ? q + 1 : q + 1 + n2nd - kDecWarps) {
              const int slot = q / nb2, k = (q - slot * nb2) * KS, n = min(KS, p.I - k), e = sm.list[slot];
              if (!((sm.mask[e] >> t) & 1u)) continue;
              const int64_t row = static_cast<int64_t>(e) * p.H + r0 + r;
              const uint8_t* scales = p.s2 + row * sb2 + k / 32;
              if (pass == 0) beyond |= mx4_beyond(scales, n / 32);
              else sum = fmaf(sm.weight[e][t], fp4_dot(p.w2 + row * rb2 + k / 2, scales,
                                                       p.act + (static_cast<int64_t>(slot) * p.M + t) * p.I + k, n), sum);
            }
          }
          if (beyond) v = sum;
        }
        const int64_t at = static_cast<int64_t>(t) * p.H + r0 + r;
        if (p.ksplit == 1) p.out[at] = static_cast<uint16_t>(pack2<BF16>(v, 0.0f));
        else __stcg(p.partial + static_cast<int64_t>(ks) * p.M * p.H + at, v);
      }
    }
    __syncthreads();
  }
  cp_async_wait<0>();
  if (p.ksplit > 1 && second) {
    // whoever comes last of the CTAs that share these rows adds their sums, in the order of their shares of K
    if (threadIdx.x == 0) {
      __threadfence();
      sm.last = atomicAdd(p.control + DC_GROUP + group, 1u) == static_cast<unsigned int>(p.ksplit) - 1u;
      __threadfence();
    }
    __syncthreads();
    if (sm.last) {
      const int rows = row1 - row0;
      for (int i = threadIdx.x; i < rows * p.M; i += kDecThreads) {
        const int64_t at = static_cast<int64_t>(i / rows) * p.H + row0 + i % rows;
        float v = 0.0f;
        for (int s = 0; s < p.ksplit; ++s) v += __ldcg(p.partial + static_cast<int64_t>(s) * p.M * p.H + at);
        p.out[at] = static_cast<uint16_t>(pack2<BF16>(v, 0.0f));
      }
      if (threadIdx.x == 0) p.control[DC_GROUP + group] = 0;
    }
  }
  decode_finish(p, base, epoch);
}

// ---- host ----------------------------------------------------------------------------------------------------
// GEMM2: CTAs per row range, so that a range has about 14 rows.  With fewer the warps' steps hold few bytes and their
// number (active experts * I / 8 warps) times the latency of one is what the product takes: 16 tokens, 64 experts,
// H = I = 512, 1.7 rows per CTA: 68 us, with eight CTAs per range 47.
static int decode_ksplit(int grid, int H) {
  const int k = (grid * 14 + H / 2) / H;
  return k < 1 ? 1 : (k > 16 ? 16 : k);
}
struct DecodeWs {
  size_t logits, partial, act, total;
};
static DecodeWs decode_ws(int64_t M, int H, int I, int E, int topk) {
  auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
  DecodeWs w;
  const int64_t active = M * topk < E ? M * topk : E;
  w.logits = up((DC_GROUP + kDecMaxGroups) * sizeof(unsigned int));  // control words first
  // the tagged logits always have the same place, so that no other call's data is ever taken for one
  w.partial = w.logits + static_cast<size_t>(kDecTokens) * kDecMaxExperts * sizeof(unsigned long long);
  w.act = w.partial + up(static_cast<size_t>(M) * (14 * kDecMaxGroups + H) * sizeof(float));   // ksplit * H of them each
  w.total = w.act + up(static_cast<size_t>(active) * M * I * 2);
  return w;
}

// control words and tagged logits: the same for all sizes
size_t moe_decode_state() { return decode_ws(1, 1, 1, 1, 1).partial; }

size_t moe_decode_workspace(int64_t M, int H, int I, int E, int topk) {
  if (M <= 0 || M > kDecTokens || H <= 0 || I <= 0 || E <= 0 || topk <= 0 || topk > E) return 0;
  return decode_ws(M, H, I, E, topk).total;
}

// HI: more than 8 tokens, the second half of the MMA's row side is used
template <bool BF16, int WF, bool HI, bool RAGGED>
static int launch_decode_rows(const DecodeParams& p, cudaStream_t st) {
  auto kern = moe_decode_kernel<BF16, WF, HI, RAGGED>;
  constexpr int smem = sizeof(DecodeSmem<WF, HI>);
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
    grid = std::min(per_sm, DecodeCfg<WF, HI>::TWO ? 2 : 1) * di.sm_count;
    grids[di.device].store(grid, std::memory_order_release);
  }
  DecodeParams q = p;
  q.ksplit = decode_ksplit(grid, p.H);
  q.groups = grid / q.ksplit;
  if (grid > kDecMaxGroups) return FR_ERR_UNSUPPORTED;
  // router: as many groups of tokens per expert as leave every CTA at most one (expert, group)
  const int groups = std::max(1, std::min(p.M, grid / p.E));
  q.tokens_per_unit = (p.M + groups - 1) / groups;
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

template <bool BF16, int WF>
static int launch_decode(const DecodeParams& p, cudaStream_t st) {
  const int per_line = WF == WF_16BIT ? 64 : 256;       // elements in 128 bytes
  if (p.H % per_line || p.I % (2 * per_line))
    return p.M > 8 ? launch_decode_rows<BF16, WF, true, true>(p, st) : launch_decode_rows<BF16, WF, false, true>(p, st);
  return p.M > 8 ? launch_decode_rows<BF16, WF, true, false>(p, st) : launch_decode_rows<BF16, WF, false, false>(p, st);
}

int moe_decode_dispatch(const void* x, const void* gate, int64_t gsh, int64_t gse, const void* w1, const void* s1,
                        const float* g1, const void* w2, const void* s2, const float* g2, int dtype, int block,
                        int64_t M, int H, int I, int E, int topk, int renormalize, void* out, float* tw, int32_t* ti,
                        void* workspace, size_t workspace_bytes, cudaStream_t st) {
  if (M < 0 || H <= 0 || I <= 0 || E <= 0 || topk <= 0 || topk > E) return FR_ERR_ARG;
  if (block != 0 && block != 16 && block != 32) return FR_ERR_ARG;
  if ((tw == nullptr) != (ti == nullptr)) return FR_ERR_ARG;
  if (dtype != FR_F16 && dtype != FR_BF16) return FR_ERR_UNSUPPORTED;
  if (M > kDecTokens || E > kDecMaxExperts || H > (1 << 22) || I > (1 << 22)) return FR_ERR_UNSUPPORTED;
  if (block == 32 && dtype != FR_BF16) return FR_ERR_UNSUPPORTED;     // E8M0 scales reach beyond fp16
  const int unit = block ? 32 : 8;                                    // 16 bytes of a weight row
  if (H % unit || I % unit) return FR_ERR_ALIGN;
  if (M == 0) return FR_OK;
  if (!x || !gate || !w1 || !w2 || !out || (block && (!s1 || !s2))) return FR_ERR_ARG;
  for (const void* q : {x, w1, w2})
    if (reinterpret_cast<uintptr_t>(q) & 15) return FR_ERR_ALIGN;
  const DecodeWs ws = decode_ws(M, H, I, E, topk);
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
  // the largest copy that every row's start allows (a step's scales are 16 bytes, or 8 for blocks of 32)
  auto scale_copy = [&](const void* s, int k) {
    const uintptr_t u = reinterpret_cast<uintptr_t>(s) | static_cast<uintptr_t>(k / (block ? block : 1));
    return block == 0 ? 0 : (block == 16 && !(u & 15)) ? 16 : !(u & 7) ? 8 : !(u & 3) ? 4 : 0;
  };
  p.scale_copy1 = scale_copy(s1, H);
  p.scale_copy2 = scale_copy(s2, I);
  p.out = static_cast<uint16_t*>(out);
  p.tw = tw;
  p.ti = ti;
  p.control = reinterpret_cast<unsigned int*>(base);
  p.logits = reinterpret_cast<unsigned long long*>(base + ws.logits);
  p.partial = reinterpret_cast<float*>(base + ws.partial);
  p.act = reinterpret_cast<uint16_t*>(base + ws.act);
  const bool bf = dtype == FR_BF16;
  if (block == 0) return bf ? launch_decode<true, WF_16BIT>(p, st) : launch_decode<false, WF_16BIT>(p, st);
  if (block == 16) return bf ? launch_decode<true, WF_NV4>(p, st) : launch_decode<false, WF_NV4>(p, st);
  return launch_decode<true, WF_MX4>(p, st);
}

}  // namespace fr
