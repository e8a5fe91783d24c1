// Microscaled 4-bit floating point: E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two per byte with
// the even element in the low half, and one scale per block of consecutive elements of a row:
//   block 16: scale E4M3, and one fp32 scale per matrix:  value = code * scale * global
//   block 32: scale E8M0 (a power of two):                value = code * scale
// This file holds the conversions; the product of two such matrices is in fr_fp4_gemm.cu.
#include "fr_common.cuh"

namespace fr {

constexpr float kFp4GlobalDiv = 2688.0f;                 // 448 * 6: the largest scale times the largest code
constexpr float kFp4GlobalMin = 7.70371977754894e-34f;   // 2^-110: 1 / (smallest E4M3 * global) stays finite
constexpr uint32_t kF32Inf = 0x7F800000u;

__device__ __forceinline__ float f32_pow2(int e) {   // 2^e, -127 <= e <= 127
  return __uint_as_float(e > -127 ? static_cast<uint32_t>(e + 127) << 23 : 0x00400000u);
}

// E4M3 byte -> fp32 (0x7F / 0xFF are NaN); E8M0 byte -> fp32 (0xFF is NaN)
__device__ __forceinline__ float e4m3_f32(uint32_t b) {
  if ((b & 0x7Fu) == 0x7Fu) return __uint_as_float(0x7FC00000u);
  // the fields of E4M3 placed in fp32 are the value times 2^-120, subnormals included
  const float v = __uint_as_float(((b & 0x7Fu) << 20) | ((b & 0x80u) << 24));
  return __fmul_rn(v, 1.329227995784916e36f);        // 2^120
}
__device__ __forceinline__ float e8m0_f32(uint32_t b) {
  return b == 0xFFu ? __uint_as_float(0x7FC00000u) : f32_pow2(static_cast<int>(b) - 127);
}

// eight values -> eight codes, nearest, ties to even, saturated at 6; element i in bits 4i..4i+3
__device__ __forceinline__ uint32_t cvt8_e2m1(const float (&v)[8]) {
  uint32_t r;
  asm("{\n"
      ".reg .b8 b0, b1, b2, b3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      "mov.b32 %0, {b0, b1, b2, b3};\n"
      "}\n"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// eight codes -> eight values as four half2 (every E2M1 value is exact in fp16)
__device__ __forceinline__ void cvt8_f16(uint32_t codes, uint32_t (&h)[4]) {
  asm("{\n"
      ".reg .b8 b0, b1, b2, b3;\n"
      "mov.b32 {b0, b1, b2, b3}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n"
      "}\n"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
}

__device__ __forceinline__ void cvt4_f16(uint16_t codes, uint32_t (&h)[2]) {
  asm("{\n"
      ".reg .b8 b0, b1;\n"
      "mov.b16 {b0, b1}, %2;\n"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n"
      "}\n"
      : "=r"(h[0]), "=r"(h[1])
      : "h"(codes));
}

__device__ __forceinline__ uint8_t cvt_e4m3(float v) {   // nearest even, saturated at 448; v is not NaN
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
  return static_cast<uint8_t>(r);
}

struct Fp4QuantParams {
  const void* x;
  int64_t ld_mat, ld_row;    // elements
  int64_t rows;
  int groups;                // cols / 16
  float* partial;            // [mats][parts] largest magnitude of the finite blocks (bits of a non-negative fp32)
  int parts;
  int own_global;            // 1: the global scale comes from the data and is written; 0: it is read; block 16 only
  float* global_scale;       // [mats]
  uint8_t* q;
  uint8_t* scale;
};

// sixteen consecutive elements of a row as fp32
template <int DT, bool VEC>
__device__ __forceinline__ void load16(const void* x, int64_t at, float (&v)[16]) {
  if constexpr (DT == FR_F32) {
    const float* p = static_cast<const float*>(x) + at;
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(p) + i);
        v[4 * i] = f.x;
        v[4 * i + 1] = f.y;
        v[4 * i + 2] = f.z;
        v[4 * i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = __ldg(p + i);
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(x) + at;
    uint32_t w[8];
    if constexpr (VEC) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(p)), b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
      w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i] = static_cast<uint32_t>(__ldg(p + 2 * i)) | (static_cast<uint32_t>(__ldg(p + 2 * i + 1)) << 16);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = unpack2<DT == FR_BF16>(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

// bits of the largest magnitude; as unsigned integers infinities and NaN compare above every finite value
__device__ __forceinline__ uint32_t amax_bits16(const float (&v)[16]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return m;
}

__device__ __forceinline__ uint32_t block_max(uint32_t m, uint32_t* red) {
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  uint32_t t = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) t = max(t, red[w]);
  __syncthreads();
  return t;
}

__device__ __forceinline__ float fp4_global(uint32_t amax) {
  return amax == 0 ? 1.0f : fmaxf(__fdiv_rn(__uint_as_float(amax), kFp4GlobalDiv), kFp4GlobalMin);
}

// Largest magnitude of each matrix over its finite blocks of 16: one partial per CTA, read back by the kernel below
// (no atomics, nothing to clear first).
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) fp4_amax_kernel(const Fp4QuantParams p) {
  __shared__ uint32_t red[8];
  const int64_t mat = blockIdx.y, total = p.rows * p.groups;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  uint32_t m = 0;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
    const int64_t row = i / p.groups, g = i - row * p.groups;
    float v[16];
    load16<DT, VEC>(p.x, mat * p.ld_mat + row * p.ld_row + g * 16, v);
    const uint32_t a = amax_bits16(v);
    if (a < kF32Inf) m = max(m, a);
  }
  m = block_max(m, red);
  if (threadIdx.x == 0) p.partial[mat * p.parts + blockIdx.x] = __uint_as_float(m);
}

// One thread quantises sixteen elements.  SMALL: one CTA per matrix finds the global scale itself first (a few rows:
// one launch instead of two).  The scale of a block that holds an infinity or a NaN is NaN and its codes are zero.
template <int DT, bool VEC, int BLOCK, bool SMALL>
__global__ void __launch_bounds__(256) fp4_quantize_kernel(const Fp4QuantParams p) {
  __shared__ uint32_t red[8];
  const int64_t mat = blockIdx.y, total = p.rows * p.groups;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  float global = 1.0f, six_g = 6.0f;
  if constexpr (BLOCK == 16) {
    if (p.own_global) {
      uint32_t m = 0;
      if constexpr (SMALL) {
        for (int64_t i = threadIdx.x; i < total; i += blockDim.x) {
          const int64_t row = i / p.groups, g = i - row * p.groups;
          float v[16];
          load16<DT, VEC>(p.x, mat * p.ld_mat + row * p.ld_row + g * 16, v);
          const uint32_t a = amax_bits16(v);
          if (a < kF32Inf) m = max(m, a);
        }
      } else {
        for (int i = threadIdx.x; i < p.parts; i += blockDim.x)
          m = max(m, __float_as_uint(__ldcg(p.partial + mat * p.parts + i)));
      }
      global = fp4_global(block_max(m, red));
      if (blockIdx.x == 0 && threadIdx.x == 0) p.global_scale[mat] = global;
    } else {
      global = __ldg(p.global_scale + mat);
    }
    six_g = __fmul_rn(6.0f, global);
  }
  // every lane of a warp takes part in the exchange below, so the bound of the loop is the warp's
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * blockDim.x + (threadIdx.x & ~31); i0 < total; i0 += step) {
    const int64_t i = i0 + (threadIdx.x & 31);
    const bool in = i < total;
    const int64_t row = in ? i / p.groups : 0, g = in ? i - row * p.groups : 0;
    float v[16];
    if (in) {
      load16<DT, VEC>(p.x, mat * p.ld_mat + row * p.ld_row + g * 16, v);
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = 0.0f;
    }
    uint32_t a = amax_bits16(v);
    if constexpr (BLOCK == 32) a = max(a, __shfl_xor_sync(0xffffffffu, a, 1));   // groups is even: both in one row
    if (!in) continue;
    float inv;
    uint8_t sc;
    if constexpr (BLOCK == 16) {
      sc = cvt_e4m3(__fdiv_rn(__uint_as_float(a < kF32Inf ? a : 0u), six_g));
      const float unit = __fmul_rn(e4m3_f32(sc), global);
      const bool ok = unit >= 1.17549435e-38f;       // also false for a NaN: the block becomes zero
      inv = ok ? __frcp_rn(unit) : 0.0f;
      if (!ok) sc = 0;
      if (a >= kF32Inf) sc = 0x7F;
    } else {
      // 2^(floor(log2 amax) - 2): the largest element lands in [4, 8) and saturates at 6
      int e = static_cast<int>(a >> 23) - 127 - 2;
      e = e < -127 ? -127 : e;
      sc = static_cast<uint8_t>(e + 127);
      inv = a < kF32Inf ? f32_pow2(-e) : 0.0f;
      if (a >= kF32Inf) sc = 0xFF;
    }
    uint2 codes = make_uint2(0, 0);
    if (inv != 0.0f && a < kF32Inf) {
      float lo[8], hi[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        lo[k] = __fmul_rn(v[k], inv);
        hi[k] = __fmul_rn(v[8 + k], inv);
      }
      codes = make_uint2(cvt8_e2m1(lo), cvt8_e2m1(hi));
    }
    reinterpret_cast<uint2*>(p.q)[mat * total + i] = codes;
    if constexpr (BLOCK == 16) p.scale[mat * total + i] = sc;
    else if (!(i & 1)) p.scale[(mat * total + i) >> 1] = sc;
  }
}

// value = code * (scale * global), the product of the scales rounded to fp32 first.  A thread writes 16 bytes, so that a
// warp's store covers whole lines (sixteen elements per thread, two half-sector stores: 42 us for 16384 x 4096 to fp16).
template <int DT, int BLOCK>
__global__ void __launch_bounds__(256) fp4_dequantize_kernel(const uint8_t* __restrict__ q,
                                                             const uint8_t* __restrict__ scale,
                                                             const float* __restrict__ global_scale, int64_t per_mat,
                                                             void* __restrict__ out) {
  constexpr int N = DT == FR_F32 ? 4 : 8;            // elements per thread
  constexpr int U = 4;                               // loads in flight
  const int64_t mat = blockIdx.y;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const float global = (BLOCK == 16 && global_scale) ? __ldg(global_scale + mat) : 1.0f;
  for (int64_t j0 = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; j0 < per_mat; j0 += U * step) {
    uint32_t code[U];
    uint8_t sc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t j = j0 + u * step, i = mat * per_mat + j;
      if (j < per_mat) {
        if constexpr (N == 8) code[u] = __ldg(reinterpret_cast<const uint32_t*>(q) + i);
        else code[u] = __ldg(reinterpret_cast<const uint16_t*>(q) + i);
        sc[u] = __ldg(scale + i / (BLOCK / N));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t j = j0 + u * step, i = mat * per_mat + j;
      if (j >= per_mat) break;
      const float unit = BLOCK == 16 ? __fmul_rn(e4m3_f32(sc[u]), global) : e8m0_f32(sc[u]);
      if constexpr (N == 4) {
        uint32_t h[2];
        cvt4_f16(static_cast<uint16_t>(code[u]), h);
        const float2 a = unpack2<false>(h[0]), b = unpack2<false>(h[1]);
        reinterpret_cast<float4*>(out)[i] =
            make_float4(__fmul_rn(a.x, unit), __fmul_rn(a.y, unit), __fmul_rn(b.x, unit), __fmul_rn(b.y, unit));
      } else {
        uint32_t h[4], r[4];
        cvt8_f16(code[u], h);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 v = unpack2<false>(h[k]);
          r[k] = pack2<DT == FR_BF16>(__fmul_rn(v.x, unit), __fmul_rn(v.y, unit));
        }
        reinterpret_cast<uint4*>(out)[i] = make_uint4(r[0], r[1], r[2], r[3]);
      }
    }
  }
}

// CTAs per matrix of the amax pass; also the number of partials the quantising kernel reads back
static int fp4_parts(int64_t mats, int64_t rows, int64_t cols) {
  const int64_t groups = rows * (cols / 16);
  int64_t want = (groups + 255) / 256;
  int64_t cap = 1184 / (mats < 1 ? 1 : mats);       // eight CTAs per SM over all matrices
  cap = cap < 8 ? 8 : cap;
  return static_cast<int>(want < 1 ? 1 : (want < cap ? want : cap));
}
// a matrix of at most this many elements is handled by one CTA in one launch (8 x 4096: 1.5 us of one SM's loads)
constexpr int64_t kFp4SmallElems = 32768;

template <int DT, bool VEC, int BLOCK>
static int fp4_quantize_launch(Fp4QuantParams p, int64_t mats, int64_t cols, cudaStream_t st) {
  const int64_t groups = p.rows * p.groups;
  if constexpr (BLOCK == 16) {
    if (p.own_global && p.rows * cols <= kFp4SmallElems) {
      fp4_quantize_kernel<DT, VEC, 16, true><<<dim3(1, static_cast<unsigned>(mats)), 256, 0, st>>>(p);
      return static_cast<int>(cudaGetLastError());
    }
    if (p.own_global) {
      fp4_amax_kernel<DT, VEC><<<dim3(p.parts, static_cast<unsigned>(mats)), 256, 0, st>>>(p);
      FR_CUDA_OK(cudaGetLastError());
    }
  }
  int64_t ctas = (groups + 255) / 256;
  const int64_t cap = 16 * 148;
  if (ctas > cap) ctas = cap;
  fp4_quantize_kernel<DT, VEC, BLOCK, false><<<dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(mats)), 256, 0,
                                               st>>>(p);
  return static_cast<int>(cudaGetLastError());
}

template <int DT>
static int fp4_quantize_block(const Fp4QuantParams& p, int64_t mats, int64_t cols, int block, bool vec,
                              cudaStream_t st) {
  if (block == 16)
    return vec ? fp4_quantize_launch<DT, true, 16>(p, mats, cols, st) : fp4_quantize_launch<DT, false, 16>(p, mats, cols, st);
  return vec ? fp4_quantize_launch<DT, true, 32>(p, mats, cols, st) : fp4_quantize_launch<DT, false, 32>(p, mats, cols, st);
}

size_t fp4_quantize_workspace(int64_t mats, int64_t rows, int64_t cols) {
  if (mats <= 0 || rows <= 0 || cols <= 0 || rows * cols <= kFp4SmallElems) return 0;
  return (static_cast<size_t>(mats) * fp4_parts(mats, rows, cols) * sizeof(float) + 255) & ~size_t(255);
}

int fp4_quantize_dispatch(const void* x, int dtype, int64_t mats, int64_t rows, int64_t cols, int64_t ld_mat,
                          int64_t ld_row, int block, float* global_scale, int own_global, void* q, void* scale,
                          void* workspace, size_t workspace_bytes, cudaStream_t st) {
  if (mats < 0 || rows < 0 || cols <= 0 || (block != 16 && block != 32)) return FR_ERR_ARG;
  if (mats == 0 || rows == 0) return FR_OK;
  if (!x || !q || !scale || (block == 16 && !global_scale)) return FR_ERR_ARG;
  if (dtype != FR_F16 && dtype != FR_BF16 && dtype != FR_F32) return FR_ERR_UNSUPPORTED;
  if (cols % block || mats > 65535 || cols > (int64_t(1) << 30)) return FR_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(q) & 7)) return FR_ERR_ALIGN;
  if (block == 16 && own_global) {
    const size_t need = fp4_quantize_workspace(mats, rows, cols);
    if (need && (!workspace || workspace_bytes < need)) return FR_ERR_WORKSPACE;
  }
  Fp4QuantParams p;
  p.x = x;
  p.ld_mat = ld_mat;
  p.ld_row = ld_row;
  p.rows = rows;
  p.groups = static_cast<int>(cols / 16);
  p.partial = static_cast<float*>(workspace);
  p.parts = fp4_parts(mats, rows, cols);
  p.own_global = own_global;
  p.global_scale = global_scale;
  p.q = static_cast<uint8_t*>(q);
  p.scale = static_cast<uint8_t*>(scale);
  const int elt = dtype == FR_F32 ? 4 : 2;
  const bool vec = !(reinterpret_cast<uintptr_t>(x) & 15) && (ld_row * elt) % 16 == 0 && (mats == 1 || (ld_mat * elt) % 16 == 0);
  switch (dtype) {
    case FR_F16: return fp4_quantize_block<FR_F16>(p, mats, cols, block, vec, st);
    case FR_BF16: return fp4_quantize_block<FR_BF16>(p, mats, cols, block, vec, st);
    default: return fp4_quantize_block<FR_F32>(p, mats, cols, block, vec, st);
  }
}

template <int BLOCK>
static int fp4_dequantize_launch(const void* q, const void* scale, const float* global_scale, int64_t mats,
                                 int64_t elems, int dtype, void* out, cudaStream_t st) {
  const int64_t per_mat = elems / (dtype == FR_F32 ? 4 : 8);
  int64_t ctas = (per_mat + 255) / 256;
  if (ctas > 16 * 148) ctas = 16 * 148;
  const dim3 grid(static_cast<unsigned>(ctas), static_cast<unsigned>(mats));
  const uint8_t* qv = static_cast<const uint8_t*>(q);
  const uint8_t* sv = static_cast<const uint8_t*>(scale);
  switch (dtype) {
    case FR_F16: fp4_dequantize_kernel<FR_F16, BLOCK><<<grid, 256, 0, st>>>(qv, sv, global_scale, per_mat, out); break;
    case FR_BF16: fp4_dequantize_kernel<FR_BF16, BLOCK><<<grid, 256, 0, st>>>(qv, sv, global_scale, per_mat, out); break;
    default: fp4_dequantize_kernel<FR_F32, BLOCK><<<grid, 256, 0, st>>>(qv, sv, global_scale, per_mat, out); break;
  }
  return static_cast<int>(cudaGetLastError());
}

int fp4_dequantize_dispatch(const void* q, const void* scale, const float* global_scale, int64_t mats, int64_t rows,
                            int64_t cols, int block, int dtype, void* out, cudaStream_t st) {
  if (mats < 0 || rows < 0 || cols <= 0 || (block != 16 && block != 32)) return FR_ERR_ARG;
  if (mats == 0 || rows == 0) return FR_OK;
  if (!q || !scale || !out) return FR_ERR_ARG;
  if (dtype != FR_F16 && dtype != FR_BF16 && dtype != FR_F32) return FR_ERR_UNSUPPORTED;
  if (cols % block || mats > 65535) return FR_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(q) & 7) || (reinterpret_cast<uintptr_t>(out) & 15)) return FR_ERR_ALIGN;
  return block == 16 ? fp4_dequantize_launch<16>(q, scale, global_scale, mats, rows * cols, dtype, out, st)
                     : fp4_dequantize_launch<32>(q, scale, global_scale, mats, rows * cols, dtype, out, st);
}

}  // namespace fr
