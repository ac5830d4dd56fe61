// Block-scaled fp8 (e4m3) operands on gfx950: the quantizer's arithmetic, the resident weight layout and the matrix
// products, shared by the dense and the expert kernels.
#pragma once

#include "common.hpp"

typedef int intx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int FP8_BLOCK = 128;  // values per scale along K; rows per weight scale along N

// A block's scale: its largest magnitude lands on the largest e4m3 value. An infinite value makes the scale infinite and
// its row's results NaN; a NaN does not reach amax and becomes the NaN code itself.
__device__ __forceinline__ float fp8_scale(float amax) { return fmaxf(amax / 448.0f, 1e-12f); }

// The largest of 16 neighbouring lanes' values, in all of them: rotations inside the vector instruction.
template <int CTRL>
__device__ __forceinline__ float fp8_rotated(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float fp8_max16(float x) {
  x = fmaxf(x, fp8_rotated<0x121>(x));  // by 1, 2, 4 and 8 lanes
  x = fmaxf(x, fp8_rotated<0x122>(x));
  x = fmaxf(x, fp8_rotated<0x124>(x));
  return fmaxf(x, fp8_rotated<0x128>(x));
}

// x / s as an f32 number, with the reciprocal of s taken once per block: the residual of the product with the reciprocal
// corrects it to the rounded quotient. Codes are rounded from that number, so that they do not depend on how a division
// is carried out: ties are common, since x and amax have few bits.
struct Fp8Div {
  float r, s;
  __device__ __forceinline__ explicit Fp8Div(float scale) {
    const bool inf = scale > 3.4e38f;
    r = inf ? 0.f : 1.0f / scale;
    s = inf ? 0.f : scale;
  }
  __device__ __forceinline__ float operator()(float x) const {
    const float q = x * r;
    return __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-q, s, x), r, q), x);  // (-0 stays -0)
  }
};
// Four quotients to their codes (nearest even; |q| <= 448 up to a rounding, which stays on the largest code).
__device__ __forceinline__ uint32_t fp8_codes4(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

// The resident layout of a weight [N, K]: blocks of 32 rows and 128 K-values, 4 KB each, [N/32][K/128], rows and K padded
// with zeros to multiples of 128. Inside a block 16-byte chunk c = 4s + 2h + j of row r lies at ((2s + j)·2 + h)·512 + 16·r:
// each of a wave's four loads of a block is 1 KB in one piece, lane 32h + r holding chunk (s, j) of its row, which is also
// the operand layout of the 32×32 products. Scales [N/128][K/128].
__host__ __device__ inline int64_t fp8_offset(int64_t r, int64_t k, int kt) {
  const int c = (int)(k % 128) / 16;
  return ((r / 32) * kt + k / 128) * 4096 + (((c >> 2) * 2 + (c & 1)) * 2 + ((c >> 1) & 1)) * 512 + (r % 32) * 16 + k % 16;
}

// One operand of a 32-row, 128-value block: as it lies (products of fp8 codes), or widened to bf16, which holds every code
// exactly. The fp8 products (2·64 K-values) are twice as fast, but align the terms of a sum to the largest and cut them
// there: 1.4e-5 of a result's size on normally distributed codes (2^-16), where the bf16 products' sums are those of f32.
// That is far below a bf16 or fp16 rounding; results that stay f32 take the bf16 products, those of one block of K, and those
// that are quantized again (a code that flips is a sixteenth of its value) in front of fp16 results or in tiles of few rows:
// one token's result of 8 experts is then off by 1.6e-3 of its size, as the bf16 rounding alone has it, instead of 3.8e-3,
// for 19.2 us instead of 18.1. In tiles of many rows, where the products are what bounds the time, the flips of a bf16
// layer's codes stay: 2.3e-3 instead of 1.7e-3.
template <bool EXACT>
struct Fp8Frag;
template <>
struct Fp8Frag<false> {
  intx8 f[2];
  __device__ __forceinline__ void set(int s, intx4 j0, intx4 j1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[s][i] = j0[i];
      f[s][4 + i] = j1[i];
    }
  }
};
template <>
struct Fp8Frag<true> {
  bf16x8 f[8];
  __device__ __forceinline__ void widen(int at, int lo, int hi) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    f[at] = bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
  __device__ __forceinline__ void set(int s, intx4 j0, intx4 j1) {
    widen(4 * s, j0[0], j0[1]);
    widen(4 * s + 1, j0[2], j0[3]);
    widen(4 * s + 2, j1[0], j1[1]);
    widen(4 * s + 3, j1[2], j1[3]);
  }
};
// The 32 × 32 product of two blocks' codes, by halves of the block: rows 8·(r/4) + 4·(lane/32) + r%4 of `a` in register r, column lane%32 of `b`.
// With the weight as `a` a lane holds one token's results for 16 outputs: one scale of its own, and one of the weight that
// is the same for all.
__device__ __forceinline__ floatx16 fp8_half(const Fp8Frag<false> &a, const Fp8Frag<false> &b, int s, floatx16 p) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a.f[s], b.f[s], p, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ floatx16 fp8_half(const Fp8Frag<true> &a, const Fp8Frag<true> &b, int s, floatx16 p) {
#pragma unroll
  for (int i = 0; i < 4; ++i) p = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.f[4 * s + i], b.f[4 * s + i], p, 0, 0, 0);
  return p;
}
template <bool EXACT>
__device__ __forceinline__ floatx16 fp8_product(const Fp8Frag<EXACT> &a, const Fp8Frag<EXACT> &b) {
  return fp8_half(a, b, 1, fp8_half(a, b, 0, floatx16{}));
}

// silu(g) · u in f32: g / (1 + e^-g) · u. Behind products of the fp8 instructions (2^-16), by the exponential and reciprocal
// instructions, whose steps of 2^-23 or so (|g|·2^-24 for the exponent's) are nothing to that: a tenth of an expert tile's
// time for the exact forms.
template <bool EXACT>
__device__ __forceinline__ float fp8_silu_mul(float g, float u) {
  if constexpr (EXACT) return g / (1.0f + expf(-g)) * u;
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504f)) * u;
}

// Four f32 values to a type's bits, by the conversion instructions (nearest even; a NaN stays one).
template <int DT>
__device__ __forceinline__ void fp8_encode4(void *to, const float *v) {
  if constexpr (DT == RK_DTYPE_BF16) {
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    *(bf16x4 *)to = bf16x4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
  } else {
    dt_store_vec<DT, 4>(to, 0, v);
  }
}
// Four consecutive values of a row of c (element type known at run time), `n` of them inside the row. In one store at any
// address, which gfx950 has: the rows of an odd length begin anywhere.
__device__ __forceinline__ void fp8_store4(void *c, int dt, int64_t at, const float *v, int n) {
  if (n >= 4) {
    typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef uint32_t words2 __attribute__((ext_vector_type(2), aligned(2)));
    uint16_t h[4] __attribute__((aligned(8)));
    if (dt == RK_DTYPE_F32) {
      *(words4 *)((float *)c + at) = words4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
      return;
    }
    if (dt == RK_DTYPE_F16) fp8_encode4<RK_DTYPE_F16>(h, v);
    else fp8_encode4<RK_DTYPE_BF16>(h, v);
    *(words2 *)((uint16_t *)c + at) = __builtin_bit_cast(uintx2, h);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n) {
      if (dt == RK_DTYPE_F32) dt_store<RK_DTYPE_F32>(c, at + e, v[e]);
      else if (dt == RK_DTYPE_F16) dt_store<RK_DTYPE_F16>(c, at + e, v[e]);
      else dt_store<RK_DTYPE_BF16>(c, at + e, v[e]);
    }
}
