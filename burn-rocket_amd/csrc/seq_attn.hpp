// Device helpers of the attention kernels on batches of sequences: the fp16 and
// bf16 operand forms, and where 16-key blocks of K and V lie.
#pragma once

#include "attn_common.hpp"

#define ALWAYS_INLINE __attribute__((always_inline))

namespace {
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));

// D += A·B on 16x16 tiles, 32 deep; operands as 16-byte registers.
template <int DT>
__device__ __forceinline__ floatx4 mfma16(uintx4 a, uintx4 b, floatx4 c) {
  if constexpr (DT == RK_DTYPE_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// Two values rounded to nearest even, packed.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (DT == RK_DTYPE_F16)
    return __builtin_bit_cast(uint32_t, half2_{(f16)x, (f16)y});
  else
    return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)x, (__bf16)y});
}
// Two probabilities as two values of the type each: cut off to the type, and what that
// leaves. Together they hold 2^-16 of the value (bf16; fp16 2^-20): with one value, as
// accurate as a result's own rounding, results of rows with few keys that nearly cancel
// were off by up to 9e-2 (bf16) and 1.1e-2 (fp16) of their size, above the 1e-2 that the
// single-sequence attention is held to.
template <int DT>
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
  if constexpr (DT == RK_DTYPE_F16) {
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(minus_half_lo(hi, x), minus_half_hi(hi, y)));
  } else {
    const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
    hi = __builtin_amdgcn_perm(b, a, 0x07060302);  // the upper halves
    lo = pack2<DT>(x - __uint_as_float(a & 0xffff0000u), y - __uint_as_float(b & 0xffff0000u));
  }
}
// Probabilities are kept times 2^P_BIAS: fp16's smallest normal value is then
// 2^-20 of the largest one, the sums have the same factor.
constexpr float P_BIAS = 6.0f;

// Four values of column l % 16 from four consecutive 16-value rows in LDS (the
// transposing read): p is this lane's 8 bytes of row (l % 16) / 4.
__device__ __forceinline__ shortx4 lds_read_tr16(const uint8_t *p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4 *)(p));
}
__device__ __forceinline__ uintx4 join8(shortx4 a, shortx4 b) {
  return __builtin_bit_cast(uintx4, shortx8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
}

// Where the 16-key blocks of an item's keys lie, for one kv head: a lane knows one
// block, and a wave that needs block i takes its descriptor from lane i. Keys from the
// item's end on (which no row of its tile sees, or another part has) and blocks below
// the first key that one sees read as zeros. V's keys below it in its own block do too
// (hidden_below): a probability of 0 times a NaN or an infinity would reach every row.
struct KeyBlocks {
  uint32_t lo, hi, bytes;
};
// The block from key key0 on; page: its page id (paged).
template <bool PAGED>
__device__ __forceinline__ KeyBlocks key_blocks(const SeqAttnArgs &a, const SeqItem &it, const void *base,
                                                int64_t tok_stride, int kvh, int key0, int page) {
  const int rows = key0 + 15 < it.k_lo ? 0 : max(0, min(16, it.k_end - key0));
  const int D = a.head_dim;
  int64_t at;
  KeyBlocks b;  // (strides are below SEQ_MAX_STRIDE)
  if constexpr (PAGED) {
    at = ((((int64_t)page * a.n_kv_heads + kvh) << a.page_log2) + (key0 & ((1 << a.page_log2) - 1))) * D;
    b.bytes = (uint32_t)(rows * D * 2);
  } else {
    at = (int64_t)(it.tok0 + key0) * tok_stride + (int64_t)kvh * D;
    b.bytes = rows > 0 ? (uint32_t)(((rows - 1) * (int)tok_stride + D) * 2) : 0;
  }
  const uint64_t addr = (uint64_t)base + (uint64_t)at * 2;
  b.lo = (uint32_t)addr;
  b.hi = (uint32_t)(addr >> 32) & 0xffff;
  return b;
}
// Whether row `row` of the block from key key0 on lies below the first key that a row of
// the item's tile sees.
__device__ __forceinline__ bool hidden_below(const SeqItem &it, int key0, int row) { return row < it.k_lo - key0; }
__device__ __forceinline__ rsrc_t block_rsrc(const KeyBlocks &b, int i) {
  const uint32_t lo = __builtin_amdgcn_readlane(b.lo, i), hi = __builtin_amdgcn_readlane(b.hi, i);
  return __builtin_amdgcn_make_buffer_rsrc((void *)((uint64_t)hi << 32 | lo), (short)0, __builtin_amdgcn_readlane(b.bytes, i),
                                           RSRC_WORD3);
}
}  // namespace
