// K and V in 4 bits: blocks of 32 dims that share a power of two (OCP Microscaling Formats 1.0, MXFP4: E2M1 elements, E8M0
// scales), and what its kernels share.
//
// A block of values x with the largest magnitude m: e = floor(log2 m) - 2 (so that m lies in [4, 8) units), at least -127; the
// code of x is that of the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 to |x| / 2^e, ties to the even code, 6 for more, and x's sign
// in bit 3. Dims 2 i and 2 i + 1 are the low and high half of byte i of the row's D / 2; e + 127 is byte b of its D / 32, or
// 255 where the block holds an infinity or a NaN: all of it is NaN then.
//
// The value of a code, 2 bits of significand times a power of two, is exact in bf16: v_cvt_scalef32_pk_bf16_fp4 gives two,
// taking bits 30..23 of its scale operand (a byte shifted there, whatever the other bits are) as the exponent. Measured:
// two values an instruction at full rate.
//
// The matrix instructions that take 4 bits as they are were not used for the scores: they take the other operand in 8
// bits at most (a query would be two such pieces) and align a sum's products to about 2^-13 of its largest: scores off by 4.5e-6
// and at most 8e-5 of unit variance, where bf16 operands gave 9e-8.
#pragma once

#include "mla_common.h"
#include "mla_device.h"

namespace mla {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// A pool's codes [pages, ps, Hkv, D / 2] and scales [pages, ps, Hkv, D / 32], strides in bytes
struct Mx4View {
  uint8_t *codes, *scales;
  int64_t c_page, c_tok, c_head, s_page, s_tok, s_head;
};

// Rows into pools, or out of them
struct Mx4Rows {
  const __bf16 *k, *v;   // [T, Hkv, D]: store
  __bf16 *k_out, *v_out;  // [T, Hkv, D]: load
  int64_t k_stride_t, k_stride_h, v_stride_t, v_stride_h;
  Mx4View k_pool, v_pool;
  const void* indices;  // [T]
  int32_t index_bits, rows, kv_heads, log2_ps;
  int64_t pool_rows;
};
hipError_t launch_mx4_rows(const Mx4Rows& p, int dim, bool load, hipStream_t stream);

// 8 values of a word of codes; the scale in bits 30..23
__device__ __forceinline__ u32x4 mx4_values(uint32_t codes, uint32_t scale) {
  const float f = __uint_as_float(scale);
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, f, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, f, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, f, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, f, 3))};
}

}  // namespace mla
