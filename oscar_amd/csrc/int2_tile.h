// The 32-token key tiles of the packed INT2 history as operands of the 32x32x16 MFMA: the
// history values with the reference's rounding, looked up per code, and the element order
// that they, the current chunk's rows and the queries share (attn_decode.hip,
// attn_weights.hip).
#pragma once

#include "common.h"

namespace oscar {

typedef _Float16 __attribute__((ext_vector_type(2))) f16x2;
typedef __bf16 __attribute__((ext_vector_type(2))) bf16x2;
typedef float __attribute__((ext_vector_type(2))) f32x2;

// Query dtype QT (OSCAR_BF16 or OSCAR_F16): the dtype of the QK operands, of the
// slow tiles' V values and of P in their PV.
//
// reference history rounding q_dtype(fp16(x)) (streaming_attention.py:124) of a pair
// (a -> low half, b -> high half) with the packed RNE conversions v_cvt_pk_f16_f32
// (/ v_cvt_f32_f16 / v_cvt_pk_bf16_f32 for bf16 queries)
template <int QT>
__device__ __forceinline__ unsigned hist_pair(float a, float b) {
  const f16x2 h = __builtin_convertvector(f32x2{a, b}, f16x2);
  if constexpr (QT == OSCAR_F16) {
    return __builtin_bit_cast(unsigned, h);
  } else {
    const f32x2 w = __builtin_convertvector(h, f32x2);
    return __builtin_bit_cast(unsigned, __builtin_convertvector(w, bf16x2));
  }
}
// pair (RNE) of two floats in the query dtype, and the value of its half k
template <int QT>
__device__ __forceinline__ unsigned q_pair(float a, float b) {
  if constexpr (QT == OSCAR_F16) return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, f16x2));
  else return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
template <int QT>
__device__ __forceinline__ float q_half(unsigned pair, int k) {
  const unsigned bits = k ? pair >> 16 : pair & 0xffffu;
  if constexpr (QT == OSCAR_F16) return f16_bits_to_f32(bits);
  else return __uint_as_float(bits << 16);
}
// 8 query-dtype elements (one MFMA operand per lane)
template <int QT> struct QVec { typedef bf16x8 type; };
template <> struct QVec<OSCAR_F16> { typedef f16x8 type; };
// C += A B (32x32x16 MFMA) with operands in the query dtype, given as packed words
template <int QT>
__device__ __forceinline__ f32x16 mma16(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (QT == OSCAR_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

// token of S^T output register r for lane half g (also the O^T row of register r)
__device__ __forceinline__ int out_tok(int r, int g) { return 8 * (r >> 2) + 4 * g + (r & 3); }

// history value table of one token, q_dtype(fp16(c*scale + zero)) for c = 0..3
template <int QT>
__device__ __forceinline__ void value_table(unsigned scale_zero, unsigned& lo, unsigned& hi) {
  const float s = f16_bits_to_f32(scale_zero & 0xffff), z = f16_bits_to_f32(scale_zero >> 16);
  float v[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] = __fadd_rn(__fmul_rn((float)c, s), z);  // mul, then add
  lo = hist_pair<QT>(v[0], v[1]);
  hi = hist_pair<QT>(v[2], v[3]);
}

// bf16 pairs of 16 elements (lo = e0..e7, hi = e8..e15) in the K-step order of lut16:
// (e0,e4) (e1,e5) (e2,e6) (e3,e7) | (e8,e12) (e9,e13) (e10,e14) (e11,e15)
__device__ __forceinline__ void kpairs16(const u32x4& lo, const u32x4& hi, unsigned o[8]) {
  o[0] = __builtin_amdgcn_perm(lo[2], lo[0], 0x05040100u);
  o[1] = __builtin_amdgcn_perm(lo[2], lo[0], 0x07060302u);
  o[2] = __builtin_amdgcn_perm(lo[3], lo[1], 0x05040100u);
  o[3] = __builtin_amdgcn_perm(lo[3], lo[1], 0x07060302u);
  o[4] = __builtin_amdgcn_perm(hi[2], hi[0], 0x05040100u);
  o[5] = __builtin_amdgcn_perm(hi[2], hi[0], 0x07060302u);
  o[6] = __builtin_amdgcn_perm(hi[3], hi[1], 0x05040100u);
  o[7] = __builtin_amdgcn_perm(hi[3], hi[1], 0x07060302u);
}

// the four history values of a token as byte tables: t_lo = low bytes of the 16-bit
// values for codes 0..3, t_hi = their high bytes
template <int QT>
__device__ __forceinline__ void byte_tables(unsigned scale_zero, unsigned& t_lo, unsigned& t_hi) {
  unsigned lo, hi;
  value_table<QT>(scale_zero, lo, hi);
  t_lo = __builtin_amdgcn_perm(hi, lo, 0x06040200u);
  t_hi = __builtin_amdgcn_perm(hi, lo, 0x07050301u);
}

// bf16 values of the 16 codes of one code dword (byte j holds elements 4j..4j+3 at
// bits 2k), in the pair order of kpairs16.  Per k: the four codes 4j + k as bytes
// select table bytes directly (v_perm_b32 selectors 0..3), one perm each for the low
// and high bytes, then two perms interleave them into bf16 pairs: 23 VALU per dword.
__device__ __forceinline__ void lut16(unsigned w, unsigned t_lo, unsigned t_hi, unsigned o[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const unsigned x = (w >> (2 * k)) & 0x03030303u;
    const unsigned lo = __builtin_amdgcn_perm(t_hi, t_lo, x);
    const unsigned hi = __builtin_amdgcn_perm(t_lo, t_hi, x);
    o[k] = __builtin_amdgcn_perm(hi, lo, 0x05010400u);      // (e_k, e_4+k)
    o[4 + k] = __builtin_amdgcn_perm(hi, lo, 0x07030602u);  // (e_8+k, e_12+k)
  }
}

}  // namespace oscar
