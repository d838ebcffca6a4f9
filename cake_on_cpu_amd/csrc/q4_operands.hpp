// q4_operands.hpp -- codes and rows of x as the matrix pipe takes them: what the kernels of the
// 4-bit linear layer share.
//
// Codes are whole numbers 0..15, exact in 16-bit floats, so the products go to the matrix pipe as
// x . code and the group's scale and zero point are applied to the 32-bit sums behind it:
//   y[m][n] = sum over groups g of s[n][g] * (sum_k x[m][k] code[n][k] - z[n][g] * sum_k x[m][k]).
// No weight is rounded.  (Codes less their zero point would keep the two sums from cancelling, but bf16 pairs
// have no addition: through fp32 it is 20 vector instructions for 8 codes in place of 7.)  The sums are larger
// than what they stand for, up to 15 x 128 of the largest x before the scale is applied, so where x reaches as
// far as fp32 does, codes and column sums count in units of 2^-12 (exact, by the unpacking's own scale) and the
// result is multiplied by 2^12 at its end: no sum overflows where the values do not.  x is exact as well:
// 16-bit types go in as they are, a 32-bit x as three bf16 pieces (its leading, middle and last 8 significant
// bits, cut, not rounded, so that no piece overflows) that take three rows of the product and are added up at
// the end.
#pragma once

#include "low_bits.hpp"

namespace cake {

template <int TYPE> struct Codes;   // what the matrix pipe multiplies: code * UNIT
template <> struct Codes<CAKE_HIP_F16> {
    typedef f16x8 V;
    static constexpr float UNIT = 1.f, UNPACK = 512.f * UNIT;
    static __device__ __forceinline__ unsigned pair(unsigned bytes, bool upper)
    {
        return upper ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, UNPACK, true))
                     : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, UNPACK, false));
    }
    static constexpr unsigned ONES = 0x3C003C00u;   // UNIT
    static __device__ __forceinline__ floatx4 mfma(uintx4 a, uintx4 b, floatx4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
};
template <> struct Codes<CAKE_HIP_BF16> {
    typedef bf16x8 V;
    static constexpr float UNIT = 0x1p-12f, UNPACK = 512.f * UNIT;
    static __device__ __forceinline__ unsigned pair(unsigned bytes, bool upper)
    {
        return upper ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes, UNPACK, true))
                     : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes, UNPACK, false));
    }
    static constexpr unsigned ONES = 0x39803980u;   // UNIT
    static __device__ __forceinline__ floatx4 mfma(uintx4 a, uintx4 b, floatx4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
};
template <> struct Codes<CAKE_HIP_F32> : Codes<CAKE_HIP_BF16> {};

template <int TYPE> constexpr int pieces_of() { return TYPE == CAKE_HIP_F32 ? 3 : 1; }

template <int TYPE>
__device__ __forceinline__ uintx4 unpack_codes(unsigned word)
{
    const unsigned low = word & 0x0F0F0F0Fu, high = (word >> 4) & 0x0F0F0F0Fu;
    uintx4 b;
    b[0] = Codes<TYPE>::pair(low, false);
    b[1] = Codes<TYPE>::pair(low, true);
    b[2] = Codes<TYPE>::pair(high, false);
    b[3] = Codes<TYPE>::pair(high, true);
    return b;
}

// Eight consecutive elements of a row of x, zero from `left` on.  Rows start at any element: the
// hardware's 16-byte loads take any address.
template <int TYPE>
__device__ __forceinline__ void load_eight(const typename Element<TYPE>::T* at, int left, typename Element<TYPE>::T (&v)[8])
{
    typedef typename Element<TYPE>::T T;
    if (left >= 8) {
        __builtin_memcpy(v, at, sizeof v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < left ? at[e] : (T)0.f;
    }
}

// piece p of eight elements as the matrix pipe takes them
template <int TYPE>
__device__ __forceinline__ uintx4 piece_of(const typename Element<TYPE>::T (&v)[8], int p)
{
    uintx4 out;
    if constexpr (TYPE == CAKE_HIP_F32) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            unsigned half[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float rest = v[e + j];
                unsigned cut = __builtin_bit_cast(unsigned, rest) & 0xFFFF0000u;
                for (int i = 0; i < p; ++i) {
                    rest -= __builtin_bit_cast(float, cut);   // exact: the bits behind the cut
                    cut = __builtin_bit_cast(unsigned, rest) & 0xFFFF0000u;
                }
                half[j] = cut;
            }
            out[e / 2] = (half[0] >> 16) | half[1];
        }
    } else {
        struct alignas(16) Eight { typename Element<TYPE>::T e[8]; } all;
#pragma unroll
        for (int e = 0; e < 8; ++e) all.e[e] = v[e];
        out = __builtin_bit_cast(uintx4, all);
    }
    return out;
}

}  // namespace cake
