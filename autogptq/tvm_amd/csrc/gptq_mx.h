// MXFP4 rows of a key/value cache: what the kernels that write and read them share.
//
// A head's dim values are padded with zeros to whole groups of 32.  A group is 32 codes of 4 bits, a sign and one of 0, 1/2, 1, 3/2, 2,
// 3, 4, 6 (value 2 j in the low half of byte j), and a power of two 2^e, kept as the byte e + 127; 255 makes the group NaN.  A
// row is 16 bytes a group, and its scales lie in a word of their own of 2, 4 or 8 bytes.
//
// Why this form: gfx950 turns two codes and their power of two into two values of fp16 or bf16 in one instruction, exactly (a value has
// two bits of mantissa, and the exponents that a write chooses keep it within the type), so that a row from the cache is an operand of the
// matrix instructions without a rounding of its own.  An error of 0.112 sigma of normal values at 4.25 bits; groups of 32 keep a few large
// channels, as rotated keys have them, to themselves.
#pragma once
#include <hip/hip_runtime.h>

#include "gptq_unpack.h"

namespace gptq {

__host__ __device__ constexpr int mx_groups(int dim) { return (dim + 31) / 32; }
__host__ __device__ constexpr int mx_scale_bytes(int dim) { return dim <= 64 ? 2 : dim <= 128 ? 4 : 8; }

// The two values of byte B of `codes` as 16-bit values of type E.  Of the scale only the exponent counts, so that it may be any
// word with the scale's byte in bits 23 to 30.
template <typename E, int B>
__device__ __forceinline__ uint32_t mx_pair(uint32_t codes, uint32_t scale)
{
    const float s = __builtin_bit_cast(float, scale);
    if constexpr (__is_same(E, _Float16)) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, B));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, B));
}
// the eight values of a word of codes
template <typename E>
__device__ __forceinline__ u4 mx_values(uint32_t codes, uint32_t scale)
{
    return (u4){mx_pair<E, 0>(codes, scale), mx_pair<E, 1>(codes, scale), mx_pair<E, 2>(codes, scale), mx_pair<E, 3>(codes, scale)};
}

// byte `b` of a word of scales to where mx_pair wants it (the rest of the word goes around)
__device__ __forceinline__ uint32_t mx_scale(uint32_t word, uint32_t turn) { return __builtin_amdgcn_alignbit(word, word, turn); }
__device__ __forceinline__ uint32_t mx_turn(int b) { return (8u * (uint32_t)b + 9u) & 31u; }

}  // namespace gptq
