// Keys and values held in 4 bits: the numbers, the pages' layout and the conversions.
//
// A number is a 4-bit float (sign, two exponent bits, one mantissa bit: 0, 1/2, 1, 3/2, 2, 3,
// 4, 6 and their negatives) times its block's scale, a power of two. A block is 32 consecutive
// features of a head; its scale is 2^(floor(log2 m) - 2) for the block's largest magnitude m,
// kept as the biased exponent in a byte, so that m / scale is in [4, 8). Numbers round to the
// nearest, ties to the even code, and those past 6 (m / scale above 7 loses at most a quarter)
// become 6. A scale is no smaller than 2^-23 for f16 rows, whose smallest number is then half
// of it, and 2^-100 for others: every cached number is one of the rows' type, and of bf16, so
// that the matrix cores take it exactly. A block with an infinity or NaN, or rotated past the
// type's range, has scale byte 255: all of it reads as NaN. 17 bytes a block, 4.25 bits a
// number: against bf16 a decode step reads 3.76 times as many tokens in its time.
//
// gfx950 converts a pair of codes with its scale in one full-rate instruction (measured:
// 4.7 cycles a wave against 4.4 of an addition), so a K or V operand of a matrix
// instruction costs one vector instruction for each two numbers. The layout serves them:
// 16 tokens of a head stand together (a tile), codes first, then scales, keys and values
// each in an order in which a wave's loads are contiguous and what a lane loads is what it
// feeds to v_mfma_f32_16x16x32_bf16:
//   K: codes [token][feature]; scales [token][block]. Lane (c, g) = (lane % 16, lane / 16)
//      takes D/4 features of token c, of block g (of each 128 features; 64-wide heads: the
//      16 from 16g on): the contraction runs over features in an order of its own, which
//      the query operand follows.
//   V: codes [feature part][g][c][token 4g..4g+3][features]: lane (c, g) takes 8 features
//      (64-wide heads: 4) from 8c on of tokens 4g..4g+3, with parts of 128 features; scales
//      [block][token]. A token's codes are whole words of its own, so an append touches no
//      other token's.
#pragma once

#include "ckv_internal.h"

namespace ckv {

// Bytes of a tile: 16 tokens of one head of `head_dim` features, keys or values.
__host__ __device__ constexpr uint32_t fp4_tile_bytes(uint32_t head_dim)
{
    return 8 * head_dim + head_dim / 2;
}
constexpr uint32_t fp4_tile = 16; // tokens

__host__ __device__ constexpr bool fp4_head_dim(size_t head_dim)
{
    return head_dim == 64 || head_dim == 128 || head_dim == 256;
}

// The first byte of the tile that holds `slot`'s token of a head, within a layer.
__host__ __device__ inline uint64_t fp4_tile_at(uint32_t slot, uint32_t head, uint32_t block_size,
                                                uint32_t kv_heads, uint32_t head_dim)
{
    const uint64_t page = slot / block_size;
    const uint32_t tile = slot % block_size / fp4_tile, tiles = block_size / fp4_tile;
    return ((page * kv_heads + head) * tiles + tile) * fp4_tile_bytes(head_dim);
}

// Places within a tile: of token t's codes of the 8 features from 8w on (`v`: in V's order),
// of 64-wide heads' values also the four from 8w + 4 on (+ 8), and of a block's scale.
__host__ __device__ constexpr uint32_t fp4_word_at(uint32_t head_dim, uint32_t t, uint32_t w, bool v)
{
    if (!v)
        return t * (head_dim / 2) + 4 * w;
    if (head_dim == 64)
        return t / 4 * 128 + 2 * w * 8 + t % 4 * 2;
    return w / 16 * 1024 + t / 4 * 256 + w % 16 * 16 + t % 4 * 4;
}
__host__ __device__ constexpr uint32_t fp4_scale_at(uint32_t head_dim, uint32_t t, uint32_t block, bool v)
{
    return 8 * head_dim + (v ? block * fp4_tile + t : t * (head_dim / 32) + block);
}

constexpr int fp4_least_exponent(int dtype)
{
    return dtype == CKV_F16 ? -23 : -100;
}

#if defined(__HIPCC__)
namespace {

typedef __bf16 fp4_bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 fp4_f16x2_t __attribute__((ext_vector_type(2)));

// The scale byte of a block from the biased exponent (of 127) of its largest magnitude, 255
// for an infinity or NaN, and for what f16 has no number for: rotated rows reach 2^16.
template <int DT>
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t biased)
{
    constexpr int least = 127 + fp4_least_exponent(DT);
    return biased >= (DT == CKV_F16 ? 127u + 16 : 255u) ? 255 : (uint32_t)max((int)biased - 2, least);
}

__device__ __forceinline__ float fp4_scale(uint32_t byte)
{
    return __builtin_bit_cast(float, byte << 23); // 255: the conversions below give NaN
}

// Byte SEL of a code word, two numbers times the scale, as a packed pair.
template <int SEL>
__device__ __forceinline__ uint32_t fp4_bf16_pair(uint32_t word, float scale)
{
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, SEL));
}
template <int SEL, bool F16>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t word, float scale)
{
    if constexpr (F16)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, SEL));
    else
        return fp4_bf16_pair<SEL>(word, scale);
}

// Eight numbers as 16-bit pairs.
template <bool F16>
__device__ __forceinline__ uint4 fp4_eight(uint32_t word, float scale)
{
    return make_uint4(fp4_pair<0, F16>(word, scale), fp4_pair<1, F16>(word, scale),
                      fp4_pair<2, F16>(word, scale), fp4_pair<3, F16>(word, scale));
}

// Codes of eight floats over a scale.
__device__ __forceinline__ uint32_t fp4_codes(const float (&x)[8], float scale)
{
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
}

// A double in (-8, 8) as the float on the same side of every 4-bit border: cut off, with
// the last bit set where something was. (Rounded to the nearest, it could meet a border.)
// Under 1/8 only the sign counts.
__device__ __forceinline__ float fp4_side(double y)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, y);
    const uint32_t hi = (uint32_t)(b >> 32), lo = (uint32_t)b;
    const uint32_t magnitude = (hi & 0x7FFFFFFFu) < 0x3FC00000u
        ? 0
        : (((hi & 0x7FFFFFFFu) - (896u << 20)) << 3) | (lo >> 29) | ((lo & 0x1FFFFFFFu) != 0);
    return __builtin_bit_cast(float, (hi & 0x80000000u) | magnitude);
}

} // namespace
#endif

} // namespace ckv
