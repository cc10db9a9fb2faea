// The results of a wave's 32 query rows on their way from accumulators to memory: the
// epilogue of the windowed prefill kernels. HIP device code only.
#pragma once

#include "ckv_internal.h"
#include "prefill_tile.h"

namespace ckv {
namespace {

// An accumulator holds four features of each row: stored from there, an instruction
// writes 16 or 32 bytes (two lanes) of each of 32 rows 4 KB apart, and the L2 takes a
// request for every one. So the floats go through LDS, a wave's own part of the stages,
// and leave as whole rows, 16 bytes a lane (32 prompts of 128 rows, half of whose bytes
// are outputs, 19.0 and 15.0 us; 64 of 64 14.6 and 12.9).
template <int D>
constexpr uint32_t row_floats = D + 4; // a row's pitch in LDS: 16 rows on other banks

// Rows 0 .. n_rows - 1 but those of `skip`, from `tile` [32][row_floats], times
// sigmoid(gate), rounded once, to out[row * stride + feature]. (Unrolled no further: the
// code that follows the key blocks is fetched cold.)
template <int D, int DT, class T>
__device__ __forceinline__ void store_rows(const float* tile, uint32_t lane, uint32_t n_rows,
                                           uint32_t skip, T* out, size_t stride, const T* gate)
{
    constexpr uint32_t each = 16 / sizeof(T), lanes = D / each, rows = 64 / lanes;
    const uint32_t f = lane % lanes * each;
#pragma unroll 2
    for (uint32_t i = 0; i < 32 / rows; ++i) {
        const uint32_t r = i * rows + lane / lanes;
        float x[each];
#pragma unroll
        for (uint32_t j = 0; j < each; j += 4)
            *reinterpret_cast<float4*>(x + j) =
                *reinterpret_cast<const float4*>(tile + r * row_floats<D> + f + j);
        if (r >= n_rows || skip >> r & 1)
            continue;
        const size_t at = r * stride + f;
        uint4 w;
        if constexpr (DT == CKV_F32) {
            if (gate) { // sigmoid_mul (src/qwen/qwen_layer.cc:204) in the epilogue
                const float4 v = *reinterpret_cast<const float4*>(gate + at);
                x[0] *= sigmoid(v.x);
                x[1] *= sigmoid(v.y);
                x[2] *= sigmoid(v.z);
                x[3] *= sigmoid(v.w);
            }
            w = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                           __float_as_uint(x[3]));
        } else {
            constexpr bool F16 = DT == CKV_F16;
            if (gate) {
                const uint4 v = *reinterpret_cast<const uint4*>(gate + at);
                const uint32_t words[4] = { v.x, v.y, v.z, v.w };
#pragma unroll
                for (uint32_t e = 0; e < each; ++e)
                    x[e] *= sigmoid(half_value<F16>((uint16_t)(words[e / 2] >> (16 * (e % 2)))));
            }
            w = make_uint4(pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3]), pack2<F16>(x[4], x[5]),
                           pack2<F16>(x[6], x[7]));
        }
        *reinterpret_cast<uint4*>(out + at) = w;
    }
}

} // namespace
} // namespace ckv
