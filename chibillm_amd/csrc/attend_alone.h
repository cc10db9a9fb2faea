// Attention of single query rows by vector arithmetic: what a wave of the matrix-core
// prefill kernels falls back to for rows to which a tile gave a value that is not
// finite. HIP device code only.
#pragma once

#include <cfloat>
#include <type_traits>

#include "ckv_internal.h"
#include "prefill_records.h"
#include "prefill_tile.h"

namespace ckv {
namespace {

template <bool F16>
__device__ __forceinline__ float word_value(uint32_t w, int e)
{
    if constexpr (F16)
        return half_value<true>(static_cast<uint16_t>(w >> (16 * e)));
    else
        return __builtin_bit_cast(float, e ? w & 0xFFFF0000u : w << 16);
}

// Sum over each row of 16 lanes, result in every lane of the row.
__device__ __forceinline__ float row16_sum(float v)
{
    auto add = [&](int moved) { v += __builtin_bit_cast(float, moved); };
    const auto bits = [&]() { return __builtin_bit_cast(int, v); };
    add(__builtin_amdgcn_mov_dpp(bits(), 0xB1, 0xF, 0xF, true));  // quad_perm [1,0,3,2]
    add(__builtin_amdgcn_mov_dpp(bits(), 0x4E, 0xF, 0xF, true));  // quad_perm [2,3,0,1]
    add(__builtin_amdgcn_mov_dpp(bits(), 0x141, 0xF, 0xF, true)); // row_half_mirror
    add(__builtin_amdgcn_mov_dpp(bits(), 0x140, 0xF, 0xF, true)); // row_mirror
    return v;
}

// Up to alone_queries rows of one query head (bits of `rows`, from row r0 on) against
// their keys by vector arithmetic: what a wave falls back to for the queries to
// which the tile gave a value that is not finite. A product with P^T
// multiplies every key of a block for all its queries, so an infinity or NaN
// in a V row also meets the zeros of the queries that do not attend it (and of a
// low term), and 0 * inf is NaN; the decode kernels give such a row only to the
// queries that attend it, and so does this. Sixteen lanes hold a row, four rows
// a step, the next step's in flight; finite results never come here. An infinity
// early in a shared prefix sends every query of a launch here, so a K/V row read
// and widened serves several queries: with one in the first page of each
// sequence the launch below takes 1.81 ms (two at a time 2.29, eight 1.96, one
// 5.84; the general path took 3.93 for these rows). The cost grows with the
// rows' positions, as theirs did. (The launch is that of kernels_prefill_wide.hip.)
// WINDOW: the keys that no row of them attends are passed over by the page.
constexpr uint32_t alone_queries = 4;

template <int D, int DT, bool WINDOW, class T>
__device__ __forceinline__ void attend_alone(const T* __restrict__ keys,
                                             const T* __restrict__ values,
                                             const uint32_t* __restrict__ table, uint32_t F,
                                             uint32_t rows, uint32_t pos0, const T* q,
                                             size_t q_stride, float c, const T* gate, T* out,
                                             uint32_t lane, key_window window)
{
    constexpr bool F32 = DT == CKV_F32, F16 = DT == CKV_F16;
    constexpr uint32_t page_tokens = 16;
    constexpr uint32_t each = D / 16, Q = alone_queries, W = each * sizeof(T) / 16;
    const uint32_t f = (lane & 15) * each, sub = lane >> 4;
    struct words {
        u32x4_t w[W];
    };
    auto load = [&](const T* at) {
        words r;
#pragma unroll
        for (uint32_t i = 0; i < W; ++i)
            r.w[i] = reinterpret_cast<const u32x4_t*>(at + f)[i];
        return r;
    };
    auto widen = [](const words& r, float (&x)[each]) {
#pragma unroll
        for (uint32_t i = 0; i < each; ++i)
            if constexpr (F32)
                x[i] = __builtin_bit_cast(float, (uint32_t)r.w[i / 4][i % 4]);
            else
                x[i] = word_value<F16>(r.w[i / 8][i / 2 % 4], i % 2);
    };
    auto weight = [&](float ms, float to) { return __builtin_amdgcn_exp2f((ms - to) * c); };
    // the rows (the first again in the places left over) and their states, which
    // start at the lowest finite maximum: without keys a state weighs 0 or holds 0
    uint32_t row[Q], count = 0;
    float qf[Q][each], acc[Q][each], m[Q], l[Q];
#pragma unroll
    for (uint32_t i = 0; i < Q; ++i) {
        row[i] = rows ? __builtin_ctz(rows) : row[0];
        count += rows != 0;
        rows &= rows - (rows != 0);
        widen(load(q + row[i] * q_stride), qf[i]);
        m[i] = -FLT_MAX;
        l[i] = 0.0f;
#pragma unroll
        for (uint32_t j = 0; j < each; ++j)
            acc[i][j] = 0.0f;
    }
    const uint32_t last = pos0 + row[count - 1]; // the rows ascend
    // the first row's gap, which every row has: keys [gap_begin, gap_end)
    const window_gap gap = WINDOW
        ? window_gap_of(window_low(pos0 + row[0], window), window.sinks, page_tokens)
        : window_gap {};
    const uint32_t gap_begin = gap.kept * page_tokens;
    const uint32_t gap_end = gap_begin + gap.skip * page_tokens;
    const uint32_t first = WINDOW && !gap_begin ? gap_end : 0;
    uint32_t page = table[first / page_tokens];
    auto at_key = [&](uint32_t key) { // in the page at hand; past the last key, that one
        return ((uint64_t)page * page_tokens + min(key, last) % page_tokens) * F;
    };
    words k_next = load(keys + at_key(first + sub)), v_next = load(values + at_key(first + sub));
#pragma unroll 1
    for (uint32_t key0 = first, next; key0 <= last; key0 = next) {
        const words k_now = k_next, v_now = v_next;
        const uint32_t key = key0 + sub;
        next = key0 + 4;
        if (WINDOW && next == gap_begin)
            next = gap_end;
        if (next <= last) {
            if (next % page_tokens == 0)
                page = table[next / page_tokens];
            k_next = load(keys + at_key(next + sub));
            v_next = load(values + at_key(next + sub));
        }
        float x[each], s[Q];
        widen(k_now, x);
#pragma unroll
        for (uint32_t i = 0; i < Q; ++i) {
            s[i] = 0.0f;
#pragma unroll
            for (uint32_t j = 0; j < each; ++j)
                s[i] = __builtin_fmaf(qf[i][j], x[j], s[i]);
            s[i] = row16_sum(s[i]);
        }
        widen(v_now, x);
#pragma unroll
        for (uint32_t i = 0; i < Q; ++i)
            if (key <= pos0 + row[i]
                && (!WINDOW || key >= window_low(pos0 + row[i], window) || key < window.sinks)) {
                const float m_new = fmaxf(m[i], s[i]);
                const float keep = weight(m[i], m_new), w = weight(s[i], m_new);
                m[i] = m_new;
                l[i] = l[i] * keep + w;
#pragma unroll
                for (uint32_t j = 0; j < each; ++j)
                    acc[i][j] = acc[i][j] * keep + w * x[j];
            }
    }
#pragma unroll
    for (uint32_t i = 0; i < Q; ++i) {
#pragma unroll
        for (uint32_t d = 16; d < 64; d *= 2) {
            const float m_other = __shfl_xor(m[i], d), l_other = __shfl_xor(l[i], d);
            const float m_new = fmaxf(m[i], m_other);
            const float keep = weight(m[i], m_new), w = weight(m_other, m_new);
            m[i] = m_new;
            l[i] = l[i] * keep + l_other * w;
#pragma unroll
            for (uint32_t j = 0; j < each; ++j) {
                const float other = __shfl_xor(acc[i][j], d);
                acc[i][j] = acc[i][j] * keep + other * w;
            }
        }
        if (i >= count || sub)
            continue;
        const float inv = 1.0f / l[i];
        const size_t at = row[i] * q_stride + f;
#pragma unroll
        for (uint32_t j = 0; j < each; j += 2) {
            float y[2] = { acc[i][j] * inv, acc[i][j + 1] * inv };
            if (gate)
                for (int e = 0; e < 2; ++e) {
                    if constexpr (F32)
                        y[e] *= sigmoid(gate[at + j + e]);
                    else
                        y[e] *= sigmoid(half_value<F16>(gate[at + j + e]));
                }
            if constexpr (F32)
                *reinterpret_cast<float2*>(out + at + j) = make_float2(y[0], y[1]);
            else
                *reinterpret_cast<uint32_t*>(out + at + j) = pack2<F16>(y[0], y[1]);
        }
    }
}

} // namespace
} // namespace ckv
