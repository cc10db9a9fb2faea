// Rotary embedding in its forms (pairs of halves or of neighbours, part of the head,
// frequencies scaled for long contexts, lengths by a magnitude), its fusion with the KV
// append, and the append to and the reading of a cache held in 4 bits (fp4.h).
//
// Within each head of a row, pair j < rotary/2 is elements (j, j + rotary/2) or
// (2j, 2j + 1); a row at position p turns it by p * step[j] (rotation_table; exact
// fractions of a turn, rope_turns.h) and multiplies it by the magnitude; elements past
// the rotary width are copied. Queries, keys and values of a layer go through one launch.
//
// A key on its way to 4 bits is turned in 64 bits: which code it gets then depends on no
// rounding before its own (its angle holds to 2^-50 of a radian), whatever the order of
// the operations, and the caches of two programs agree. That costs little: the device
// does as many 64-bit products a clock as 32-bit ones, and the angle's 20 serve a row's
// heads together.
#include "ckv_internal.h"
#include "fp4.h"
#include "rope_turns.h"

#include <cmath>

namespace ckv {
namespace {

constexpr uint32_t block_threads = 256;

// Sine and cosine of a turned angle in 64 bits: the quadrant from the turn's top bits,
// the Taylor series of the rest (an eighth of a turn at most) to x^15 and x^16, cut off
// below 2^-54.
__device__ __forceinline__ void sincos_turn64(uint64_t step, uint64_t position, double& s, double& c)
{
    const uint64_t turn = step * position; // of 2^64
    const uint64_t quadrant = (turn + (1ull << 61)) >> 62;
    const double x = (double)(int64_t)(turn - (quadrant << 62)) * 3.4061215800304775e-19; // 2 pi / 2^64
    const double z = x * x;
    double ps = fma(z, -1.0 / 1307674368000.0, 1.0 / 6227020800.0);
    ps = fma(z, ps, -1.0 / 39916800.0);
    ps = fma(z, ps, 1.0 / 362880.0);
    ps = fma(z, ps, -1.0 / 5040.0);
    ps = fma(z, ps, 1.0 / 120.0);
    ps = fma(z, ps, -1.0 / 6.0);
    ps = fma(x * z, ps, x);
    double pc = fma(z, 1.0 / 20922789888000.0, -1.0 / 87178291200.0);
    pc = fma(z, pc, 1.0 / 479001600.0);
    pc = fma(z, pc, -1.0 / 3628800.0);
    pc = fma(z, pc, 1.0 / 40320.0);
    pc = fma(z, pc, -1.0 / 720.0);
    pc = fma(z, pc, 1.0 / 24.0);
    pc = fma(z, pc, -0.5);
    pc = fma(z, pc, 1.0);
    const double a = quadrant & 1 ? pc : ps, b = quadrant & 1 ? ps : pc;
    s = quadrant & 2 ? -a : a;
    c = (quadrant + 1) & 2 ? -b : b;
}

// Rows whose rotary and head widths are whole pairs of 16-byte words: a thread takes two
// words of PER heads of a row, with the pairs p0 .. p0 + each - 1: a word of the first half
// and the one it is turned with, or the two words of neighbouring pairs; past the rotary
// width two words that are copied. Heads from q_heads on are keys, whose values go along.
template <int DT, bool PAIRS, int PER>
__device__ __forceinline__ void rotate_words(uint64_t item, const pool_view& p,
                                             const uint32_t* __restrict__ slots, uint32_t layer,
                                             const rotate_rows& x, uint32_t rows, uint32_t q_heads,
                                             uint32_t heads, const rotation_table& by,
                                             const uint32_t* __restrict__ positions)
{
    using E = turn_element<DT>;
    using T = typename E::type;
    constexpr uint32_t each = 16 / sizeof(T); // elements of a word
    union word {
        uint4 v;
        T e[each];
    };
    const uint32_t d = p.head_dim, half = by.rotary / 2;
    const uint32_t groups = d / (2 * each), parts = (heads + PER - 1) / PER;
    const uint32_t row = (uint32_t)(item / (groups * parts));
    if (row >= rows)
        return;
    const uint32_t rest = (uint32_t)(item % (groups * parts));
    const uint32_t p0 = rest % groups * each, head0 = rest / groups * PER;
    const bool turned = p0 < half;
    const uint32_t at = turned && !PAIRS ? p0 : 2 * p0, apart = turned && !PAIRS ? half : each;
    const uint64_t q_row = (uint64_t)row * q_heads * d, k_row = (uint64_t)row * p.features;
    word a[PER], b[PER];
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const uint32_t h = min(head0 + i, heads - 1); // past the last head: it again
        const T* src = (h < q_heads ? static_cast<const T*>(x.queries) + q_row + h * d
                                    : static_cast<const T*>(x.keys) + k_row + (h - q_heads) * d)
            + at;
        a[i].v = *reinterpret_cast<const uint4*>(src);
        b[i].v = *reinterpret_cast<const uint4*>(src + apart);
    }
    const uint64_t slot_row = heads > q_heads && head0 + PER > q_heads // rotated alone, rows have no slots
        ? layer * p.layer_elems + (uint64_t)slots[row] * p.features
        : 0;
    float c[each], s[each];
    if (turned) {
#pragma unroll
        for (uint32_t e = 0; e < each; ++e) {
            sincos_turn(by.turns.step[p0 + e], positions[row], s[e], c[e]);
            s[e] *= by.magnitude;
            c[e] *= by.magnitude;
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const uint32_t h = head0 + i;
        if (h >= heads)
            break;
        float fa[each], fb[each];
#pragma unroll
        for (uint32_t e = 0; e < each; ++e) {
            fa[e] = E::load(a[i].e[e]);
            fb[e] = E::load(b[i].e[e]);
        }
        if (turned) {
#pragma unroll
            for (uint32_t e = 0; e < each; ++e) {
                float& first = PAIRS ? (2 * e < each ? fa : fb)[2 * e % each] : fa[e];
                float& second = PAIRS ? (2 * e < each ? fa : fb)[2 * e % each + 1] : fb[e];
                rope_pair(first, second, c[e], s[e], first, second);
            }
        }
        if (x.float_queries && h < q_heads) {
            float* to = static_cast<float*>(x.rotated) + q_row + h * d + at;
#pragma unroll
            for (uint32_t e = 0; e < each; e += 4) {
                *reinterpret_cast<float4*>(to + e) = make_float4(fa[e], fa[e + 1], fa[e + 2], fa[e + 3]);
                *reinterpret_cast<float4*>(to + apart + e) = make_float4(fb[e], fb[e + 1], fb[e + 2], fb[e + 3]);
            }
            continue;
        }
        if (turned) {
#pragma unroll
            for (uint32_t e = 0; e < each; ++e) {
                a[i].e[e] = E::store(fa[e]);
                b[i].e[e] = E::store(fb[e]);
            }
        }
        T* dst;
        if (h < q_heads) {
            dst = static_cast<T*>(x.rotated) + q_row + h * d + at;
        } else {
            const uint32_t in_row = (h - q_heads) * d + at;
            const T* vs = static_cast<const T*>(x.values) + k_row + in_row;
            T* vd = static_cast<T*>(p.values) + slot_row + in_row;
            const uint4 va = *reinterpret_cast<const uint4*>(vs);
            const uint4 vb = *reinterpret_cast<const uint4*>(vs + apart);
            *reinterpret_cast<uint4*>(vd) = va;
            *reinterpret_cast<uint4*>(vd + apart) = vb;
            if (x.held_values) {
                T* hv = static_cast<T*>(x.held_values) + k_row + in_row;
                *reinterpret_cast<uint4*>(hv) = va;
                *reinterpret_cast<uint4*>(hv + apart) = vb;
            }
            if (x.held_keys) {
                T* hk = static_cast<T*>(x.held_keys) + k_row + in_row;
                *reinterpret_cast<uint4*>(hk) = a[i].v;
                *reinterpret_cast<uint4*>(hk + apart) = b[i].v;
            }
            dst = static_cast<T*>(p.keys) + slot_row + in_row;
        }
        *reinterpret_cast<uint4*>(dst) = a[i].v;
        *reinterpret_cast<uint4*>(dst + apart) = b[i].v;
    }
}

template <int DT, bool PAIRS, int PER>
__global__ __launch_bounds__(block_threads) void rotate_words_kernel(
    pool_view p, const uint32_t* __restrict__ slots, uint32_t layer, rotate_rows x, uint32_t rows,
    uint32_t q_heads, uint32_t heads, rotation_table by, const uint32_t* __restrict__ positions)
{
    rotate_words<DT, PAIRS, PER>((uint64_t)blockIdx.x * block_threads + threadIdx.x, p, slots, layer,
                                 x, rows, q_heads, heads, by, positions);
}

// Any other geometry: one thread per (head, pair) and grid row per row.
template <int DT>
__global__ __launch_bounds__(block_threads) void rotate_pairs_kernel(
    pool_view p, const uint32_t* __restrict__ slots, uint32_t layer, rotate_rows x, uint32_t rows,
    uint32_t q_heads, uint32_t heads, rotation_table by, const uint32_t* __restrict__ positions)
{
    using E = turn_element<DT>;
    using T = typename E::type;
    const uint32_t d = p.head_dim, half = by.rotary / 2, pairs = (d + 1) / 2;
    const uint32_t t = blockIdx.x * block_threads + threadIdx.x;
    const uint32_t head = t / pairs, pair = t % pairs;
    if (head >= heads)
        return;
    const bool query = head < q_heads, turned = pair < half;
    // the pair's two elements within the head (of an odd head's last pair one)
    const uint32_t a = turned && !by.neighbours ? pair : 2 * pair;
    const uint32_t b = turned && !by.neighbours ? pair + half : min(a + 1, d - 1);
    const uint32_t at = query ? head * d : (head - q_heads) * d; // the head in its row
    for (uint32_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const uint64_t width = query ? (uint64_t)q_heads * d : p.features;
        const T* src = static_cast<const T*>(query ? x.queries : x.keys) + row * width + at;
        T o1 = src[a], o2 = src[b];
        float r1 = E::load(o1), r2 = E::load(o2);
        if (turned) {
            float s, c;
            sincos_turn(by.turns.step[pair], positions[row], s, c);
            rope_pair(r1, r2, c * by.magnitude, s * by.magnitude, r1, r2);
            o1 = E::store(r1);
            o2 = E::store(r2);
        }
        if (query && x.float_queries) {
            float* dst = static_cast<float*>(x.rotated) + row * width + at;
            dst[a] = r1;
            dst[b] = r2;
            continue;
        }
        const auto put = [&](void* to, uint64_t first, T v1, T v2) {
            T* dst = static_cast<T*>(to) + first;
            dst[a] = v1;
            dst[b] = v2;
        };
        if (query) {
            put(x.rotated, row * width + at, o1, o2);
        } else {
            const uint64_t in = row * width + at;
            const uint64_t dst = layer * p.layer_elems + (uint64_t)slots[row] * p.features + at;
            const T* vs = static_cast<const T*>(x.values) + in;
            const T v1 = vs[a], v2 = vs[b];
            put(p.keys, dst, o1, o2);
            put(p.values, dst, v1, v2);
            if (x.held_keys)
                put(x.held_keys, in, o1, o2);
            if (x.held_values)
                put(x.held_values, in, v1, v2);
        }
    }
}

// Eight elements of a row; VECTOR: read in 16-byte words.
template <int DT>
union eight {
    using T = typename turn_element<DT>::type;
    uint4 v[sizeof(T) / 2];
    T e[8];
    __device__ __forceinline__ float at(uint32_t i) const { return turn_element<DT>::load(e[i]); }
};

template <int DT, bool VECTOR>
__device__ __forceinline__ eight<DT> load_eight(const void* base, uint64_t at)
{
    using T = typename eight<DT>::T;
    const T* src = static_cast<const T*>(base) + at;
    eight<DT> x;
    if constexpr (VECTOR) {
#pragma unroll
        for (uint32_t i = 0; i < sizeof(T) / 2; ++i)
            x.v[i] = reinterpret_cast<const uint4*>(src)[i];
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            x.e[i] = src[i];
    }
    return x;
}

// Eight numbers of a code word as the rows' type.
template <int DT, bool VECTOR>
__device__ __forceinline__ void store_codes(void* base, uint64_t at, uint32_t word, float scale)
{
    using T = typename turn_element<DT>::type;
    T* dst = static_cast<T*>(base) + at;
    const uint4 h = fp4_eight<DT == CKV_F16>(word, scale);
    const uint32_t w[4] = { h.x, h.y, h.z, h.w };
    T e[8];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
        if constexpr (DT == CKV_F32)
            e[i] = __builtin_bit_cast(float, i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
        else
            e[i] = (T)(w[i / 2] >> (16 * (i % 2)));
    if constexpr (VECTOR && DT == CKV_F32) {
        reinterpret_cast<float4*>(dst)[0] = make_float4(e[0], e[1], e[2], e[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(e[4], e[5], e[6], e[7]);
    } else if constexpr (VECTOR) {
        *reinterpret_cast<uint4*>(dst) = h;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            dst[i] = e[i];
    }
}

// The largest of a block's four lanes.
__device__ __forceinline__ uint32_t block_max(uint32_t v)
{
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true)); // quad_perm [1,0,3,2]
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true)); // quad_perm [2,3,0,1]
}

// A row's code word `w` and, from the block's first lane, the scale into a tile.
__device__ __forceinline__ void store_fp4(uint8_t* tile, uint32_t d, uint32_t token, uint32_t w, bool v,
                                          uint32_t codes, uint32_t byte)
{
    uint8_t* at = tile + fp4_word_at(d, token, w, v);
    if (v && d == 64) {
        *reinterpret_cast<uint16_t*>(at) = (uint16_t)codes;
        *reinterpret_cast<uint16_t*>(at + 8) = (uint16_t)(codes >> 16);
    } else {
        *reinterpret_cast<uint32_t*>(at) = codes;
    }
    if (w % 4 == 0)
        tile[fp4_scale_at(d, token, w / 4, v)] = (uint8_t)byte;
}

// One thread per (row, PER kv heads, word of 8 features), the four words of a block in
// neighbouring lanes; the word's angles serve its heads. VECTOR: rows in 16-byte words,
// rotary a multiple of 16.
template <int DT, bool PAIRS, bool VECTOR, int PER>
__device__ __forceinline__ void fp4_append(uint64_t item, const pool_view& p,
                                           const uint32_t* __restrict__ slots, uint32_t layer,
                                           const rotate_rows& x, uint32_t rows,
                                           const rotation_table& by,
                                           const uint32_t* __restrict__ positions)
{
    constexpr uint32_t angles = PAIRS ? 4 : 8; // of a word's features
    const uint32_t d = p.head_dim, half = by.rotary / 2, words = d / 8;
    const uint32_t parts = (p.kv_heads + PER - 1) / PER;
    const uint32_t row = (uint32_t)(item / (words * parts));
    if (row >= rows) // whole blocks of lanes
        return;
    const uint32_t rest = (uint32_t)(item % (words * parts));
    const uint32_t w = rest % words, head0 = rest / words * PER, f0 = 8 * w;
    const uint64_t at_row = (uint64_t)row * p.features + f0;
    const bool turned = f0 < by.rotary;
    eight<DT> k[PER], other[PAIRS ? 1 : PER], v[PER];
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const uint64_t at = at_row + min(head0 + i, p.kv_heads - 1) * d; // past the last head: it again
        k[i] = load_eight<DT, VECTOR>(x.keys, at);
        v[i] = load_eight<DT, VECTOR>(x.values, at);
        if constexpr (!PAIRS) {
            if (turned) {
                if constexpr (VECTOR) {
                    other[i] = load_eight<DT, true>(x.keys, f0 < half ? at + half : at - half);
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) {
                        const uint32_t f = f0 + e, o = f < half ? f + half : f < by.rotary ? f - half : f;
                        other[i].e[e] = static_cast<const typename eight<DT>::T*>(x.keys)[at - f0 + o];
                    }
                }
            }
        }
    }
    const uint32_t slot = slots[row], position = positions[row];
    double s[angles], c[angles];
    if (turned) {
#pragma unroll
        for (uint32_t e = 0; e < angles; ++e) {
            const uint32_t f = PAIRS ? f0 + 2 * e : f0 + e;
            if (!VECTOR && f >= by.rotary)
                break;
            sincos_turn64(by.turns.step[PAIRS ? f / 2 : f < half ? f : f - half], position, s[e], c[e]);
            s[e] *= by.magnitude64;
            c[e] *= by.magnitude64;
        }
    }
    const uint64_t layer_at = layer * ((uint64_t)p.blocks * p.block_size / fp4_tile * p.kv_heads * fp4_tile_bytes(d));
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const uint32_t head = head0 + i;
        if (head >= p.kv_heads)
            break;
        double y[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e)
            y[e] = k[i].at(e);
        if (turned) {
#pragma unroll
            for (uint32_t e = 0; e < angles; ++e) {
                const uint32_t f = PAIRS ? f0 + 2 * e : f0 + e;
                if (!VECTOR && f >= by.rotary)
                    break;
                if constexpr (PAIRS) {
                    const double a = y[2 * e], b = y[2 * e + 1];
                    y[2 * e] = a * c[e] - b * s[e];
                    y[2 * e + 1] = b * c[e] + a * s[e];
                } else {
                    const double o = other[i].at(e);
                    y[e] = f < half ? y[e] * c[e] - o * s[e] : y[e] * c[e] + o * s[e];
                }
            }
        }
        // the largest magnitudes' exponents, biased as a float's
        uint32_t largest_k = 0, largest_v = 0;
        float u[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            u[e] = v[i].at(e);
            largest_k = max(largest_k, (uint32_t)(__builtin_bit_cast(uint64_t, y[e]) >> 32) & 0x7FFFFFFFu);
            largest_v = max(largest_v, __builtin_bit_cast(uint32_t, u[e]) & 0x7FFFFFFFu);
        }
        const uint32_t byte_k = fp4_scale_byte<DT>((uint32_t)max((int)(block_max(largest_k) >> 20) - 896, 0));
        const uint32_t byte_v = fp4_scale_byte<DT>(block_max(largest_v) >> 23);
        const double to_unit = __builtin_bit_cast(double, (uint64_t)(1023 + 127 - byte_k) << 52);
        float z[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e)
            z[e] = fp4_side(y[e] * to_unit);
        const uint32_t codes_k = byte_k == 255 ? 0 : fp4_codes(z, 1.0f);
        const uint32_t codes_v = byte_v == 255 ? 0 : fp4_codes(u, fp4_scale(byte_v));
        const uint64_t tile = layer_at + fp4_tile_at(slot, head, p.block_size, p.kv_heads, d);
        store_fp4(static_cast<uint8_t*>(p.keys) + tile, d, slot % fp4_tile, w, false, codes_k, byte_k);
        store_fp4(static_cast<uint8_t*>(p.values) + tile, d, slot % fp4_tile, w, true, codes_v, byte_v);
        if (x.held_keys)
            store_codes<DT, VECTOR>(x.held_keys, at_row + head * d, codes_k, fp4_scale(byte_k));
        if (x.held_values)
            store_codes<DT, VECTOR>(x.held_values, at_row + head * d, codes_v, fp4_scale(byte_v));
    }
}

// The first `append_blocks` workgroups append, the others rotate queries.
template <int DT, bool PAIRS, int PER>
__global__ __launch_bounds__(block_threads) void fp4_rotate_append_kernel(
    pool_view p, const uint32_t* __restrict__ slots, uint32_t layer, rotate_rows x, uint32_t rows,
    uint32_t q_heads, rotation_table by, const uint32_t* __restrict__ positions, uint32_t append_blocks)
{
    if (blockIdx.x < append_blocks)
        fp4_append<DT, PAIRS, true, PER>((uint64_t)blockIdx.x * block_threads + threadIdx.x, p, slots, layer,
                                    x, rows, by, positions);
    else
        rotate_words<DT, PAIRS, 4>((uint64_t)(blockIdx.x - append_blocks) * block_threads + threadIdx.x,
                                   p, slots, layer, x, rows, q_heads, q_heads, by, positions);
}

template <int DT, bool PAIRS>
__global__ __launch_bounds__(block_threads) void fp4_append_any_kernel(
    pool_view p, const uint32_t* __restrict__ slots, uint32_t layer, rotate_rows x, uint32_t rows,
    rotation_table by, const uint32_t* __restrict__ positions)
{
    fp4_append<DT, PAIRS, false, 1>((uint64_t)blockIdx.x * block_threads + threadIdx.x, p, slots, layer, x,
                                 rows, by, positions);
}

// Tokens 0 .. n_tokens - 1 of a sequence as rows: one thread per (token, kv head, word).
template <int DT, bool VECTOR>
__global__ __launch_bounds__(block_threads) void fp4_gather_kernel(
    pool_view p, const uint32_t* __restrict__ table, uint32_t layer, uint32_t n_tokens, void* out_keys,
    void* out_values)
{
    const uint32_t d = p.head_dim, words = d / 8;
    const uint64_t item = (uint64_t)blockIdx.x * block_threads + threadIdx.x;
    const uint32_t token = (uint32_t)(item / (words * p.kv_heads));
    if (token >= n_tokens)
        return;
    const uint32_t rest = (uint32_t)(item % (words * p.kv_heads)), w = rest % words, head = rest / words;
    const uint32_t slot = table[token / p.block_size] * p.block_size + token % p.block_size;
    const uint64_t at = layer * ((uint64_t)p.blocks * p.block_size / fp4_tile * p.kv_heads * fp4_tile_bytes(d))
        + fp4_tile_at(slot, head, p.block_size, p.kv_heads, d);
    const uint64_t to = (uint64_t)token * p.features + head * d + 8 * w;
    const uint32_t in = slot % fp4_tile;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const uint8_t* tile = static_cast<const uint8_t*>(v ? p.values : p.keys) + at;
        const uint8_t* word = tile + fp4_word_at(d, in, w, v);
        const uint32_t codes = v && d == 64
            ? *reinterpret_cast<const uint16_t*>(word) | (uint32_t)*reinterpret_cast<const uint16_t*>(word + 8) << 16
            : *reinterpret_cast<const uint32_t*>(word);
        store_codes<DT, VECTOR>(v ? out_values : out_keys, to, codes,
                                fp4_scale(tile[fp4_scale_at(d, in, w / 4, v)]));
    }
}

bool aligned16(const void* ptr)
{
    return reinterpret_cast<uintptr_t>(ptr) % 16 == 0;
}

// The instantiation for a row type and a pairing.
template <class Call>
auto of_type(int dtype, Call&& call)
{
    return dtype == CKV_F32 ? call(std::integral_constant<int, CKV_F32> {})
        : dtype == CKV_BF16 ? call(std::integral_constant<int, CKV_BF16> {})
                            : call(std::integral_constant<int, CKV_F16> {});
}

hipError_t grid_of(uint64_t threads, uint32_t& blocks)
{
    const uint64_t n = (threads + block_threads - 1) / block_threads;
    blocks = (uint32_t)n;
    return n > 0x7FFFFFFFull ? hipErrorInvalidValue : hipSuccess;
}

// Rows of 16-byte words whose rotary and head widths are whole pairs of them.
bool in_words(const pool_view& p, const rotate_rows& x, uint32_t rotary, bool appended)
{
    const uint32_t each = 16 / p.elem_size;
    return p.head_dim % (2 * each) == 0 && rotary % (2 * each) == 0 && aligned16(x.queries)
        && aligned16(x.rotated) && aligned16(x.keys) && aligned16(x.values) && aligned16(x.held_keys)
        && aligned16(x.held_values) && (!appended || (aligned16(p.keys) && aligned16(p.values)));
}

} // namespace

hipError_t launch_rotate(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                         const rotate_rows& x, uint32_t rows, uint32_t q_heads, const rotation_table& by)
{
    const uint32_t heads = q_heads + (x.keys ? p.kv_heads : 0);
    if (!rows || !heads)
        return hipSuccess;
    uint32_t blocks = 0;
    if (in_words(p, x, by.rotary, x.keys != nullptr)) {
        const uint64_t words = (uint64_t)rows * (p.head_dim / (32 / p.elem_size)); // of a head's halves
        // four heads share their angles, unless that leaves under two workgroups a compute unit
        const bool four = words * heads / 4 >= 512 * block_threads;
        if (const hipError_t e = grid_of(words * (four ? (heads + 3) / 4 : heads), blocks))
            return e;
        of_type(p.dtype, [&](auto dt) {
            constexpr int DT = decltype(dt)::value;
            auto* kernel = by.neighbours ? (four ? rotate_words_kernel<DT, true, 4> : rotate_words_kernel<DT, true, 1>)
                                         : (four ? rotate_words_kernel<DT, false, 4> : rotate_words_kernel<DT, false, 1>);
            kernel<<<blocks, block_threads, 0, s>>>(p, m.slots, layer, x, rows, q_heads, heads, by, m.positions);
        });
        return hipGetLastError();
    }
    if (const hipError_t e = grid_of((uint64_t)heads * ((p.head_dim + 1) / 2), blocks))
        return e;
    const dim3 grid(blocks, rows < 65535 ? rows : 65535);
    of_type(p.dtype, [&](auto dt) {
        rotate_pairs_kernel<decltype(dt)::value><<<grid, block_threads, 0, s>>>(
            p, m.slots, layer, x, rows, q_heads, heads, by, m.positions);
    });
    return hipGetLastError();
}

hipError_t launch_fp4_append(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                             const rotate_rows& x, uint32_t rows, uint32_t q_heads,
                             const rotation_table& by)
{
    if (!rows)
        return hipSuccess;
    uint32_t append = 0, queries = 0;
    const uint64_t words = (uint64_t)rows * (p.head_dim / 8);
    if (by.rotary % 16 == 0 && in_words(p, x, by.rotary, false)) {
        // four heads share their angles, unless that leaves under two workgroups a compute unit
        const bool four = words * ((p.kv_heads + 3) / 4) >= 512 * block_threads;
        if (const hipError_t e = grid_of(words * (four ? (p.kv_heads + 3) / 4 : p.kv_heads), append))
            return e;
        if (const hipError_t e = grid_of((uint64_t)rows * (p.head_dim / (32 / p.elem_size)) * ((q_heads + 3) / 4), queries))
            return e;
        if ((uint64_t)append + queries > 0x7FFFFFFFull)
            return hipErrorInvalidValue;
        of_type(p.dtype, [&](auto dt) {
            constexpr int DT = decltype(dt)::value;
            auto* kernel = by.neighbours
                ? (four ? fp4_rotate_append_kernel<DT, true, 4> : fp4_rotate_append_kernel<DT, true, 1>)
                : (four ? fp4_rotate_append_kernel<DT, false, 4> : fp4_rotate_append_kernel<DT, false, 1>);
            kernel<<<append + queries, block_threads, 0, s>>>(p, m.slots, layer, x, rows, q_heads, by,
                                                              m.positions, append);
        });
        return hipGetLastError();
    }
    if (const hipError_t e = grid_of(words * p.kv_heads, append))
        return e;
    of_type(p.dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        auto* kernel = by.neighbours ? fp4_append_any_kernel<DT, true> : fp4_append_any_kernel<DT, false>;
        kernel<<<append, block_threads, 0, s>>>(p, m.slots, layer, x, rows, by, m.positions);
    });
    if (const hipError_t e = hipGetLastError(); e != hipSuccess || !q_heads)
        return e;
    rotate_rows alone {};
    alone.queries = x.queries;
    alone.rotated = x.rotated;
    alone.float_queries = x.float_queries;
    return launch_rotate(s, p, m, 0, alone, rows, q_heads, by);
}

hipError_t launch_fp4_gather(hipStream_t s, const pool_view& p, const uint32_t* table, uint32_t layer,
                             uint32_t n_tokens, void* out_keys, void* out_values)
{
    if (!n_tokens)
        return hipSuccess;
    uint32_t blocks = 0;
    if (const hipError_t e = grid_of((uint64_t)n_tokens * p.kv_heads * (p.head_dim / 8), blocks))
        return e;
    const bool vector = aligned16(out_keys) && aligned16(out_values);
    of_type(p.dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        auto* kernel = vector ? fp4_gather_kernel<DT, true> : fp4_gather_kernel<DT, false>;
        kernel<<<blocks, block_threads, 0, s>>>(p, table, layer, n_tokens, out_keys, out_values);
    });
    return hipGetLastError();
}

void rotation_steps(const long double* turns, uint32_t rotary, rotation_table& out)
{
    for (uint32_t j = 0; j < rotary / 2; ++j) {
        const long double part = turns[j] - std::floor(turns[j]); // whole turns fall away
        out.turns.step[j] = (uint64_t)(part * 0x1p64L);
    }
}

} // namespace ckv
