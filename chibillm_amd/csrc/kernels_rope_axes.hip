// Rotary embedding of rows whose tokens have a position on several axes (time,
// height and width of images and video), and its fusion with the KV append.
//
// Within each head of a row, pair j < rotary/2 rotates elements j and j + rotary/2
// by positions[axis[j]][row] * theta^(-2j/rotary), as ckv_rope does by the row's one
// position; elements past the rotary width are copied. Queries, keys and values of a
// layer go through one launch: rotated queries to a buffer, rotated keys and the
// values into the rows' slots.
//
// Bound by HBM from a few hundred rows on: each row is read and written once. Measured
// on MI355X, 16 q and 8 kv heads of 128, bf16: 4,096 rows 14.9 us, 4.5 TB/s read and
// written (an element a thread with every angle computed for each head, 24.6 us); 1,531
// fp16 rows of 8 q and 2 kv heads of 256, 64 of them rotated, 6.5 us; 6 rows take 3.3 us
// on the GPU, a launch's own time, and a call 6.1.
#include "ckv_internal.h"
#include "rope_turns.h"

#include <cmath>

namespace ckv {
namespace {

constexpr uint32_t block_threads = 256;

// Rows whose rotary and head widths are whole pairs of 16-byte words: a thread takes
// one word of a head's first half and the one it is turned with (or two words past the
// rotary width, of its halves likewise) in PER heads of a row, whose angles it computes
// once, with the rows' words in flight meanwhile.
template <int DT, int PER>
__global__ __launch_bounds__(block_threads) void rope_axes_words_kernel(
    pool_view p, const uint32_t* __restrict__ slots, uint32_t layer, axes_rows x, uint32_t rows,
    uint32_t q_heads, uint32_t heads, uint32_t rotary, turn_table turns, axis_table axes,
    const uint32_t* __restrict__ positions)
{
    using E = turn_element<DT>;
    using T = typename E::type;
    constexpr uint32_t each = 16 / sizeof(T); // elements of a word
    union word {
        uint4 v;
        T e[each];
    };
    const uint32_t d = p.head_dim, half = rotary / 2;
    const uint32_t groups = d / (2 * each), parts = (heads + PER - 1) / PER;
    const uint64_t item = (uint64_t)blockIdx.x * block_threads + threadIdx.x;
    const uint32_t row = (uint32_t)(item / (groups * parts));
    if (row >= rows)
        return;
    const uint32_t rest = (uint32_t)(item % (groups * parts));
    const uint32_t p0 = rest % groups * each, head0 = rest / groups * PER;
    const bool turned = p0 < half;
    const uint32_t at = turned ? p0 : half + p0, apart = turned ? half : (d - rotary) / 2;
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
        for (uint32_t e = 0; e < each; ++e)
            sincos_turn(turns.step[p0 + e],
                        positions[(uint64_t)axes.axis[p0 + e] * rows + row], s[e], c[e]);
    }
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const uint32_t h = head0 + i;
        if (h >= heads)
            break;
        if (turned) {
#pragma unroll
            for (uint32_t e = 0; e < each; ++e) {
                float r1, r2;
                rope_pair(E::load(a[i].e[e]), E::load(b[i].e[e]), c[e], s[e], r1, r2);
                a[i].e[e] = E::store(r1);
                b[i].e[e] = E::store(r2);
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
            dst = static_cast<T*>(p.keys) + slot_row + in_row;
        }
        *reinterpret_cast<uint4*>(dst) = a[i].v;
        *reinterpret_cast<uint4*>(dst + apart) = b[i].v;
    }
}

// Any other geometry: one thread per (head, pair) and grid row per row: heads
// 0 .. q_heads - 1 are the query row's, the next kv_heads the key's and value's.
template <int DT>
__global__ __launch_bounds__(block_threads) void rope_axes_kernel(
    pool_view p, const uint32_t* __restrict__ slots, uint32_t layer, axes_rows x, uint32_t rows,
    uint32_t q_heads, uint32_t heads, uint32_t rotary, turn_table turns, axis_table axes,
    const uint32_t* __restrict__ positions)
{
    using E = turn_element<DT>;
    using T = typename E::type;
    const uint32_t d = p.head_dim, half = rotary / 2;
    const uint32_t t = blockIdx.x * block_threads + threadIdx.x;
    const uint32_t head = t / (d / 2), pair = t % (d / 2);
    if (head >= heads)
        return;
    const bool query = head < q_heads, turned = pair < half;
    // the pair's two elements within the head
    const uint32_t a = turned ? pair : rotary + 2 * (pair - half), b = turned ? pair + half : a + 1;
    const uint32_t at = query ? head * d : (head - q_heads) * d; // the head in its row
    for (uint32_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const uint64_t width = query ? (uint64_t)q_heads * d : p.features;
        const T* src = static_cast<const T*>(query ? x.queries : x.keys) + row * width + at;
        T o1 = src[a], o2 = src[b];
        if (turned) {
            float s, c, r1, r2;
            sincos_turn(turns.step[pair], positions[(uint64_t)axes.axis[pair] * rows + row], s, c);
            rope_pair(E::load(o1), E::load(o2), c, s, r1, r2);
            o1 = E::store(r1);
            o2 = E::store(r2);
        }
        if (query) {
            T* dst = static_cast<T*>(x.rotated) + row * width + at;
            dst[a] = o1;
            dst[b] = o2;
        } else {
            const uint64_t dst = layer * p.layer_elems + (uint64_t)slots[row] * p.features + at;
            T* kc = static_cast<T*>(p.keys) + dst;
            T* vc = static_cast<T*>(p.values) + dst;
            const T* vs = static_cast<const T*>(x.values) + row * width + at;
            kc[a] = o1;
            kc[b] = o2;
            vc[a] = vs[a];
            vc[b] = vs[b];
        }
    }
}

} // namespace

void turn_steps(float theta, uint32_t rotary, turn_table& out)
{
    // the 64 bits of a long double's significand; 256 products keep 2^-55 of a step
    const long double ratio = std::pow((long double)theta, -2.0L / rotary);
    long double turn = 1.0L / (2.0L * 3.14159265358979323846264338327950288L);
    for (uint32_t pair = 0; pair < rotary / 2; ++pair, turn *= ratio) {
        // whole turns per position fall away
        const long double part = turn < 1.0L ? turn : turn - std::floor(turn);
        out.step[pair] = (uint64_t)(part * 0x1p64L);
    }
}

uint32_t rope_axes_heads(const pool_view& p, const axes_rows& x, uint32_t rows, uint32_t heads,
                         uint32_t rotary)
{
    const uint32_t each = 16 / p.elem_size;
    const auto aligned = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 16 == 0; };
    if (p.head_dim % (2 * each) || rotary % (2 * each) || !aligned(x.queries) || !aligned(x.rotated)
        || !aligned(x.keys) || !aligned(x.values)
        || (x.keys && (!aligned(p.keys) || !aligned(p.values))))
        return 0;
    const uint64_t words = (uint64_t)rows * (p.head_dim / (2 * each)); // of a head's halves
    return words * heads / 4 >= 512 * block_threads ? 4 : 1;
}

hipError_t launch_rope_axes(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                            const axes_rows& x, uint32_t rows, uint32_t q_heads, uint32_t rotary,
                            const turn_table& turns, const axis_table& axes,
                            const uint32_t* positions)
{
    const uint32_t heads = q_heads + (x.keys ? p.kv_heads : 0);
    if (!rows || !heads)
        return hipSuccess;
    if (const uint32_t per = rope_axes_heads(p, x, rows, heads, rotary)) {
        const uint64_t words = (uint64_t)rows * (p.head_dim / (32 / p.elem_size)); // of a head's halves
        const bool four = per == 4;
        const uint64_t parts = four ? (heads + 3) / 4 : heads;
        const uint64_t blocks = (words * parts + block_threads - 1) / block_threads;
        if (blocks > 0x7FFFFFFFull)
            return hipErrorInvalidValue;
        auto* kernel = p.dtype == CKV_F32
            ? (four ? rope_axes_words_kernel<CKV_F32, 4> : rope_axes_words_kernel<CKV_F32, 1>)
            : p.dtype == CKV_BF16
            ? (four ? rope_axes_words_kernel<CKV_BF16, 4> : rope_axes_words_kernel<CKV_BF16, 1>)
            : (four ? rope_axes_words_kernel<CKV_F16, 4> : rope_axes_words_kernel<CKV_F16, 1>);
        kernel<<<(uint32_t)blocks, block_threads, 0, s>>>(p, m.slots, layer, x, rows, q_heads, heads,
                                                          rotary, turns, axes, positions);
        return hipGetLastError();
    }
    const uint64_t threads = (uint64_t)heads * (p.head_dim / 2);
    const uint64_t blocks = (threads + block_threads - 1) / block_threads;
    if (blocks > 0x7FFFFFFFull)
        return hipErrorInvalidValue;
    const dim3 grid((uint32_t)blocks, rows < 65535 ? rows : 65535);
    auto* kernel = p.dtype == CKV_F32 ? rope_axes_kernel<CKV_F32>
        : p.dtype == CKV_BF16         ? rope_axes_kernel<CKV_BF16>
                                      : rope_axes_kernel<CKV_F16>;
    kernel<<<grid, block_threads, 0, s>>>(p, m.slots, layer, x, rows, q_heads, heads, rotary, turns,
                                          axes, positions);
    return hipGetLastError();
}

} // namespace ckv
