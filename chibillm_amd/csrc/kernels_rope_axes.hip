// Rotary embedding of rows whose tokens have a position on several axes (time,
// height and width of images and video), and its fusion with the KV append.
//
// Within each head of a row, pair j < rotary/2 rotates elements j and j + rotary/2
// by positions[axis[j]][row] * theta^(-2j/rotary), as ckv_rope does by the row's one
// position; elements past the rotary width are copied. Queries, keys and values of a
// layer go through one launch: rotated queries to a buffer, rotated keys and the
// values into the rows' slots.
#include "ckv_internal.h"
#include "rope_turns.h"

#include <cmath>

namespace ckv {
namespace {

constexpr uint32_t block_threads = 256;

// One thread per (head, pair) and grid row per row: heads 0 .. q_heads - 1 are the
// query row's, the next kv_heads the key's and value's.
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
        // whole turns per position fall away; a fraction that rounds to one does too
        const long double scaled = std::ldexp(turn - std::floor(turn), 64);
        out.step[pair] = scaled >= 0x1p64L ? 0 : (uint64_t)scaled;
    }
}

hipError_t launch_rope_axes(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                            const axes_rows& x, uint32_t rows, uint32_t q_heads, uint32_t rotary,
                            const turn_table& turns, const axis_table& axes,
                            const uint32_t* positions)
{
    const uint32_t heads = q_heads + (x.keys ? p.kv_heads : 0);
    if (!rows || !heads)
        return hipSuccess;
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
