// Compaction: kept tokens' K and V rows move to other slots of every layer, and the
// moved keys turn to their new positions.
//
// A cached key was rotated at its old position; turning each pair by (new position -
// old) * frequency gives the key rotated at the new one, with one more rounding to
// the pool's type. Values, elements past the rotary width and keys that keep their
// position are copied bit for bit.
//
// In place, a move may overwrite a slot that another move reads. A run's moves are
// done in order, a chunk at a time: a workgroup reads a chunk's rows into registers,
// waits until all of them have arrived, and writes them. One workgroup walks a run
// for one head of one layer of K or V, so nothing else touches the bytes it reads.
#include "ckv_internal.h"
#include "prefill_records.h"
#include "rope_turns.h"

#include <algorithm>

namespace ckv {
namespace {

constexpr uint32_t block_threads = 256;
constexpr uint32_t items = 8; // pairs a thread holds

template <int DT>
__global__ __launch_bounds__(block_threads) void compact_kernel(pool_view p, compact_moves m,
                                                               uint32_t rotary, turn_table turns)
{
    using E = turn_element<DT>;
    using T = typename E::type;
    const uint32_t d = p.head_dim, half = rotary / 2, pairs = (d + 1) / 2;
    const uint32_t head = blockIdx.x % p.kv_heads, run = blockIdx.x / p.kv_heads;
    const uint64_t base = blockIdx.y * p.layer_elems + (uint64_t)head * d;
    const bool keys = blockIdx.z == 0;
    T* rows = static_cast<T*>(keys ? p.keys : p.values) + base;
    const uint32_t first = m.runs[2 * run], count = m.runs[2 * run + 1];
    const uint64_t total = (uint64_t)count * pairs;
    for (uint64_t i0 = 0; i0 < total; i0 += items * block_threads) {
        T x[items], y[items];
#pragma unroll
        for (uint32_t k = 0; k < items; ++k) {
            const uint64_t i = i0 + k * block_threads + threadIdx.x;
            if (i >= total)
                continue;
            const uint32_t move = first + (uint32_t)(i / pairs), pair = (uint32_t)(i % pairs);
            const uint32_t a = pair < half ? pair : rotary + 2 * (pair - half);
            const uint32_t b = pair < half ? pair + half : min(a + 1, d - 1);
            const T* src = rows + (uint64_t)m.from[move] * p.features;
            x[k] = src[a];
            y[k] = src[b];
        }
        wait_vector_memory();
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < items; ++k) {
            const uint64_t i = i0 + k * block_threads + threadIdx.x;
            if (i >= total)
                continue;
            const uint32_t move = first + (uint32_t)(i / pairs), pair = (uint32_t)(i % pairs);
            const uint32_t a = pair < half ? pair : rotary + 2 * (pair - half);
            const uint32_t b = pair < half ? pair + half : min(a + 1, d - 1);
            T* dst = rows + (uint64_t)m.to[move] * p.features;
            const int32_t shift = m.shift[move];
            if (keys && shift && pair < half) {
                float s, c, r1, r2;
                sincos_turn(turns.step[pair], (uint64_t)(int64_t)shift, s, c);
                rope_pair(E::load(x[k]), E::load(y[k]), c, s, r1, r2);
                x[k] = E::store(r1);
                y[k] = E::store(r2);
            }
            dst[a] = x[k];
            dst[b] = y[k];
        }
    }
}

} // namespace

const char* plan_compaction(move_marks& marks, size_t slots, const uint32_t* from,
                            const uint32_t* to, const int32_t* shift, const uint32_t* counts,
                            size_t n_sequences, std::vector<uint32_t>& kept,
                            std::vector<uint32_t>& runs, int& status)
{
    size_t n = 0;
    for (size_t q = 0; q < n_sequences; ++q)
        n += counts[q];
    status = CKV_E_CACHE_SLOT_OUT_OF_RANGE;
    for (size_t i = 0; i < n; ++i)
        if (from[i] >= slots || to[i] >= slots)
            return "a move's slot is outside the pool";
    if (marks.written.size() < slots) {
        for (auto* v : { &marks.read, &marks.first, &marks.last, &marks.written })
            v->assign(slots, 0);
        marks.generation = 0;
    }
    if (++marks.generation == 0) {
        std::fill(marks.read.begin(), marks.read.end(), 0);
        std::fill(marks.written.begin(), marks.written.end(), 0);
        marks.generation = 1;
    }
    const uint32_t g = marks.generation;
    for (size_t i = 0; i < n; ++i) {
        if (marks.read[from[i]] != g)
            marks.first[from[i]] = (uint32_t)i;
        marks.read[from[i]] = g;
        marks.last[from[i]] = (uint32_t)i;
    }
    status = CKV_E_UNSUPPORTED_ALIASING;
    for (size_t q = 0, begin = 0; q < n_sequences; begin += counts[q], ++q) {
        const size_t end = begin + counts[q], first = kept.size();
        bool free = true; // no target is read by another move
        for (size_t i = begin; i < end; ++i) {
            if (marks.written[to[i]] == g)
                return "two moves share a target";
            marks.written[to[i]] = g;
            if (marks.read[to[i]] == g) {
                if (marks.first[to[i]] < begin || marks.last[to[i]] > i)
                    return "a move's target is read by a later move or another sequence";
                free = free && marks.first[to[i]] == i;
            }
            if (from[i] != to[i] || (shift && shift[i]))
                kept.push_back((uint32_t)i);
        }
        const size_t moves = kept.size() - first;
        const size_t each = free ? compact_run : std::max<size_t>(moves, 1);
        for (size_t at = 0; at < moves; at += each)
            runs.insert(runs.end(), { (uint32_t)(first + at), (uint32_t)std::min(each, moves - at) });
    }
    status = CKV_OK;
    return nullptr;
}

hipError_t launch_compact(hipStream_t s, const pool_view& p, uint32_t layers,
                          const compact_moves& moves, uint32_t rotary, const turn_table& turns)
{
    if (!moves.n_runs)
        return hipSuccess;
    const uint64_t blocks = (uint64_t)moves.n_runs * p.kv_heads;
    if (blocks > 0x7FFFFFFFull || layers > 65535)
        return hipErrorInvalidValue;
    const dim3 grid((uint32_t)blocks, layers, 2);
    auto* kernel = p.dtype == CKV_F32 ? compact_kernel<CKV_F32>
        : p.dtype == CKV_BF16         ? compact_kernel<CKV_BF16>
                                      : compact_kernel<CKV_F16>;
    kernel<<<grid, block_threads, 0, s>>>(p, moves, rotary, turns);
    return hipGetLastError();
}

} // namespace ckv
