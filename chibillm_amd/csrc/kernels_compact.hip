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
// for some heads of one layer of K or V, so nothing else touches the bytes it reads.
// Runs are made so that a move and the one that overwrites its source share a run: kept
// tokens that move towards the front form chains, the writer of a slot after its reader,
// short where many tokens leave (a fraction f kept: log n / log 1/f moves). A long chain,
// where few leave, is cut into several runs once it would take longer than one launch
// more, which saves the sources that other runs overwrite to spare rows first.
//
// Bound by HBM, each row read and written once. Measured on MI355X, 8 kv heads of 128,
// bf16: 28 layers of 1,010 moves (the newer half of 2,011 tokens to behind the first
// four) 53.5 us, 4.3 TB/s; 12 layers of 7,600 moves of six sequences to fresh pages or in
// place 156 us, a device copy's 4.76 TB/s; one of 2,000 tokens leaving 4 layers, a chain
// that is cut, 32 us where its bytes take 14, leaving 28 layers, uncut, 109 and 96.
#include "ckv_internal.h"
#include "prefill_records.h"
#include "rope_turns.h"

#include <algorithm>

namespace ckv {
namespace {

constexpr uint32_t block_threads = 256;

// A workgroup's saved rows: those of its layer of K or V.
template <class T>
__device__ __forceinline__ T* spare_rows(const pool_view& p, const compact_moves& m)
{
    return static_cast<T*>(m.spare)
        + ((uint64_t)blockIdx.z * gridDim.y + blockIdx.y) * m.n_spare * p.features;
}

// The row of a slot, or of spare_slot + a saved row.
template <class T>
__device__ __forceinline__ T* moved_row(T* base, T* spare, uint32_t slot, uint32_t features)
{
    return (slot & spare_slot ? spare : base) + (uint64_t)(slot & ~spare_slot) * features;
}

// Rows whose rotary and head widths are whole pairs of 16-byte words: a thread moves a
// word of a head's first half and the one it is turned with (or two words past the
// rotary width, of its halves likewise) for `ahead` tokens at a time. The workgroup goes
// through `heads` heads of a chunk of tokens, whose angles it computes once, then to the
// next chunk; the next head's rows are in flight while this one's are turned and
// written. Rows are read and written once: past the caches, as checkpoints are.
constexpr uint32_t ahead = 2;

template <int DT>
__global__ __launch_bounds__(block_threads) void compact_rows_kernel(pool_view p, compact_moves m,
                                                                    uint32_t rotary, uint32_t heads,
                                                                    turn_table turns)
{
    using E = turn_element<DT>;
    using T = typename E::type;
    constexpr uint32_t each = 16 / sizeof(T); // elements of a word
    union word {
        u32x4_t v;
        T e[each];
    };
    struct slots {
        uint32_t from[ahead], to[ahead];
        int32_t shift[ahead];
        bool live[ahead];
    };
    struct rows {
        word a[ahead], b[ahead];
    };
    const uint32_t d = p.head_dim, half = rotary / 2;
    const uint32_t groups = d / (2 * each), step = block_threads / groups; // tokens side by side
    const uint32_t t = threadIdx.x / groups, p0 = threadIdx.x % groups * each;
    const bool turned = p0 < half;
    const uint32_t at = turned ? p0 : half + p0, apart = turned ? half : (d - rotary) / 2;
    const uint32_t parts = p.kv_heads / heads;
    const uint32_t run = blockIdx.x / parts, head0 = blockIdx.x % parts * heads;
    const bool keys = blockIdx.z == 0;
    T* base = static_cast<T*>(keys ? p.keys : p.values) + blockIdx.y * p.layer_elems + head0 * d + at;
    T* spare = spare_rows<T>(p, m) + head0 * d + at;
    auto row_of = [&](uint32_t slot) { return moved_row(base, spare, slot, p.features); };
    const uint32_t first = m.runs[2 * run], count = m.runs[2 * run + 1];
    const uint32_t chunk = ahead * step;

    auto slots_of = [&](uint32_t i0) {
        slots s;
#pragma unroll
        for (uint32_t k = 0; k < ahead; ++k) {
            const uint32_t i = i0 + k * step + t, move = first + min(i, count - 1);
            s.live[k] = t < step && i < count;
            s.from[k] = m.from[move];
            s.to[k] = m.to[move];
            s.shift[k] = m.shift[move];
        }
        return s;
    };
    auto read = [&](const slots& s, uint32_t h) {
        rows x;
#pragma unroll
        for (uint32_t k = 0; k < ahead; ++k) {
            const T* src = row_of(s.from[k]) + h * d;
            x.a[k].v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(src));
            x.b[k].v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(src + apart));
        }
        return x;
    };
    uint64_t turn[each]; // of the thread's pairs
#pragma unroll
    for (uint32_t e = 0; e < each; ++e) {
        turn[e] = turned ? turns.step[p0 + e] : 0;
        asm volatile("" : "+v"(turn[e])); // read once, not beside the rows in flight
    }
    slots now = slots_of(0), next = slots_of(chunk);
    rows x = read(now, 0);
    for (uint32_t i0 = 0; i0 < count; i0 += chunk) {
        const slots later = slots_of(i0 + 2 * chunk);
        float c[ahead][each], sn[ahead][each];
        if (keys && turned) {
#pragma unroll
            for (uint32_t k = 0; k < ahead; ++k)
#pragma unroll
                for (uint32_t e = 0; e < each; ++e)
                    sincos_turn(turn[e], (uint64_t)(int64_t)now.shift[k], sn[k][e], c[k][e]);
        }
        for (uint32_t h = 0; h < heads; ++h) {
            // every wave's rows of this chunk and head have arrived: they may be overwritten
#pragma unroll
            for (uint32_t k = 0; k < ahead; ++k)
                asm volatile("" : "+v"(x.a[k].v), "+v"(x.b[k].v)::"memory");
            __syncthreads();
            // (past the run's end its last row again, which is not written)
            const bool same = h + 1 < heads;
            slots ahead_of = next;
#pragma unroll
            for (uint32_t k = 0; k < ahead; ++k)
                ahead_of.from[k] = same ? now.from[k] : next.from[k];
            const rows y = read(ahead_of, same ? h + 1 : 0);
#pragma unroll
            for (uint32_t k = 0; k < ahead; ++k) {
                if (keys && turned && now.shift[k]) {
#pragma unroll
                    for (uint32_t e = 0; e < each; ++e) {
                        float r1, r2;
                        rope_pair(E::load(x.a[k].e[e]), E::load(x.b[k].e[e]), c[k][e], sn[k][e], r1, r2);
                        x.a[k].e[e] = E::store(r1);
                        x.b[k].e[e] = E::store(r2);
                    }
                }
                if (now.live[k]) {
                    T* dst = row_of(now.to[k]) + h * d;
                    __builtin_nontemporal_store(x.a[k].v, reinterpret_cast<u32x4_t*>(dst));
                    __builtin_nontemporal_store(x.b[k].v, reinterpret_cast<u32x4_t*>(dst + apart));
                }
            }
            x = y;
        }
        now = next;
        next = later;
    }
}

// Any other geometry, an element at a time.
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
    T* spare = spare_rows<T>(p, m) + head * d;
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
            const T* src = moved_row(rows, spare, m.from[move], p.features);
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
            T* dst = moved_row(rows, spare, m.to[move], p.features);
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

// Words from pinned host memory, 8 bytes a thread, past every cache: the host wrote them
// since the GPU last read there.
__global__ __launch_bounds__(block_threads) void fetch_kernel(uint64_t* __restrict__ to,
                                                              const uint64_t* __restrict__ from,
                                                              uint32_t n)
{
    const uint32_t i = blockIdx.x * block_threads + threadIdx.x;
    if (i < n)
        to[i] = __hip_atomic_load(from + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

} // namespace

hipError_t launch_fetch(hipStream_t s, uint32_t* to, const void* pinned, size_t words)
{
    void* from = nullptr;
    if (const hipError_t e = hipHostGetDevicePointer(&from, const_cast<void*>(pinned), 0))
        return e;
    const uint64_t n = words / 2, blocks = (n + block_threads - 1) / block_threads;
    if (words % 2 || n > 0xFFFFFFFFull)
        return hipErrorInvalidValue;
    fetch_kernel<<<(uint32_t)blocks, block_threads, 0, s>>>(reinterpret_cast<uint64_t*>(to),
                                                            static_cast<const uint64_t*>(from),
                                                            (uint32_t)n);
    return hipGetLastError();
}

// Measured on MI355X: bytes pass at 4.5 TB/s, a run's chunk takes 2.9 us, and a launch
// more costs 8 us where bytes are moving.
compact_cost compact_cost_of(const pool_view& p, uint32_t layers)
{
    const double row = (double)p.features * p.elem_size;
    const double chunk = ahead * block_threads * 32.0 / ((double)p.head_dim * p.elem_size);
    return { 4.0 * row * layers / 4.5e6, 2.9 / std::max(chunk, 1.0), 8.0 };
}

const char* plan_compaction(move_marks& marks, size_t slots, const uint32_t* from,
                            const uint32_t* to, const int32_t* shift, const uint32_t* counts,
                            size_t n_sequences, const compact_cost& cost, compact_plan& plan,
                            int& status)
{
    size_t n = 0;
    for (size_t q = 0; q < n_sequences; ++q)
        n += counts[q];
    auto& at_slot = marks.at_slot;
    if (at_slot.size() < slots) {
        at_slot.assign(slots, {});
        marks.generation = 0;
    }
    if (++marks.generation == 0) {
        std::fill(at_slot.begin(), at_slot.end(), move_marks::mark {});
        marks.generation = 1;
    }
    const uint32_t g = marks.generation;
    status = CKV_E_CACHE_SLOT_OUT_OF_RANGE;
    for (size_t i = 0; i < n; ++i) {
        if (from[i] >= slots || to[i] >= slots)
            return "a move's slot is outside the pool";
        auto& m = at_slot[from[i]];
        if (m.read != g) {
            m.read = g;
            m.first = (uint32_t)i;
        }
        m.last = (uint32_t)i;
    }
    // Chains: a move joins the chain of the move that reads its target first, if that
    // chain has fewer than `most` moves.
    std::vector<uint32_t> &chain = marks.chain, &reader = marks.reader, &sizes = marks.sizes;
    chain.resize(n);
    reader.resize(n);
    sizes.assign(n, 0);
    uint32_t n_chains = 0;
    auto follow = [&](uint32_t i, uint32_t most) { // (selects: no branch would guess it)
        const uint32_t r = reader[i];
        chain[i] = n_chains;
        const uint32_t other = chain[r];
        const bool joins = r < i && sizes[other] < most;
        chain[i] = joins ? other : n_chains;
        n_chains += !joins;
        ++sizes[chain[i]];
    };
    status = CKV_E_UNSUPPORTED_ALIASING;
    for (size_t q = 0, begin = 0; q < n_sequences; begin += counts[q], ++q)
        for (size_t i = begin; i < begin + counts[q]; ++i) {
            auto& m = at_slot[to[i]];
            if (m.written == g)
                return "two moves share a target";
            m.written = g;
            m.writer = (uint32_t)i;
            const bool read = m.read == g;
            if (read & ((m.first < begin) | (m.last > i)))
                return "a move's target is read by a later move or another sequence";
            reader[i] = read ? m.first : (uint32_t)i; // the move itself: none
            if (from[i] != to[i] || (shift && shift[i]))
                follow((uint32_t)i, UINT32_MAX);
            else
                chain[i] = UINT32_MAX; // changes nothing
        }
    status = CKV_OK;
    if (!n_chains)
        return nullptr;
    sizes.resize(n_chains);
    const double longest = cost.move_in_run * *std::max_element(sizes.begin(), sizes.end());
    const double others = std::max(cost.move_bytes * (double)n, cost.move_in_run * compact_run);
    if (longest > others + cost.launch) {
        sizes.assign(n, 0);
        n_chains = 0;
        for (uint32_t i = 0; i < n; ++i)
            if (chain[i] != UINT32_MAX)
                follow(i, compact_run);
        sizes.resize(n_chains);
    }
    // Chains in the order of their first moves, as many to a run as it takes; a longer one
    // has a run of its own.
    std::vector<uint32_t> run_of(sizes.size()), begins { 0 };
    uint32_t held = 0; // moves of the run that takes chains, the last of them
    bool open = false;
    uint32_t taking = 0;
    for (size_t c = 0; c < sizes.size(); ++c) {
        if (sizes[c] <= compact_run && open && held + sizes[c] <= compact_run) {
            run_of[c] = taking;
            held += sizes[c];
        } else {
            run_of[c] = (uint32_t)begins.size() - 1;
            begins.push_back(0);
            if (sizes[c] <= compact_run) {
                taking = run_of[c];
                held = sizes[c];
                open = true;
            }
        }
        begins[run_of[c] + 1] += sizes[c];
    }
    for (size_t r = 1; r < begins.size(); ++r)
        begins[r] += begins[r - 1];
    plan.kept.resize(begins.back());
    plan.spare.assign(plan.kept.size(), UINT32_MAX);
    std::vector<uint32_t> next(begins.begin(), begins.end() - 1);
    for (size_t i = 0; i < n; ++i) {
        if (chain[i] == UINT32_MAX)
            continue;
        const uint32_t run = run_of[chain[i]], at = next[run]++;
        plan.kept[at] = (uint32_t)i;
        const auto& m = at_slot[from[i]];
        const uint32_t writer = m.written == g ? m.writer : (uint32_t)i;
        if (chain[writer] != UINT32_MAX && run_of[chain[writer]] != run) {
            plan.spare[at] = (uint32_t)plan.saved.size();
            plan.saved.push_back((uint32_t)i);
        }
    }
    const uint32_t kept = (uint32_t)plan.kept.size(), saved = (uint32_t)plan.saved.size();
    for (uint32_t at = 0; at < saved; at += compact_run)
        plan.runs.insert(plan.runs.end(), { kept + at, std::min(compact_run, saved - at) });
    if (saved)
        plan.launches.push_back((uint32_t)plan.runs.size() / 2);
    for (size_t r = 0; r + 1 < begins.size(); ++r)
        plan.runs.insert(plan.runs.end(), { begins[r], begins[r + 1] - begins[r] });
    plan.launches.push_back((uint32_t)begins.size() - 1);
    return nullptr;
}

uint32_t compact_heads(const pool_view& p, uint32_t layers, uint32_t n_runs, uint32_t rotary)
{
    const uint32_t each = 16 / p.elem_size;
    const auto aligned = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 16 == 0; };
    if (p.head_dim % (2 * each) || rotary % (2 * each) || p.head_dim / (2 * each) > block_threads
        || !aligned(p.keys) || !aligned(p.values))
        return 0;
    uint32_t heads = p.kv_heads;
    while (heads % 2 == 0 && (uint64_t)n_runs * layers * 2 * (p.kv_heads / heads) < 2048)
        heads /= 2;
    return heads;
}

hipError_t launch_compact(hipStream_t s, const pool_view& p, uint32_t layers,
                          const compact_moves& moves, uint32_t rotary, const turn_table& turns)
{
    if (!moves.n_runs)
        return hipSuccess;
    const uint32_t in_words = compact_heads(p, layers, moves.n_runs, rotary);
    const uint32_t heads = std::max(in_words, 1u);
    const uint64_t blocks = (uint64_t)moves.n_runs * (p.kv_heads / heads);
    if (blocks > 0x7FFFFFFFull || layers > 65535)
        return hipErrorInvalidValue;
    const dim3 grid((uint32_t)blocks, layers, 2);
    if (in_words) {
        auto* kernel = p.dtype == CKV_F32 ? compact_rows_kernel<CKV_F32>
            : p.dtype == CKV_BF16         ? compact_rows_kernel<CKV_BF16>
                                          : compact_rows_kernel<CKV_F16>;
        kernel<<<grid, block_threads, 0, s>>>(p, moves, rotary, heads, turns);
        return hipGetLastError();
    }
    auto* kernel = p.dtype == CKV_F32 ? compact_kernel<CKV_F32>
        : p.dtype == CKV_BF16         ? compact_kernel<CKV_BF16>
                                      : compact_kernel<CKV_F16>;
    kernel<<<grid, block_threads, 0, s>>>(p, moves, rotary, turns);
    return hipGetLastError();
}

} // namespace ckv
