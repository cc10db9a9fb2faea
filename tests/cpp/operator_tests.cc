// Windowed attention, rotation on several axes and compaction on the CPU: the window's
// arithmetic against its definition, the fixed-point turns against long doubles, the
// runs that moves are cut into, and what the entry points refuse (over a pool without
// a GPU: every call here ends in its checks).
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <random>

#include "check.h"
#include "ckv_internal.h"

namespace {

using namespace ckv;

bool attends(uint32_t p, uint32_t t, key_window w)
{
    return t <= p && ((uint64_t)t + w.window > p || t < w.sinks);
}

// The units that a kernel walks are those with a key the row attends, in order.
TEST("window: the units walked are those with a key the row attends")
{
    for (const uint32_t unit : { 1u, 8u, 16u, 32u })
        for (const uint32_t window : { 1u, 2u, 7u, 15u, 16u, 17u, 40u, 64u, 300u, UINT32_MAX })
            for (const uint32_t sinks : { 0u, 1u, 4u, 15u, 16u, 17u, 33u, 250u, UINT32_MAX })
                for (uint32_t p = 0; p < 280; p = p < 70 ? p + 1 : p + 13) {
                    const key_window w { window, sinks };
                    const window_gap gap = window_gap_of(window_low(p, w), sinks, unit);
                    const uint32_t units = p / unit + 1;
                    REQUIRE(gap.kept + gap.skip < units);
                    for (uint32_t u = 0; u < units; ++u) {
                        bool some = false;
                        for (uint32_t t = u * unit; t < (u + 1) * unit; ++t)
                            some = some || attends(p, t, w);
                        const bool walked = u < gap.kept || u >= gap.kept + gap.skip;
                        CHECK(walked == some);
                    }
                }
    // positions near the type's end
    const key_window w { 100, 4 };
    CHECK(window_low(0xFFFFFFF0u, w) == 0xFFFFFFF0u - 99u);
    CHECK(window_low(99, w) == 0);
    CHECK(window_low(100, w) == 1);
    CHECK(window_low(0xFFFFFFF0u, all_keys) == 0);
}

// A position's turn, as the device takes it from the steps, within 2^-32 of a turn of
// the angle in long double, for positions as far as 32 bits go.
TEST("rope axes: fixed-point turns match long doubles at every position")
{
    const long double two_pi = 2.0L * 3.14159265358979323846264338327950288L;
    for (const float theta : { 1e4f, 1e6f, 1e7f, 2.5f, 0.5f })
        for (const uint32_t rotary : { 2u, 16u, 64u, 128u, 512u }) {
            turn_table t {};
            turn_steps(theta, rotary, t);
            for (uint32_t j = 0; j < rotary / 2; j += rotary > 64 ? 7 : 1) {
                const long double step = std::pow((long double)theta, -2.0L * j / rotary) / two_pi;
                for (const int64_t p : { 0LL, 1LL, 2LL, 1000LL, 131071LL, 5000011LL, -1LL, -4096LL, 4294967295LL }) {
                    const uint64_t turn = t.step[j] * (uint64_t)p;
                    const long double got = (long double)turn / 0x1p64L;
                    // step * p in long double is good to |p| 2^-62 of a turn
                    long double off = got - (step * p - std::floor(step * p));
                    off -= std::round(off);
                    CHECK(std::fabs(off) < 0x1p-32L + std::fabs((long double)p) * 0x1p-55L * (step > 1 ? step : 1));
                }
            }
        }
}

struct plan : compact_plan {
    int status = -1;
    bool refused = false;
};

plan compaction(move_marks& marks, size_t slots, const std::vector<uint32_t>& from,
                const std::vector<uint32_t>& to, const std::vector<uint32_t>& counts,
                const int32_t* shift = nullptr, const compact_cost& cost = { 0.007, 0.05, 8.0 })
{
    plan p;
    p.refused = plan_compaction(marks, slots, from.data(), to.data(), shift, counts.data(),
                                counts.size(), cost, p, p.status) != nullptr;
    return p;
}

// Launches one after another, their runs concurrently, each in its order, leave what all
// reads before all writes do. A run's moves are interleaved with the other runs' as two
// steps, a read of up to 32 of them and then their writes.
void run_and_compare(const plan& p, uint32_t slots, const std::vector<uint32_t>& from,
                     const std::vector<uint32_t>& to, std::mt19937_64& rng)
{
    REQUIRE(!p.refused && p.status == CKV_OK);
    std::vector<uint32_t> want(slots), got(slots);
    for (uint32_t i = 0; i < slots; ++i)
        want[i] = got[i] = 1000 + i;
    for (size_t i = 0; i < from.size(); ++i)
        want[to[i]] = 1000 + from[i];
    std::vector<int> done(from.size(), 0);
    size_t first = 0;
    REQUIRE(p.launches.size() == (p.kept.empty() ? 0 : p.saved.empty() ? 1 : 2));
    REQUIRE(p.spare.size() == p.kept.size());
    std::vector<uint32_t> spare(p.saved.size(), 0);
    for (const uint32_t n : p.launches) {
        struct walk {
            uint32_t at, end;
            std::vector<uint32_t> held;
        };
        std::vector<walk> runs;
        for (size_t r = first; r < first + n; ++r)
            runs.push_back({ p.runs[2 * r], p.runs[2 * r] + p.runs[2 * r + 1], {} });
        first += n;
        while (!runs.empty()) {
            const size_t r = rng() % runs.size();
            walk& w = runs[r];
            const uint32_t k = std::min<uint32_t>(32, w.end - w.at);
            if (w.held.empty()) {
                for (uint32_t j = 0; j < k; ++j) {
                    const uint32_t at = w.at + j, kept = (uint32_t)p.kept.size();
                    w.held.push_back(at >= kept                 ? got[from[p.saved.at(at - kept)]]
                                         : p.spare[at] != UINT32_MAX ? spare.at(p.spare[at])
                                                                     : got[from[p.kept[at]]]);
                }
            } else {
                for (uint32_t j = 0; j < k; ++j) {
                    if (w.at + j >= p.kept.size()) {
                        spare.at(w.at + j - p.kept.size()) = w.held[j];
                        continue;
                    }
                    const uint32_t i = p.kept[w.at + j];
                    REQUIRE(!done[i]);
                    done[i] = 1;
                    got[to[i]] = w.held[j];
                }
                w.held.clear();
                w.at += k;
                if (w.at == w.end)
                    runs.erase(runs.begin() + r);
            }
        }
    }
    REQUIRE(2 * first == p.runs.size());
    for (const uint32_t i : p.kept)
        CHECK(done[i]);
    CHECK(got == want);
}

TEST("compaction: concurrent runs leave what reads before writes do")
{
    std::mt19937_64 rng(7);
    move_marks marks;
    for (int trial = 0; trial < 400; ++trial) {
        const uint32_t each = trial % 4 ? 200 : 1500, slots = 3 * each;
        std::vector<uint32_t> order(slots), from, to, counts;
        for (uint32_t i = 0; i < slots; ++i)
            order[i] = i;
        std::shuffle(order.begin(), order.end(), rng);
        for (uint32_t q = 0; q < 3; ++q) { // a sequence: slots of its own
            const uint32_t* at = order.data() + each * q;
            uint32_t n = 0;
            const bool fresh = rng() % 3 == 0;
            const uint32_t of = fresh ? each / 2 : each, kind = rng() % 4;
            for (uint32_t t = 0; t < of; ++t) {
                const bool keep = kind == 0 ? rng() % 5 != 0
                    : kind == 1             ? t < 4 || t >= of / 2
                    : kind == 2             ? t != 3
                                            : t < 20 || t >= 90; // 70 leave
                if (keep) {
                    from.push_back(at[t]);
                    to.push_back(at[fresh ? of + n : n]);
                    ++n;
                }
            }
            counts.push_back(n);
        }
        // rates that favour cutting chains, none, and either
        const compact_cost costs[] = { { 0.0, 1.0, 0.1 }, { 1.0, 0.0, 9.0 }, { 0.007, 0.05, 8.0 } };
        run_and_compare(compaction(marks, slots, from, to, counts, nullptr, costs[trial % 3]), slots, from,
                        to, rng);
    }
    // slots read several times, and moves that change a key where it stands
    for (int trial = 0; trial < 200; ++trial) {
        std::vector<uint32_t> from, to;
        std::vector<int32_t> shift;
        for (uint32_t i = 0; i < 150; ++i) {
            to.push_back(i);
            from.push_back(i + rng() % 3 * (rng() % 40));
            shift.push_back(-(int32_t)(rng() % 3));
        }
        const plan p = compaction(marks, 250, from, to, { 150 }, shift.data());
        run_and_compare(p, 250, from, to, rng);
    }
}

TEST("compaction: chains share runs, and one that is too long is cut")
{
    move_marks marks;
    std::vector<uint32_t> from, to;
    for (uint32_t t = 0; t < 2000; ++t)
        if (t < 4 || t >= 1000) {
            to.push_back((uint32_t)to.size());
            from.push_back(t);
        }
    plan p = compaction(marks, 2000, from, to, { (uint32_t)to.size() });
    // 1004 tokens but for the first 4, 8 of them in chains of two
    CHECK(p.launches.size() == 1 && p.kept.size() == 1000 && p.saved.empty());
    CHECK(p.launches[0] == (1000 + 63) / 64);
    from.clear();
    to.clear();
    for (uint32_t t = 0; t < 2000; ++t)
        if (t != 4) {
            to.push_back((uint32_t)to.size());
            from.push_back(t);
        }
    // one chain: in one run where launches cost more, else cut where each run ends
    p = compaction(marks, 2000, from, to, { (uint32_t)to.size() }, nullptr, { 0.007, 0.05, 100.0 });
    CHECK(p.launches.size() == 1 && p.launches[0] == 1 && p.kept.size() == 1995);
    p = compaction(marks, 2000, from, to, { (uint32_t)to.size() });
    CHECK(p.launches.size() == 2 && p.kept.size() == 1995 && p.saved.size() == (1995 + 63) / 64 - 1);
    CHECK(p.launches[0] == 1 && p.launches[1] == (1995 + 63) / 64);
}

TEST("compaction: unsafe moves are refused")
{
    move_marks marks;
    const size_t n = 64;
    CHECK(compaction(marks, n, { 3, 64 }, { 1, 2 }, { 2 }).status == CKV_E_CACHE_SLOT_OUT_OF_RANGE);
    CHECK(compaction(marks, n, { 3, 4 }, { 1, 99 }, { 2 }).status == CKV_E_CACHE_SLOT_OUT_OF_RANGE);
    CHECK(compaction(marks, n, { 3, 4 }, { 1, 1 }, { 2 }).status == CKV_E_UNSUPPORTED_ALIASING);
    // a target read by a later move, and by another sequence before or after it
    CHECK(compaction(marks, n, { 3, 4 }, { 4, 5 }, { 2 }).status == CKV_E_UNSUPPORTED_ALIASING);
    CHECK(compaction(marks, n, { 3, 4 }, { 4, 5 }, { 1, 1 }).status == CKV_E_UNSUPPORTED_ALIASING);
    CHECK(compaction(marks, n, { 3, 4 }, { 5, 3 }, { 1, 1 }).status == CKV_E_UNSUPPORTED_ALIASING);
    // towards the front, and one slot read twice
    CHECK(compaction(marks, n, { 3, 4 }, { 2, 3 }, { 2 }).status == CKV_OK);
    CHECK(compaction(marks, n, { 3, 3 }, { 1, 2 }, { 2 }).status == CKV_OK);
    // an exchange is none: its second move reads what the first wrote
    CHECK(compaction(marks, n, { 3, 4 }, { 4, 3 }, { 2 }).status == CKV_E_UNSUPPORTED_ALIASING);
    // moves that change nothing are left out; with a shift they are not
    CHECK(compaction(marks, n, { 3, 4 }, { 3, 4 }, { 2 }).kept.empty());
    const int32_t shift[] = { 0, -2 };
    CHECK(compaction(marks, n, { 3, 4 }, { 3, 4 }, { 2 }, shift).kept == std::vector<uint32_t> { 1 });
    // the generation's wrap forgets old marks
    marks.generation = UINT32_MAX;
    CHECK(compaction(marks, n, { 3, 4 }, { 2, 3 }, { 2 }).status == CKV_OK);
    CHECK(marks.generation == 1);
}

// Every argument that the entry points refuse, over a batch of two rows.
TEST("entry points: what is refused")
{
    ckv_context ctx;
    ckv_pool pool;
    pool.ctx = &ctx;
    pool.layers = 2;
    pool.blocks = 8;
    pool.block_size = 16;
    pool.kv_heads = 2;
    pool.head_dim = 128;
    int x[4]; // never read: no call gets that far
    void *k = x, *v = x + 1, *q = x + 2, *o = x + 3;
    const size_t rows = 2;
    auto attend = [&](size_t layer, const void* q, size_t heads, size_t window, const void* gate,
                      void* out, size_t n) {
        return ckv_attention_window(&pool, layer, q, heads, 1.0f, window, 4, gate, out, n);
    };
    CHECK(ckv_attention_window(nullptr, 0, q, 4, 1.0f, 8, 0, nullptr, o, 1) == CKV_E_INVALID_ARGUMENT);
    CHECK(attend(0, q, 4, 8, nullptr, o, rows) == CKV_E_NO_TABLES);
    CHECK(ckv_rope_axes_upload(&pool, nullptr, 3, rows) == CKV_E_INVALID_ARGUMENT);
    const uint32_t positions[8] = {};
    CHECK(ckv_rope_axes_upload(&pool, positions, 3, rows) == CKV_E_NO_TABLES);
    pool.uploaded = true;
    pool.positions = { 40, 50 };
    pool.last_position = 50;
    CHECK(attend(0, nullptr, 4, 8, nullptr, o, rows) == CKV_E_INVALID_ARGUMENT);
    CHECK(attend(0, q, 4, 8, nullptr, nullptr, rows) == CKV_E_INVALID_ARGUMENT);
    CHECK(attend(0, q, 4, 8, nullptr, o, 3) == CKV_E_POSITION_COUNT_MISMATCH);
    CHECK(attend(0, q, 0, 8, nullptr, o, rows) == CKV_E_INVALID_HEAD_COUNT);
    CHECK(attend(0, q, 3, 8, nullptr, o, rows) == CKV_E_INVALID_KV_HEAD_MAPPING);
    CHECK(attend(2, q, 4, 8, nullptr, o, rows) == CKV_E_CACHE_LAYER_OUT_OF_RANGE);
    CHECK(attend(0, q, 4, 0, nullptr, o, rows) == CKV_E_INVALID_ARGUMENT);
    CHECK(attend(0, q, 4, 8, q, o, rows) == CKV_E_UNSUPPORTED_ALIASING);
    CHECK(attend(0, q, 4, 8, o, o, rows) == CKV_E_UNSUPPORTED_ALIASING);
    auto append = [&](size_t layer, const void* k, const void* v, size_t window, size_t n) {
        const int a = ckv_append_decode_window(&pool, layer, k, v, q, 4, 1.0f, window, 4, nullptr, o, n);
        const int b = ckv_rope_append_decode_window(&pool, layer, k, v, q, 4, 1.0f, 1e4f, 0, window, 4,
                                                    nullptr, o, n);
        CHECK(a == b);
        return a;
    };
    CHECK(append(0, k, v, 8, rows) == CKV_E_NO_TABLES); // no slots
    pool.has_slots = true;
    pool.slot_rows = rows;
    CHECK(append(0, nullptr, v, 8, rows) == CKV_E_INVALID_ARGUMENT);
    CHECK(append(0, k, nullptr, 8, rows) == CKV_E_INVALID_ARGUMENT);
    CHECK(append(0, k, v, 8, 3) == CKV_E_CACHE_SLOT_COUNT_MISMATCH);
    CHECK(append(2, k, v, 8, rows) == CKV_E_CACHE_LAYER_OUT_OF_RANGE);
    CHECK(append(0, k, v, 0, rows) == CKV_E_INVALID_ARGUMENT);
    auto rope_window = [&](float theta, size_t rotary) {
        return ckv_rope_append_decode_window(&pool, 0, k, v, q, 4, 1.0f, theta, rotary, 8, 4, nullptr,
                                             o, rows);
    };
    CHECK(rope_window(0.0f, 0) == CKV_E_INVALID_ROPE_THETA);
    CHECK(rope_window(1e4f, 3) == CKV_E_INVALID_HEAD_DIMENSION);

    CHECK(ckv_rope_axes_upload(&pool, positions, 0, rows) == CKV_E_INVALID_ARGUMENT);
    CHECK(ckv_rope_axes_upload(&pool, positions, 5, rows) == CKV_E_INVALID_ARGUMENT);
    CHECK(ckv_rope_axes_upload(&pool, positions, 3, 1) == CKV_E_POSITION_COUNT_MISMATCH);
    uint8_t axis[64] = {};
    auto axes = [&](size_t heads, float theta, size_t rotary, const uint8_t* a, size_t n = rows) {
        const int one = ckv_rope_axes(&pool, q, o, heads, theta, rotary, a, n);
        return one;
    };
    CHECK(axes(4, 1e4f, 0, axis) == CKV_E_NO_TABLES); // before the upload
    pool.axes = 3;
    CHECK(axes(4, 1e4f, 0, axis, 3) == CKV_E_POSITION_COUNT_MISMATCH);
    CHECK(axes(0, 1e4f, 0, axis) == CKV_E_INVALID_HEAD_COUNT);
    CHECK(axes(4, 1e4f, 130, axis) == CKV_E_INVALID_HEAD_DIMENSION);
    CHECK(axes(4, 1e4f, 7, axis) == CKV_E_INVALID_HEAD_DIMENSION);
    CHECK(axes(4, -1.0f, 0, axis) == CKV_E_INVALID_ROPE_THETA);
    CHECK(axes(4, INFINITY, 0, axis) == CKV_E_INVALID_ROPE_THETA);
    CHECK(axes(4, 1e4f, 0, nullptr) == CKV_E_INVALID_ARGUMENT);
    axis[63] = 3;
    CHECK(axes(4, 1e4f, 0, axis) == CKV_E_INVALID_ARGUMENT);
    auto axes_append = [&](const void* queries, void* rotated, size_t heads, const void* keys) {
        return ckv_rope_axes_append(&pool, 0, queries, rotated, heads, keys, v, 1e4f, 0, axis, rows);
    };
    CHECK(axes_append(q, o, 4, k) == CKV_E_INVALID_ARGUMENT); // axis 3 again
    axis[63] = 0;
    CHECK(axes_append(nullptr, o, 4, k) == CKV_E_INVALID_ARGUMENT);
    CHECK(axes_append(q, nullptr, 4, k) == CKV_E_INVALID_ARGUMENT);
    CHECK(axes_append(q, k, 4, k) == CKV_E_UNSUPPORTED_ALIASING);
    CHECK(axes_append(q, v, 4, k) == CKV_E_UNSUPPORTED_ALIASING);
    pool.head_dim = 1024;
    CHECK(axes(4, 1e4f, 0, axis) == CKV_E_INVALID_HEAD_DIMENSION);
    pool.head_dim = 128;

    const uint32_t from[] = { 5, 6 }, to[] = { 1, 2 }, counts[] = { 2 };
    const int32_t shift[] = { -4, -4 };
    CHECK(ckv_compact(nullptr, from, to, shift, counts, 1, 1e4f, 0) == CKV_E_INVALID_ARGUMENT);
    CHECK(ckv_compact(&pool, from, to, shift, nullptr, 1, 1e4f, 0) == CKV_E_INVALID_ARGUMENT);
    CHECK(ckv_compact(&pool, nullptr, to, shift, counts, 1, 1e4f, 0) == CKV_E_INVALID_ARGUMENT);
    CHECK(ckv_compact(&pool, from, nullptr, shift, counts, 1, 1e4f, 0) == CKV_E_INVALID_ARGUMENT);
    CHECK(ckv_compact(&pool, from, to, shift, counts, 1, 0.0f, 0) == CKV_E_INVALID_ROPE_THETA);
    CHECK(ckv_compact(&pool, from, to, shift, counts, 1, 1e4f, 129) == CKV_E_INVALID_HEAD_DIMENSION);
    CHECK(ckv_compact(&pool, from, to, shift, counts, 1, 1e4f, 256) == CKV_E_INVALID_HEAD_DIMENSION);
    const uint32_t far[] = { 5, 128 }, same[] = { 1, 1 };
    CHECK(ckv_compact(&pool, far, to, nullptr, counts, 1, 0.0f, 0) == CKV_E_CACHE_SLOT_OUT_OF_RANGE);
    CHECK(ckv_compact(&pool, from, same, nullptr, counts, 1, 0.0f, 0) == CKV_E_UNSUPPORTED_ALIASING);
    const uint32_t many[] = { UINT32_MAX, UINT32_MAX };
    CHECK(ckv_compact(&pool, from, to, nullptr, many, 2, 0.0f, 0) == CKV_E_UNSUPPORTED_ALIASING);
    // nothing to do
    const uint32_t none[] = { 0 };
    CHECK(ckv_compact(&pool, nullptr, nullptr, nullptr, none, 1, 0.0f, 0) == CKV_OK);
    {
        const size_t blocks = pool.blocks;
        pool.blocks = (size_t(1) << 31) / pool.block_size + 1; // a slot past what the move lists hold
        CHECK(ckv_compact(&pool, from, to, nullptr, counts, 1, 0.0f, 0) == CKV_E_INVALID_ARGUMENT);
        pool.blocks = blocks;
    }
    CHECK(ckv_compact(&pool, from, from, nullptr, counts, 1, 0.0f, 0) == CKV_OK);
    pool.positions.clear();
    CHECK(attend(0, nullptr, 4, 8, nullptr, nullptr, 0) == CKV_OK);
}

// Head counts whose rows pass 32 bits, or that wrap once kv heads are added, reach no launch.
TEST("entry points: rows too wide for 32 bits are refused")
{
    ckv_context ctx;
    ckv_pool pool;
    pool.ctx = &ctx;
    pool.layers = 1;
    pool.blocks = 8;
    pool.block_size = 16;
    pool.kv_heads = 2;
    pool.head_dim = 128;
    pool.uploaded = pool.has_slots = true;
    pool.positions = { 40, 50 };
    pool.last_position = 50;
    pool.slot_rows = 2;
    pool.axes = 1;
    int x[4]; // never read
    const uint8_t axis[64] = {};
    for (const size_t heads : { (size_t)1 << 25, (size_t)1 << 32, (size_t)1 << 57, ((size_t)1 << 57) + 2,
                                SIZE_MAX - 1, SIZE_MAX - 3 }) {
        CHECK(ckv_rope_axes(&pool, x, x + 1, heads, 1e4f, 0, axis, 2) == CKV_E_INVALID_ARGUMENT);
        CHECK(ckv_rope_axes_append(&pool, 0, x, x, heads, x + 1, x + 2, 1e4f, 0, axis, 2)
              == CKV_E_INVALID_ARGUMENT);
        CHECK(ckv_rope(&pool, x, x + 1, heads, 1e4f, 0, 2) == CKV_E_INVALID_ARGUMENT);
        CHECK(ckv_attention_window(&pool, 0, x, heads, 1.0f, 8, 0, nullptr, x + 1, 2)
              == CKV_E_INVALID_ARGUMENT);
        CHECK(ckv_append_decode_window(&pool, 0, x, x + 1, x + 2, heads, 1.0f, 8, 0, nullptr, x + 3, 2)
              == CKV_E_INVALID_ARGUMENT);
        CHECK(ckv_attention(&pool, 0, x, heads, 1.0f, x + 1, 2) == CKV_E_INVALID_ARGUMENT);
        CHECK(ckv_append_decode(&pool, 0, x, x + 1, x + 2, heads, 1.0f, x + 3, 2) == CKV_E_INVALID_ARGUMENT);
        CHECK(ckv_append_decode_noalloc(&pool, 0, x, x + 1, x + 2, heads, 1.0f, x + 3, 2)
              == CKV_E_INVALID_ARGUMENT);
    }
}

// The forms that the device tests of large batches mean to reach, at their sizes
// (tests/test_gpu_operators_large.py).
TEST("launch forms: heads a workgroup of a compaction and a thread of a rotation take")
{
    auto pool = [](int dtype, uint32_t kv_heads, uint32_t head_dim) {
        pool_view p {};
        p.dtype = dtype;
        p.elem_size = dtype == CKV_F32 ? 4 : 2;
        p.kv_heads = kv_heads;
        p.head_dim = head_dim;
        p.features = kv_heads * head_dim;
        return p;
    };
    auto runs = [](uint32_t moves) { return (moves + compact_run - 1) / compact_run; };
    CHECK(compact_heads(pool(CKV_BF16, 8, 64), 12, runs(6000), 64) == 8);
    CHECK(compact_heads(pool(CKV_BF16, 8, 64), 12, runs(3500), 64) == 4);
    CHECK(compact_heads(pool(CKV_F32, 8, 64), 12, runs(1800), 32) == 2);
    CHECK(compact_heads(pool(CKV_F16, 8, 64), 12, runs(1000), 0) == 1);
    CHECK(compact_heads(pool(CKV_F32, 4, 128), 16, runs(4200), 128) == 4);
    CHECK(compact_heads(pool(CKV_F16, 3, 256), 2, runs(900), 64) == 3); // an odd number never halves
    CHECK(compact_heads(pool(CKV_F16, 6, 256), 2, runs(900), 64) == 3);
    CHECK(compact_heads(pool(CKV_F32, 3, 33), 12, runs(6000), 0) == 0);
    CHECK(compact_heads(pool(CKV_BF16, 8, 64), 12, runs(6000), 24) == 0);
    pool_view odd = pool(CKV_BF16, 8, 64);
    odd.values = reinterpret_cast<void*>(8);
    CHECK(compact_heads(odd, 12, runs(6000), 64) == 0);
    const axes_rows x {};
    CHECK(rope_axes_heads(pool(CKV_BF16, 8, 128), x, 4200, 16, 128) == 4);
    CHECK(rope_axes_heads(pool(CKV_BF16, 7, 128), x, 4700, 14, 48) == 4);
    CHECK(rope_axes_heads(pool(CKV_F16, 3, 256), x, 5500, 6, 64) == 4);
    CHECK(rope_axes_heads(pool(CKV_F32, 5, 64), x, 13200, 5, 64) == 4);
    CHECK(rope_axes_heads(pool(CKV_BF16, 8, 128), x, 4000, 16, 128) == 1);
    CHECK(rope_axes_heads(pool(CKV_BF16, 8, 128), x, 4200, 16, 24) == 0);
    axes_rows unaligned {};
    unaligned.rotated = reinterpret_cast<void*>(2);
    CHECK(rope_axes_heads(pool(CKV_BF16, 8, 128), unaligned, 4200, 16, 128) == 0);
}

constexpr uint32_t page = 16;

// The plan of rows at `positions` behind a window, its structure checked: a row's chunks
// cover the pages that hold a key it attends, each once and in order, with the row's own
// position, its records behind one another, and workgroups linked through every entry.
decode_plan_shape window_plan_of(const std::vector<uint32_t>& positions, key_window w, uint32_t kv_heads,
                                 int cus, int dtype, uint32_t head_dim)
{
    const size_t rows = positions.size();
    std::vector<uint32_t> left(rows), offsets(rows);
    for (size_t r = 0, at = 0; r < rows; at += positions[r] / page + 1, ++r) {
        left[r] = positions[r] - window_gap_of(window_low(positions[r], w), w.sinks, page).skip * page;
        offsets[r] = (uint32_t)at;
    }
    const decode_plan_shape s = shape_window_plan(left, page, kv_heads, cus, window_form_of(dtype, head_dim));
    std::vector<uint32_t> plan(plan_entry_words * s.n_items, 0xDEADBEEFu), first(rows, 0xDEADBEEFu),
        cut(s.n_cut, 0xDEADBEEFu);
    std::vector<uint64_t> scratch;
    write_decode_plan(left, offsets, page, s, scratch, plan.data(), first.data(), cut.data());
    place_window_plan(positions, s, plan.data());
    REQUIRE(s.n_wgs >= 1 && s.n_wgs <= s.n_items);
    std::vector<int> reached(s.n_items, 0);
    struct piece {
        uint32_t chunk, first, end, of;
    };
    std::vector<std::vector<piece>> pieces(rows);
    for (uint32_t wg = 0; wg < s.n_wgs; ++wg)
        for (uint32_t at = wg; at != plan_last;) {
            REQUIRE(at < s.n_items && !reached[at]++);
            const uint32_t* e = &plan[plan_entry_words * at];
            REQUIRE(e[0] < rows);
            CHECK(e[2] == positions[e[0]] && e[3] == offsets[e[0]] + e[4]);
            pieces[e[0]].push_back({ e[1], e[4], e[5], e[6] });
            at = e[7];
        }
    CHECK(std::count(reached.begin(), reached.end(), 1) == (std::ptrdiff_t)s.n_items);
    uint32_t records = 0, cuts = 0;
    std::vector<int> taken(s.n_records, 0);
    for (size_t r = 0; r < rows; ++r) {
        auto& of = pieces[r];
        std::sort(of.begin(), of.end(), [](const piece& a, const piece& b) { return a.chunk < b.chunk; });
        const window_gap gap = window_gap_of(window_low(positions[r], w), w.sinks, page);
        std::vector<uint32_t> read;
        uint32_t at = 0;
        for (size_t c = 0; c < of.size(); ++c) {
            REQUIRE(of[c].chunk == c && of[c].of == of.size() && of[c].first == at && of[c].end > at);
            at = of[c].end;
            for (uint32_t u = of[c].first; u < of[c].end; ++u)
                read.push_back(u < gap.kept ? u : u + gap.skip);
        }
        std::vector<uint32_t> want;
        for (uint32_t u = 0; u <= positions[r] / page; ++u) {
            bool some = false;
            for (uint32_t t = u * page; t < (u + 1) * page; ++t)
                some = some || attends(positions[r], t, w);
            if (some)
                want.push_back(u);
        }
        CHECK(read == want);
        if (of.size() > 1) {
            ++cuts;
            records += (uint32_t)of.size();
            for (size_t c = 0; c < of.size(); ++c) {
                REQUIRE(first[r] + c < s.n_records);
                CHECK(!taken[first[r] + c]++);
            }
            CHECK(std::count(cut.begin(), cut.end(), (uint32_t)r) == 1);
        }
    }
    CHECK(records == s.n_records && cuts == s.n_cut);
    return s;
}

TEST("window plan: every row's attended pages once, at any size")
{
    std::mt19937_64 rng(11);
    for (int trial = 0; trial < 600; ++trial) {
        const uint32_t kv_heads = 1u << rng() % 4, rows = 1 + rng() % (trial % 5 ? 40 : 200);
        const int cus = trial % 3 ? 256 : 1 + (int)(rng() % 300);
        const key_window w { 1 + (uint32_t)(rng() % (trial % 2 ? 2100 : 90)), (uint32_t)(rng() % 3 * (rng() % 70)) };
        const uint32_t high = 40 + rng() % 5000;
        std::vector<uint32_t> positions(rows);
        for (auto& p : positions)
            p = rng() % high;
        const int dtype = (int)(rng() % 3);
        window_plan_of(positions, w, kv_heads, cus, dtype, rng() % 2 ? 128 : 256);
    }
}

TEST("window plan: halves of rows of equal length, from one to one and a half units per compute unit")
{
    const key_window w { 1024, 4 };
    auto rows = [](size_t n) {
        std::vector<uint32_t> p(n);
        for (size_t r = 0; r < n; ++r)
            p[r] = 1500 + 211 * (uint32_t)r % 9000;
        return p;
    };
    for (const size_t n : { 33u, 40u, 48u }) { // 8 kv heads: 264 to 384 units
        const decode_plan_shape s = window_plan_of(rows(n), w, 8, 256, CKV_BF16, 128);
        CHECK(s.n_cut == n && s.n_records == 2 * n && (s.split_pages == 33 || s.split_pages == 34));
    }
    // one unit per compute unit or fewer is cut as any small batch is, more than one and a half stay whole
    CHECK(window_plan_of(rows(49), w, 8, 256, CKV_BF16, 128).n_cut == 0);
    CHECK(window_plan_of(rows(64), w, 8, 256, CKV_BF16, 128).n_cut == 0);
    CHECK(window_plan_of(rows(80), w, 8, 256, CKV_F16, 128).n_cut == 0);
    CHECK(window_plan_of(rows(32), w, 8, 256, CKV_BF16, 128).n_records != 64);
    // 32 pages behind 512 tokens are too few to halve, 256-wide rows of 17 are not
    CHECK(window_plan_of(rows(40), { 490, 0 }, 8, 256, CKV_BF16, 128).n_records == 0);
    CHECK(window_plan_of(rows(40), { 272, 4 }, 8, 256, CKV_BF16, 256).n_records == 80);
    CHECK(window_plan_of(rows(40), w, 8, 256, CKV_F32, 128).n_records != 80);
    // rows of unequal length are not halved
    std::vector<uint32_t> uneven = rows(40);
    for (size_t r = 0; r < 20; ++r)
        uneven[r] = 100;
    CHECK(window_plan_of(uneven, w, 8, 256, CKV_BF16, 128).n_records != 80);
}

TEST("window plan: pieces of small batches, an eighth of the longest row")
{
    auto pieces = [](size_t n, uint32_t window, int dtype, uint32_t head_dim) {
        return window_plan_of(std::vector<uint32_t>(n, 4000), { window, 0 }, 8, 256, dtype, head_dim).split_pages;
    };
    CHECK(pieces(4, 512, CKV_BF16, 128) == 4 || pieces(4, 512, CKV_BF16, 128) == 5);
    CHECK(pieces(1, 256, CKV_BF16, 128) == 4); // 17 pages
    CHECK(pieces(1, 241, CKV_BF16, 128) == 12); // 16: the pieces of a batch without a window
    CHECK(window_plan_of({ 4000 }, { 177, 0 }, 8, 256, CKV_BF16, 128).n_records == 0); // 12 stay whole
    CHECK(pieces(2, 2000, CKV_BF16, 128) >= 12);
    CHECK(pieces(3, 300, CKV_F32, 128) >= 4 && pieces(3, 300, CKV_F32, 128) < 8);
}

TEST("window decode: waves of a workgroup")
{
    if (std::getenv("CKV_DECODE_WAVES"))
        return;
    auto waves = [](uint32_t head_dim, uint32_t group, int dtype, uint32_t units, uint32_t split) {
        return decode_window_waves(head_dim, group, dtype, units, 256, 65, split);
    };
    CHECK(waves(128, 2, CKV_F32, 400, 0) == 4);
    CHECK(waves(128, 2, CKV_BF16, 40, 4) == 4);    // pieces of four pages
    CHECK(waves(128, 2, CKV_BF16, 200, 0) == 16);  // a workgroup to a compute unit and to spare
    CHECK(waves(128, 4, CKV_BF16, 200, 0) == 8);
    CHECK(waves(128, 2, CKV_BF16, 768, 33) == 4);  // halves of 48 rows
    CHECK(waves(128, 8, CKV_BF16, 768, 33) == 8);
    CHECK(waves(128, 2, CKV_BF16, 400, 0) == 8);   // whole rows, one to two units per compute unit
    CHECK(waves(128, 2, CKV_BF16, 640, 0) == 4);   // more
    CHECK(waves(128, 4, CKV_BF16, 640, 0) == 4);
    CHECK(waves(128, 8, CKV_BF16, 512, 0) == 4);
    CHECK(waves(128, 8, CKV_BF16, 640, 0) == 8);
    CHECK(waves(256, 4, CKV_BF16, 640, 0) == 8);
}

} // namespace
