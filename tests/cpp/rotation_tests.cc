// What the calls of scaled rotations, whole prompts and 4-bit pools refuse, over pools without
// device memory, and the work lists of tiles. Each case gives the status a caller gets.
#include <algorithm>
#include <cmath>
#include <limits>

#include "check.h"
#include "ckv_internal.h"

using namespace ckv;

namespace {

struct two_rows {
    ckv_context ctx;
    ckv_pool pool;
    int x[8]; // never read: no call gets that far
    two_rows()
    {
        pool.ctx = &ctx;
        pool.layers = 2;
        pool.blocks = 8;
        pool.block_size = 16;
        pool.kv_heads = 2;
        pool.head_dim = 128;
        pool.dtype = CKV_BF16;
    }
    void upload()
    {
        pool.uploaded = pool.has_slots = true;
        pool.positions = { 0, 1 };
        pool.row_offsets = { 0, 0 };
        pool.last_position = 1;
        pool.slot_rows = 2;
    }
};

ckv_rotation plain()
{
    ckv_rotation r {};
    r.theta = 1e4f;
    return r;
}

} // namespace

TEST("rotations: arguments that are refused")
{
    two_rows t;
    ckv_pool* p = &t.pool;
    void *q = t.x, *o = t.x + 1, *k = t.x + 2, *v = t.x + 3, *a = t.x + 4, *b = t.x + 5;
    ckv_rotation r = plain();
    CHECK(ckv_rotate(nullptr, &r, q, o, 2, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(ckv_rotate(p, &r, q, o, 2, 2) == CKV_E_NO_TABLES);
    CHECK(ckv_rotate_append(p, 0, &r, q, o, 4, k, v, a, b, 2) == CKV_E_NO_TABLES);
    CHECK(ckv_rotate_append_decode(p, 0, &r, k, v, q, 4, 1.0f, nullptr, a, b, o, 2) == CKV_E_NO_TABLES);
    t.upload();
    CHECK(ckv_rotate(p, nullptr, q, o, 2, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(ckv_rotate(p, &r, nullptr, o, 2, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(ckv_rotate(p, &r, q, nullptr, 2, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(ckv_rotate(p, &r, q, o, 2, 3) == CKV_E_POSITION_COUNT_MISMATCH);
    CHECK(ckv_rotate(p, &r, q, o, 0, 2) == CKV_E_INVALID_HEAD_COUNT);
    for (const size_t heads : { (size_t)1 << 25, (size_t)1 << 57, SIZE_MAX })
        CHECK(ckv_rotate(p, &r, q, o, heads, 2) == CKV_E_INVALID_ARGUMENT);
    // every check of the rotation holds in each call that takes one
    const auto all = [&](const ckv_rotation& x) {
        const int one = ckv_rotate(p, &x, q, o, 2, 2);
        CHECK(one == ckv_rotate_append(p, 0, &x, q, o, 4, k, v, a, b, 2));
        CHECK(one == ckv_rotate_append_decode(p, 0, &x, k, v, q, 4, 1.0f, nullptr, a, b, o, 2));
        return one;
    };
    const float inf = std::numeric_limits<float>::infinity(), nan = std::nanf("");
    for (const uint32_t width : { 3u, 130u, 1u, UINT32_MAX }) {
        r = plain();
        r.rotary_dim = width;
        CHECK(all(r) == CKV_E_INVALID_HEAD_DIMENSION);
    }
    for (const float theta : { 0.0f, -1.0f, inf, nan }) {
        r = plain();
        r.theta = theta;
        CHECK(all(r) == CKV_E_INVALID_ROPE_THETA);
    }
    for (const int wrong : { -1, 2 }) {
        r = plain();
        r.layout = wrong;
        CHECK(all(r) == CKV_E_INVALID_ARGUMENT);
        r = plain();
        r.scaling = wrong < 0 ? wrong : 4;
        CHECK(all(r) == CKV_E_INVALID_ARGUMENT);
    }
    for (const int scaling : { CKV_SCALING_LINEAR, CKV_SCALING_BANDS, CKV_SCALING_YARN }) {
        ckv_rotation good = plain();
        good.scaling = scaling;
        good.factor = 4.0f;
        good.low = 1.0f;
        good.high = 32.0f;
        good.original = 4096;
        for (const float wrong : { 0.0f, -2.0f, inf, nan }) {
            r = good;
            r.factor = wrong;
            CHECK(all(r) == CKV_E_INVALID_ARGUMENT);
        }
        for (const float wrong : { -1.0f, inf, nan }) {
            r = good;
            r.magnitude = wrong;
            CHECK(all(r) == CKV_E_INVALID_ARGUMENT);
        }
        if (scaling == CKV_SCALING_LINEAR)
            continue;
        for (const float wrong : { 0.0f, -1.0f, 32.0f, 40.0f, inf, nan }) {
            r = good;
            r.low = wrong;
            CHECK(all(r) == CKV_E_INVALID_ARGUMENT);
        }
        r = good;
        r.high = nan;
        CHECK(all(r) == CKV_E_INVALID_ARGUMENT);
        r = good;
        r.original = 0;
        CHECK(all(r) == CKV_E_INVALID_ARGUMENT);
        r = good;
        r.theta = 1.0f;
        if (scaling == CKV_SCALING_YARN)
            CHECK(all(r) == CKV_E_INVALID_ARGUMENT);
    }
    r = plain();
    p->head_dim = 1024; // more pairs than a rotation's table
    CHECK(all(r) == CKV_E_INVALID_HEAD_DIMENSION);
    p->head_dim = 5;
    CHECK(all(r) == CKV_E_INVALID_HEAD_DIMENSION);
}

TEST("rotated appends: arguments that are refused")
{
    two_rows t;
    t.upload();
    ckv_pool* p = &t.pool;
    void *q = t.x, *o = t.x + 1, *k = t.x + 2, *v = t.x + 3, *a = t.x + 4, *b = t.x + 5, *g = t.x + 6;
    const ckv_rotation r = plain();
    const auto put = [&](size_t layer, void* q, void* o, size_t heads, void* k, void* v, void* a, void* b, size_t n) {
        return ckv_rotate_append(p, layer, &r, q, o, heads, k, v, a, b, n);
    };
    CHECK(put(0, q, o, 4, nullptr, v, a, b, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(put(0, q, o, 4, k, nullptr, a, b, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(put(0, q, o, 4, k, v, a, b, 3) == CKV_E_CACHE_SLOT_COUNT_MISMATCH);
    CHECK(put(2, q, o, 4, k, v, a, b, 2) == CKV_E_CACHE_LAYER_OUT_OF_RANGE);
    CHECK(put(0, nullptr, o, 4, k, v, a, b, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(put(0, q, nullptr, 4, k, v, a, b, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(put(0, q, k, 4, k, v, a, b, 2) == CKV_E_UNSUPPORTED_ALIASING);
    CHECK(put(0, q, v, 4, k, v, a, b, 2) == CKV_E_UNSUPPORTED_ALIASING);
    for (void* taken : { q, o, k, v, b })
        CHECK(put(0, q, o, 4, k, v, taken, b, 2) == CKV_E_UNSUPPORTED_ALIASING);
    for (void* taken : { q, o, k, v })
        CHECK(put(0, q, o, 4, k, v, nullptr, taken, 2) == CKV_E_UNSUPPORTED_ALIASING);
    for (const size_t heads : { (size_t)1 << 25, (size_t)1 << 57, SIZE_MAX - 1, SIZE_MAX })
        CHECK(put(0, q, o, heads, k, v, a, b, 2) == CKV_E_INVALID_ARGUMENT);
    const auto step = [&](size_t layer, size_t heads, void* k, void* v, void* q, void* g, void* a, void* b, void* o, size_t n) {
        return ckv_rotate_append_decode(p, layer, &r, k, v, q, heads, 1.0f, g, a, b, o, n);
    };
    CHECK(step(0, 4, nullptr, v, q, g, a, b, o, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(step(0, 4, k, v, nullptr, g, a, b, o, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(step(0, 4, k, v, q, g, a, b, nullptr, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(step(0, 4, k, v, q, g, a, b, o, 1) == CKV_E_CACHE_SLOT_COUNT_MISMATCH);
    CHECK(step(2, 4, k, v, q, g, a, b, o, 2) == CKV_E_CACHE_LAYER_OUT_OF_RANGE);
    CHECK(step(0, 0, k, v, q, g, a, b, o, 2) == CKV_E_INVALID_HEAD_COUNT);
    CHECK(step(0, 3, k, v, q, g, a, b, o, 2) == CKV_E_INVALID_KV_HEAD_MAPPING);
    CHECK(step(0, (size_t)1 << 57, k, v, q, g, a, b, o, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(step(0, 4, k, v, q, q, a, b, o, 2) == CKV_E_UNSUPPORTED_ALIASING);
    CHECK(step(0, 4, k, v, q, o, a, b, o, 2) == CKV_E_UNSUPPORTED_ALIASING);
    for (void* taken : { q, k, v, g, o, b })
        CHECK(step(0, 4, k, v, q, g, taken, b, o, 2) == CKV_E_UNSUPPORTED_ALIASING);
}

TEST("whole prompts: arguments and batches that are refused")
{
    two_rows t;
    ckv_pool* p = &t.pool;
    void *q = t.x, *k = t.x + 1, *v = t.x + 2, *o = t.x + 3, *g = t.x + 4;
    const auto attend = [&](void* q, size_t qs, void* k, void* v, size_t ks, size_t heads, void* g, void* o, size_t n) {
        return ckv_prompt_attention(p, q, qs, k, v, ks, heads, 1.0f, g, o, n);
    };
    CHECK(ckv_prompt_attention(nullptr, q, 0, k, v, 0, 4, 1.0f, g, o, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(attend(q, 0, k, v, 0, 4, g, o, 2) == CKV_E_NO_TABLES);
    t.upload();
    for (const int none : { 0, 1, 2, 3 })
        CHECK(attend(none == 0 ? nullptr : q, 0, none == 1 ? nullptr : k, none == 2 ? nullptr : v, 0, 4, g,
                     none == 3 ? nullptr : o, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(attend(q, 0, k, v, 0, 4, g, o, 3) == CKV_E_POSITION_COUNT_MISMATCH);
    CHECK(attend(q, 0, k, v, 0, 0, g, o, 2) == CKV_E_INVALID_HEAD_COUNT);
    CHECK(attend(q, 0, k, v, 0, 3, g, o, 2) == CKV_E_INVALID_KV_HEAD_MAPPING);
    CHECK(attend(q, 0, k, v, 0, (size_t)1 << 57, g, o, 2) == CKV_E_INVALID_ARGUMENT);
    for (void* taken : { q, k, v, g })
        CHECK(attend(q, 0, k, v, 0, 4, g, taken, 2) == CKV_E_UNSUPPORTED_ALIASING);
    for (void* taken : { q, k, v })
        CHECK(attend(q, 0, k, v, 0, 4, taken, o, 2) == CKV_E_UNSUPPORTED_ALIASING);
    CHECK(attend(q, 511, k, v, 0, 4, g, o, 2) == CKV_E_INPUT_SHAPE_MISMATCH);
    CHECK(attend(q, 512, k, v, 255, 4, g, o, 2) == CKV_E_INPUT_SHAPE_MISMATCH);
    for (const size_t dim : { 32, 96, 512 }) {
        p->head_dim = dim;
        CHECK(attend(q, 0, k, v, 0, 4, g, o, 2) == CKV_E_INVALID_HEAD_DIMENSION);
    }
    p->head_dim = 128;
    const auto batch = [&](std::vector<uint32_t> positions, std::vector<uint32_t> offsets) {
        p->positions = positions;
        p->row_offsets = offsets;
        p->whole_prompts = -1;
        return attend(q, 0, k, v, 0, 4, g, o, positions.size());
    };
    CHECK(batch({ 1, 2 }, { 0, 0 }) == CKV_E_INVALID_ARGUMENT); // begins behind its first token
    CHECK(batch({ 0, 2 }, { 0, 0 }) == CKV_E_INVALID_ARGUMENT); // a token left out
    CHECK(batch({ 0, 1 }, { 0, 1 }) == CKV_E_INVALID_ARGUMENT); // of two tables
    CHECK(batch({ 0, 1, 1 }, { 0, 0, 0 }) == CKV_E_INVALID_ARGUMENT); // a token twice
    CHECK(batch({ 0, 1, 5, 6 }, { 0, 0, 1, 1 }) == CKV_E_INVALID_ARGUMENT); // a chunk among prompts
}

TEST("4-bit pools: geometries and calls that are refused")
{
    ckv_context ctx;
    ckv_pool* out = nullptr;
    int memory[8];
    const auto make = [&](size_t layers, size_t blocks, size_t size, size_t heads, size_t dim, int dtype) {
        const int a = ckv_pool_create_fp4(&ctx, layers, blocks, size, heads, dim, dtype, &out);
        CHECK(a == ckv_pool_wrap_fp4(&ctx, layers, blocks, size, heads, dim, dtype, memory, memory + 4, &out));
        CHECK(out == nullptr);
        return a;
    };
    CHECK(ckv_pool_create_fp4(nullptr, 1, 1, 16, 1, 64, CKV_BF16, &out) == CKV_E_INVALID_ARGUMENT);
    CHECK(ckv_pool_create_fp4(&ctx, 1, 1, 16, 1, 64, CKV_BF16, nullptr) == CKV_E_INVALID_ARGUMENT);
    CHECK(make(1, 1, 16, 1, 64, 17) == CKV_E_UNSUPPORTED_DTYPE);
    for (const size_t size : { 1, 8, 15, 24, 48, 8192 })
        CHECK(make(1, 1, size, 1, 64, CKV_BF16) == CKV_E_INVALID_BLOCK_SIZE);
    for (const size_t dim : { 32, 80, 96, 192, 512 })
        CHECK(make(1, 1, 16, 1, dim, CKV_F32) == CKV_E_INVALID_HEAD_DIMENSION_KV);
    CHECK(ckv_pool_wrap_fp4(&ctx, 1, 1, 16, 1, 64, CKV_BF16, nullptr, memory, &out) == CKV_E_INVALID_ARGUMENT);
    CHECK(ckv_pool_wrap_fp4(&ctx, 1, 1, 16, 1, 64, CKV_BF16, (char*)memory + 1, memory, &out) == CKV_E_INVALID_ARGUMENT);

    two_rows t;
    t.upload();
    ckv_pool* p = &t.pool;
    p->positions = { 5, 9 }; // two decode rows
    p->fp4 = true;
    void *q = t.x, *k = t.x + 1, *v = t.x + 2, *o = t.x + 3;
    size_t offset = 0;
    const uint8_t axis[64] = {};
    const uint32_t words[2] = { 0, 1 };
    CHECK(ckv_attention_window(p, 0, q, 4, 1.0f, 8, 0, nullptr, o, 2) == CKV_E_UNSUPPORTED_DTYPE);
    CHECK(ckv_append_decode_window(p, 0, k, v, q, 4, 1.0f, 8, 0, nullptr, o, 2) == CKV_E_UNSUPPORTED_DTYPE);
    CHECK(ckv_rope_append_decode_window(p, 0, k, v, q, 4, 1.0f, 1e4f, 0, 8, 0, nullptr, o, 2) == CKV_E_UNSUPPORTED_DTYPE);
    CHECK(ckv_append_decode_noalloc(p, 0, k, v, q, 4, 1.0f, o, 2) == CKV_E_UNSUPPORTED_DTYPE);
    p->axes = 1;
    CHECK(ckv_rope_axes_append(p, 0, q, o, 4, k, v, 1e4f, 0, axis, 2) == CKV_E_UNSUPPORTED_DTYPE);
    CHECK(ckv_compact(p, words, words, nullptr, words + 1, 1, 0.0f, 0) == CKV_E_UNSUPPORTED_DTYPE);
    CHECK(ckv_element_offset(p, 0, 0, 0, 0, 0, &offset) == CKV_E_UNSUPPORTED_DTYPE);
    CHECK(ckv_checkpoint_pack(p, words, 1, 16, k, v) == CKV_E_UNSUPPORTED_DTYPE);
    CHECK(ckv_checkpoint_unpack(p, words, 1, 16, k, v) == CKV_E_UNSUPPORTED_DTYPE);
    CHECK(ckv_decode_attention(p, 0, q, 2 << 19, 1.0f, o, 2) == CKV_E_INVALID_ARGUMENT); // decode rows too wide
    // what they refuse of every pool they refuse of these
    CHECK(ckv_append(p, 0, nullptr, v, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(ckv_append(p, 0, k, v, 3) == CKV_E_CACHE_SLOT_COUNT_MISMATCH);
    CHECK(ckv_attention(p, 0, q, 3, 1.0f, o, 2) == CKV_E_INVALID_KV_HEAD_MAPPING);
    CHECK(ckv_attention_gated(p, 0, q, 4, 1.0f, nullptr, o, 2) == CKV_E_INVALID_ARGUMENT);
    CHECK(ckv_gather(p, 2, 0, 0, 0, k, v) == CKV_E_CACHE_LAYER_OUT_OF_RANGE);
}

// Every row of every tile is listed with every one of its key blocks once, records and cut
// tiles have places of their own, and the longest ranges come first.
TEST("work lists: every tile's key blocks once")
{
    for (const int dtype : { CKV_BF16, CKV_F32 })
        for (const uint32_t dim : { 64u, 128u, 256u })
            for (const uint32_t heads : { 1u, 2u, 4u })
                for (const std::vector<uint32_t>& prompts : { std::vector<uint32_t> { 1 }, { 900 }, { 17, 1, 300, 64 },
                                                             { 5000 }, { 33, 8000, 1 }, std::vector<uint32_t>(600, 40) })
                    for (const uint32_t behind : { 0u, 6001u }) {
                        pool_view p {};
                        p.dtype = dtype;
                        p.head_dim = dim;
                        prompt_form form {};
                        form.waves = 4;
                        form.heads = heads;
                        std::vector<uint32_t> tiles;
                        uint32_t row = 0, table = 0;
                        for (const uint32_t n : prompts) {
                            for (uint32_t r = 0; r < n; r += 256)
                                tiles.insert(tiles.end(), { row + r, std::min(256u, n - r), behind + r, table });
                            row += n;
                            table += 7;
                        }
                        prompt_list list;
                        write_prompt_list(p, tiles, form, heads, 256, list);
                        REQUIRE(list.words.size() % prompt_entry_words == 0);
                        std::vector<uint32_t> ranges(row, 0), wanted(row, 0);
                        std::vector<bool> record(list.n_records, false);
                        uint32_t cut = 0, last = UINT32_MAX;
                        for (size_t e = 0; e < list.words.size(); e += prompt_entry_words) {
                            const uint32_t* w = &list.words[e];
                            REQUIRE(w[1] >= 1 && w[1] <= 128 / heads && w[0] + w[1] <= row);
                            const uint32_t blocks = (w[2] + w[1] - 1) / 32 + 1, length = (blocks + w[5] - 1) / w[5];
                            CHECK(w[4] < w[5] && w[5] <= blocks && w[5] <= 16);
                            CHECK(length <= last);
                            last = length;
                            for (uint32_t r = w[0]; r < w[0] + w[1]; ++r) {
                                ++ranges[r];
                                wanted[r] = w[5];
                            }
                            if (w[5] == 1)
                                continue;
                            REQUIRE(w[6] + w[5] <= list.n_records && w[7] < list.n_cut);
                            CHECK(!record[w[6] + w[4]]);
                            record[w[6] + w[4]] = true;
                            cut += w[4] == 0;
                        }
                        CHECK(ranges == wanted);
                        CHECK(std::all_of(ranges.begin(), ranges.end(), [](uint32_t n) { return n > 0; }));
                        CHECK(std::all_of(record.begin(), record.end(), [](bool x) { return x; }));
                        CHECK(cut == list.n_cut);
                        // one short prompt on an idle chip is not cut into ranges of nothing
                        if (prompts.size() == 600 && !behind)
                            CHECK(list.n_cut == 0);
                    }
}

// 256-wide heads: once a call of a 4-bit pool has met a stream capture, what appends or attends
// is refused, and what only reads the pool's metadata is not.
TEST("4-bit pools of 256-wide heads after a capture")
{
    two_rows t;
    t.pool.head_dim = 256;
    t.pool.fp4 = t.pool.captured = true;
    t.upload();
    ckv_pool* p = &t.pool;
    void *q = t.x, *o = t.x + 1, *k = t.x + 2, *v = t.x + 3, *a = t.x + 4, *b = t.x + 5;
    const ckv_rotation r = plain();
    const auto refused = [&](int status) {
        const bool told = t.ctx.last_error.find("nor after a call under one") != std::string::npos;
        t.ctx.last_error.clear();
        return status == CKV_E_INVALID_ARGUMENT && told;
    };
    CHECK(refused(ckv_append(p, 0, k, v, 2)));
    CHECK(refused(ckv_rope_append(p, 0, k, v, 1e4f, 0, 2)));
    CHECK(refused(ckv_rotate_append(p, 0, &r, q, o, 4, k, v, a, b, 2)));
    CHECK(refused(ckv_rotate_append(p, 0, nullptr, nullptr, nullptr, 0, k, v, nullptr, nullptr, 2)));
    CHECK(refused(ckv_prompt_attention(p, q, 0, k, v, 0, 4, 1.0f, nullptr, o, 2)));
    t.pool.shared_tile = true; // a chunk
    CHECK(refused(ckv_attention(p, 0, q, 4, 1.0f, o, 2)));
    CHECK(refused(ckv_attention_gated(p, 0, q, 4, 1.0f, a, o, 2)));
    CHECK(refused(ckv_prefill_attention(p, 0, q, 4, 1.0f, o, 2)));
    t.pool.shared_tile = false;
    CHECK(refused(ckv_attention(p, 0, q, 4, 1.0f, o, 2)));
    CHECK(refused(ckv_decode_attention(p, 0, q, 4, 1.0f, o, 2)));
    CHECK(refused(ckv_append_decode(p, 0, k, v, q, 4, 1.0f, o, 2)));
    CHECK(refused(ckv_rotate_append_decode(p, 0, nullptr, k, v, q, 4, 1.0f, nullptr, a, b, o, 2)));
}

// Layers that alternate between rotations find their tables; more than are kept are made anew,
// and every table is its own rotation's.
TEST("rotations kept by a pool")
{
    two_rows t;
    t.upload();
    t.pool.positions.clear(); // no rows: nothing is launched
    t.pool.slot_rows = 0;
    ckv_pool* p = &t.pool;
    std::vector<ckv_rotation> all(1, plain());
    const auto with = [&](auto change) {
        ckv_rotation r = plain();
        r.scaling = CKV_SCALING_YARN;
        r.factor = 4.0f;
        r.low = 1.0f;
        r.high = 32.0f;
        r.original = 4096;
        change(r);
        all.push_back(r);
    };
    with([](ckv_rotation&) {});
    with([](ckv_rotation& r) { r.theta = 5e5f; });
    with([](ckv_rotation& r) { r.layout = CKV_ROTARY_NEIGHBOURS; });
    with([](ckv_rotation& r) { r.rotary_dim = 64; });
    with([](ckv_rotation& r) { r.factor = 8.0f; });
    with([](ckv_rotation& r) { r.original = 8192; });
    with([](ckv_rotation& r) { r.magnitude = 2.0f; });
    with([](ckv_rotation& r) { r.low = 2.0f; });
    with([](ckv_rotation& r) { r.high = 40.0f; });
    with([](ckv_rotation& r) { r.scaling = CKV_SCALING_LINEAR; });
    const size_t most = sizeof(p->rotations) / sizeof(p->rotations[0]);
    REQUIRE(all.size() > most);
    const auto call = [&](ckv_pool* pool, const ckv_rotation& r) { return ckv_rotate(pool, &r, t.x, t.x + 1, 2, 0); };
    for (int round = 0; round < 4; ++round)
        for (size_t i = 0; i < most; ++i)
            CHECK(call(p, all[i]) == CKV_OK);
    CHECK(p->n_rotations == most && p->next_rotation == 0); // each made once
    for (int round = 0; round < 3; ++round)
        for (const ckv_rotation& r : all) {
            CHECK(call(p, r) == CKV_OK);
            two_rows fresh; // a pool that has met no other
            fresh.upload();
            fresh.pool.positions.clear();
            CHECK(call(&fresh.pool, r) == CKV_OK);
            REQUIRE(fresh.pool.n_rotations == 1);
            const auto& want = fresh.pool.rotations[0];
            size_t found = 0;
            for (uint32_t i = 0; i < p->n_rotations; ++i) {
                const auto& kept = p->rotations[i];
                if (std::memcmp(&kept.of, &want.of, sizeof(ckv_rotation)))
                    continue;
                ++found;
                const rotation_table &a = kept.table, &b = want.table;
                CHECK(std::equal(a.turns.step, a.turns.step + b.rotary / 2, b.turns.step));
                CHECK(a.magnitude == b.magnitude && a.magnitude64 == b.magnitude64 && a.rotary == b.rotary
                      && a.neighbours == b.neighbours);
            }
            CHECK(found == 1);
        }
    // one that is refused leaves them as they are
    const uint32_t next = p->next_rotation;
    ckv_rotation bad = plain();
    bad.theta = 0.0f;
    CHECK(call(p, bad) == CKV_E_INVALID_ROPE_THETA);
    CHECK(p->next_rotation == next);
}
