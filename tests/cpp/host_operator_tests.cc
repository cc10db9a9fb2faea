// GPU tests of the host layer's windowed attention, rotation on several axes and
// compaction: known answers through device tensors, the checks of their shapes, and a
// sequence whose prefix a checkpoint shares, compacted without disturbing it.
#include <array>
#include <cmath>
#include <numeric>
#include <stdexcept>

#include "check.h"
#include "hip_model_state.h"
#include "tensor_ops.h"

using namespace chibillm;

namespace {

hip_context&
gpu()
{
    static hip_context ctx = [] {
        auto c = hip_context::make(0);
        if (!c)
            throw std::runtime_error("no GPU context: " + describe_error(c.error()));
        return std::move(*c);
    }();
    return ctx;
}

device_buffer
upload(const std::vector<float>& host)
{
    auto b = device_buffer::make(gpu(), host.size() * sizeof(float));
    REQUIRE(b);
    REQUIRE(b->upload(host.data(), host.size() * sizeof(float)));
    return std::move(*b);
}

std::vector<float>
download(const void* ptr, std::size_t count)
{
    std::vector<float> out(count);
    REQUIRE(ckv_copy_to_host(gpu().get(), out.data(), ptr, count * sizeof(float)) == 0);
    return out;
}

device_tensor
view(const device_buffer& b, std::vector<std::size_t> dims)
{
    return device_tensor { b.data(), dtype::f32, std::move(dims) };
}

template <typename R, typename C>
bool
error_is(const R& r, C code)
{
    return !r.has_value() && r.error() == code;
}

} // namespace

TEST("window: a row sees its last tokens and the sinks")
{
    auto c = hip_kv_cache::make(gpu(), { 1, 2, 4, 1, 2 }, kv_dtype::f32);
    REQUIRE(c);
    // equal keys: the output is the mean of the values a row attends
    const std::vector<float> keys(16, 1.0f);
    std::vector<float> values(16);
    for (int t = 0; t < 8; ++t)
        values[2 * t] = values[2 * t + 1] = static_cast<float>(1 << t);
    REQUIRE(ckv_copy_to_device(gpu().get(), c->keys(), keys.data(), 64) == 0);
    REQUIRE(ckv_copy_to_device(gpu().get(), c->values(), values.data(), 64) == 0);
    const std::vector<std::uint32_t> pos { 7 }, table { 0, 1 }, off { 0 }, len { 2 };
    REQUIRE(upload_attention_metadata(*c, { pos, {}, table, off, len }));
    auto q = upload({ 1, 0 }), o = upload({ 0, 0 });
    auto out = view(o, { 1, 2 });
    auto mean = [&](std::size_t window, std::size_t sinks) {
        REQUIRE(paged_attention_window(*c, view(q, { 1, 2 }), 0, 1, window, sinks, out));
        return download(o.data(), 2)[0];
    };
    auto near = [](float a, float b) { return std::fabs(a - b) <= 1e-5f * b; };
    CHECK(near(mean(1, 0), 128));
    CHECK(near(mean(3, 0), (32 + 64 + 128) / 3.0f));
    CHECK(near(mean(2, 2), (1 + 2 + 64 + 128) / 4.0f));
    CHECK(near(mean(100, 0), 255 / 8.0f));
    CHECK(error_is(paged_attention_window(*c, view(q, { 1, 2 }), 0, 1, 0, 0, out),
                   tensor_op_errc::backend_failure));
    auto narrow = view(q, { 1, 1 });
    CHECK(error_is(paged_attention_window(*c, view(q, { 1, 2 }), 0, 1, 1, 0, out, &narrow),
                   tensor_op_errc::input_shape_mismatch));
    auto gate = upload({ 0, 1000 });
    auto gv = view(gate, { 1, 2 });
    REQUIRE(paged_attention_window(*c, view(q, { 1, 2 }), 0, 1, 1, 0, out, &gv));
    const auto gated = download(o.data(), 2);
    CHECK(near(gated[0], 64) && near(gated[1], 128));

    // a decode row stored first
    const std::vector<std::uint32_t> slots { 7 };
    REQUIRE(upload_attention_metadata(*c, { pos, slots, table, off, len }));
    auto k = upload({ 1, 1 }), v = upload({ 6, 6 });
    REQUIRE(store_kv_and_attend_window(*c, view(k, { 1, 2 }), view(v, { 1, 2 }), view(q, { 1, 2 }), 0, 1,
                                       2, 1, out));
    CHECK(near(download(o.data(), 2)[1], (1 + 64 + 6) / 3.0f));
    CHECK(error_is(store_kv_and_attend_window(*c, view(k, { 1, 2 }), view(v, { 2, 1 }), view(q, { 1, 2 }),
                                              0, 1, 2, 1, out),
                   tensor_op_errc::input_shape_mismatch));
}

TEST("rope axes: each pair turns by its own axis")
{
    auto c = hip_kv_cache::make(gpu(), { 1, 1, 4, 1, 4 }, kv_dtype::f32);
    REQUIRE(c);
    const std::vector<std::uint32_t> pos { 0, 1 }, slots { 0, 1 }, table { 0 }, off { 0, 0 }, len { 1, 1 };
    REQUIRE(upload_attention_metadata(*c, { pos, slots, table, off, len }));
    const std::vector<std::uint32_t> axes { 3, 5, 70, 90 }; // two rows on two axes
    const std::array<std::uint8_t, 2> pair_axis { 1, 0 };
    auto x = upload({ 1, 2, 3, 4, 5, 6, 7, 8 }), y = upload(std::vector<float>(8, 0.0f));
    auto in = view(x, { 2, 4 }), out = view(y, { 2, 4 });
    CHECK(error_is(rope_axes(*c, in, 1, 100.0f, pair_axis, out), tensor_op_errc::backend_failure));
    CHECK(error_is(upload_rope_axes(*c, std::span(axes).first(3), 2), tensor_op_errc::position_count_mismatch));
    CHECK(error_is(upload_rope_axes(*c, std::span(axes).first(2), 2), tensor_op_errc::position_count_mismatch));
    REQUIRE(upload_rope_axes(*c, axes, 2));
    CHECK(error_is(rope_axes(*c, in, 1, 100.0f, std::span(pair_axis).first(1), out),
                   tensor_op_errc::invalid_head_dimension));
    CHECK(error_is(rope_axes(*c, in, 2, 100.0f, pair_axis, out), tensor_op_errc::invalid_head_dimension));
    REQUIRE(rope_axes(*c, in, 1, 100.0f, pair_axis, out));
    auto want = [&](int row, int e) { // theta 100, rotary 4: 1 and 1/10 radian a position
        const double a = row ? (e % 2 ? 5 * 0.1 : 90.0) : (e % 2 ? 3 * 0.1 : 70.0);
        const double lo = 4 * row + 1 + e % 2, hi = lo + 2;
        return e < 2 ? lo * std::cos(a) - hi * std::sin(a) : hi * std::cos(a) + lo * std::sin(a);
    };
    const auto got = download(y.data(), 8);
    for (int i = 0; i < 8; ++i)
        CHECK(std::fabs(got[i] - want(i / 4, i % 4)) < 1e-5);
    auto values = upload({ 9, 9, 9, 9, 8, 8, 8, 8 });
    REQUIRE(store_kv_rotated_axes(*c, in, out, 1, in, view(values, { 2, 4 }), 0, 100.0f, pair_axis));
    CHECK(download(y.data(), 8) == got);
    CHECK(download(c->keys(), 8) == got);
    CHECK(download(c->values(), 8)[5] == 8.0f);
    CHECK(error_is(store_kv_rotated_axes(*c, in, out, 2, in, view(values, { 2, 4 }), 0, 100.0f, pair_axis),
                   tensor_op_errc::invalid_head_dimension));
}

TEST("compaction: a sequence drops its middle beside a checkpoint that shares its pages")
{
    const std::size_t bs = 4, layers = 2, width = 2;
    auto made = hip_model_state::make(gpu(), { layers, 12, bs, 1, width }, kv_dtype::f32);
    REQUIRE(made);
    hip_model_state& state = **made;
    hip_kv_cache& c = state.cache();
    std::vector<float> keys(c.element_count()), values(c.element_count());
    std::iota(keys.begin(), keys.end(), 1.0f);
    std::iota(values.begin(), values.end(), 5001.0f);
    REQUIRE(ckv_copy_to_device(gpu().get(), c.keys(), keys.data(), keys.size() * 4) == 0);
    REQUIRE(ckv_copy_to_device(gpu().get(), c.values(), values.data(), values.size() * 4) == 0);
    const seq_id id { 1 };
    REQUIRE(state.reserve(id, 18)); // 5 pages
    const std::vector<block_id> before(state.resources(id).blocks.begin(), state.resources(id).blocks.end());
    auto saved = state.checkpoint(id, 10); // shares the first 3
    REQUIRE(saved);
    const std::size_t free_before = state.pages().free_block_count();

    const std::vector<std::uint32_t> unordered { 0, 3, 2 }, past { 0, 20 };
    CHECK(error_is(state.compact(id, unordered), state_errc::invalid_reservation));
    CHECK(error_is(state.compact(id, past), state_errc::invalid_reservation));
    CHECK(error_is(state.compact(id, {}), state_errc::invalid_reservation));
    CHECK(error_is(state.compact(seq_id { 9 }, std::vector<std::uint32_t> { 0 }), state_errc::invalid_reservation));
    CHECK(error_is(state.compact(id, std::vector<std::uint32_t> { 0 }, -1.0f), state_errc::invalid_reservation));
    CHECK(error_is(state.compact(id, std::vector<std::uint32_t> { 0 }, 10.0f, 3), state_errc::invalid_reservation));

    // the first page stays as it is and shared; the second and third change: own pages
    std::vector<std::uint32_t> kept { 0, 1, 2, 3, 5, 9, 12, 13, 16, 17 };
    REQUIRE(state.compact(id, kept, 10.0f));
    const std::vector<block_id> after(state.resources(id).blocks.begin(), state.resources(id).blocks.end());
    REQUIRE(after.size() == 3);
    CHECK(after[0] == before[0] && after[1] != before[1] && after[2] != before[2]);
    CHECK(state.pages().refcount(before[0]) == 2 && state.pages().refcount(before[1]) == 1);
    CHECK(state.pages().free_block_count() == free_before - 2 + 2); // two taken, two given back
    auto got_k = download(c.keys(), keys.size()), got_v = download(c.values(), values.size());
    auto at = [&](std::size_t layer, const std::vector<block_id>& table, std::size_t t) {
        return (layer * 12 * bs + table[t / bs] * bs + t % bs) * width;
    };
    for (std::size_t layer = 0; layer < layers; ++layer)
        for (std::size_t i = 0; i < kept.size(); ++i) {
            const std::size_t s = at(layer, before, kept[i]), d = at(layer, after, i);
            const double a = static_cast<double>(i) - kept[i]; // rotary 2: a radian a position
            const double k0 = keys[s] * std::cos(a) - keys[s + 1] * std::sin(a);
            const double k1 = keys[s + 1] * std::cos(a) + keys[s] * std::sin(a);
            CHECK(std::fabs(got_k[d] - k0) <= 1e-6 * 2 * keys[s + 1]);
            CHECK(std::fabs(got_k[d + 1] - k1) <= 1e-6 * 2 * keys[s + 1]);
            CHECK(got_v[d] == values[s] && got_v[d + 1] == values[s + 1]);
        }
    // the checkpoint's pages hold what they held: a sequence restored from it has them
    const seq_id other { 2 };
    REQUIRE(state.reserve(other, 1));
    REQUIRE(state.restore(other, **saved));
    const std::vector<block_id> restored(state.resources(other).blocks.begin(), state.resources(other).blocks.end());
    got_k = download(c.keys(), keys.size());
    for (std::size_t layer = 0; layer < layers; ++layer)
        for (std::size_t t = 0; t < 10; ++t)
            CHECK(got_k[at(layer, restored, t)] == keys[at(layer, before, t)]);
    // in place now: nothing is shared past the first page
    kept = { 0, 1, 2, 3, 7, 8, 9 };
    const auto held = download(c.values(), values.size());
    REQUIRE(state.compact(id, kept));
    CHECK(state.resources(id).blocks.size() == 2 && state.resources(id).blocks[1] == after[1]);
    got_v = download(c.values(), values.size());
    for (std::size_t i = 0; i < kept.size(); ++i)
        CHECK(got_v[at(1, after, i)] == held[at(1, after, kept[i])]);
    // a shared last page that is not full becomes the sequence's own though nothing moves
    saved->reset();
    auto tail = state.checkpoint(id, 7);
    REQUIRE(tail);
    const block_id shared = state.resources(id).blocks[1];
    REQUIRE(state.compact(id, std::vector<std::uint32_t> { 0, 1, 2, 3, 4, 5 }));
    CHECK(state.resources(id).blocks[1] != shared && state.pages().refcount(shared) == 1);
    got_v = download(c.values(), values.size());
    const std::vector<block_id> last(state.resources(id).blocks.begin(), state.resources(id).blocks.end());
    for (std::size_t i = 4; i < 6; ++i)
        CHECK(got_v[at(0, last, i)] == got_v[at(0, after, i)]);
}

TEST("compaction: a pool without a free page for a shared one is refused unchanged")
{
    auto made = hip_model_state::make(gpu(), { 1, 3, 4, 1, 2 }, kv_dtype::f32);
    REQUIRE(made);
    hip_model_state& state = **made;
    state.set_spill(false);
    REQUIRE(state.reserve(seq_id { 1 }, 12));
    auto saved = state.checkpoint(seq_id { 1 }, 12);
    REQUIRE(saved);
    const block_id first = state.resources(seq_id { 1 }).blocks[0];
    CHECK(error_is(state.compact(seq_id { 1 }, std::vector<std::uint32_t> { 1, 5 }), state_errc::capacity_exhausted));
    CHECK(state.resources(seq_id { 1 }).blocks.size() == 3 && state.resources(seq_id { 1 }).blocks[0] == first);
}

TEST("compaction: a spill for a full pool leaves the pages to the sequence")
{
    auto made = hip_model_state::make(gpu(), { 1, 3, 4, 1, 2 }, kv_dtype::f32);
    REQUIRE(made);
    hip_model_state& state = **made;
    hip_kv_cache& c = state.cache();
    std::vector<float> values(c.element_count());
    std::iota(values.begin(), values.end(), 1.0f);
    REQUIRE(ckv_copy_to_device(gpu().get(), c.values(), values.data(), values.size() * 4) == 0);
    const seq_id gone { 1 }, id { 2 };
    REQUIRE(state.reserve(gone, 4));
    auto lone = state.checkpoint(gone, 4);
    REQUIRE(lone);
    state.release(gone); // a page that the checkpoint alone holds
    REQUIRE(state.reserve(id, 8));
    auto saved = state.checkpoint(id, 8);
    REQUIRE(saved);
    const std::vector<block_id> before(state.resources(id).blocks.begin(), state.resources(id).blocks.end());
    const std::vector<std::uint32_t> kept { 0, 2, 3, 6, 7 }; // both pages change
    auto done = state.compact(id, kept);
    // one page can be had: not enough for both, and nothing changed
    CHECK(error_is(done, state_errc::capacity_exhausted));
    CHECK(state.resources(id).blocks[0] == before[0] && state.resources(id).blocks.size() == 2);
    CHECK(state.pages().free_block_count() == 1 && state.spills() == 1);
    const std::vector<std::uint32_t> one { 0, 1, 2, 3, 6, 7 }; // the second alone
    REQUIRE(state.compact(id, one));
    const std::vector<block_id> after(state.resources(id).blocks.begin(), state.resources(id).blocks.end());
    CHECK(after[0] == before[0] && after[1] != before[1]);
    const auto got = download(c.values(), values.size());
    CHECK(got[after[1] * 8] == values[before[1] * 8 + 4] && got[after[1] * 8 + 2] == values[before[1] * 8 + 6]);
    CHECK(got[before[1] * 8] == values[before[1] * 8]); // the checkpoint's
}

TEST("block_manager: truncate gives the last pages back in order")
{
    auto pages = block_manager::make(5, 2);
    REQUIRE(pages);
    REQUIRE(pages->reserve(seq_id { 7 }, 10));
    CHECK(error_is(pages->truncate(seq_id { 8 }, 2), state_errc::invalid_reservation));
    CHECK(error_is(pages->truncate(seq_id { 7 }, 0), state_errc::invalid_reservation));
    CHECK(error_is(pages->truncate(seq_id { 7 }, 11), state_errc::invalid_reservation));
    REQUIRE(pages->truncate(seq_id { 7 }, 5));
    CHECK(pages->resources(seq_id { 7 }).blocks.size() == 3 && pages->free_block_count() == 2);
    REQUIRE(pages->reserve(seq_id { 8 }, 4));
    CHECK(pages->resources(seq_id { 8 }).blocks[0] == 3 && pages->resources(seq_id { 8 }).blocks[1] == 4);
}
