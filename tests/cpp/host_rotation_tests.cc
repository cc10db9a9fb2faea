// GPU tests of the host layer's caches held in 4 bits, rotations in their forms and prompt
// attention: known answers through device tensors and the checks of their shapes.
#include <array>
#include <cmath>
#include <stdexcept>

#include "check.h"
#include "hip_kv_cache.h"
#include "tensor_ops.h"

using namespace chibillm;

namespace {

constexpr std::size_t dim = 64;

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

struct rows_of {
    device_buffer buffer;
    device_tensor tensor;
};

// Rows of `dim` floats, row r all of fill(r).
template <class F>
rows_of
rows(std::size_t n, F fill)
{
    std::vector<float> host(n * dim);
    for (std::size_t r = 0; r < n; ++r)
        for (std::size_t f = 0; f < dim; ++f)
            host[r * dim + f] = fill(r);
    auto b = device_buffer::make(gpu(), host.size() * sizeof(float));
    REQUIRE(b);
    REQUIRE(b->upload(host.data(), host.size() * sizeof(float)));
    rows_of x { std::move(*b), {} };
    x.tensor = device_tensor { x.buffer.data(), dtype::f32, { n, dim } };
    return x;
}

std::vector<float>
download(const rows_of& x)
{
    std::vector<float> out(x.tensor.dims[0] * dim);
    REQUIRE(x.buffer.download(out.data(), out.size() * sizeof(float)));
    return out;
}

template <typename R, typename C>
bool
error_is(const R& r, C code)
{
    return !r.has_value() && r.error() == code;
}

ckv_rotation
turn(float theta)
{
    ckv_rotation r {};
    r.theta = theta;
    r.layout = CKV_ROTARY_NEIGHBOURS;
    return r;
}

} // namespace

TEST("caches in 4 bits: geometry, bytes and what they refuse")
{
    CHECK(error_is(hip_kv_cache::make(gpu(), { 1, 2, 8, 1, dim }, kv_dtype::f32, kv_storage::fp4),
                   kv_cache_errc::invalid_block_size));
    CHECK(error_is(hip_kv_cache::make(gpu(), { 1, 2, 16, 1, 96 }, kv_dtype::f32, kv_storage::fp4),
                   kv_cache_errc::invalid_head_dimension));
    auto made = hip_kv_cache::make(gpu(), { 2, 3, 16, 1, dim }, kv_dtype::f32, kv_storage::fp4);
    REQUIRE(made);
    hip_kv_cache c = std::move(*made);
    CHECK(c.storage() == kv_storage::fp4);
    CHECK(c.page_bytes_all_layers() == 2 * 2 * 16 * dim / 32 * 17);
    CHECK(error_is(c.element_offset(0, 0, 0, 0, 0), kv_cache_errc::head_feature_out_of_range));
    const std::array<block_id, 1> blocks { 0 };
    CHECK(error_is(c.checkpoint(blocks, 16), state_errc::backend_failure));
    CHECK(error_is(c.export_prefix(blocks, 16), state_errc::backend_failure));
    const std::array<std::uint32_t, 1> from { 1 }, to { 0 }, counts { 1 };
    CHECK(error_is(c.compact(from, to, {}, counts, 0.0f), state_errc::invalid_reservation));
    const std::array<block_id, 1> target { 2 };
    CHECK(c.copy_pages(blocks, target));
}

TEST("a prompt and a step over a cache in 4 bits")
{
    auto c = hip_kv_cache::make(gpu(), { 1, 2, 16, 1, dim }, kv_dtype::f32, kv_storage::fp4);
    REQUIRE(c);
    const std::vector<std::uint32_t> table { 1, 0 }, pos { 0, 1, 2 }, slots { 16, 17, 18 }, off { 0, 0, 0 }, len { 2, 2, 2 };
    REQUIRE(upload_attention_metadata(*c, { pos, slots, table, off, len }));
    // queries of zeros weigh all keys alike: outputs are means of values that 4 bits hold exactly
    auto q = rows(3, [](std::size_t) { return 0.0f; });
    auto k = rows(3, [](std::size_t r) { return 1.0f + r; });
    auto v = rows(3, [](std::size_t r) { return static_cast<float>(1 << r); });
    auto turned = rows(3, [](std::size_t) { return 9.0f; }), out = rows(3, [](std::size_t) { return 9.0f; });
    auto hk = rows(3, [](std::size_t) { return 9.0f; }), hv = rows(3, [](std::size_t) { return 9.0f; });
    const ckv_rotation r = turn(1e4f);
    REQUIRE(store_kv_rotated_by(*c, &r, q.tensor, turned.tensor, 1, k.tensor, v.tensor, 0, &hk.tensor, &hv.tensor));
    const auto held = download(hv), rotated = download(hk);
    for (std::size_t i = 0; i < held.size(); ++i)
        CHECK(held[i] == static_cast<float>(1 << i / dim));
    for (std::size_t f = 0; f < dim; ++f) // position 0 turns nothing
        CHECK(rotated[f] == 1.0f);
    REQUIRE(prompt_attention(*c, turned.tensor, hk.tensor, hv.tensor, 1, out.tensor));
    const auto first = download(out);
    const float means[3] = { 1.0f, 1.5f, 7.0f / 3 };
    for (std::size_t i = 0; i < first.size(); ++i)
        CHECK(std::fabs(first[i] - means[i / dim]) <= 1e-6f * means[i / dim]);
    REQUIRE(paged_attention(*c, turned.tensor, 0, 1, out.tensor));
    const auto again = download(out);
    for (std::size_t i = 0; i < again.size(); ++i)
        CHECK(std::fabs(again[i] - means[i / dim]) <= 1e-6f * means[i / dim]);
    // one more token
    const std::vector<std::uint32_t> p1 { 3 }, s1 { 19 }, o1 { 0 }, l1 { 2 };
    REQUIRE(upload_attention_metadata(*c, { p1, s1, table, o1, l1 }));
    auto q1 = rows(1, [](std::size_t) { return 0.0f; }), v1 = rows(1, [](std::size_t) { return -3.0f; });
    auto k1 = rows(1, [](std::size_t) { return 0.5f; }), out1 = rows(1, [](std::size_t) { return 9.0f; });
    auto gate = rows(1, [](std::size_t) { return 1000.0f; });
    REQUIRE(store_kv_rotated_by_and_attend(*c, &r, k1.tensor, v1.tensor, q1.tensor, 0, 1, out1.tensor, &gate.tensor));
    for (const float x : download(out1))
        CHECK(std::fabs(x - 1.0f) <= 1e-6f);
    auto turned1 = rows(1, [](std::size_t) { return 9.0f; });
    REQUIRE(rotate(*c, r, k1.tensor, 1, turned1.tensor));
    const float s = std::sin(3.0f), co = std::cos(3.0f);
    const auto t = download(turned1);
    CHECK(std::fabs(t[0] - 0.5f * (co - s)) <= 1e-6f);
    CHECK(std::fabs(t[1] - 0.5f * (co + s)) <= 1e-6f);
}

TEST("rotations and prompts: shapes that are refused")
{
    auto c = hip_kv_cache::make(gpu(), { 1, 2, 16, 1, dim }, kv_dtype::f32, kv_storage::fp4);
    REQUIRE(c);
    const std::vector<std::uint32_t> table { 1, 0 }, pos { 0, 1 }, slots { 16, 17 }, off { 0, 0 }, len { 2, 2 };
    REQUIRE(upload_attention_metadata(*c, { pos, slots, table, off, len }));
    auto zero = [](std::size_t) { return 0.0f; };
    auto q = rows(2, zero), o = rows(2, zero), k = rows(2, zero), v = rows(2, zero), one = rows(1, zero);
    device_tensor half = q.tensor, flat = q.tensor;
    half.type = dtype::bf16;
    flat.dims = { 2 * dim };
    const ckv_rotation r = turn(1e4f), none = turn(0.0f);
    CHECK(error_is(rotate(*c, r, flat, 1, o.tensor), tensor_op_errc::invalid_rank));
    CHECK(error_is(rotate(*c, r, half, 1, o.tensor), tensor_op_errc::unsupported_dtype));
    CHECK(error_is(rotate(*c, r, q.tensor, 1, one.tensor), tensor_op_errc::output_shape_mismatch));
    CHECK(error_is(rotate(*c, r, q.tensor, 2, o.tensor), tensor_op_errc::invalid_head_dimension));
    CHECK(error_is(rotate(*c, none, q.tensor, 1, o.tensor), tensor_op_errc::invalid_rope_theta));
    CHECK(error_is(store_kv_rotated_by(*c, &r, one.tensor, one.tensor, 1, k.tensor, v.tensor, 0),
                   tensor_op_errc::position_count_mismatch));
    CHECK(error_is(store_kv_rotated_by(*c, &r, q.tensor, o.tensor, 1, k.tensor, v.tensor, 1),
                   tensor_op_errc::cache_layer_out_of_range));
    CHECK(error_is(store_kv_rotated_by(*c, &r, q.tensor, o.tensor, 1, k.tensor, v.tensor, 0, &one.tensor),
                   tensor_op_errc::output_shape_mismatch));
    CHECK(error_is(store_kv_rotated_by(*c, &r, q.tensor, o.tensor, 1, k.tensor, v.tensor, 0, &k.tensor),
                   tensor_op_errc::unsupported_aliasing));
    CHECK(error_is(store_kv_rotated_by_and_attend(*c, &r, k.tensor, v.tensor, q.tensor, 0, 2, o.tensor),
                   tensor_op_errc::cache_head_dimension_mismatch));
    CHECK(error_is(prompt_attention(*c, q.tensor, k.tensor, one.tensor, 1, o.tensor),
                   tensor_op_errc::input_shape_mismatch));
    CHECK(error_is(prompt_attention(*c, one.tensor, k.tensor, v.tensor, 1, one.tensor),
                   tensor_op_errc::position_count_mismatch));
    CHECK(error_is(prompt_attention(*c, q.tensor, k.tensor, v.tensor, 1, q.tensor),
                   tensor_op_errc::unsupported_aliasing));
}

TEST("element offsets: a cache in 4 bits says why it has none")
{
    auto c = hip_kv_cache::make(gpu(), { 1, 2, 16, 1, dim }, kv_dtype::f32, kv_storage::fp4);
    auto floats = hip_kv_cache::make(gpu(), { 1, 2, 16, 1, dim }, kv_dtype::f32);
    REQUIRE(c && floats);
    const auto none = c->element_offset(0, 0, 0, 0, 0), outside = floats->element_offset(0, 0, 0, 0, dim);
    REQUIRE(!none && !outside);
    CHECK(none.error().detail == "held in 4 bits");
    CHECK(outside.error() == kv_cache_errc::head_feature_out_of_range && outside.error().detail.empty());
}
