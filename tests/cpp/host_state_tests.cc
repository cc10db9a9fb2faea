// CPU tests of hip_model_state's compaction: what a refusal leaves behind. libckv's entry points
// that it calls are replaced here (a program's own definitions come before a library's), so that a
// compaction can be made to fail and its moves can be carried out on host arrays.
#include <algorithm>
#include <cstdlib>
#include <numeric>

#include "check.h"
#include "hip_model_state.h"

using namespace chibillm;

namespace {

// One value per slot stands for a token's rows of every layer.
struct fake_device {
    std::vector<float> rows;
    int compact_status = 0; // what the next compactions answer
    std::size_t compactions = 0;
} device;

} // namespace

struct ckv_context {};
struct ckv_pool {};

extern "C" {
int ckv_context_create(int, ckv_context** out)
{
    *out = new ckv_context;
    return 0;
}
int ckv_context_destroy(ckv_context* ctx)
{
    delete ctx;
    return 0;
}
const char* ckv_last_error(const ckv_context*) { return "fake"; }
int ckv_pool_create(ckv_context*, size_t, size_t blocks, size_t block_size, size_t, size_t, int,
                    ckv_pool** out)
{
    device = {};
    device.rows.resize(blocks * block_size);
    std::iota(device.rows.begin(), device.rows.end(), 1.0f);
    *out = new ckv_pool;
    return 0;
}
int ckv_pool_destroy(ckv_pool* pool)
{
    delete pool;
    return 0;
}
int ckv_host_alloc(ckv_context*, size_t bytes, void** out)
{
    *out = std::malloc(bytes ? bytes : 1);
    return 0;
}
int ckv_host_free(ckv_context*, void* ptr)
{
    std::free(ptr);
    return 0;
}
int ckv_checkpoint_export(ckv_pool*, const uint32_t*, size_t, size_t, void*, void*) { return 0; }
int ckv_copy_blocks(ckv_pool*, const uint32_t*, const uint32_t*, size_t) { return 0; }
int ckv_compact(ckv_pool*, const uint32_t* from, const uint32_t* to, const int32_t*,
                const uint32_t* counts, size_t n_sequences, float, size_t)
{
    ++device.compactions;
    if (device.compact_status)
        return device.compact_status;
    const std::vector<float> before = device.rows;
    for (uint32_t i = 0, n = std::accumulate(counts, counts + n_sequences, 0u); i < n; ++i)
        device.rows.at(to[i]) = before.at(from[i]);
    return 0;
}
}

namespace {

hip_context&
context()
{
    static hip_context ctx = std::move(*hip_context::make(0));
    return ctx;
}

std::unique_ptr<hip_model_state>
make_state(std::size_t pages, std::size_t page)
{
    auto made = hip_model_state::make(context(), { 1, pages, page, 1, 2 }, kv_dtype::f32);
    REQUIRE(made);
    return std::move(*made);
}

std::vector<block_id>
table_of(const hip_model_state& state, seq_id id)
{
    const auto held = state.resources(id).blocks;
    return { held.begin(), held.end() };
}

} // namespace

TEST("compaction: one that the library refuses leaves tables, references and free pages as they were")
{
    const seq_id id { 1 }, next { 2 };
    const std::vector<std::uint32_t> kept { 0, 1, 2, 3, 5, 9, 12 }; // changes the second page of two
    for (const auto& [status, code] : { std::pair { CKV_E_TENSOR_ALLOCATION_FAILED, state_errc::allocation_failed },
                                        std::pair { CKV_E_INVALID_ARGUMENT, state_errc::invalid_reservation },
                                        std::pair { CKV_E_HIP_FAILURE, state_errc::backend_failure } }) {
        auto state = make_state(8, 4);
        REQUIRE(state->reserve(id, 14));
        auto saved = state->checkpoint(id, 8); // shares the first two pages
        REQUIRE(saved);
        const auto before = table_of(*state, id);
        const std::size_t free_before = state->pages().free_block_count();
        device.compact_status = status;
        const auto refused = state->compact(id, kept);
        CHECK(!refused && refused.error() == code);
        CHECK(device.compactions == 1);
        CHECK(table_of(*state, id) == before);
        CHECK(state->pages().refcount(before[1]) == 2);
        CHECK(state->pages().free_block_count() == free_before);
        // the free pages in their order too
        REQUIRE(state->reserve(next, 4));
        CHECK(table_of(*state, next) == std::vector<block_id> { 4 });
        // and the sequence can be compacted once there is nothing in the way
        device.compact_status = 0;
        REQUIRE(state->compact(id, kept));
        const auto after = table_of(*state, id);
        REQUIRE(after.size() == 2);
        CHECK(after[0] == before[0] && after[1] == 5 && state->pages().refcount(before[1]) == 1);
        for (std::size_t i = 0; i < kept.size(); ++i)
            CHECK(device.rows[after[i / 4] * 4 + i % 4] == 1.0f + before[kept[i] / 4] * 4 + kept[i] % 4);
    }
}

TEST("block_manager: borrowed pages are placed or go back as if never taken")
{
    auto pages = block_manager::make(4, 2);
    REQUIRE(pages);
    REQUIRE(pages->reserve(seq_id { 1 }, 4));
    CHECK(!pages->borrow(3));
    auto some = pages->borrow(2);
    REQUIRE(some);
    CHECK(*some == std::vector<block_id>({ 2, 3 }) && pages->free_block_count() == 0);
    pages->give_back(*some);
    CHECK(pages->free_block_count() == 2 && pages->refcount(2) == 0);
    some = pages->borrow(1);
    REQUIRE(some && (*some)[0] == 2);
    pages->put(seq_id { 1 }, 1, 2);
    CHECK(pages->resources(seq_id { 1 }).blocks[1] == 2 && pages->refcount(1) == 0 && pages->refcount(2) == 1);
}
