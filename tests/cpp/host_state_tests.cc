// CPU tests of hip_model_state's compaction: what a refusal leaves behind, and the engine that goes
// on with a compacted sequence. libckv's entry points
// that it calls are replaced here (a program's own definitions come before a library's), so that a
// compaction can be made to fail and its moves can be carried out on host arrays.
#include <algorithm>
#include <cstdlib>
#include <numeric>

#include "check.h"
#include "hip_model_state.h"
#include "inference_engine.h"

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
        // and the sequence can be compacted once there is nothing in the way, but for the device's
        device.compact_status = 0;
        if (status == CKV_E_HIP_FAILURE) {
            CHECK(!state->compact(id, kept));
            continue;
        }
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

// ---- the engine over a compacted sequence ---------------------------------------------------

namespace {

// Writes every row's token into its slot and samples from what a row attends: the tokens at the
// positions before it, which have to be the ones the test expects (history).
struct slot_runner final : model_runner {
    std::size_t pages = 16, page = 4;
    mutable hip_model_state* state = nullptr;
    std::unordered_map<seq_id, std::vector<token_id>> history;
    std::vector<seq_id> batch_ids;
    const std::vector<std::uint32_t>* compact_inside = nullptr;

    const model_info& info() const noexcept override
    {
        static const model_info value { "slots", 256, -1 };
        return value;
    }
    result<std::unique_ptr<model_state>, model_runner_error> make_state(scheduler_config) const override
    {
        auto made = ::make_state(pages, page);
        state = made.get();
        return std::unique_ptr<model_state>(std::move(made));
    }
    result<std::vector<token_id>, model_runner_error> execute(const model_batch& batch, model_state&) override
    {
        batch_ids.clear();
        const auto md = prepare_paged_batch(batch, 256, pages, page);
        if (!md)
            return fail(model_runner_errc::inconsistent_batch);
        std::vector<token_id> samples;
        for (const auto& item : batch.items) {
            batch_ids.push_back(item.id);
            auto& seen = history[item.id];
            for (std::size_t r = item.token_offset; r < item.token_offset + item.token_count; ++r) {
                CHECK(batch.positions[r] == seen.size());
                seen.push_back(batch.tokens[r]);
                device.rows.at(md->slots[r]) = static_cast<float>(batch.tokens[r]);
            }
            for (std::size_t p = 0; p < seen.size(); ++p)
                CHECK(device.rows.at(item.block_table.at(p / page) * page + p % page) == static_cast<float>(seen[p]));
            if (compact_inside)
                CHECK(!state->compact(item.id, *compact_inside));
            if (item.logits_index)
                samples.push_back(100 + static_cast<token_id>(seen.size()) % 50);
        }
        return samples;
    }
    void keep(seq_id id, const std::vector<std::uint32_t>& kept)
    {
        std::vector<token_id> left;
        for (const std::uint32_t p : kept)
            left.push_back(history[id].at(p));
        history[id] = left;
    }
};

scheduler_config
slot_config()
{
    scheduler_config c;
    c.max_sequences = 2;
    c.max_batch_tokens = 8;
    c.kv_block_count = 16;
    c.kv_block_size = 4;
    c.prefill_chunk_tokens = 8;
    c.prefix_cache_min_tokens = 4;
    return c;
}

seq
prompt_of(seq_id id, token_id first, std::size_t n, std::size_t max_new, std::vector<std::size_t> boundaries = {})
{
    std::vector<token_id> tokens(n);
    std::iota(tokens.begin(), tokens.end(), first);
    auto s = seq::make(id, std::move(tokens), generation_params { max_new, true }, std::move(boundaries));
    REQUIRE(s);
    return std::move(*s);
}

} // namespace

TEST("engine: a sequence compacted behind the scheduler's back is refused, not continued at its old positions")
{
    slot_runner runner;
    auto config = slot_config();
    config.prefix_cache_bytes = 0;
    auto engine = inference_engine::make(config, runner);
    REQUIRE(engine);
    REQUIRE(engine->add(prompt_of(1, 1, 6, 20)));
    for (int i = 0; i < 6; ++i)
        REQUIRE(engine->step());
    REQUIRE(engine->find_sequence(1)->processed_token_count() == 11);
    const std::vector<std::uint32_t> kept { 0, 1, 7, 8 };
    REQUIRE(runner.state->compact(1, kept));
    runner.batch_ids.clear();
    const auto stepped = engine->step(); // at position 11 of a cache that holds four tokens
    CHECK(!stepped && stepped.error() == inference_engine_errc::model_execution_failed);
    CHECK(runner.batch_ids.empty());
    REQUIRE(engine->cancel(1));
    CHECK(runner.state->pages().free_block_count() == 16);
}

TEST("engine: compacted sequences go on behind what they kept")
{
    slot_runner runner;
    auto engine = inference_engine::make(slot_config(), runner);
    REQUIRE(engine);
    REQUIRE(engine->add(prompt_of(1, 1, 10, 25, { 4 })));
    REQUIRE(engine->step()); // the prompt up to its boundary, whose prefix is published
    CHECK(engine->engine_scheduler().prefixes().entry_count() == 1);
    for (int i = 0; i < 9; ++i)
        REQUIRE(engine->step());
    const seq* s = engine->find_sequence(1);
    REQUIRE(s->processed_token_count() == 18 && s->next_position() == 18);
    // positions that hold nothing yet, none, out of order; other sequences
    const std::vector<std::uint32_t> past { 0, 18 }, unordered { 3, 2 }, one { 0 };
    CHECK(!engine->compact(1, past) && !engine->compact(1, {}) && !engine->compact(1, unordered));
    CHECK(!engine->compact(9, one));
    const std::vector<std::uint32_t> kept { 0, 1, 2, 3, 9, 14, 15, 16, 17 };
    runner.compact_inside = &one; // a batch is under way: refused, and the step goes on
    REQUIRE(engine->step());
    runner.compact_inside = nullptr;
    REQUIRE(s->next_position() == 19);
    REQUIRE(engine->compact(1, kept));
    runner.keep(1, kept);
    CHECK(s->next_position() == 9 && s->processed_token_count() == 19 && s->dropped_token_count() == 10);
    CHECK(runner.state->resources(1).blocks.size() == 3);
    // a second sequence from the prefix that the first published: its pages are as they were
    REQUIRE(engine->add(prompt_of(2, 1, 12, 4, { 8 })));
    CHECK(engine->find_sequence(2)->cached_token_count() == 4);
    runner.history[2] = { 1, 2, 3, 4 };
    REQUIRE(engine->step());
    // compacted while it waits for the rest of its prompt; no more of it is published
    REQUIRE(engine->step());
    const seq* other = engine->find_sequence(2);
    REQUIRE(other->status() == seq_status::waiting || other->status() == seq_status::running);
    const std::size_t entries = engine->engine_scheduler().prefixes().entry_count();
    const std::vector<std::uint32_t> ends { 0, static_cast<std::uint32_t>(other->next_position() - 1) };
    REQUIRE(engine->compact(2, ends));
    runner.keep(2, ends);
    for (int i = 0; i < 4; ++i)
        REQUIRE(engine->step());
    CHECK(engine->engine_scheduler().prefixes().entry_count() == entries);
    // once more, in place, then to the end
    const std::vector<std::uint32_t> again { 0, 3, 4, 8, static_cast<std::uint32_t>(s->next_position() - 1) };
    REQUIRE(engine->compact(1, again));
    runner.keep(1, again);
    while (!engine->is_finished())
        REQUIRE(engine->step());
    CHECK(s->completion_token_count() == 25 && engine->find_sequence(2)->completion_token_count() == 4);
    CHECK(!engine->compact(1, one)); // finished
    // the prefix cache alone holds pages now: the one page of the published prefix
    CHECK(runner.state->pages().free_block_count() == 16 - entries);
}

TEST("engine: a prefix is not published from a compacted cache")
{
    slot_runner runner;
    auto config = slot_config();
    config.prefill_chunk_tokens = 4;
    auto engine = inference_engine::make(config, runner);
    REQUIRE(engine);
    REQUIRE(engine->add(prompt_of(1, 1, 15, 3, { 12 })));
    REQUIRE(engine->add(prompt_of(2, 101, 15, 3, { 12 })));
    REQUIRE(engine->step()); // four tokens of each
    const std::vector<std::uint32_t> kept { 0, 3 };
    REQUIRE(engine->compact(1, kept));
    runner.keep(1, kept);
    while (!engine->is_finished())
        REQUIRE(engine->step());
    CHECK(engine->engine_scheduler().prefixes().entry_count() == 1); // the second's alone
    REQUIRE(engine->add(prompt_of(3, 1, 15, 1)));
    CHECK(engine->find_sequence(3)->cached_token_count() == 0);
}

TEST("engine: after a device's failure in a compaction the sequence can only be cancelled")
{
    slot_runner runner;
    auto config = slot_config();
    config.prefix_cache_bytes = 0;
    auto engine = inference_engine::make(config, runner);
    REQUIRE(engine);
    REQUIRE(engine->add(prompt_of(1, 1, 6, 20)));
    for (int i = 0; i < 3; ++i)
        REQUIRE(engine->step());
    const std::vector<std::uint32_t> kept { 0, 5 };
    device.compact_status = CKV_E_INVALID_ARGUMENT; // refused: nothing happened
    CHECK(!engine->compact(1, kept));
    REQUIRE(engine->step());
    device.compact_status = CKV_E_HIP_FAILURE;
    CHECK(!engine->compact(1, kept));
    device.compact_status = 0;
    CHECK(!engine->compact(1, kept) && !engine->step());
    REQUIRE(engine->cancel(1));
    CHECK(runner.state->pages().free_block_count() == 16);
    REQUIRE(engine->add(prompt_of(2, 1, 3, 2)));
    while (!engine->is_finished())
        REQUIRE(engine->step());
}

TEST("seq: positions kept by a compaction")
{
    auto s = seq::make(1, { 1, 2, 3, 4 }, generation_params { 5 });
    REQUIRE(s);
    CHECK(!s->keep_positions(1)); // nothing is cached yet
    REQUIRE(s->schedule_tokens(4));
    CHECK(!s->keep_positions(1));
    REQUIRE(s->commit_scheduled_tokens());
    CHECK(!s->keep_positions(0) && !s->keep_positions(5) && s->next_position() == 4);
    REQUIRE(s->keep_positions(2));
    CHECK(s->next_position() == 2 && s->dropped_token_count() == 2 && s->processed_token_count() == 4);
    REQUIRE(s->mark_running());
    REQUIRE(s->append_token(9));
    REQUIRE(s->schedule_tokens(1));
    REQUIRE(s->commit_scheduled_tokens());
    CHECK(s->next_position() == 3);
    REQUIRE(s->keep_positions(3));
    CHECK(s->next_position() == 3 && s->dropped_token_count() == 2);
    REQUIRE(s->finish(finish_reason::cancelled));
    CHECK(!s->keep_positions(1));
}
