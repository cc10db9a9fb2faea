// GPU test of the engine over a sequence that outgrows its cache: every layer call of a runner through
// the host layer (rotation, append, attention through a window with sinks), the sequence compacted
// between steps, and every output against the definition over what was kept, at its new positions.
#include <cmath>
#include <stdexcept>

#include "check.h"
#include "hip_model_state.h"
#include "inference_engine.h"
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

constexpr std::size_t width = 4, pages = 24, page = 4, window = 7, sinks = 2;
constexpr float theta = 100.0f; // pairs (0, 2) and (1, 3) turn by 1 and 0.1 radian a position

// What a token projects to, of part 0 (query), 1 (key) and 2 (value).
float
project(token_id token, int part, std::size_t feature)
{
    return static_cast<float>(std::sin(0.7 * token + 1.3 * part + 2.1 * static_cast<double>(feature)));
}

std::array<double, width>
rotated(token_id token, int part, double position)
{
    std::array<double, width> x;
    for (std::size_t j = 0; j < 2; ++j) {
        const double a = project(token, part, j), b = project(token, part, j + 2);
        const double angle = position * std::pow(static_cast<double>(theta), -0.5 * static_cast<double>(j));
        x[j] = a * std::cos(angle) - b * std::sin(angle);
        x[j + 2] = b * std::cos(angle) + a * std::sin(angle);
    }
    return x;
}

struct window_runner final : model_runner {
    mutable hip_model_state* state = nullptr;
    std::unordered_map<seq_id, std::vector<token_id>> history; // the tokens in the cache, in order
    std::size_t checked = 0;

    const model_info& info() const noexcept override
    {
        static const model_info value { "window", 512, -1 };
        return value;
    }
    result<std::unique_ptr<model_state>, model_runner_error> make_state(scheduler_config) const override
    {
        auto made = hip_model_state::make(gpu(), { 1, pages, page, 1, width }, kv_dtype::f32);
        REQUIRE(made);
        state = made->get();
        REQUIRE(state->enable_device_tables(4, pages));
        return std::unique_ptr<model_state>(std::move(*made));
    }
    result<std::vector<token_id>, model_runner_error> execute(const model_batch& batch, model_state&) override
    {
        hip_kv_cache& c = state->cache();
        const std::size_t rows = batch.tokens.size();
        REQUIRE(state->tables()->upload(batch, 512, true));
        std::vector<float> host(rows * width);
        std::array<device_buffer, 4> on_device;
        for (int part = 0; part < 4; ++part) {
            for (std::size_t i = 0; i < host.size(); ++i)
                host[i] = part < 3 ? project(batch.tokens[i / width], part, i % width) : 0.0f;
            auto b = device_buffer::make(gpu(), host.size() * 4);
            REQUIRE(b);
            REQUIRE(b->upload(host.data(), host.size() * 4));
            on_device[part] = std::move(*b);
        }
        auto view = [&](int part) {
            return device_tensor { on_device[part].data(), dtype::f32, { rows, width } };
        };
        auto q = view(0), out = view(3);
        REQUIRE(rope(c, q, 1, theta, q));
        REQUIRE(store_kv_rotated(c, view(1), view(2), 0, theta));
        REQUIRE(paged_attention_window(c, q, 0, 1, window, sinks, out));
        REQUIRE(on_device[3].download(host.data(), host.size() * 4));
        std::vector<token_id> samples;
        for (const auto& item : batch.items) {
            auto& seen = history[item.id];
            for (std::size_t r = item.token_offset; r < item.token_offset + item.token_count; ++r) {
                const std::size_t p = seen.size();
                CHECK(batch.positions[r] == p);
                seen.push_back(batch.tokens[r]);
                const auto query = rotated(batch.tokens[r], 0, static_cast<double>(p));
                double sum = 0.0, want[width] = {};
                for (std::size_t t = 0; t <= p; ++t) {
                    if (t + window <= p && t >= sinks)
                        continue;
                    const auto key = rotated(seen[t], 1, static_cast<double>(t));
                    double score = 0.0;
                    for (std::size_t f = 0; f < width; ++f)
                        score += query[f] * key[f] / 2.0; // 1 / sqrt(width)
                    const double weight = std::exp(score);
                    sum += weight;
                    for (std::size_t f = 0; f < width; ++f)
                        want[f] += weight * project(seen[t], 2, f);
                }
                // values of 1 at most; a key is rotated in 32 bits (an angle of up to 60 radians
                // is off by 60 steps of 2^-24) and turned once more: a score by under 1e-4
                for (std::size_t f = 0; f < width; ++f)
                    CHECK(std::fabs(host[r * width + f] - want[f] / sum) < 2e-4);
                ++checked;
            }
            if (item.logits_index)
                samples.push_back(10 + static_cast<token_id>(seen.size() % 40));
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

std::vector<std::uint32_t>
sinks_and_newest(std::size_t held, std::size_t newest)
{
    std::vector<std::uint32_t> kept;
    for (std::uint32_t p = 0; p < held; ++p)
        if (p < sinks || p + newest >= held)
            kept.push_back(p);
    return kept;
}

} // namespace

TEST("engine: chats that outgrow their cache, one of them from a shared prefix")
{
    scheduler_config config;
    config.max_sequences = 2;
    config.max_batch_tokens = 16;
    config.kv_block_count = pages;
    config.kv_block_size = page;
    config.prefill_chunk_tokens = 8;
    config.prefix_cache_min_tokens = 4;
    window_runner runner;
    auto engine = inference_engine::make(config, runner);
    REQUIRE(engine);
    auto add = [&](seq_id id, std::size_t prompt, std::size_t max_new) {
        std::vector<token_id> tokens(prompt);
        for (std::size_t i = 0; i < prompt; ++i)
            tokens[i] = static_cast<token_id>(3 + i % 17);
        auto s = seq::make(id, std::move(tokens), generation_params { max_new, true }, { 9 });
        REQUIRE(s);
        REQUIRE(engine->add(std::move(*s)));
    };
    add(1, 12, 40);
    for (int i = 0; i < 8; ++i)
        REQUIRE(engine->step());
    add(2, 15, 20); // shares the first nine tokens' pages
    CHECK(engine->find_sequence(2)->cached_token_count() == 9);
    runner.history[2].assign(runner.history[1].begin(), runner.history[1].begin() + 9);
    std::size_t compactions = 0;
    for (int steps = 0; !engine->is_finished(); ++steps) {
        for (const seq_id id : { seq_id { 1 }, seq_id { 2 } }) {
            const seq* s = engine->find_sequence(id);
            if (s->is_finished() || s->next_position() < 20)
                continue;
            const auto kept = sinks_and_newest(s->next_position(), 9);
            REQUIRE(engine->compact(id, kept, theta));
            runner.keep(id, kept);
            CHECK(s->next_position() == 11 && runner.state->resources(id).blocks.size() == 3);
            ++compactions;
        }
        REQUIRE(engine->step());
        REQUIRE(steps < 200);
    }
    CHECK(compactions >= 4 && runner.checked > 60);
    CHECK(engine->find_sequence(1)->completion_token_count() == 40);
    CHECK(engine->find_sequence(2)->completion_token_count() == 20);
    CHECK(runner.state->pages().free_block_count() == pages - 3); // the published prefix's
}
