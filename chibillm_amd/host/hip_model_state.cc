#include "hip_model_state.h"

#include <algorithm>
#include <limits>

#include "model_batch.h"

namespace chibillm {

result<std::unique_ptr<hip_model_state>, state_error>
hip_model_state::make(const hip_context& ctx, kv_cache_config config, kv_dtype type,
                      prefix_sharing sharing)
{
    auto pages = block_manager::make(config.block_count, config.block_size);
    if (!pages)
        return fail(state_errc::invalid_reservation, pages.error(), "block allocator");
    auto cache = hip_kv_cache::make(ctx, config, type);
    if (!cache)
        return fail(state_errc::backend_failure, cache.error(), "KV cache");
    return std::unique_ptr<hip_model_state>(new hip_model_state(
        std::make_shared<block_manager>(std::move(*pages)), std::move(*cache), sharing));
}

result<void, state_error>
hip_model_state::reserve(seq_id id, std::size_t tokens)
{
    auto reserved = pages_->reserve(id, tokens);
    if (reserved || reserved.error().code != state_errc::capacity_exhausted || !spill_)
        return reserved;
    const std::size_t bs = pages_->block_size();
    const std::size_t required = tokens ? 1 + (tokens - 1) / bs : 0;
    const std::size_t held = pages_->resources(id).blocks.size();
    if (required <= held || !spill_for(required - held))
        return reserved;
    return pages_->reserve(id, tokens);
}

bool
hip_model_state::spill_for(std::size_t pages) noexcept
try {
    // passes until no checkpoint frees a page: spilling one checkpoint can
    // leave an older one (a shorter prefix of the same pages) the only holder
    for (bool progress = true; progress && pages_->free_block_count() < pages;) {
        progress = false;
        for (shared_prefix_checkpoint* saved : *live_) {
            if (pages_->free_block_count() >= pages)
                break;
            if (saved->is_spilled())
                continue;
            // only pages that nothing else references come free
            std::size_t freed = 0;
            for (const block_id b : saved->pages)
                freed += pages_->refcount(b) == 1;
            if (!freed)
                continue;
            // the export is queued before any later write of the freed pages
            auto exported = cache_.export_prefix(saved->pages, saved->token_count);
            if (!exported)
                return false;
            saved->spilled = std::move(*exported);
            pages_->drop(saved->pages);
            saved->pages.clear();
            ++spills_;
            spilled_pages_ += freed;
            progress = true;
        }
    }
    return pages_->free_block_count() >= pages;
} catch (const std::bad_alloc&) {
    return false;
}

result<void, state_error>
hip_model_state::compact(seq_id id, std::span<const std::uint32_t> kept, float theta,
                         std::size_t rotary)
{
    const std::size_t bs = cache_.block_size();
    const auto held = resources(id).blocks;
    if (in_batch_ || kept.empty() || kept.back() / bs >= held.size())
        return fail(state_errc::invalid_reservation);
    if (const auto at = next_.find(id); at != next_.end() && at->second == no_position)
        return fail(state_errc::invalid_reservation);
    for (std::size_t i = 1; i < kept.size(); ++i)
        if (kept[i] <= kept[i - 1])
            return fail(state_errc::invalid_reservation);
    const std::size_t width = rotary ? rotary : cache_.head_dimension();
    if (!(theta >= 0.0f) || theta == std::numeric_limits<float>::infinity()
        || (theta > 0.0f && (width % 2 || width > cache_.head_dimension() || width > 512)))
        return fail(state_errc::invalid_reservation);
    // the pages that change, or that later tokens will fill, have to be the sequence's own
    const std::vector<block_id> old(held.begin(), held.end());
    const std::size_t n = kept.size(), pages = (n - 1) / bs + 1;
    const auto shared = [&] {
        std::vector<std::size_t> found;
        for (std::size_t j = 0; j < pages; ++j) {
            const std::size_t last = std::min(n, (j + 1) * bs) - 1;
            // tokens ascend: a page's last one moves if any does
            if (pages_->refcount(old[j]) > 1 && (kept[last] != last || last % bs != bs - 1))
                found.push_back(j);
        }
        return found;
    };
    std::vector<std::size_t> forks = shared();
    if (forks.size() > pages_->free_block_count() && spill_) {
        spill_for(forks.size()); // which may leave pages to this sequence alone
        forks = shared();
    }
    const std::uint32_t size = static_cast<std::uint32_t>(bs), count = static_cast<std::uint32_t>(n);
    std::vector<std::uint32_t> from(n), to(n);
    std::vector<std::int32_t> shift(theta > 0.0f ? n : 0);
    std::vector<block_id> table = old;
    // the pages that take the shared ones' place enter the sequence's table once the moves
    // are accepted; until then a failure gives them back
    struct borrowed_pages {
        block_manager& owner;
        std::vector<block_id> pages;
        ~borrowed_pages() { owner.give_back(pages); }
    } fresh { *pages_, {} };
    CL_TRY_ASSIGN(fresh.pages, pages_->borrow(forks.size()));
    for (std::size_t k = 0; k < forks.size(); ++k)
        table[forks[k]] = fresh.pages[k];
    for (std::uint32_t i = 0; i < count; ++i) {
        from[i] = old[kept[i] / size] * size + kept[i] % size;
        to[i] = table[i / size] * size + i % size;
        if (!shift.empty())
            shift[i] = static_cast<std::int32_t>(i - kept[i]);
    }
    std::size_t& next = next_.try_emplace(id, no_position).first->second;
    const std::size_t before = std::exchange(next, no_position);
    if (auto done = cache_.compact(from, to, shift, std::span(&count, 1), theta, rotary); !done) {
        if (done.error() != state_errc::backend_failure) {
            if (before == no_position)
                next_.erase(id);
            else
                next = before;
        }
        return fail(std::move(done.error()));
    }
    next = n;
    for (std::size_t k = 0; k < forks.size(); ++k)
        pages_->put(id, forks[k], fresh.pages[k]);
    fresh.pages.clear();
    return pages_->truncate(id, n);
}

result<void, state_error>
hip_model_state::begin_batch(const model_batch& batch)
{
    begun_.clear();
    if (!next_.empty())
        for (const model_batch_item& item : batch.items) {
            const auto at = next_.find(item.id);
            if (at == next_.end())
                continue;
            if (at->second == no_position || item.token_offset >= batch.positions.size()
                || batch.positions[item.token_offset] != at->second)
                return fail(state_errc::invalid_reservation);
            begun_.emplace_back(item.id, at->second + item.token_count);
        }
    in_batch_ = true;
    return {};
}

void
hip_model_state::commit_batch() noexcept
{
    for (const auto& [id, next] : begun_)
        if (const auto at = next_.find(id); at != next_.end())
            at->second = next;
    abort_batch();
}

void
hip_model_state::abort_batch() noexcept
{
    begun_.clear();
    in_batch_ = false;
}

std::size_t
hip_model_state::checkpoint_bytes(std::size_t tokens) const noexcept
{
    if (sharing_ != prefix_sharing::shared_pages)
        return cache_.checkpoint_bytes(tokens);
    if (!tokens || tokens > cache_.block_count() * cache_.block_size())
        return 0;
    // the pages a shared checkpoint keeps alive
    return (1 + (tokens - 1) / cache_.block_size()) * cache_.page_bytes_all_layers();
}

result<std::unique_ptr<model_checkpoint>, state_error>
hip_model_state::checkpoint(seq_id id, std::size_t tokens) const
{
    const auto table = resources(id).blocks;
    if (sharing_ == prefix_sharing::packed_copy) {
        auto saved = cache_.checkpoint(table, tokens);
        if (!saved)
            return fail(saved.error());
        return std::unique_ptr<model_checkpoint>(std::move(*saved));
    }
    if (sharing_ == prefix_sharing::host_copy) {
        auto saved = cache_.export_prefix(table, tokens);
        if (!saved)
            return fail(saved.error());
        return std::unique_ptr<model_checkpoint>(std::move(*saved));
    }
    const std::size_t bytes = checkpoint_bytes(tokens);
    if (!bytes)
        return fail(state_errc::invalid_reservation);
    const std::size_t needed = 1 + (tokens - 1) / cache_.block_size();
    if (table.size() < needed)
        return fail(state_errc::invalid_reservation);
    std::vector<block_id> held(table.begin(), table.begin() + needed);
    CL_TRY(pages_->retain(held));
    return std::unique_ptr<model_checkpoint>(
        std::make_unique<shared_prefix_checkpoint>(pages_, live_, std::move(held), tokens, bytes));
}

result<void, state_error>
hip_model_state::restore(seq_id id, const model_checkpoint& saved)
{
    const host_kv_checkpoint* host = dynamic_cast<const host_kv_checkpoint*>(&saved);
    if (const auto* shared = dynamic_cast<const shared_prefix_checkpoint*>(&saved)) {
        if (!shared->is_spilled())
            return restore_shared(id, *shared);
        host = shared->spilled.get();
    }
    if (host) { // reserve, copy in from host memory
        CL_TRY(reserve(id, host->token_count));
        return cache_.import_prefix(resources(id).blocks, *host);
    }
    const auto* packed = dynamic_cast<const kv_cache_checkpoint*>(&saved);
    if (!packed)
        return fail(state_errc::invalid_reservation);
    // the reference path (src/metal/metal_model_state.h:60-68): reserve, copy in
    CL_TRY(reserve(id, packed->token_count));
    return cache_.restore(resources(id).blocks, *packed);
}

result<void, state_error>
hip_model_state::restore_shared(seq_id id, const shared_prefix_checkpoint& saved)
{
    const std::size_t bs = cache_.block_size();
    const auto own = resources(id).blocks;
    // a fresh reservation holds exactly the one page admission reserved
    if (saved.owner != pages_ || own.size() != 1 || saved.pages.empty())
        return fail(state_errc::invalid_reservation);
    const block_id fresh = own[0];
    const std::size_t full = saved.token_count / bs;
    const bool partial_tail = saved.token_count % bs != 0;
    if (partial_tail) {
        // copy-on-write of the shared tail page into the sequence's own page,
        // which follows the shared full pages in its table
        const block_id tail = saved.pages[full];
        CL_TRY(cache_.copy_pages(std::span(&tail, 1), std::span(&fresh, 1)));
        ++cow_copies_;
    }
    // the own page now covers positions [full * bs, (full + 1) * bs)
    return pages_->share_prefix(id, std::span(saved.pages).first(full));
}

} // namespace chibillm
