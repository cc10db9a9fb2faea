// Internal declarations of libckv: context/pool state and kernel launchers.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <map>
#include <memory>
#include <string>
#include <vector>

#include "ckv.h"

namespace ckv {

// Geometry of one KV tensor as the kernels see it. Element index of
// (layer, slot, kv_head, feature) is (layer*slot_count + slot)*F + kv_head*D + feature.
struct pool_view {
    void* keys;
    void* values;
    uint64_t layer_elems; // blocks * block_size * F
    uint32_t blocks;
    uint32_t block_size;
    uint32_t kv_heads;
    uint32_t head_dim;
    uint32_t features; // kv_heads * head_dim
    uint32_t elem_size;
    int dtype; // ckv_dtype
};

// The keys a row at position p attends: those at t <= p with t > p - window or
// t < sinks. all_keys: every t <= p.
struct key_window {
    uint32_t window; // at least 1: a row attends itself
    uint32_t sinks;
};
constexpr key_window all_keys { UINT32_MAX, 0 };

// The window's first key.
__host__ __device__ inline uint32_t window_low(uint32_t position, key_window w)
{
    return position >= w.window ? position - w.window + 1 : 0;
}

// Of a row's units of `unit` tokens (tokens, pages or key blocks) in order, those
// that hold no key it attends: `skip` of them from unit `kept` on. What a kernel
// walks is the row's other units: unit u < kept as it is, a later one skip on.
struct window_gap {
    uint32_t kept, skip;
};
__host__ __device__ inline window_gap window_gap_of(uint32_t low, uint32_t sinks, uint32_t unit)
{
    const uint32_t first = low / unit; // the window's first unit
    const uint32_t held = sinks < low ? sinks / unit + (sinks % unit != 0) : first;
    const uint32_t kept = held < first ? held : first;
    return { kept, first - kept };
}

// Device pointers into the uploaded metadata block (one H2D copy per upload).
struct meta_view {
    const uint32_t* table;
    const uint32_t* offsets;
    const uint32_t* lengths;
    const uint32_t* positions;
    const uint32_t* slots;
    const uint32_t* items; // decode work list: (row, chunk) pairs
    const uint32_t* row_first; // first work item of each row
    const uint32_t* row_count; // work items (chunks) of each row
    // prefill query tiles, tile_entry_words each: (first row, row count, the
    // first row's position, the rows' table offset)
    const uint32_t* tiles;
    // fast decode plan, plan_entry_words per entry: a segment (pages
    // [first, end) of a row) per entry, (row, the segment's chunk index in
    // the row, the row's position, the flat table index of page `first`,
    // first, end, the row's chunk count, the workgroup's next entry or
    // plan_last). Workgroup w (per kv head) starts at entry w. A workgroup
    // needs nothing else from the batch to issue its first page loads.
    const uint32_t* plan;
    const uint32_t* split_first; // first partial record of each row cut into chunks
    const uint32_t* cut;         // the rows cut into chunks
    uint32_t n_entries;
    uint32_t rows;
    uint32_t n_items;
    uint32_t chunk; // tokens per decode work item, a multiple of 16
    uint32_t n_tiles;
    uint32_t tile_blocks; // 32-key blocks the batch's shortest query tile attends (host side)
    uint32_t row_blocks[3]; // runs of 32, 64 and 128 rows the tiles fall into (host side)
    uint32_t mean_pages; // pages attended per row, mean over the batch (host side)
    uint32_t n_plan;      // workgroups per kv head of the fast decode (the entries they start at)
    uint32_t n_segments;  // entries of plan
    uint32_t split_pages; // the plan's pages per chunk or per workgroup; 0: one row per workgroup
    uint32_t n_records;   // partial records of the rows cut into chunks
    uint32_t n_cut;       // rows cut into chunks
    key_window window = all_keys;
    uint32_t longest_blocks; // 32-key blocks the longest of a window's tiles attends (host side)
};

// Device scratch of the fast decode's cut rows: a partial record
// [max, denominator, 0, 0, acc[head_dim]] per (record, q head), written by the
// chunks, and an arrival counter per (record, kv head), of which a cut row
// uses the one at (its first record, kv head). The counters must be zero
// before a launch and every launch leaves them zero (the row's last chunk
// resets its counter), so they are cleared once, when allocated.
struct split_scratch {
    float* records;
    uint32_t* arrivals;
};

constexpr size_t tile_entry_words = 4;

// Device scratch of a prefill launch whose tiles' key blocks are split
// between workgroups: a record [max, denominator, 0, 0, acc[128]] per (share,
// query vector), and an arrival counter per (tile, workgroup row range, kv
// head), zero before a launch and left zero by it. n_split = 1: no split;
// a tile's keys are cut into at most n_split ranges of at least min_blocks
// 32-key blocks.
struct prefill_split {
    float* records;
    uint32_t* arrivals;
    uint32_t n_split;
    uint32_t min_blocks;
};
constexpr uint32_t prefill_record_floats = 128 + 4;
constexpr uint32_t split_min_blocks = 8; // default of prefill_split::min_blocks
constexpr uint32_t split_max = 8;        // shares a tile's keys are split into at most

// A tile (or a workgroup's rows of it) whose keys span n_blocks 32-key
// blocks is cut into at most n_split ranges of at least min_blocks each;
// prefill_range_count gives how many. A tile shorter than three ranges' worth
// is not cut (1): the handoff's round trips would cost more than the blocks
// it takes off the longest range. n_split and min_blocks are at least 1
// (prefill_plan).
__host__ __device__ inline uint32_t prefill_range_count(uint32_t n_blocks, uint32_t n_split,
                                                        uint32_t min_blocks)
{
    const uint32_t by_length = n_blocks / min_blocks;
    return n_blocks >= 3 * min_blocks ? (by_length < n_split ? by_length : n_split) : 1;
}

// The key blocks [begin, end) of range `part` of n ranges. Range 0 starts at
// block 0, of which every query attends some key where there is no window; through
// one it may attend none there, but itself in some range. 32-bit:
// n_blocks < 2^27 (positions are 32-bit) and part < 16 (prompts' ranges; others' split_max).
__host__ __device__ inline void prefill_range_bounds(uint32_t n_blocks, uint32_t n, uint32_t part,
                                                     uint32_t& begin, uint32_t& end)
{
    begin = part * n_blocks / n;
    end = (part + 1) * n_blocks / n;
}

// Largest query tile, in rows (positions): the prefill kernel covers a tile
// with G workgroups of 256/G rows for GQA group size G.
constexpr uint32_t prefill_tile_rows = 256;

// Inverse RoPE frequencies of one (theta, rotary width), by value as a kernel
// argument; head_dim is at most 1024, so rotary/2 <= 512.
constexpr uint32_t max_rope_pairs = 512;
struct rope_table {
    float inv_freq[max_rope_pairs];
};
// The first N of them, all that a head of 2N features uses: the fused decode's
// kernel argument.
template <int N>
struct rope_pairs {
    float inv_freq[N];
};

// Turns of a position's angle on each rotary pair: the fraction of a whole turn
// by which a step of one position turns the pair, times 2^64, so that a position's
// angle modulo a turn is one 64-bit product (rope_turns.h). By value as a kernel
// argument, like rope_table.
constexpr uint32_t max_turn_pairs = 256;
struct turn_table {
    uint64_t step[max_turn_pairs];
};
// The axis whose position turns each pair.
constexpr uint32_t max_axes = 4;
struct axis_table {
    uint8_t axis[max_turn_pairs];
};

// A rotation of rows (kernels_rotate.hip): how far a position turns each pair, how the
// pairs stand, and what turned pairs are multiplied by.
struct rotation_table {
    turn_table turns;
    double magnitude64;
    float magnitude;
    uint32_t rotary;     // 0: no rotation
    uint32_t neighbours; // pairs (2j, 2j + 1), else (j, j + rotary / 2)
};

// One rotary pair (a, b) -> (a cos - b sin, b cos + a sin), written once with
// explicit fused multiply-adds for every kernel that rotates (ckv_rope,
// ckv_rope_append, the fused decode).
__device__ __forceinline__ void rope_pair(float a, float b, float c, float s, float& ra, float& rb)
{
    ra = __builtin_fmaf(a, c, -(b * s));
    rb = __builtin_fmaf(b, c, a * s);
}

// The moves of a compaction that read each slot (the first and the last) and the one
// that writes it, by the generation of the call that marked them; and its moves' chains.
struct move_marks {
    struct mark {
        uint32_t read = 0, first = 0, last = 0, written = 0, writer = 0;
    };
    std::vector<mark> at_slot;
    std::vector<uint32_t> chain, reader, sizes;
    uint32_t generation = 0;
};

// A batch through a window: the same rows with the plan, the work list or the tiles of
// what the window leaves of them, each derived at the first launch that takes it and
// kept, in buffers of their own, until the next batch: a model's layers of several
// windows, and graphs that captured them, find theirs.
struct window_batch {
    uint32_t tile_rows = 0; // the tiles' rows at most; 0: decode rows
    bool plan_ready = false, work_ready = false, tiles_ready = false;
    bool work_multi = false;
    meta_view meta {};
    uint32_t *d_plan = nullptr, *d_work = nullptr, *d_tiles = nullptr;
    size_t d_plan_words = 0, d_work_words = 0, d_tiles_words = 0;
};

// A batch's work list of kernels_prompt.hip for one form of launch, made and kept as a
// window_batch's.
struct prompt_batch {
    bool ready = false;
    uint32_t q_heads = 0, waves = 0, heads = 0;
    bool paged_kernel = false, fp4 = false;
    meta_view meta {};
    uint32_t n_records = 0, n_cut = 0;
    uint32_t* d_list = nullptr;
    size_t d_list_words = 0;
};

struct pending_timing {
    const char* name;
    hipEvent_t start;
    hipEvent_t stop;
};

struct profile_total {
    double ms = 0.0;
    uint64_t launches = 0;
};

// ---- elementwise (kernels_rope.hip) ------------------------------------------------
// out[i] = in[i] * sigmoid(gate[i]) over n elements of dtype (src/tensor/tensor_ops.cc:289-296)
hipError_t launch_sigmoid_mul(hipStream_t s, int dtype, const void* gate, const void* in,
                              void* out, uint64_t n);

// ---- launchers (kernels_rope.hip) --------------------------------------------------
// theta^(-2j/rotary) in float for j < rotary/2 (src/metal/metal_kernels.mm:186-191)
void rope_frequencies(float theta, uint32_t rotary, rope_table& out);
// rows of `heads` heads of the pool's head_dim and dtype, at the uploaded positions
hipError_t launch_rope(hipStream_t s, const pool_view& p, const meta_view& m, const void* in,
                       void* out, uint32_t rows, uint32_t heads, uint32_t rotary,
                       const rope_table& freq);
// rotated key rows and the value rows into the uploaded slots of `layer`
hipError_t launch_rope_append(hipStream_t s, const pool_view& p, const meta_view& m,
                              uint32_t layer, const void* keys, const void* values, uint32_t rows,
                              uint32_t rotary, const rope_table& freq);

} // namespace ckv

struct ckv_context {
    int device = 0;
    int cu_count = 0;
    hipStream_t own_stream = nullptr;
    hipStream_t stream = nullptr;
    std::string last_error;

    // pinned staging for metadata uploads: a ring of slots, each reused once
    // the copy last made from it has completed, so the host can prepare the
    // next uploads while earlier ones wait in the stream behind kernels
    static constexpr int staging_slots = 4;
    struct staging_slot {
        void* pinned = nullptr;
        size_t bytes = 0;
        hipEvent_t done = nullptr;
        bool pending = false;
    };
    staging_slot staging[staging_slots];
    int staging_next = 0; // the slot stage() hands out

    // this device's copy of the no-allocation entry point's scratch array
    // (its device address, from hipGetSymbolAddress at context creation; null
    // if that failed)
    void* noalloc_scratch = nullptr;

    // device and pinned host allocations and frees made by the library on
    // this context (ckv_debug_allocations)
    uint64_t allocations = 0;

    // A call that takes launches under capture into account runs on a stream being
    // captured: it is refused what it would upload or allocate.
    bool in_capture = false;

    bool profile = false;
    std::vector<ckv::pending_timing> pending;
    std::vector<hipEvent_t> spare_events;
    std::map<std::string, ckv::profile_total> totals;
};

struct ckv_pool {
    ckv_context* ctx = nullptr;
    size_t layers = 0, blocks = 0, block_size = 0, kv_heads = 0, head_dim = 0;
    int dtype = CKV_BF16;
    size_t elem_size = 2;
    void* keys = nullptr;
    void* values = nullptr;
    size_t bytes_each = 0;
    bool owned = false;
    bool fp4 = false; // keys and values held in 4 bits (fp4.h); dtype is the rows'

    // host state of the current batch
    bool uploaded = false;
    bool has_slots = false;
    size_t n_entries = 0; // entries of the table the rows index
    size_t slot_rows = 0; // rows with an uploaded slot (0 without slots)
    std::vector<uint32_t> positions;
    uint32_t last_position = 0; // the largest of them
    std::vector<uint32_t> row_offsets; // each row's table offset (the decode plan's entries)
    std::vector<uint32_t> tiles; // the batch's query tiles (meta_view::tiles)
    bool shared_tile = false;
    bool fusable = false; // slots are the rows' own positions, one row per table range
    // while fusable: each row's own table index (offset + position / block_size)
    // and its uploaded slot, so a table patch can tell whether the fused
    // append still writes where ckv_append would
    std::vector<uint32_t> own_index, own_slot;
    // derived when a decode launch first needs them: the fast decode's plan
    // (uploaded with the batch when the batch goes to the decode kernel
    // anyway) and the generic path's split-KV work list
    bool plan_ready = false;
    bool work_ready = false;
    bool work_multi = false; // some row has more than one chunk: partials are merged
    std::vector<uint32_t> scratch; // host staging of the derived arrays
    std::vector<uint64_t> sort_keys;
    std::vector<uint32_t> stamp; // distinctness checks (all_distinct)
    uint32_t stamp_generation = 0;
    // pages the fused append writes, by page id: the generation that marked
    // them and the table index each is written through (own_pages_clash)
    std::vector<uint32_t> own_stamp, own_at;
    uint32_t own_generation = 0;

    // device copies
    uint32_t* d_meta = nullptr;
    size_t d_meta_words = 0;
    uint32_t* d_plan = nullptr; // the plan of a batch uploaded without it
    size_t d_plan_words = 0;
    uint32_t* d_work = nullptr;
    size_t d_work_words = 0;
    ckv::meta_view meta {};

    // device-resident sequence tables (ckv_seq_tables_*): seq_max rows of
    // seq_cap page ids. The host keeps a mirror of the entries and the rows'
    // lengths; entries written since the last batch upload are pending
    // (listed once each in `dirty`) and go up with the next batch.
    bool device_tables = false; // the current batch indexes the sequence tables
    uint32_t* d_seq = nullptr;
    size_t d_seq_words = 0;
    size_t seq_max = 0, seq_cap = 0;
    std::vector<uint32_t> seq_len, seq_host, dirty;
    std::vector<uint8_t> seq_dirty;

    // the current batch through each window it was attended through, then spare ones
    std::vector<std::unique_ptr<ckv::window_batch>> windows;
    size_t n_windows = 0;
    std::vector<std::unique_ptr<ckv::prompt_batch>> prompts; // the same of work lists
    size_t n_prompts = 0;
    std::vector<uint32_t> window_positions; // positions less the tokens of the skipped units

    // the batch rows' positions on several axes ([axes][rows], ckv_rope_axes_upload)
    uint32_t axes = 0;
    uint32_t* d_axes = nullptr;
    size_t d_axes_words = 0;

    ckv::turn_table turns {}; // of the last theta and rotary width (turns_of)
    float turns_theta = 0.0f;
    uint32_t turns_rotary = 0;

    // the tables of the last few ckv_rotations: layers that alternate between some find theirs
    struct kept_rotation {
        ckv_rotation of;
        ckv::rotation_table table;
    };
    kept_rotation rotations[8] = {};
    uint32_t n_rotations = 0, next_rotation = 0;
    int whole_prompts = -1; // whether the batch's rows are whole prompts; -1: not yet looked at

    ckv::move_marks marks; // of ckv_compact's slots
    uint8_t* d_spare = nullptr; // rows it saves
    size_t d_spare_bytes = 0;

    // A captured launch keeps reading what it was given whenever its graph is replayed.
    // captured: a call of the pool that takes launches under capture into account was
    // made under one; buffers that grow from then on leave the old one to the graphs,
    // until the pool goes.
    bool captured = false;
    std::vector<void*> retired;

    // device scratch
    float* d_partials = nullptr;
    size_t d_partials_bytes = 0;
    uint32_t* d_arrivals = nullptr; // the fast decode's arrival counters (zero between launches)
    size_t d_arrivals_words = 0;
    float* d_pre_records = nullptr; // the split prefill's records
    size_t d_pre_records_floats = 0;
    uint32_t* d_pre_arrivals = nullptr; // its arrival counters (zero between launches)
    size_t d_pre_arrivals_words = 0;
    uint32_t* d_pairs = nullptr; // block-id pairs / patch pairs
    size_t d_pairs_words = 0;
    char* d_spill = nullptr; // staging of checkpoint export/import
    size_t d_spill_bytes = 0;
    char* d_rope_q = nullptr; // rotated queries of the unfused ckv_rope_append_decode
    size_t d_rope_q_bytes = 0;
};

namespace ckv {

// ---- launchers (kernels_copy.hip) ------------------------------------------
hipError_t launch_store_kv(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                           const void* keys, const void* values, uint32_t rows);
hipError_t launch_gather(hipStream_t s, const pool_view& p, const uint32_t* table,
                         uint32_t layer, uint32_t n_tokens, void* out_keys, void* out_values);
hipError_t launch_copy_blocks(hipStream_t s, const pool_view& p, uint32_t layers,
                              const uint32_t* pairs, uint32_t n);
hipError_t launch_checkpoint(hipStream_t s, const pool_view& p, uint32_t layers,
                             const uint32_t* blocks, uint32_t tokens, void* packed_keys,
                             void* packed_values, bool unpack);
hipError_t launch_table_patch(hipStream_t s, uint32_t* table, const uint32_t* pairs, uint32_t n);
// dst[0..n) = value (a kernel, not hipMemsetAsync: callers may capture it)
hipError_t launch_fill(hipStream_t s, uint32_t* dst, uint32_t value, uint32_t n);
// Expands a batch given as items into per-row metadata. `items` holds five
// sections of n_items words: sequence, first position, token count, first
// row, table length. Rows get offset seq*cap, the item's length, position
// first + j and (with_slots) slot seq_table[seq*cap + pos/bs]*bs + pos%bs.
hipError_t launch_expand_batch(hipStream_t s, const uint32_t* items, uint32_t n_items,
                               uint32_t rows, const uint32_t* seq_table, uint32_t cap,
                               uint32_t block_size, bool with_slots, uint32_t* offsets,
                               uint32_t* lengths, uint32_t* positions, uint32_t* slots);

// ---- decode plan (kernels_decode.hip) -------------------------------------------
// The fast decode's plan of a batch, from its rows' positions: which pages
// each workgroup covers, as segments of rows, and each cut row's first
// partial record. A row per workgroup (longest first) while that keeps every
// compute unit busy; otherwise, when one workgroup per (row, kv head) would
// leave the batch bound by its longest rows (a row holds more than half of
// one compute unit's share of the batch's pages), the batch's pages in row
// order are dealt out evenly to as many workgroups as the GPU holds at once,
// each taking a run of whole rows and row pieces (balanced). The fixed form
// cuts each row into chunks of split_pages pages, a workgroup per chunk.
// CKV_DECODE_SPLIT=<pages> forces the fixed form (0: no cut),
// CKV_DECODE_BALANCE=<pages> the balanced form with that many pages per
// workgroup.
struct decode_plan_shape {
    uint32_t split_pages; // pages per chunk (fixed) or per workgroup (balanced); 0: no cut
    uint32_t n_items;     // plan entries (segments)
    uint32_t n_records;
    uint32_t n_cut;
    uint32_t n_wgs;       // workgroups per kv head
    uint32_t n_deal;      // balanced: the workgroups per kv head the pages are dealt to
    uint64_t deal_work;   // balanced: the work dealt out (pages and segment costs)
    bool balanced;
};
struct decode_form {
    uint32_t per_cu;      // workgroups a compute unit holds
    uint32_t min_pages;   // shortest chunk cut, but for the rest of a row
    uint32_t max_chunks;  // most chunks of a row
    uint32_t uncut_slack; // pages by which a row may exceed the share and stay whole
    bool few_waves;       // workgroups too small to read a whole row at full rate
};
decode_form decode_form_of(int dtype, uint32_t head_dim);
decode_plan_shape shape_decode_plan(const std::vector<uint32_t>& positions, uint32_t block_size,
                                    uint32_t kv_heads, int cu_count,
                                    const decode_form& form = decode_form_of(CKV_BF16, 128),
                                    uint64_t chunk = 0); // fixed chunks of so many pages
// The plan of rows through a window, from their positions without its gaps.
decode_form window_form_of(int dtype, uint32_t head_dim);
decode_plan_shape shape_window_plan(const std::vector<uint32_t>& positions, uint32_t block_size,
                                    uint32_t kv_heads, int cu_count, decode_form form);
// Waves per workgroup of the fast decode for a launch of `units` (plan
// workgroup, kv head) workgroups: a plan's split_pages (0 when no row is cut)
// and the batch's mean row pages decide it; CKV_DECODE_WAVES overrides.
uint32_t decode_fast_waves(uint32_t group, int dtype, uint32_t units, int cu_count,
                           uint32_t mean_pages, uint32_t split_pages);
constexpr size_t plan_entry_words = 8;
constexpr uint32_t plan_last = 0xFFFFFFFFu; // no next entry
// Writes shape.n_items plan entries to plan, rows words to split_first and the
// shape.n_cut cut rows to cut; offsets are the rows' table offsets.
void write_decode_plan(const std::vector<uint32_t>& positions,
                       const std::vector<uint32_t>& offsets, uint32_t block_size,
                       const decode_plan_shape& shape, std::vector<uint64_t>& sort_keys,
                       uint32_t* plan, uint32_t* split_first, uint32_t* cut);

// ---- launchers (kernels_decode.hip) ------------------------------------------
// Returns hipErrorInvalidValue when no kernel fits the geometry. The fast
// path (decode_fast_applies) merges a chunk's waves in the workgroup; when the
// plan cuts rows into chunks it needs `split` (records of m.n_records x q_heads)
// and launches a merge of the cut rows after the chunks; the generic path
// writes partials for rows with several chunks and needs a merge launch.
// gate (optional, same shape and dtype as out): out = attention * sigmoid(gate),
// the sigmoid_mul of src/qwen/qwen_layer.cc:204 in the epilogue.
hipError_t launch_decode(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                         const void* q, uint32_t q_heads, float scale, void* out,
                         float* partials, int cu_count, const void* gate = nullptr,
                         split_scratch split = {});
bool decode_fast_applies(const pool_view& p, uint32_t q_heads, const void* q, const void* out);
// store_kv + fast decode in one launch; the caller has checked
// decode_fast_applies, 16-byte aligned inputs, and that every row's slot is
// its position's slot with no two rows on one table range.
// With `rope` (rotary a multiple of 16 up to 128, rotary/16 a power of two)
// the queries and the new keys are rotated inside the kernel first.
hipError_t launch_append_decode(hipStream_t s, const pool_view& p, const meta_view& m,
                                uint32_t layer, const void* k_in, const void* v_in, const void* q,
                                uint32_t q_heads, float scale, void* out, const void* gate,
                                int cu_count, split_scratch split, const rope_table* rope = nullptr,
                                uint32_t rotary = 0);
hipError_t launch_merge(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t q_heads,
                        void* out, const float* partials, const void* gate = nullptr);
bool decode_uses_fast_path(const pool_view& p, uint32_t q_heads);
// The fast decode of a batch through a window (m.window), its arguments already
// checked and scaled by launch_decode and launch_append_decode.
hipError_t launch_window_fast(hipStream_t s, const pool_view& p, const meta_view& m,
                              uint32_t layer, const void* q, uint32_t q_heads, float scale_log2,
                              void* out, const void* k_in, const void* v_in, const void* gate,
                              int cu_count, split_scratch split, const rope_table* rope,
                              uint32_t rotary);
// Waves per workgroup of the fast decode through a window (decode_fast_waves's arguments).
uint32_t decode_window_waves(uint32_t head_dim, uint32_t group, int dtype, uint32_t units,
                             int cu_count, uint32_t mean_pages, uint32_t split_pages);
// Sets every entry of a plan written from the window's positions to its row's position.
void place_window_plan(const std::vector<uint32_t>& positions, const decode_plan_shape& shape,
                       uint32_t* plan);
// Floats per (work item, q head) partial record: [max, denominator, 0, 0, acc[head_dim]].
uint32_t partial_record_floats(uint32_t head_dim);

// ---- launchers (kernels_prefill.hip, kernels_prefill_wide.hip, kernels_prefill_f32.hip) ----
// MFMA prefill: head_dim 128 (16-bit pools: or 256), 16-token pages, GQA group
// 1/2/4/8, 16-byte aligned pools, queries and output; bf16/fp16 products on
// v_mfma_f32_32x32x16, f32 ones on v_mfma_f32_32x32x2_f32.
bool prefill_supported(const pool_view& p, uint32_t q_heads, const void* q, const void* out);
// How a 16-bit prefill launch runs: workgroup waves (8, or 4 when 8-wave
// workgroups would not give every compute unit one) and the key split of the
// 4-wave form (1: none), with the records and counters that split needs.
struct prefill_shape_info {
    uint32_t waves;
    uint32_t n_split;
    uint32_t min_blocks;
    uint64_t records_floats;
    uint64_t counters;
};
prefill_shape_info prefill_plan(const pool_view& p, const meta_view& m, uint32_t q_heads,
                                int cu_count);
hipError_t launch_prefill(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                          const void* q, uint32_t q_heads, float scale, void* out,
                          const void* gate, const prefill_shape_info& plan,
                          prefill_split split);
// Rows of a workgroup of the windowed prefill: its tiles have at most so many.
uint32_t prefill_window_rows(const pool_view& p, uint32_t q_heads);
// The same for 16-bit pools of 256-wide heads (kernels_prefill_wide.hip).
prefill_shape_info prefill_wide_plan(const pool_view& p, const meta_view& m, uint32_t q_heads,
                                     int cu_count, uint32_t min_blocks);
hipError_t launch_prefill_wide(hipStream_t s, const pool_view& p, const meta_view& m,
                               uint32_t layer, const void* q, uint32_t q_heads, float scale,
                               void* out, const void* gate, prefill_split split);
hipError_t launch_prefill_f32(hipStream_t s, const pool_view& p, const meta_view& m,
                              uint32_t layer, const void* q, uint32_t q_heads, float scale,
                              void* out, const void* gate, prefill_split split);

// ---- launchers (kernels_rope.hip) --------------------------------------------------
// theta^(-2j/rotary) in float for j < rotary/2 (src/metal/metal_kernels.mm:186-191)
void rope_frequencies(float theta, uint32_t rotary, rope_table& out);
// rows of `heads` heads of the pool's head_dim and dtype, at the uploaded positions
hipError_t launch_rope(hipStream_t s, const pool_view& p, const meta_view& m, const void* in,
                       void* out, uint32_t rows, uint32_t heads, uint32_t rotary,
                       const rope_table& freq);
// rotated key rows and the value rows into the uploaded slots of `layer`
hipError_t launch_rope_append(hipStream_t s, const pool_view& p, const meta_view& m,
                              uint32_t layer, const void* keys, const void* values, uint32_t rows,
                              uint32_t rotary, const rope_table& freq);

// ---- launchers (kernels_rope_axes.hip) ----------------------------------------------
// theta^(-2j/rotary) of a radian per position, as turn_table's steps
void turn_steps(float theta, uint32_t rotary, turn_table& out);
// Query rows [rows, q_heads, head_dim] rotated into `rotated` and, with keys, key
// rows rotated and value rows copied into the uploaded slots of `layer`; pair j
// turns by positions[axis[j]][row]. q_heads 0: keys and values alone.
struct axes_rows {
    const void* queries;
    void* rotated;
    const void* keys;
    const void* values;
};
// Heads of a row that a thread of the launch takes in 16-byte words: four, unless that
// leaves fewer than two workgroups per compute unit; 0: the rows go pair by pair.
uint32_t rope_axes_heads(const pool_view& p, const axes_rows& x, uint32_t rows, uint32_t heads,
                         uint32_t rotary);
hipError_t launch_rope_axes(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                            const axes_rows& x, uint32_t rows, uint32_t q_heads, uint32_t rotary,
                            const turn_table& turns, const axis_table& axes,
                            const uint32_t* positions);

// ---- launchers (kernels_compact.hip) --------------------------------------------------
// Moves of a compaction on the device: `runs` holds n_runs (first move, moves), each
// run's moves in order, and the moves' source slots, target slots and position
// shifts. A run's moves may overwrite what the same run reads at or before them;
// nothing a run reads or writes is written by another. Slots from spare_slot on are rows
// of `spare`, n_spare for each layer of K, then of V.
constexpr uint32_t spare_slot = 0x80000000u;
struct compact_moves {
    const uint32_t* runs;
    const uint32_t* from;
    const uint32_t* to;
    const int32_t* shift;
    uint32_t n_runs;
    void* spare;
    uint32_t n_spare;
};
// Checks the moves of ckv_compact (of at most spare_slot slots) and cuts them into runs.
// `kept` are the moves that change something, run by run; `runs` pairs (first of kept,
// how many), in the order of their launches, whose numbers of runs `launches` holds. The
// runs of one launch depend on each other in no way. Where some of kept read what another
// run writes, `saved` are those moves and `spare` the place in it of each of kept
// (UINT32_MAX: none): the first of two launches copies their sources to spare rows, its
// runs counting on from the end of kept. Returns null, or why the moves are refused, with
// the status.
constexpr uint32_t compact_run = 64;
struct compact_plan {
    std::vector<uint32_t> kept, spare, saved, runs, launches;
};
// What a move costs, in microseconds: its bytes and its share of a run done in order; and
// a launch.
struct compact_cost {
    double move_bytes, move_in_run, launch;
};
compact_cost compact_cost_of(const pool_view& p, uint32_t layers);
const char* plan_compaction(move_marks& marks, size_t slots, const uint32_t* from,
                            const uint32_t* to, const int32_t* shift, const uint32_t* counts,
                            size_t n_sequences, const compact_cost& cost, compact_plan& plan,
                            int& status);
// Words (an even number, both arrays aligned to 8 bytes) from pinned host memory, read
// by a kernel: between two kernels a copy of 120 KB takes 14 us on MI355X, of 16 KB 5.
hipError_t launch_fetch(hipStream_t s, uint32_t* to, const void* pinned, size_t words);
// The kv heads that a workgroup of the compaction in 16-byte words goes through: all of
// them, unless that leaves fewer workgroups than keep the memory busy; 0: the geometry is
// moved an element at a time.
uint32_t compact_heads(const pool_view& p, uint32_t layers, uint32_t n_runs, uint32_t rotary);
hipError_t launch_compact(hipStream_t s, const pool_view& p, uint32_t layers,
                          const compact_moves& moves, uint32_t rotary, const turn_table& turns);

// ---- launchers (kernels_rotate.hip) ----------------------------------------------------
// Query rows rotated into `rotated` and, with keys, key rows rotated and value rows copied
// into the uploaded slots of `layer`, and both also into held_keys and held_values where
// these are given. q_heads 0: keys and values alone.
struct rotate_rows {
    const void* queries;
    void* rotated;
    const void* keys;
    const void* values;
    void* held_keys;
    void* held_values;
    bool float_queries; // `rotated` holds floats, whatever the rows' type
};
hipError_t launch_rotate(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                         const rotate_rows& x, uint32_t rows, uint32_t q_heads,
                         const rotation_table& by);
// The same into a pool held in 4 bits; held rows are as the cache holds them.
hipError_t launch_fp4_append(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                             const rotate_rows& x, uint32_t rows, uint32_t q_heads,
                             const rotation_table& by);
hipError_t launch_fp4_gather(hipStream_t s, const pool_view& p, const uint32_t* table,
                             uint32_t layer, uint32_t n_tokens, void* out_keys, void* out_values);
// The fractions of a turn of turns[j] (turns a position on pair j) as steps.
void rotation_steps(const long double* turns, uint32_t rotary, rotation_table& out);

// ---- launchers (kernels_fp4_decode.hip) -------------------------------------------------
decode_form fp4_decode_form();
// (float_queries: the queries are floats, whatever the rows' type.)
// Workgroups that share a (plan workgroup, kv head): each takes at most eight query heads
// (f32 rows: four).
uint32_t fp4_decode_passes(const pool_view& p, uint32_t q_heads);
hipError_t launch_fp4_decode(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                             const void* q, bool float_queries, uint32_t q_heads, float scale,
                             void* out, const void* gate, split_scratch split);

// ---- launchers (kernels_prompt.hip) ------------------------------------------------------
// Rows of an attention of tiles; keys and values only where they are not a 4-bit pool's.
// Strides in elements. launch_prompt sets the alignments.
struct prompt_rows {
    const void* queries;
    const void* keys;
    const void* values;
    uint64_t q_stride, kv_stride;
    bool vectors, out_vectors;
};
// How a launch over the batch `m` runs: its waves (8: kernels_prefill.hip's workgroups over
// rows), and whether it is kernels_prefill.hip's at all.
struct prompt_form {
    uint32_t waves, heads; // of a workgroup
    bool paged_kernel, fp4;
    uint32_t tile_rows() const { return 32 * waves / heads; }
};
prompt_form prompt_form_of(const pool_view& p, const meta_view& m, const prompt_rows& x, uint32_t q_heads,
                           float scale, const void* out, const void* gate, bool fp4, int cu_count);
// A launch's work list: the batch's tiles cut into a workgroup's rows and, where that leaves
// compute units idle, each into ranges of its keys. An entry of prompt_entry_words for each
// range: first row, rows, first position, table offset, range, ranges, the tile's first
// record and its place among the tiles that are cut; most key blocks first.
constexpr size_t prompt_entry_words = 8;
struct prompt_list {
    std::vector<uint32_t> words;
    uint32_t n_records = 0, n_cut = 0; // for each (pass, kv head)
};
void write_prompt_list(const pool_view& p, const std::vector<uint32_t>& tiles, const prompt_form& form,
                       uint32_t q_heads, int cu_count, prompt_list& list);
hipError_t launch_prompt(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                         const prompt_rows& rows, const prompt_form& form, uint32_t q_heads,
                         float scale, void* out, const void* gate, bool fp4,
                         const prefill_split& split);
// kernels_prefill.hip's workgroups of `waves` waves over rows; the caller has checked 16-bit
// rows of 128-wide heads in 16-byte words and scale > 0.
hipError_t launch_prefill_rows(hipStream_t s, const pool_view& p, const meta_view& m,
                               const prompt_rows& x, uint32_t q_heads, float scale, void* out,
                               const void* gate, uint32_t heads, uint32_t waves,
                               const prefill_split& split);

} // namespace ckv
