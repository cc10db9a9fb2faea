// Paged GQA decode attention.
//
// Fast path (head_dim 128 or 256, 16-token pages, 1/2/4/8 q heads per KV head;
// f32 pages up to 4): one workgroup per (plan workgroup, kv_head) serves every
// q head of the KV head's GQA group, so each K/V byte is read once. Of 128-wide
// heads a wave reads four token rows per load instruction, 16 lanes per row, so lane l holds 8
// features of token 4j + l/16: 8*(l%16).. of a bf16/fp16 row (16 bytes), or
// 4*(l%16).. and 64 + 4*(l%16).. of an f32 row (two 16-byte words, each
// instruction reading 256 contiguous bytes). A score is a dot chain over the lane's 8 features
// (v_dot2 for 16-bit pairs) followed by a 16-lane DPP all-reduce (4 VALU ops).
// Each 16-lane row group keeps its own online-softmax state over its tokens;
// the four states are merged once per segment. 256-wide heads take 32 lanes a
// row, two rows per load instruction and half a page per step, which keeps the
// registers of the 128-wide form; they are read once for the whole group
// instead of once per q head by one wave (the general path): 32 rows of
// U[256, 4096] tokens, 2 kv heads, 8 q heads, rotated and gated, 607 -> 37 us. Scores are kept in the log2
// domain (scale * log2(e)) so every exponential is one v_exp_f32. Rows the
// batch plan cuts are merged in the same launch with weights 2^(m_c - M), the
// reduction of paged_attention_reduce_f32
// (src/metal/kernels/attention.metal:567-615).
//
// Generic path (any head_dim <= 1024, any page size): split-KV over token
// chunks, one wave per (chunk, kv_head), and a merge launch.
#include "decode_wg.h"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdlib>
#include <functional>

namespace ckv {
namespace {

// ---- generic path: any head_dim <= 1024, f32 / bf16 / fp16 ---------------------

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int mask = 32; mask >= 1; mask >>= 1)
        v += __shfl_xor(v, mask);
    return v;
}

constexpr int generic_max_features_per_lane = 16; // head_dim <= 1024

// Cut rows (shape_decode_plan). The balanced plan deals the batch's pages to
// as many workgroups as the GPU holds at once (decode_form::per_cu per compute
// unit), with a segment costing split_segment_pages pages and no piece shorter
// than split_min_piece; no more workgroups than rows where pieces would fall
// under the form's min_pages, and no row in more than max_chunks pieces (the
// merge of a row reads its pieces' records). With more rows than workgroups the
// round trips of the segments a workgroup runs one after another cost more than
// the balance gains, and rows are cut into fixed chunks of a quarter of a
// compute unit's share instead (the config-5 churn took 3 % longer dealing its
// batches of hundreds of rows); batches of under split_balance_min_pages pages
// per workgroup, and all of 256-wide heads, weigh the two (small_batch_span).
constexpr uint64_t split_row_pages = 10;
constexpr uint64_t split_min_piece = 4;
constexpr uint64_t split_balance_min_pages = 32;
constexpr uint64_t split_per_share = 4;
constexpr uint64_t split_segment_pages = 4;
// Pages (about 12 us of one workgroup's reads) by which the longest row may
// exceed 9/8 of a compute unit's share and still stay whole, for batches of
// one or two (row, kv head) units per compute unit, and no more than 13/8 of
// the share. Measured on one MI355X layer (fused, bf16, 8 kv heads), longest over
// share, whole and dealt out, us: 48 rows of U[200, 2000] tokens 1.21, 39.2 and
// 39.7; 56 of U[200, 2400] 1.06, 50.9 and 52.4; 64 of U[300, 3000] 0.91, 70.4 and 73.1; 36
// of U[100, 1200] 1.63, 23.6 and 21.7; 32 of U[300, 2000] 1.74, 36.5 and 30.6; 32 of
// U[1000, 3500] 1.55 (61 pages over), 60.2 and 51.5. Between 1.3 and the cap cutting
// has become the faster with its cheaper merges (32 of U[500, 1500] 1.49, 29.7
// and 27.2; 40 of U[300, 2000] 1.39, 37.7 and 35.2; 32 of U[400, 1700] 1.62, 32.2 and
// 28.5), which the line does not follow yet. Batches of fewer (row, kv head)
// units than compute units are cut (8 rows of 1,024 tokens whole: +36 %).
constexpr uint32_t split_uncut_slack = 47;
// How a pool's decode fills the GPU (decode_form). 16-bit pages of 128-wide
// heads: two 8-wave workgroups per compute unit. f32 pages: two of 4 waves; a
// whole row on 4 waves reads at a fraction of a compute unit's rate, so rows stay
// whole only while none is over 9/8 of the share and they even out (whole_rows_even):
// 48 rows of U[256, 700] tokens, longest 0.96 times the share, cut 39.0 us, whole 35.7;
// 36 of U[400, 900], 1.24 times, 35.1 and 41.4; 48 of U[256, 4096], 1.25, 130 and 170.
// 256-wide heads: one workgroup of 8 waves. With more than two q heads per kv
// head its lanes need the registers of two; with one or two, two would fit, but
// a plan for two is slower (2 kv heads, chunks for one and for two workgroups
// per compute unit, us: 32 rows of U[256, 4096] tokens 27.0 and 29.6 at one q head
// per kv head, 28.5 and 32.0 at two; 32 of 1,000 14.7 and 15.0, 16.0 and 16.3; 16 of
// U[100, 2500] 12.0 and 13.7, 13.2 and 15.1). A page is twice the bytes, so chunks may
// be shorter and the slack is half.
constexpr decode_form form_narrow { 2, 12, 32, split_uncut_slack, false };
constexpr decode_form form_f32 { 2, 8, 32, 0, true };
constexpr decode_form form_wide { 1, 4, 128, split_uncut_slack / 2, false };

// One wave per (work item, kv_head); the group's q heads are processed one
// after another, each with the per-token online softmax of
// paged_attention_f32 (src/metal/kernels/attention.metal:101-155), lanes
// striding the features.
template <int DT>
__global__ __launch_bounds__(64) void decode_generic_kernel(pool_view p, meta_view m, uint32_t layer,
                                                            const void* __restrict__ q,
                                                            uint32_t q_heads, float scale_log2,
                                                            void* __restrict__ out,
                                                            float* __restrict__ partials,
                                                            const void* __restrict__ gate)
{
    constexpr int NF = generic_max_features_per_lane;
    const uint32_t H = p.kv_heads;
    const uint32_t D = p.head_dim;
    const uint32_t kv_head = blockIdx.x % H;
    const uint32_t item = blockIdx.x / H;
    const uint32_t row = m.items[2 * item];
    const uint32_t chunk_index = m.items[2 * item + 1];
    const uint32_t position = m.positions[row];
    const uint32_t table_base = m.offsets[row];
    // the row's keys in order, without those its window skips
    const window_gap gap = window_gap_of(window_low(position, m.window), m.window.sinks, 1);
    const uint32_t begin = chunk_index * m.chunk;
    const uint32_t end = min(position + 1 - gap.skip, begin + m.chunk);
    const uint32_t lane = threadIdx.x;
    const uint32_t G = q_heads / H;
    const uint32_t bs = p.block_size;
    const uint64_t slot_count = (uint64_t)p.blocks * bs;
    const bool single = m.row_count[row] == 1;

    for (uint32_t g = 0; g < G; ++g) {
        const uint32_t qh = kv_head * G + g;
        const uint64_t q_base = ((uint64_t)row * q_heads + qh) * D;
        float qf[NF], acc[NF];
#pragma unroll
        for (int k = 0; k < NF; ++k) {
            const uint32_t f = lane + 64 * k;
            qf[k] = f < D ? load_elem<DT>(q, q_base + f) : 0.0f;
            acc[k] = 0.0f;
        }
        // (the lowest finite maximum: a score of -inf weighs 0 also where it comes first)
        float mx = -FLT_MAX, den = 0.0f;
        for (uint32_t i = begin; i < end; ++i) {
            const uint32_t t = i < gap.kept ? i : i + gap.skip;
            const uint64_t slot = (uint64_t)m.table[table_base + t / bs] * bs + t % bs;
            const uint64_t base = ((uint64_t)layer * slot_count + slot) * p.features + kv_head * D;
            float d = 0.0f;
#pragma unroll
            for (int k = 0; k < NF; ++k) {
                const uint32_t f = lane + 64 * k;
                if (f < D)
                    d += qf[k] * load_elem<DT>(p.keys, base + f);
            }
            const float score = wave_sum(d) * scale_log2;
            const float nm = fmaxf(mx, score);
            const float alpha = fast_exp2(mx - nm);
            const float w = fast_exp2(score - nm);
            den = den * alpha + w;
#pragma unroll
            for (int k = 0; k < NF; ++k) {
                const uint32_t f = lane + 64 * k;
                if (f < D)
                    acc[k] = acc[k] * alpha + w * load_elem<DT>(p.values, base + f);
            }
            mx = nm;
        }
        if (single) {
            for (int k = 0; k < NF; ++k) {
                const uint32_t f = lane + 64 * k;
                if (f < D) {
                    float o = acc[k] / den;
                    if (gate)
                        o *= sigmoid(load_elem<DT>(gate, q_base + f));
                    store_elem<DT>(out, q_base + f, o);
                }
            }
        } else {
            float* rec = partials + ((uint64_t)item * q_heads + qh) * record_floats(D);
            for (int k = 0; k < NF; ++k) {
                const uint32_t f = lane + 64 * k;
                if (f < D)
                    rec[4 + f] = acc[k];
            }
            if (lane == 0) {
                rec[0] = mx;
                rec[1] = den;
            }
        }
    }
}

// One wave per (row, q head) of rows with more than one chunk.
template <int DT>
__global__ __launch_bounds__(64) void merge_kernel(meta_view m, uint32_t q_heads, uint32_t D,
                                                   const float* __restrict__ partials,
                                                   void* __restrict__ out,
                                                   const void* __restrict__ gate)
{
    const uint32_t row = blockIdx.x / q_heads;
    const uint32_t qh = blockIdx.x % q_heads;
    const uint32_t n = m.row_count[row];
    if (n <= 1)
        return;
    const uint32_t first = m.row_first[row];
    const uint32_t stride = record_floats(D);
    const float* rec0 = partials + ((uint64_t)first * q_heads + qh) * stride;
    const uint64_t item_stride = (uint64_t)q_heads * stride;
    float M = -INFINITY;
    for (uint32_t c = 0; c < n; ++c)
        M = fmaxf(M, rec0[c * item_stride]);
    float den = 0.0f;
    for (uint32_t c = 0; c < n; ++c)
        den += rec0[c * item_stride + 1] * fast_exp2(rec0[c * item_stride] - M);
    const float inv = 1.0f / den;
    const uint64_t o_base = ((uint64_t)row * q_heads + qh) * D;
    for (uint32_t f = threadIdx.x; f < D; f += 64) {
        float a = 0.0f;
        for (uint32_t c = 0; c < n; ++c)
            a += rec0[c * item_stride + 4 + f] * fast_exp2(rec0[c * item_stride] - M);
        float o = a * inv;
        if (gate)
            o *= sigmoid(load_elem<DT>(gate, o_base + f));
        store_elem<DT>(out, o_base + f, o);
    }
}

bool aligned16(const void* ptr)
{
    return reinterpret_cast<uintptr_t>(ptr) % 16 == 0;
}

// Pages of a row at `position`, and the batch's total and longest.
void batch_pages(const std::vector<uint32_t>& positions, uint32_t block_size, uint64_t& total,
                 uint64_t& longest)
{
    total = longest = 0;
    for (const uint32_t p : positions) {
        const uint64_t pages = p / block_size + 1;
        total += pages;
        longest = std::max(longest, pages);
    }
}

// The balanced plan's segments: the batch's pages, row after row, dealt to
// `n` workgroups. A segment costs split_segment_pages pages of work besides
// its pages (its first loads and its merge wait on memory round trips), so
// the work dealt out (balanced_work) is the pages plus that cost for every
// segment, and workgroup k ends at ceil((k + 1) * work / n) of it. No row is
// cut into a piece shorter than split_min_piece pages (a workgroup takes such
// a rest with it, or ends early and leaves the row to the next one). Calls
// emit(row, first page, end page, workgroup) in row order; returns the
// workgroups used (at most n).
template <class Emit>
uint32_t balanced_segments(const std::vector<uint32_t>& positions, uint32_t block_size,
                           uint64_t work, uint64_t n, Emit&& emit)
{
    auto cut = [&](uint64_t i) { return (work * (i + 1) + n - 1) / n; };
    uint64_t k = 0; // the current workgroup's end, as an index of the cuts
    uint64_t end = cut(0), done = 0;
    uint32_t wg = 0;
    bool empty = true;
    auto next_wg = [&]() {
        ++wg;
        empty = true;
        if (k + 1 < n)
            end = cut(++k);
        while (k + 1 < n && end <= done)
            end = cut(++k);
    };
    for (size_t r = 0; r < positions.size(); ++r) {
        const uint64_t pages = positions[r] / block_size + 1;
        uint64_t pg = 0;
        while (pg < pages) {
            const uint64_t left = pages - pg;
            uint64_t take = left;
            if (k + 1 < n) { // the last workgroup takes what is left
                const uint64_t cost = done + split_segment_pages;
                take = std::min(left, end > cost ? end - cost : 0);
                if (take < left && take < split_min_piece) { // too short a piece to cut off
                    if (!empty) {
                        next_wg();
                        continue;
                    }
                    take = std::min(left, split_min_piece);
                }
                if (left - take < split_min_piece) // nor leave a short rest
                    take = left;
            }
            emit((uint32_t)r, (uint32_t)pg, (uint32_t)(pg + take), wg);
            empty = false;
            pg += take;
            done += take + split_segment_pages;
            if (k + 1 < n && done >= end)
                next_wg();
        }
    }
    return empty ? wg : wg + 1;
}

// The work balanced_segments deals out: the batch's pages plus the segment
// cost of as many segments as dealing that work makes (every row and every
// workgroup has one; found by dealing again until the count holds, at most
// four times), so the last workgroup's share comes out like the others.
uint64_t balanced_work(const std::vector<uint32_t>& positions, uint32_t block_size,
                       uint64_t total, uint64_t n)
{
    uint64_t segments = std::max<uint64_t>(positions.size(), n);
    for (int round = 0; round < 4; ++round) {
        uint64_t count = 0;
        balanced_segments(positions, block_size, total + split_segment_pages * segments, n,
                          [&](uint32_t, uint32_t, uint32_t, uint32_t) { ++count; });
        if (count == segments)
            break;
        segments = count;
    }
    return total + split_segment_pages * segments;
}

// Chunk length, in pages, of a batch too small to deal out page by page, or 0
// when it is better dealt out all the same. The times of three plans are
// weighed in tenths of a page of one workgroup alone on its compute unit (k
// workgroups there share its reads, so a page takes each k times as long; two of
// the f32 form's, too small to read at the full rate, 1.6 times): the shortest
// chunks that make at most k workgroups per compute unit take span * k for each
// k, and the balanced plan its pages and, for each row, the round trips of one
// more segment. Rows whose chunks fit one round of workgroups end together;
// with a few workgroups more than fit, the last round runs nearly alone.
// Measured on MI355X (8 kv heads of 128, us) against chunks of a quarter of a
// compute unit's share: 8 rows of 1,000 tokens 11.7 -> 10.6, 4 of 4,000 19.6 ->
// 16.0, 16 of 1,000 18.6 -> 16.0, 8 of 4,000 29.6 -> 26.0, 24 of U[100, 2500]
// 29.4 -> 26.1; f32 pages: 8 of 2,000 30.0 -> 24.8, 32 of U[64, 1000] 36.5 ->
// 26.5; 256-wide heads, 2 kv heads: 32 of U[256, 4096] 47.8 -> 35.6, 32 of 1,000
// 29.1 -> 19.6.
uint64_t small_batch_span(const std::vector<uint32_t>& positions, uint32_t block_size,
                          uint32_t kv_heads, uint64_t cus, const decode_form& form, uint64_t total,
                          uint64_t longest)
{
    const uint64_t rows = positions.size();
    // a record folded costs about an eighth of a 256-wide page (500 pages of such
    // heads in chunks of 4, 8 and 16: 17.8, 15.9 and 18.2 us)
    const uint64_t shortest = std::max<uint64_t>(
        { form.min_pages, (longest + form.max_chunks - 1) / form.max_chunks,
          (uint64_t)std::sqrt((double)longest / 8) });
    const auto tenths = [&](uint64_t k) { return form.few_waves && k == 2 ? 16 : 10 * k; };
    uint64_t best_span = 0, best = UINT64_MAX;
    uint64_t slots = 1;
    for (uint64_t k = 1; k <= form.per_cu; ++k) {
        slots = std::max<uint64_t>(1, cus * k / kv_heads);
        if (rows > slots)
            continue;
        // the shortest span of at most `slots` chunks (longest makes one per row)
        uint64_t lo = std::min(shortest, longest), hi = longest;
        while (lo < hi) {
            const uint64_t mid = (lo + hi) / 2;
            uint64_t chunks = 0;
            for (const uint32_t p : positions)
                chunks += (p / block_size + mid) / mid;
            if (chunks <= slots)
                hi = mid;
            else
                lo = mid + 1;
        }
        if (hi * tenths(k) < best) {
            best = hi * tenths(k);
            best_span = hi;
        }
    }
    // Work the balanced plan gives a compute unit, and the line below which it is
    // taken. Measured at dealt over best, dealt against chunks, us: 16-bit 0.84 (30
    // rows of U[100, 2000] tokens) 26.3 and 27.6, 0.92 (14 of U[100, 4000]) 24.3 and 25.2,
    // 0.95 (8 of U[3000, 4100]) 23.6 and 25.0, 0.96 (12 of U[500, 3000]) 19.0 and 19.8, 1.06 (16
    // of 1,000) 17.0 and 15.4; f32 0.87 (24 of U[100, 2500]) 43.9 and 45.8, 0.92 (14 of
    // U[100, 4000]) 40.4 and 41.7, 0.93 (16 of U[200, 2000]) 28.5 and 26.7, 0.94 (20 of U[1000,
    // 1300]) 36.1 and 34.0.
    const uint64_t work = tenths(form.per_cu) * (total + split_row_pages / form.per_cu * rows);
    const uint64_t dealt = (work + slots - 1) / slots, line = form.few_waves ? 92 : 97;
    if (total >= slots * form.min_pages && rows <= slots && 100 * dealt < line * best)
        return 0;
    return best_span;
}

// Whether whole rows, started longest first on the compute unit that is free
// first, leave none with more than num/den of its share of the pages. Measured on
// MI355X (16-bit pages, 8 kv heads, 65 to 112 rows) against chunks of a quarter
// of the share: at 1.10 to 1.15 times the share whole rows are 1 to 4 % faster
// (96 rows of U[100, 3000] tokens 100.2 and 103.5 us, 80 rows 86.5 and 87.9), near 1.2 the
// two tie (74 rows of U[784, 2096] 81.7 and 81.9), and past it chunks are: 72 rows
// of U[1000, 2500] (1.22) 89.4 and 93.0, 70 of U[2290, 2983] (1.33) 133 and 140, 73 of
// U[160, 216] (1.29) 17.6 and 18.3. f32 rows of one or two units per compute unit,
// against their cut plan: up to 1.17 whole rows are 2 to 13 % faster (64 rows of
// U[764, 1286], 1.01: 88.8 and 98.6; but 64 of U[245, 1833], 1.00, 95.6 and 87.0), between
// 1.2 and 1.25 they gain 20 % or lose 3 to 5 % (42 of U[276, 623] 32.0 and 39.8, 49
// of U[741, 1239] 70.1 and 66.6), past that they mostly lose (38 of U[1008, 1153], 1.61,
// 62.3 and 56.3).
bool whole_rows_even(const std::vector<uint32_t>& positions, uint32_t block_size, uint32_t kv_heads,
                     uint64_t cus, uint64_t total, uint64_t num, uint64_t den)
{
    std::vector<uint64_t> pages(positions.size());
    std::transform(positions.begin(), positions.end(), pages.begin(),
                   [&](uint32_t p) { return (uint64_t)p / block_size + 1; });
    std::sort(pages.begin(), pages.end(), std::greater<> {});
    // a row takes kv_heads compute units at once: least-loaded first of the sets
    const uint64_t sets = std::max<uint64_t>(1, cus / kv_heads);
    std::vector<uint64_t> load(sets, 0); // a min-heap
    for (const uint64_t n : pages) {
        std::pop_heap(load.begin(), load.end(), std::greater<> {});
        load.back() += n;
        std::push_heap(load.begin(), load.end(), std::greater<> {});
    }
    return den * sets * *std::max_element(load.begin(), load.end()) <= num * total;
}

uint64_t forced_pages(const char* name, bool& set)
{
    const char* v = std::getenv(name);
    set = v != nullptr;
    return v ? (uint64_t)std::max(0L, std::strtol(v, nullptr, 10)) : 0;
}

} // namespace

uint32_t decode_fast_waves(uint32_t group, int dtype, uint32_t units, int cu_count,
                           uint32_t mean_pages, uint32_t split_pages)
{
    return fast_waves(group, dtype, units, cu_count, mean_pages, split_pages);
}

decode_form decode_form_of(int dtype, uint32_t head_dim)
{
    if (dtype == CKV_F32)
        return form_f32;
    return head_dim == 256 ? form_wide : form_narrow;
}

decode_plan_shape shape_decode_plan(const std::vector<uint32_t>& positions, uint32_t block_size,
                                    uint32_t kv_heads, int cu_count, const decode_form& form,
                                    uint64_t chunk)
{
    const uint32_t rows = (uint32_t)positions.size();
    decode_plan_shape shape { 0, rows, 0, 0, rows, 0, 0, false };
    uint64_t total, longest;
    batch_pages(positions, block_size, total, longest);
    bool fixed_set, balanced_set;
    uint64_t span = forced_pages("CKV_DECODE_SPLIT", fixed_set);
    const uint64_t target = forced_pages("CKV_DECODE_BALANCE", balanced_set);
    if (chunk && !fixed_set && !balanced_set) {
        span = chunk;
        fixed_set = true;
    }
    uint64_t deal = 0; // workgroups per kv head the balanced plan deals the pages to
    if (balanced_set) {
        deal = target ? (total + target - 1) / target : 0;
    } else if (!fixed_set) {
        // a compute unit's share of the batch, in (page, kv head) units
        const uint64_t cus = (uint64_t)std::max(cu_count, 1);
        const uint64_t share = total * kv_heads / cus;
        // Rows stay whole when they give every compute unit one or two (row,
        // kv head) units and the longest is within the form's slack of the
        // share: a cut costs its merge and second segment, and the cut plan's
        // pages run about 12 % slower than a whole row's. With more units per
        // compute unit the fixed chunks balance better (the config-5 churn's
        // batches of hundreds of rows: 1.5 % faster cut), unless whole rows,
        // which start longest first, even out.
        const uint64_t units = (uint64_t)rows * kv_heads;
        const auto whole = [&]() {
            const auto even = [&](uint64_t num, uint64_t den) {
                return whole_rows_even(positions, block_size, kv_heads, cus, total, num, den);
            };
            if (units > 2 * cus)
                return 5 * longest <= 4 * share && even(6, 5);
            if (units < cus)
                return false;
            return form.few_waves
                ? longest <= share + share / 8 && even(5, 4)
                : longest <= share + std::min(share / 8 + form.uncut_slack, 5 * share / 8);
        };
        if (2 * longest > share && !whole()) {
            // as many workgroups as the GPU holds at once, but no more than a
            // row each where rows are short (pieces of at least
            // form.min_pages), nor more than max_chunks to a row
            const uint64_t slots = std::max<uint64_t>(1, cus * form.per_cu / kv_heads);
            const uint64_t piece = std::max<uint64_t>(
                form.min_pages, (longest + form.max_chunks - 1) / form.max_chunks);
            deal = std::max<uint64_t>(1, std::min(slots, std::max<uint64_t>(rows, total / piece)));
            if (rows > deal) {
                // More rows than workgroups (the balanced plan would run several
                // whole rows one after another in a workgroup, each paying its
                // round trips): fixed chunks instead, a quarter of a compute
                // unit's share, dispatched longest first.
                deal = 0;
                span = std::max({ (uint64_t)form.min_pages,
                                  (share + split_per_share - 1) / split_per_share,
                                  (longest + form.max_chunks - 1) / form.max_chunks });
                fixed_set = true;
            } else if (form.per_cu == 1 || total < deal * split_balance_min_pages) {
                span = small_batch_span(positions, block_size, kv_heads, cus, form, total, longest);
                if (span) {
                    deal = 0;
                    fixed_set = true;
                }
            }
        }
    }
    uint64_t items = 0, records = 0, cut = 0, wgs = 0, per_wg = 0;
    if (deal) {
        uint32_t run_row = UINT32_MAX;
        uint64_t run = 0;
        auto close_run = [&]() {
            records += run > 1 ? run : 0;
            cut += run > 1 ? 1 : 0;
        };
        shape.deal_work = balanced_work(positions, block_size, total, deal);
        wgs = balanced_segments(positions, block_size, shape.deal_work, deal,
                                [&](uint32_t r, uint32_t, uint32_t, uint32_t) {
                                    ++items;
                                    if (r != run_row) {
                                        close_run();
                                        run_row = r;
                                        run = 0;
                                    }
                                    ++run;
                                });
        close_run();
        shape.balanced = true;
        per_wg = balanced_set ? target : (total + deal - 1) / deal;
    } else if (fixed_set && span && span < longest) {
        for (const uint32_t p : positions) {
            const uint64_t n = (p / block_size + span) / span; // chunks of (p / bs + 1) pages
            items += n;
            records += n > 1 ? n : 0;
            cut += n > 1 ? 1 : 0;
        }
        wgs = items;
        per_wg = span;
    } else {
        return shape; // a row per workgroup
    }
    if (items > UINT32_MAX / plan_entry_words || wgs > UINT32_MAX / kv_heads
        || records > UINT32_MAX / kv_heads)
        return decode_plan_shape { 0, rows, 0, 0, rows, 0, 0, false };
    shape.split_pages = (uint32_t)per_wg;
    shape.n_deal = (uint32_t)deal;
    shape.n_items = (uint32_t)items;
    shape.n_records = (uint32_t)records;
    shape.n_cut = (uint32_t)cut;
    shape.n_wgs = (uint32_t)wgs;
    return shape;
}

// Rows behind a window are mostly equally long. With one to one and a half (row, kv
// head) units per compute unit, some hold two whole rows and most one; halves, four
// waves each (decode_wg.h), even them out. Measured on MI355X (8 kv heads, 2 q heads
// per kv head, bf16, us, whole rows at 8 waves and halves at 4): 34 rows behind a window
// of 4,096 tokens 130 and 107, of 2,048 67.7 and 58.4, of 1,024 36.6 and 32.7, of 512
// 21.0 and 19.9, of 256 12.3 and 13.0; 48 rows behind 2,048 75.0 and 69.7, behind 512
// 24.0 and 24.0; 52 rows behind 2,048 78.9 and 83.0. 256-wide heads hold one workgroup
// to a compute unit: 40 rows of 8 kv heads, 4 q heads each, behind 1,024 tokens 91 and
// 65, behind 256 30.7 and 24.5; 160 of 2 kv heads, 2 each, 67.7 and 61.1, 21.8 and 22.4.
constexpr uint64_t window_half_pages = 33, window_half_pages_wide = 17;

// Small batches of 128-wide 16-bit rows are cut into pieces of an eighth of the longest
// row, 4 to 12 pages, where all others are of at least 12: us at 12 and now (8 kv heads,
// bf16), 4 rows behind 512 tokens 7.0 and 6.4, 1 behind 256 6.8 and 6.0, 8 behind 256 6.6
// and 6.1. Where the longest row has up to 16 pages, pieces stay at 12 or more (16 rows
// behind 128, whole 6.1 and in halves 6.5).
constexpr uint64_t window_long_pages = 16;

decode_form window_form_of(int dtype, uint32_t head_dim)
{
    decode_form form = decode_form_of(dtype, head_dim);
    // f32 rows behind a window are few pages: pieces of 4 rather than 8 fill more of the
    // GPU where they have room (3 rows behind 300 tokens: 128-wide heads 6.6 and 6.0 us,
    // 256-wide 12.7 and 9.4; 12 behind 600: 256-wide 15.4 and 11.7)
    if (dtype == CKV_F32)
        form.min_pages = std::min(form.min_pages, 4u);
    return form;
}

decode_plan_shape shape_window_plan(const std::vector<uint32_t>& positions, uint32_t block_size,
                                    uint32_t kv_heads, int cu_count, decode_form form)
{
    uint64_t total, longest;
    batch_pages(positions, block_size, total, longest);
    if (form.min_pages == form_narrow.min_pages && longest > window_long_pages)
        form.min_pages = (uint32_t)std::clamp<uint64_t>(longest / 8, 4, form_narrow.min_pages);
    const uint64_t rows = positions.size(), cus = (uint64_t)std::max(cu_count, 1);
    const bool even = 8 * total >= 7 * longest * rows;
    const uint64_t least = form.per_cu == 1 ? window_half_pages_wide : window_half_pages;
    const bool halves = !form.few_waves && even && longest >= least
        && rows * kv_heads > cus && 2 * rows * kv_heads <= 3 * cus;
    return shape_decode_plan(positions, block_size, kv_heads, cu_count, form,
                             halves ? (longest + 1) / 2 : 0);
}

void write_decode_plan(const std::vector<uint32_t>& positions,
                       const std::vector<uint32_t>& offsets, uint32_t block_size,
                       const decode_plan_shape& shape, std::vector<uint64_t>& sort_keys,
                       uint32_t* plan, uint32_t* split_first, uint32_t* cut)
{
    const size_t rows = positions.size();
    const uint32_t span = shape.split_pages;
    auto entry = [&](size_t at, uint32_t r, uint32_t chunk, uint32_t first, uint32_t end,
                     uint32_t n_chunks, uint32_t next) {
        uint32_t* e = plan + plan_entry_words * at;
        e[0] = r;
        e[1] = chunk;
        e[2] = positions[r];
        e[3] = offsets[r] + first;
        e[4] = first;
        e[5] = end;
        e[6] = n_chunks;
        e[7] = next;
    };
    auto pages_of = [&](size_t r) { return positions[r] / block_size + 1; };
    if (!span) {
        // rows by decreasing position (ties in row order): the longest first
        sort_keys.resize(rows);
        for (size_t r = 0; r < rows; ++r)
            sort_keys[r] = ((uint64_t)(UINT32_MAX - positions[r]) << 32) | r;
        std::sort(sort_keys.begin(), sort_keys.end());
        for (size_t r = 0; r < rows; ++r) {
            const uint32_t row = (uint32_t)sort_keys[r];
            entry(r, row, 0, 0, pages_of(row), 1, plan_last);
            split_first[r] = 0;
        }
        return;
    }
    if (shape.balanced) {
        // the segments in row order, two words each: (row, first), (end, workgroup)
        sort_keys.clear();
        balanced_segments(positions, block_size, shape.deal_work, shape.n_deal,
                          [&](uint32_t r, uint32_t first, uint32_t end, uint32_t wg) {
                              sort_keys.push_back(((uint64_t)r << 32) | first);
                              sort_keys.push_back(((uint64_t)end << 32) | wg);
                          });
        // Dealt workgroup w runs as plan workgroup slot_of[w]: its first
        // segment is entry slot_of[w], its others follow the first segments in
        // order, each entry linking to the next.
        const size_t n = sort_keys.size() / 2;
        auto row_at = [&](size_t i) { return (uint32_t)(sort_keys[2 * i] >> 32); };
        auto wg_at = [&](size_t i) { return (uint32_t)sort_keys[2 * i + 1]; };
        // Workgroups with more segments take the lower slots: workgroups start
        // in slot order, one per compute unit before a second, and the second
        // to start on a compute unit loses issue to the first, so a workgroup
        // paying an extra segment's round trips should not also be the younger
        // (bit-identical; 32 rows of U[384, 3072] tokens 6 % faster, U[256,
        // 2560] 4 %, config 2 0.3 %).
        std::vector<uint32_t> segs(shape.n_wgs, 0), slot_of(shape.n_wgs);
        for (size_t i = 0; i < n; ++i)
            ++segs[wg_at(i)];
        {
            std::vector<uint32_t> order(shape.n_wgs);
            for (uint32_t w = 0; w < shape.n_wgs; ++w)
                order[w] = w;
            std::stable_sort(order.begin(), order.end(),
                             [&](uint32_t a, uint32_t b) { return segs[a] > segs[b]; });
            for (uint32_t k = 0; k < shape.n_wgs; ++k)
                slot_of[order[k]] = k;
        }
        std::fill(split_first, split_first + rows, 0u);
        size_t more = shape.n_wgs, n_cut = 0;
        uint32_t record = 0, run = 0, chunk = 0;
        for (size_t i = 0; i < n; ++i) {
            const uint32_t r = row_at(i), wg = wg_at(i);
            if (i == 0 || r != row_at(i - 1)) { // a row's first segment: count its segments
                run = 1;
                while (i + run < n && row_at(i + run) == r)
                    ++run;
                chunk = 0;
                if (run > 1) {
                    split_first[r] = record;
                    record += run;
                    cut[n_cut++] = r;
                }
            }
            const size_t at = i == 0 || wg != wg_at(i - 1) ? slot_of[wg] : more++;
            const uint32_t next = i + 1 < n && wg_at(i + 1) == wg ? (uint32_t)more : plan_last;
            const uint32_t first = (uint32_t)sort_keys[2 * i];
            const uint32_t end = (uint32_t)(sort_keys[2 * i + 1] >> 32);
            entry(at, r, chunk++, first, end, run, next);
        }
        return;
    }
    // fixed chunks by decreasing page count: the full chunks of every row (row
    // after row), then the short last chunks, longest first
    uint32_t record = 0;
    size_t at = 0, n_cut = 0;
    auto chunk_entry = [&](size_t at, uint32_t r, uint32_t c) {
        const uint32_t pages = pages_of(r);
        entry(at, r, c, c * span, std::min(c * span + span, pages), (pages + span - 1) / span,
              plan_last);
    };
    sort_keys.clear();
    for (size_t r = 0; r < rows; ++r) {
        const uint32_t pages = pages_of(r);
        const uint32_t n = (pages + span - 1) / span, full = pages / span;
        split_first[r] = n > 1 ? record : 0;
        record += n > 1 ? n : 0;
        if (n > 1)
            cut[n_cut++] = (uint32_t)r;
        for (uint32_t c = 0; c < full; ++c, ++at)
            chunk_entry(at, (uint32_t)r, c);
        if (full < n)
            sort_keys.push_back(((uint64_t)(span - (pages - full * span)) << 32) | r);
    }
    std::sort(sort_keys.begin(), sort_keys.end());
    for (const uint64_t key : sort_keys) {
        const uint32_t r = (uint32_t)key;
        chunk_entry(at++, r, pages_of(r) / span); // the last chunk
    }
}

bool decode_uses_fast_path(const pool_view& p, uint32_t q_heads)
{
    const uint32_t G = q_heads / p.kv_heads;
    // f32 at G = 8 runs as two passes of G = 4 (launch_fast<8>)
    return (p.head_dim == 128 || p.head_dim == 256) && p.block_size == 16
        && (G == 1 || G == 2 || G == 4 || G == 8)
        && (fast_fits(G, p.dtype) || (G == 8 && p.dtype == CKV_F32)) && aligned16(p.keys)
        && aligned16(p.values);
}

bool decode_fast_applies(const pool_view& p, uint32_t q_heads, const void* q, const void* out)
{
    return decode_uses_fast_path(p, q_heads) && aligned16(q) && aligned16(out);
}

hipError_t launch_decode(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                         const void* q, uint32_t q_heads, float scale, void* out,
                         float* partials, int cu_count, const void* gate, split_scratch split)
{
    if (!m.rows)
        return hipSuccess;
    const float scale_log2 = scale * log2e;
    if (decode_fast_applies(p, q_heads, q, out)) {
        const void* no_row = nullptr;
        if (m.window.window != all_keys.window)
            return launch_window_fast(s, p, m, layer, q, q_heads, scale_log2, out, no_row, no_row,
                                      gate, cu_count, split, nullptr, 0);
        return launch_width<false>(p.head_dim, q_heads / p.kv_heads, s, p, m, layer, q, q_heads,
                            scale_log2, out, p.dtype, no_row, no_row, gate, cu_count, split);
    }
    if (p.head_dim > 64u * generic_max_features_per_lane)
        return hipErrorInvalidValue;
    const dim3 grid(m.n_items * p.kv_heads), block(64);
    switch (p.dtype) {
    case CKV_F32:
        decode_generic_kernel<CKV_F32><<<grid, block, 0, s>>>(p, m, layer, q, q_heads, scale_log2,
                                                              out, partials, gate);
        break;
    case CKV_BF16:
        decode_generic_kernel<CKV_BF16><<<grid, block, 0, s>>>(p, m, layer, q, q_heads,
                                                               scale_log2, out, partials, gate);
        break;
    default:
        decode_generic_kernel<CKV_F16><<<grid, block, 0, s>>>(p, m, layer, q, q_heads, scale_log2,
                                                              out, partials, gate);
        break;
    }
    return hipGetLastError();
}

hipError_t launch_append_decode(hipStream_t s, const pool_view& p, const meta_view& m,
                                uint32_t layer, const void* k_in, const void* v_in, const void* q,
                                uint32_t q_heads, float scale, void* out, const void* gate,
                                int cu_count, split_scratch split, const rope_table* rope,
                                uint32_t rotary)
{
    if (!m.rows)
        return hipSuccess;
    if (rope && (rotary < 16 || rotary > p.head_dim || (rotary & (rotary - 1)) != 0))
        return hipErrorInvalidValue;
    const float scale_log2 = scale * log2e;
    if (m.window.window != all_keys.window)
        return launch_window_fast(s, p, m, layer, q, q_heads, scale_log2, out, k_in, v_in, gate,
                                  cu_count, split, rope, rotary);
    return launch_width<false>(p.head_dim, q_heads / p.kv_heads, s, p, m, layer, q, q_heads, scale_log2,
                        out, p.dtype, k_in, v_in, gate, cu_count, split, rope, rotary);
}

hipError_t launch_merge(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t q_heads,
                        void* out, const float* partials, const void* gate)
{
    const dim3 grid(m.rows * q_heads), block(64);
    switch (p.dtype) {
    case CKV_F32:
        merge_kernel<CKV_F32><<<grid, block, 0, s>>>(m, q_heads, p.head_dim, partials, out, gate);
        break;
    case CKV_BF16:
        merge_kernel<CKV_BF16><<<grid, block, 0, s>>>(m, q_heads, p.head_dim, partials, out, gate);
        break;
    default:
        merge_kernel<CKV_F16><<<grid, block, 0, s>>>(m, q_heads, p.head_dim, partials, out, gate);
        break;
    }
    return hipGetLastError();
}

void place_window_plan(const std::vector<uint32_t>& positions, const decode_plan_shape& shape,
                       uint32_t* plan)
{
    for (size_t i = 0; i < shape.n_items; ++i)
        plan[plan_entry_words * i + 2] = positions[plan[plan_entry_words * i]];
}

uint32_t partial_record_floats(uint32_t head_dim)
{
    return record_floats(head_dim);
}

} // namespace ckv
