// Chunked-prefill causal attention over f32 pages on the matrix cores (gfx950).
//
// The maths of paged_flash_attention_prefill_f32
// (src/metal/kernels/attention.metal:246-444) in f32 throughout, as the
// reference computes it: q.k, the softmax and P.V in fp32, the products on
// v_mfma_f32_32x32x2_f32 (exact fp32 products, fp32 accumulation).
//
// Decomposition as for 16-bit pools: one workgroup of eight waves owns
// (256/G rows of a query tile, one kv head) and all G query heads of the
// head's GQA group; wave w holds the q-block (head w % G, rows 32*(w/G)..+31).
// Per 32-key block (two pages) and wave:
//   S^T[key][query] = K . Q^T   64 products of 2 features: A = K from LDS
//                                (lane (m, h) gives features 64h + j of key m),
//                                B = Q^T held in registers (lane (n, h):
//                                features 64h + j of query n), in two
//                                independent accumulator chains.
//   softmax                     lane (n, h) holds query n's scores of keys
//                                8*(r/4) + 4h + r%4 (its accumulator element
//                                r); the lane 32 apart holds the other 16.
//   O^T[feature][query] += V^T . P^T   step i takes key 8*(i/4) + 4h + i%4 in
//                                lane half h, so the B operand is the lane's
//                                own probability i; the A operand of
//                                accumulator c (0..3) is V[key][4m + c], so one
//                                16-byte LDS read feeds four products and row m
//                                of accumulator c is feature 4m + c.
// A product takes 64 cycles, so a block's 128 per wave (8,192 cycles) bound
// the kernel: the softmax's vector work and the LDS reads (32 KiB per wave and
// block) hide behind them.
//
// Staging: each block's K and V rows pass through registers into LDS (two
// stages; rows padded to 528 bytes, so the 32 key rows one K read touches
// start 16 bytes apart in the banks), the next block's loads in flight while
// the current one is multiplied, one barrier per block. Keys past the tile's
// last position are staged as zeros and never read from the pool.
//
// A launch that leaves compute units idle splits each long tile's key blocks
// between up to 8 workgroups, as the 16-bit kernel does (kernels_prefill.hip):
// each stores its unnormalised state as 16-byte records, and the last to
// arrive folds them in range order.
#include <algorithm>
#include <type_traits>

#include "attend_alone.h"
#include "ckv_internal.h"
#include "prefill_records.h"
#include "store_rows.h"

namespace ckv {
namespace {

constexpr uint32_t dim = 128;
constexpr uint32_t page_tokens = 16;
constexpr uint32_t block_keys = 32;
constexpr uint32_t row_pitch = dim * 4 + 16;              // bytes per staged key row
constexpr uint32_t tensor_bytes = block_keys * row_pitch; // one block of K (or V)
constexpr uint32_t stage_bytes = 2 * tensor_bytes;        // K, then V
constexpr uint32_t n_stages = 2;

__device__ __forceinline__ f32x16_t mfma(float a, float b, const f32x16_t& c)
{
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

// WINDOW (4 waves): rows attend through md.window, as in kernels_prefill.hip. A window's
// tiles are short chains of dear blocks: workgroups of half the rows have half the chain
// to a block and two share a compute unit (2 chunks of 220 and 300 rows behind 1,000
// tokens, window 512: 65 us with 8 waves, 45 with 4).
// RANGES: the launch may cut a tile's keys; a window's launch that does not stores its
// results as whole rows (store_rows.h).
template <int G, bool WINDOW, bool RANGES = true, int waves = WINDOW ? 4 : 8>
__global__ __launch_bounds__(64 * waves, 2) void prefill_f32_kernel(
    pool_view p, meta_view md, uint32_t layer, const float* __restrict__ q,
    float* __restrict__ out, uint32_t q_heads, float c, const float* __restrict__ gate,
    prefill_split split_scratch)
{
    __shared__ __attribute__((aligned(16))) uint8_t lds[n_stages * stage_bytes];
    static_assert(waves == 8 || G <= 4, "a workgroup covers every q head of its group, or 4 of 8");
    constexpr uint32_t tile_rows = 32 * waves / G;

    const uint32_t kv_heads = p.kv_heads;
    const uint32_t kvh = blockIdx.x % kv_heads;
    const uint32_t group = WINDOW ? q_heads / kv_heads : G;
    const uint32_t passes = WINDOW ? group / G : 1; // workgroups a GQA group takes
    const uint32_t pass = WINDOW ? blockIdx.x / kv_heads % passes : 0;
    const uint32_t of_pass = blockIdx.x / (kv_heads * passes);
    // key ranges vary slowest: every tile's first range is dispatched first
    const uint32_t n_split = split_scratch.n_split;
    constexpr uint32_t subs = WINDOW ? 1 : G; // a window's tiles are of a workgroup's rows
    const uint32_t n_rest = md.n_tiles * subs;
    const uint32_t rest = of_pass % n_rest;
    const uint32_t part = of_pass / n_rest; // this workgroup's range of the keys
    const uint32_t sub = rest % subs;
    const uint32_t tile = rest / subs;
    // the tile: first row, rows, first position, table offset
    const uint4 te = *reinterpret_cast<const uint4*>(md.tiles + tile_entry_words * tile);
    const uint32_t count = te.y;
    const uint32_t r0 = sub * tile_rows;
    if (r0 >= count)
        return;
    const uint32_t nrows = min(tile_rows, count - r0);
    const uint32_t row0 = te.x + r0;
    const uint32_t pos0 = te.z + r0; // positions are consecutive inside a tile
    const uint32_t pos_last = pos0 + nrows - 1;
    const uint32_t* table = md.table + te.w;
    // the first row's window begins at `low`, no later row's before it
    const key_window window = md.window;
    const uint32_t low = WINDOW ? window_low(pos0, window) : 0;
    const window_gap gap = WINDOW ? window_gap_of(low, window.sinks, block_keys) : window_gap {};
    auto in_table = [&](uint32_t kb) { return WINDOW && kb >= gap.kept ? kb + gap.skip : kb; };
    auto some_row_attends = [&](uint32_t key) {
        return key <= pos_last && (!WINDOW || key >= low || key < window.sinks);
    };
    const uint32_t n_blocks = pos_last / block_keys + 1 - gap.skip;
    const uint32_t last_entry = pos_last / page_tokens;
    // key blocks [kb_begin, kb_end) of this workgroup
    const uint32_t n_parts =
        RANGES ? prefill_range_count(n_blocks, n_split, split_scratch.min_blocks) : 1;
    if (part >= n_parts)
        return;
    uint32_t kb_begin, kb_end;
    prefill_range_bounds(n_blocks, n_parts, part, kb_begin, kb_end);

    const uint32_t tid = threadIdx.x;
    const uint32_t lane = tid & 63, wave = tid >> 6;
    const uint32_t n = lane & 31, h = lane >> 5;
    const uint64_t q_stride = (uint64_t)q_heads * dim;

    // this wave's q-block: head kvh * G + wave % G, tile rows 32 * (wave / G) + n
    const uint32_t head = kvh * group + pass * G + wave % G;
    const uint32_t row = (wave / G) * 32 + n;
    const bool valid = row < nrows;
    const uint32_t qpos = pos0 + min(row, nrows - 1);
    const uint64_t qoff = (uint64_t)(row0 + min(row, nrows - 1)) * q_stride + (uint64_t)head * dim;
    // the q-block's first position, wave-uniform: blocks ending before it need
    // no mask (a scalar branch; 1.2 % faster on config 4)
    const uint32_t pos_lo = __builtin_amdgcn_readfirstlane(pos0 + (wave / G) * 32);

    // Q^T operands: features 64h .. 64h + 63 of query n
    float qr[64];
#pragma unroll
    for (int t = 0; t < 16; ++t) {
        const float4 v = valid ? *reinterpret_cast<const float4*>(q + qoff + 64 * h + 4 * t)
                               : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        qr[4 * t] = v.x;
        qr[4 * t + 1] = v.y;
        qr[4 * t + 2] = v.z;
        qr[4 * t + 3] = v.w;
    }

    // Staging: thread t moves 16 bytes of key rows t/32, t/32 + 2 waves, ... of each page
    // of the block, of K and of V.
    const uint64_t page_bytes = (uint64_t)page_tokens * p.features * 4;
    const uint64_t layer_bytes = p.layer_elems * 4;
    const uint8_t* kbase = static_cast<const uint8_t*>(p.keys) + layer * layer_bytes + kvh * dim * 4;
    const uint8_t* vbase = static_cast<const uint8_t*>(p.values) + layer * layer_bytes + kvh * dim * 4;
    constexpr uint32_t step = 2 * waves, each = page_tokens / step; // rows of a page a thread moves
    const uint32_t sr = tid >> 5;
    const uint32_t scol = (tid & 31) * 16;
    const uint64_t srow = (uint64_t)sr * p.features * 4 + scol;
    const uint64_t srow_step = (uint64_t)step * p.features * 4;
    // the staged 16 bytes of each page's K and V rows
    uint4 k_a[each], k_b[each], v_a[each], v_b[each];
    auto fetch = [&](uint32_t kb) __attribute__((always_inline)) {
        const uint32_t key0 = in_table(kb) * block_keys;
        const uint64_t pa = table[2 * in_table(kb)];
        const uint64_t pb = table[min(2 * in_table(kb) + 1, last_entry)];
#pragma unroll
        for (uint32_t i = 0; i < each; ++i) {
            const uint64_t at = srow + i * srow_step;
            k_a[i] = k_b[i] = v_a[i] = v_b[i] = make_uint4(0, 0, 0, 0);
            if (some_row_attends(key0 + sr + i * step)) {
                k_a[i] = *reinterpret_cast<const uint4*>(kbase + pa * page_bytes + at);
                v_a[i] = *reinterpret_cast<const uint4*>(vbase + pa * page_bytes + at);
            }
            if (some_row_attends(key0 + 16 + sr + i * step)) {
                k_b[i] = *reinterpret_cast<const uint4*>(kbase + pb * page_bytes + at);
                v_b[i] = *reinterpret_cast<const uint4*>(vbase + pb * page_bytes + at);
            }
        }
    };
    auto store = [&](uint32_t kb) __attribute__((always_inline)) {
        uint8_t* st = lds + (kb % n_stages) * stage_bytes + sr * row_pitch + scol;
#pragma unroll
        for (uint32_t i = 0; i < each; ++i, st += step * row_pitch) {
            *reinterpret_cast<uint4*>(st) = k_a[i];
            *reinterpret_cast<uint4*>(st + 16 * row_pitch) = k_b[i];
            *reinterpret_cast<uint4*>(st + tensor_bytes) = v_a[i];
            *reinterpret_cast<uint4*>(st + tensor_bytes + 16 * row_pitch) = v_b[i];
        }
    };

    f32x16_t o[4];
#pragma unroll
    for (int a = 0; a < 4; ++a)
        o[a] = f32x16_t {};
    float m = -__builtin_inff(), l = 0.0f; // running maximum (log2 units), denominator share

    const uint32_t q_low = WINDOW ? window_low(qpos, window) : 0;
    const uint32_t low_hi = WINDOW
        ? __builtin_amdgcn_readfirstlane(
              window_low(pos0 + min((wave / G) * 32 + 31, nrows - 1), window))
        : 0;
    // Whether some row of the wave attends a key of the block (uniform over the wave). A
    // block costs a wave 3.4 us, so those of the tile's other rows are left to them.
    const uint32_t pos_hi = __builtin_amdgcn_readfirstlane(
        pos0 + min((wave / G) * 32 + 31, nrows - 1));
    const uint32_t low_lo = WINDOW ? window_low(pos_lo, window) : 0;
    auto needed = [&](uint32_t kb) {
        const uint32_t key0 = in_table(kb) * block_keys;
        return pos_lo <= pos_hi && key0 <= pos_hi
            && (key0 + block_keys - 1 >= low_lo || key0 < window.sinks);
    };
    auto attend = [&](uint32_t kb) __attribute__((always_inline)) {
        const uint8_t* st = lds + (kb % n_stages) * stage_bytes;
        // S^T = K . Q^T
        const uint8_t* kr = st + n * row_pitch + h * 256;
        f32x16_t s0 = {}, s1 = {};
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            const float4 kv = *reinterpret_cast<const float4*>(kr + 16 * t);
            s0 = mfma(kv.x, qr[4 * t], s0);
            s1 = mfma(kv.y, qr[4 * t + 1], s1);
            s0 = mfma(kv.z, qr[4 * t + 2], s0);
            s1 = mfma(kv.w, qr[4 * t + 3], s1);
        }
        // causal mask, scores in log2 units, the block maximum of the query
        const uint32_t key0 = in_table(kb) * block_keys;
        float s[16];
        float mx = -__builtin_inff();
        if (WINDOW && key0 < low_hi && key0 + block_keys - 1 >= window.sinks) {
            // some row's window begins past the block's first key, and not all of it are sinks
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const uint32_t key = key0 + 8 * (r >> 2) + 4 * h + (r & 3);
                s[r] = key <= qpos && (key >= q_low || key < window.sinks) ? (s0[r] + s1[r]) * c
                                                                           : -__builtin_inff();
                mx = fmaxf(mx, s[r]);
            }
        } else if (key0 + block_keys - 1 <= pos_lo) { // every key precedes every query
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = (s0[r] + s1[r]) * c;
                mx = fmaxf(mx, s[r]);
            }
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const uint32_t key = key0 + 8 * (r >> 2) + 4 * h + (r & 3);
                s[r] = key <= qpos ? (s0[r] + s1[r]) * c : -__builtin_inff();
                mx = fmaxf(mx, s[r]);
            }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        if (__any(mx > m)) {
            const float m_new = fmaxf(m, mx);
            const float alpha = m_new == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
            l *= alpha;
#pragma unroll
            for (int a = 0; a < 4; ++a)
                o[a] *= alpha;
            m = m_new;
        }
        // a range of the keys may hold none a query attends yet (m = -inf)
        const float mm = m == -__builtin_inff() ? 0.0f : m;
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = __builtin_amdgcn_exp2f(s[r] - mm);
            sum += s[r];
        }
        l += sum;
        // O^T += V^T . P^T
        const uint8_t* vr = st + tensor_bytes + 16 * n;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t key = 8 * (i >> 2) + 4 * h + (i & 3);
            const float4 vv = *reinterpret_cast<const float4*>(vr + key * row_pitch);
            o[0] = mfma(vv.x, s[i], o[0]);
            o[1] = mfma(vv.y, s[i], o[1]);
            o[2] = mfma(vv.z, s[i], o[2]);
            o[3] = mfma(vv.w, s[i], o[3]);
        }
    };

    fetch(kb_begin);
    store(kb_begin);
    __syncthreads();
    for (uint32_t kb = kb_begin; kb < kb_end; ++kb) {
        const bool more = kb + 1 < kb_end; // workgroup-uniform
        if (more)
            fetch(kb + 1);
        if (!WINDOW || needed(kb))
            attend(kb);
        if (more)
            store(kb + 1); // stage (kb + 1) % 2 was last read in iteration kb - 1
        __syncthreads();
    }

    float lt = l + __shfl_xor(l, 32); // the query's denominator (both lane halves)
    if (RANGES && n_parts > 1) {
        // A range of a split tile: its record is 33 chunks of 4 floats per query
        // vector, chunk 0 = [max (log2 units), denominator, 0, 0] and chunk
        // 1 + j = features 4j .. 4j + 3 (lane half h, element r of the four
        // accumulators: chunk 1 + 8 (r / 4) + 4h + r % 4), chunk-major with the
        // workgroup's 256 query vectors consecutive. The range that arrives
        // last folds every range's record in range order, two per round trip,
        // with weights 2^(m_s - M).
        const uint32_t pair = (rest * passes + pass) * kv_heads + kvh;
        const uint32_t qv = wave * 32 + n;
        constexpr uint32_t QV = 32 * waves, chunks = prefill_record_floats / 4;
        const __amdgpu_buffer_rsrc_t rs = record_rsrc(
            split_scratch.records + (uint64_t)pair * n_split * (chunks * QV * 4),
            n_split * chunks * QV * 16);
        auto off = [&](uint32_t share, uint32_t chunk) {
            return ((share * chunks + chunk) * QV + qv) * 16u;
        };
#pragma unroll
        for (int r = 0; r < 16; ++r)
            agent_store4(rs, off(part, 1 + 8 * (r >> 2) + 4 * h + (r & 3)), o[0][r], o[1][r],
                         o[2][r], o[3][r]);
        if (h == 0)
            agent_store4(rs, off(part, 0), m, lt, 0.0f, 0.0f);
        wait_vector_memory();
        __syncthreads(); // also: every wave is past its LDS reads
        uint32_t* const last_flag = reinterpret_cast<uint32_t*>(lds);
        if (tid == 0) {
            const uint32_t before = __hip_atomic_fetch_add(split_scratch.arrivals + pair, 1u,
                                                           __ATOMIC_RELAXED,
                                                           __HIP_MEMORY_SCOPE_AGENT);
            const uint32_t last = before == n_parts - 1;
            if (last)
                __hip_atomic_store(split_scratch.arrivals + pair, 0u, __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
            *last_flag = last;
        }
        __syncthreads();
        if (!*last_flag)
            return;
        auto weight = [&](float ms, float to) { // 0 for a range that attended nothing
            return ms == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ms - to);
        };
        float M = -__builtin_inff();
        lt = 0.0f;
#pragma unroll
        for (int a = 0; a < 4; ++a)
            o[a] = f32x16_t {};
        for (uint32_t sh = 0; sh < n_parts; sh += 2) {
            const uint32_t s1 = min(sh + 1, n_parts - 1);
            const u32x4_t ha = agent_load4(rs, off(sh, 0)), hb = agent_load4(rs, off(s1, 0));
            u32x4_t va[16], vb[16];
#pragma unroll
            for (int r = 0; r < 16; ++r)
                va[r] = agent_load4(rs, off(sh, 1 + 8 * (r >> 2) + 4 * h + (r & 3)));
#pragma unroll
            for (int r = 0; r < 16; ++r)
                vb[r] = agent_load4(rs, off(s1, 1 + 8 * (r >> 2) + 4 * h + (r & 3)));
            const float ma = __uint_as_float(ha[0]);
            const float mb = sh + 1 < n_parts ? __uint_as_float(hb[0]) : -__builtin_inff();
            const float m_new = fmaxf(M, fmaxf(ma, mb));
            const float keep = weight(M, m_new), wa = weight(ma, m_new), wb = weight(mb, m_new);
            M = m_new;
            lt = lt * keep + __uint_as_float(ha[1]) * wa;
            lt += __uint_as_float(hb[1]) * wb;
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    float acc = o[a][r] * keep;
                    acc += __uint_as_float(va[r][a]) * wa;
                    o[a][r] = acc + __uint_as_float(vb[r][a]) * wb;
                }
        }
        // lt > 0 for a valid row: some range holds the row's own key
    }

    const float inv = 1.0f / lt;
    float* dst = out + qoff;
    uint32_t alone = 0; // the q-block's rows that are attended again
    if constexpr (WINDOW) {
        // 0 unless some result of the query is infinite or NaN (either lane half)
        float odd = inv * 0.0f;
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                odd = __builtin_fmaf(o[a][r], 0.0f, odd);
        const uint64_t odd_lanes = __ballot(valid && odd != 0.0f);
        alone = (uint32_t)odd_lanes | (uint32_t)(odd_lanes >> 32);
    }
    if constexpr (!RANGES) {
        wait_vector_memory();
        __syncthreads(); // every wave is past its LDS reads
        static_assert(waves * 32 * row_floats<dim> * sizeof(float) <= n_stages * stage_bytes);
        float* tile_out = reinterpret_cast<float*>(lds) + wave * (32 * row_floats<dim>);
#pragma unroll
        for (int r = 0; r < 16; ++r)
            *reinterpret_cast<float4*>(tile_out + n * row_floats<dim> + 32 * (r >> 2) + 16 * h + 4 * (r & 3)) =
                make_float4(o[0][r] * inv, o[1][r] * inv, o[2][r] * inv, o[3][r] * inv);
        const uint32_t before = (wave / G) * 32;
        const size_t first = (size_t)(row0 + before) * q_stride + (size_t)head * dim;
        store_rows<dim, CKV_F32>(tile_out, lane, nrows > before ? nrows - before : 0, alone, out + first,
                                 q_stride, gate ? gate + first : nullptr);
    } else if (valid && !(alone >> n & 1)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            // features 4 * (8 * (r / 4) + 4h + r % 4) + 0..3: accumulators 0..3
            const uint32_t f = 32 * (r >> 2) + 16 * h + 4 * (r & 3);
            float x[4] = { o[0][r] * inv, o[1][r] * inv, o[2][r] * inv, o[3][r] * inv };
            if (gate) { // sigmoid_mul (src/qwen/qwen_layer.cc:204) in the epilogue
                const float4 gv = *reinterpret_cast<const float4*>(gate + qoff + f);
                x[0] *= sigmoid(gv.x);
                x[1] *= sigmoid(gv.y);
                x[2] *= sigmoid(gv.z);
                x[3] *= sigmoid(gv.w);
            }
            *reinterpret_cast<float4*>(dst + f) = make_float4(x[0], x[1], x[2], x[3]);
        }
    }
    if constexpr (WINDOW) {
        if (__builtin_expect(alone == 0, 1))
            return;
        const size_t first = (size_t)(row0 + (wave / G) * 32) * q_stride + (size_t)head * dim;
        for (uint32_t left = alone; left;) {
            uint32_t some = left; // the lowest alone_queries of them
#pragma unroll
            for (uint32_t i = 0; i < alone_queries; ++i)
                left &= left - 1;
            some ^= left;
            attend_alone<dim, CKV_F32, true>(
                reinterpret_cast<const float*>(kbase), reinterpret_cast<const float*>(vbase), table,
                p.features, __builtin_amdgcn_readfirstlane(some), pos_lo, q + first, q_stride, c,
                gate ? gate + first : nullptr, out + first, lane, window);
        }
    }
}

template <int G, bool WINDOW>
hipError_t launch_g(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                    const void* q, uint32_t q_heads, float c, void* out, uint32_t grid,
                    const void* gate, prefill_split split)
{
    auto* kernel = prefill_f32_kernel<G, WINDOW>;
    if constexpr (WINDOW)
        if (split.n_split == 1)
            kernel = prefill_f32_kernel<G, true, false>;
    kernel<<<grid, WINDOW ? 256 : 512, 0, s>>>(p, m, layer, static_cast<const float*>(q),
                                               static_cast<float*>(out), q_heads, c,
                                               static_cast<const float*>(gate), split);
    return hipGetLastError();
}

} // namespace

hipError_t launch_prefill_f32(hipStream_t s, const pool_view& p, const meta_view& m,
                              uint32_t layer, const void* q, uint32_t q_heads, float scale,
                              void* out, const void* gate, prefill_split split)
{
    const uint32_t group = q_heads / p.kv_heads;
    if (split.n_split < 1 || split.min_blocks < 1
        || (split.n_split > 1 && (!split.records || !split.arrivals)))
        return hipErrorInvalidValue;
    const bool windowed = m.window.window != all_keys.window;
    const uint64_t per_tile = windowed ? group / std::min(group, 4u) : group;
    const uint64_t grid = (uint64_t)m.n_tiles * per_tile * p.kv_heads * split.n_split;
    if (!grid)
        return hipSuccess;
    if (grid > 0x7FFFFFFFull)
        return hipErrorInvalidValue;
    const float c = scale * log2e;
    const uint32_t n = (uint32_t)grid;
    const auto launch = [&](auto windowed) {
        constexpr bool WINDOW = decltype(windowed)::value;
        switch (group) {
        case 1:
            return launch_g<1, WINDOW>(s, p, m, layer, q, q_heads, c, out, n, gate, split);
        case 2:
            return launch_g<2, WINDOW>(s, p, m, layer, q, q_heads, c, out, n, gate, split);
        case 4:
            return launch_g<4, WINDOW>(s, p, m, layer, q, q_heads, c, out, n, gate, split);
        case 8:
            if constexpr (WINDOW) // two workgroups of 4 heads
                return launch_g<4, WINDOW>(s, p, m, layer, q, q_heads, c, out, n, gate, split);
            else
                return launch_g<8, WINDOW>(s, p, m, layer, q, q_heads, c, out, n, gate, split);
        default:
            return hipErrorInvalidValue;
        }
    };
    return windowed ? launch(std::true_type {}) : launch(std::false_type {});
}

} // namespace ckv
