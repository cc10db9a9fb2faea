// Causal attention of tiles of query rows over keys that are not 16-bit pages: a cache held
// in 4 bits (fp4.h), or the batch's own rows (whole prompts, packed one after another).
// gfx950 matrix cores.
//
// A query row at position p attends keys 0..p of its sequence, softmax(q.k * scale)
// weighted sum of v, online over blocks of 32 keys. The shape is that of the paged prefill's
// workgroups of four waves (kernels_prefill.hip): each wave has 32 query vectors (32 rows of
// one head), the waves share a kv head's key blocks through LDS, and per block
//   S^T[key][query] = K . Q^T      D/16 x v_mfma_f32_32x32x16
//   O^T[feature][query] += V^T . P^T  D/16 of them, P^T straight from registers
// with S(kb) on the matrix cores while the vector ALU turns S(kb - 1) into probabilities.
// Probabilities enter P.V in the rows' type. Against 64 bits that rounding and the result's own
// come to 1.27 times the result's own in nine fp16 prompts of 17 to 900 rows, 1.33 in bf16 ones of
// 6,000 and 8,192 and 1.41 in 512 bf16 rows behind 6,000 tokens of 4 bits (a second term for
// what the first left would cost half as many products again).
//
// Staging goes through registers, a block ahead: 4-bit codes become the rows' type on the
// way, exactly, once for the four waves; rows of any stride and alignment are taken as they
// are. Three LDS stages, one barrier a block.
//
// Float rows enter as three bf16 terms, each the rounding of what those before it left: 24
// bits, or what is left above bf16's smallest number (values of 2^-115, 2^-120 and 2^-126 come out
// 1.1e-6, 3.6e-5 and 2.4e-3 of themselves off). Of queries and probabilities always, of keys and values where they are rows (4-bit
// numbers are bf16's): 6 or 3 products of terms in place of one of floats, which takes 16
// times as long as one of these. On v_mfma_f32_32x32x2 (exact products) 200 rows behind
// 1,500 tokens of 4 bits took 53 us and take 27, 4 x 512 behind 3,000 456 and 148, two
// prompts of 3,000 rows 641 and 425, five of up to 700 of 64-wide heads 22 and 15.5; errors
// against 64 bits are the same. Over 4-bit pages of 256-wide heads the terms of a query are
// more than a lane's registers: 240 bytes of them spill, and 2 x 300 rows behind 2,000 tokens
// take 80 us where they took 254, 8 x 512 264 where 771. Rows of 256-wide heads have a kernel of
// their own below.
//
// Keys past the tile's last position are staged as zeros. A masked key's probability is 0,
// which meets its value in P.V all the same: where that is infinite or NaN, the rows that
// got something that is not finite are attended again alone, by vector arithmetic over the
// keys they attend.
#include "ckv_internal.h"
#include "fp4.h"
#include "prefill_records.h"
#include "prefill_tile.h"
#include "store_rows.h"

#include <algorithm>
#include <array>
#include <cfloat>
#include <cstdlib>
#include <type_traits>

namespace ckv {
namespace {

// What keys and values are: a 4-bit pool's, rows in 16-byte words, or rows of any alignment.
enum source { FROM_FP4, FROM_WORDS, FROM_ROWS };

constexpr uint32_t block_keys = 32;
constexpr uint32_t prompt_most_ranges = 16; // of a tile's keys
constexpr uint32_t n_waves = 4, n_threads = 64 * n_waves;

// Where a tile's keys are. Sequence positions are rows of `keys` and `values` (ROWS), or go
// through a block table to 4-bit tiles.
struct key_source {
    const uint8_t* keys;
    const uint8_t* values;
    const uint32_t* table;
    uint64_t stride; // bytes of a row
    uint32_t page_log, kv_heads, kvh; // (a page is 2^page_log tiles)
};

// The first byte of a tile of the sequence, within the layer.
template <int D>
__device__ __forceinline__ uint64_t tile_offset(const key_source& s, uint32_t tile)
{
    const uint64_t page = (uint64_t)s.table[tile >> s.page_log] * s.kv_heads + s.kvh;
    return ((page << s.page_log) + (tile & ((1u << s.page_log) - 1))) * fp4_tile_bytes(D);
}

__device__ __forceinline__ float word_half(uint32_t w, int e, bool f16)
{
    return f16 ? half_value<true>((uint16_t)(w >> (16 * e)))
               : __builtin_bit_cast(float, e ? w & 0xFFFF0000u : w << 16);
}

// D/16 features from `f` on of a key's (or value's) row, as floats.
template <int D, int DT, bool FP4>
__device__ __forceinline__ void load_features(const key_source& s, uint32_t key, uint32_t f, bool v,
                                              float (&x)[D / 16])
{
    constexpr uint32_t each = D / 16;
    if constexpr (FP4) {
        const uint8_t* tile = (v ? s.values : s.keys) + tile_offset<D>(s, key / fp4_tile);
        const uint32_t t = key % fp4_tile;
#pragma unroll
        for (uint32_t i = 0; i < each; i += 4) { // four features: half a word
            const uint8_t* at = tile + fp4_word_at(D, t, (f + i) / 8, v) + ((f + i) % 8 ? (v && D == 64 ? 8 : 2) : 0);
            const uint32_t codes = *reinterpret_cast<const uint16_t*>(at);
            const float scale = fp4_scale(tile[fp4_scale_at(D, t, (f + i) / 32, v)]);
            const uint32_t lo = fp4_bf16_pair<0>(codes, scale), hi = fp4_bf16_pair<1>(codes, scale);
            x[i] = word_half(lo, 0, false);
            x[i + 1] = word_half(lo, 1, false);
            x[i + 2] = word_half(hi, 0, false);
            x[i + 3] = word_half(hi, 1, false);
        }
    } else {
        const uint8_t* row = (v ? s.values : s.keys) + key * s.stride;
#pragma unroll
        for (uint32_t i = 0; i < each; ++i)
            if constexpr (DT == CKV_F32)
                x[i] = reinterpret_cast<const float*>(row)[f + i];
            else
                x[i] = half_value<DT == CKV_F16>(reinterpret_cast<const uint16_t*>(row)[f + i]);
    }
}

// One query row by vector arithmetic, four keys a step, sixteen lanes a key.
template <int D, int DT, bool FP4, class T>
__device__ __forceinline__ void attend_row(const key_source& s, uint32_t position, const T* q, float c,
                                           const T* gate, T* out, uint32_t lane)
{
// (a score's product joined with the subtraction of its own rounding weighs more than 1, and
// takes the largest floats to infinity)
#pragma clang fp contract(off)
    constexpr uint32_t each = D / 16;
    const uint32_t f = (lane & 15) * each, sub = lane >> 4;
    float qf[each], acc[each], m = -FLT_MAX, l = 0.0f;
    auto element = [](const T* at) {
        if constexpr (DT == CKV_F32)
            return *at;
        else
            return half_value<DT == CKV_F16>(*at);
    };
#pragma unroll
    for (uint32_t j = 0; j < each; ++j) {
        qf[j] = element(q + f + j);
        acc[j] = 0.0f;
    }
    auto weight = [&](float a, float b) { return __builtin_amdgcn_exp2f(a - b); };
#pragma unroll 1
    for (uint32_t key0 = 0; key0 <= position; key0 += 4) {
        const uint32_t key = min(key0 + sub, position);
        float x[each], score = 0.0f;
        load_features<D, DT, FP4>(s, key, f, false, x);
#pragma unroll
        for (uint32_t j = 0; j < each; ++j)
            score = __builtin_fmaf(qf[j], x[j], score);
#pragma unroll
        for (uint32_t d = 1; d < 16; d *= 2)
            score += __shfl_xor(score, d);
        score *= c;
        load_features<D, DT, FP4>(s, key, f, true, x);
        if (key0 + sub <= position) {
            const float m_new = fmaxf(m, score);
            const float keep = weight(m, m_new), w = weight(score, m_new);
            m = m_new;
            l = l * keep + w;
#pragma unroll
            for (uint32_t j = 0; j < each; ++j)
                acc[j] = acc[j] * keep + w * x[j];
        }
    }
#pragma unroll
    for (uint32_t d = 16; d < 64; d *= 2) {
        const float m_other = __shfl_xor(m, d), l_other = __shfl_xor(l, d);
        const float m_new = fmaxf(m, m_other);
        const float keep = weight(m, m_new), w = weight(m_other, m_new);
        m = m_new;
        l = l * keep + l_other * w;
#pragma unroll
        for (uint32_t j = 0; j < each; ++j) {
            const float other = __shfl_xor(acc[j], d);
            acc[j] = acc[j] * keep + other * w;
        }
    }
    if (sub)
        return;
#pragma unroll
    for (uint32_t j = 0; j < each; ++j) {
        float y = acc[j] / l;
        if (gate)
            y *= sigmoid(element(gate + f + j));
        if constexpr (DT == CKV_F32)
            out[f + j] = y;
        else
            out[f + j] = (uint16_t)pack2<DT == CKV_F16>(y, 0.0f);
    }
}

// A workgroup's part of a launch.
struct tile_part {
    uint32_t kvh, pass, part, n_parts;
    uint32_t records, arrival; // of this (tile, pass, kv head)
    uint32_t row0, nrows, pos0, pos_last;
    uint32_t table; // the sequence's first table entry
    uint32_t n_blocks, kb_begin, kb_end;
};

// Workgroups run over kv heads, then passes, then the list's entries.
__device__ __forceinline__ tile_part part_of(const meta_view& md, uint32_t kv_heads, uint32_t passes)
{
    tile_part w;
    w.kvh = blockIdx.x % kv_heads;
    const uint32_t rest = blockIdx.x / kv_heads;
    w.pass = rest % passes;
    const uint4* e = reinterpret_cast<const uint4*>(md.tiles + prompt_entry_words * (rest / passes));
    const uint4 tile = e[0], range = e[1];
    w.row0 = tile.x;
    w.nrows = tile.y;
    w.pos0 = tile.z;
    w.table = tile.w;
    w.part = range.x;
    w.n_parts = range.y;
    const uint32_t units = passes * kv_heads, unit = w.pass * kv_heads + w.kvh;
    w.records = range.z * units + unit * w.n_parts;
    w.arrival = range.w * units + unit;
    w.pos_last = w.pos0 + w.nrows - 1;
    w.n_blocks = w.pos_last / block_keys + 1;
    prefill_range_bounds(w.n_blocks, w.n_parts, w.part, w.kb_begin, w.kb_end);
    return w;
}

// The state of a query vector's range of keys, as records in chunks of four floats, chunk 0
// [max, denominator, 0, 0], chunk-major over the workgroup's 128 vectors. The range that
// arrives last folds all, in their order. Lane (n, g) of the accumulator layout holds
// features 32mt + 8quad + 4g + e in o[mt][4quad + e]. Returns false for the others.
template <int D>
__device__ __forceinline__ bool fold_ranges(const prefill_split& split, const tile_part& w, uint32_t qv,
                                            uint32_t g, uint32_t tid, float c, float m, float& lt,
                                            f32x16_t (&o)[D / 32], uint32_t* last_flag)
{
    constexpr uint32_t QV = 32 * n_waves, chunks = (D + 4) / 4;
    const __amdgpu_buffer_rsrc_t rs = record_rsrc(
        split.records + (uint64_t)w.records * (chunks * QV * 4), w.n_parts * chunks * QV * 16);
    auto off = [&](uint32_t share, uint32_t chunk) { return ((share * chunks + chunk) * QV + qv) * 16u; };
#pragma unroll
    for (int mt = 0; mt < D / 32; ++mt)
#pragma unroll
        for (int quad = 0; quad < 4; ++quad) {
            const f32x16_t& acc = o[mt];
            agent_store4(rs, off(w.part, 1 + 8 * mt + 2 * quad + g), acc[4 * quad], acc[4 * quad + 1],
                         acc[4 * quad + 2], acc[4 * quad + 3]);
        }
    if (g == 0)
        agent_store4(rs, off(w.part, 0), m, lt, 0.0f, 0.0f);
    wait_vector_memory();
    __syncthreads(); // also: every wave is past its LDS reads
    if (tid == 0) {
        const uint32_t before = __hip_atomic_fetch_add(split.arrivals + w.arrival, 1u, __ATOMIC_RELAXED,
                                                       __HIP_MEMORY_SCOPE_AGENT);
        const uint32_t last = before == w.n_parts - 1;
        if (last)
            __hip_atomic_store(split.arrivals + w.arrival, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *last_flag = last;
    }
    __syncthreads();
    if (!*last_flag)
        return false;
    float M = -__builtin_inff();
    auto weight = [&](float ms, float to) { // 0 for a range that attended nothing
        return ms == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((ms - to) * c);
    };
    lt = 0.0f;
#pragma unroll
    for (int mt = 0; mt < D / 32; ++mt)
        o[mt] = f32x16_t {};
#pragma unroll 1
    for (uint32_t s = 0; s < w.n_parts; ++s) {
        const u32x4_t head = agent_load4(rs, off(s, 0));
        u32x4_t v[D / 8];
#pragma unroll
        for (int j = 0; j < D / 8; ++j)
            v[j] = agent_load4(rs, off(s, 1 + 2 * j + g));
        const float ms = __uint_as_float(head[0]);
        const float m_new = fmaxf(M, ms);
        const float keep = weight(M, m_new), take = weight(ms, m_new);
        M = m_new;
        lt = lt * keep + __uint_as_float(head[1]) * take;
#pragma unroll
        for (int j = 0; j < D / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                o[j / 4][4 * (j % 4) + e] = o[j / 4][4 * (j % 4) + e] * keep + __uint_as_float(v[j][e]) * take;
    }
    return true;
}

// Eight floats as `N` words of packed bf16 terms each: the rounding of what those before it left.
template <int N>
__device__ __forceinline__ void terms_of(float a, float b, uint32_t (&w)[N])
{
#pragma unroll
    for (int t = 0; t < N; ++t) {
        w[t] = pack2<false>(a, b);
        a -= __builtin_bit_cast(float, w[t] << 16);
        b -= __builtin_bit_cast(float, w[t] & 0xFFFF0000u);
    }
}
template <int N>
__device__ __forceinline__ void terms_of(const float (&x)[8], uint4 (&out)[N])
{
    uint32_t w[4][N];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        terms_of<N>(x[2 * i], x[2 * i + 1], w[i]);
#pragma unroll
    for (int t = 0; t < N; ++t)
        out[t] = make_uint4(w[0][t], w[1][t], w[2][t], w[3][t]);
}

// What a thread holds of a block on its way to LDS: rows, eight elements at a time, or 4-bit
// codes.
template <bool F32>
struct eight_of { // (native vectors: arrays of uint4 are not kept in registers)
    u32x4_t w[F32 ? 2 : 1];
};
template <int D, bool FP4, bool F32>
struct staged {
    static constexpr uint32_t per = D / 64; // of K, and of V: 32 rows of D/8
    eight_of<F32> k[per], v[per];
};
template <int D, bool F32>
struct staged<D, true, F32> {
    // 4-byte words of K or of V: threads below half take K, the others V
    static constexpr uint32_t words = D / 32;
    uint32_t code[words];
    uint32_t scale[D == 256 ? 2 : 1];
};

// GH heads of a GQA group share a workgroup: 128 / GH rows.
template <int D, int GH, int DT, source SRC>
__global__ __launch_bounds__(n_threads, D == 256 || (D == 128 && DT == CKV_F32) ? 1 : 2) void prompt_kernel(
    pool_view p, meta_view md, uint32_t layer, prompt_rows x, void* __restrict__ out_rows, uint32_t q_heads,
    float c, uint32_t q_and, uint32_t q_xor, const void* __restrict__ gate_rows, prefill_split split)
{
    constexpr bool FP4 = SRC == FROM_FP4, F32 = DT == CKV_F32, F16 = DT == CKV_F16;
    using T = std::conditional_t<F32, float, uint16_t>;
    T* const out = static_cast<T*>(out_rows);
    const T* const gate = static_cast<const T*>(gate_rows);
    constexpr int KS = D / 16, MT = D / 32;
    // terms of queries and probabilities, and of keys and values (4-bit numbers are bf16's)
    constexpr int TQ = F32 ? 3 : 1, TK = F32 && !FP4 ? 3 : 1;
    constexpr uint32_t n_stages = 3;
    // K stage: chunk i (features 8i .. 8i + 7) holds the block's keys in the LDS rows of the
    // A operand, 16 bytes each; 16 more bytes a chunk spread a key's chunks over the banks.
    constexpr uint32_t k_chunk = block_keys * 16 + 16, k_bytes = D / 8 * k_chunk;
    // V stage: rows as they are, read transposed; key k is row (k / 4) % 4 of group
    // k % 4 + 4 * (k / 16), 64 bytes between groups (kernels_prefill.hip).
    constexpr uint32_t v_row = 2 * D, v_group = 4 * v_row + 64, v_bytes = 8 * v_group;
    constexpr uint32_t plane = k_bytes + v_bytes, stage_bytes = TK * plane; // a plane for each term
    constexpr uint32_t out_bytes = n_waves * 32 * row_floats<D> * 4;
    constexpr uint32_t lds_bytes = n_stages * stage_bytes > out_bytes ? n_stages * stage_bytes : out_bytes;
    __shared__ __attribute__((aligned(16))) uint8_t lds[lds_bytes];
    const uint32_t group = q_heads / p.kv_heads;
    const tile_part w = part_of(md, p.kv_heads, group / GH);
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t n = lane & 31, g = lane >> 5;
    const uint32_t head = w.kvh * group + w.pass * GH + wave % GH, rb = wave / GH;
    const uint32_t row = rb * 32 + n;
    const bool valid = row < w.nrows;
    const uint32_t qpos = w.pos0 + min(row, w.nrows - 1);
    const uint32_t pos_lo = w.pos0 + rb * 32;

    key_source s;
    if constexpr (FP4) {
        const uint64_t layer_bytes = (uint64_t)p.blocks * p.block_size / fp4_tile * p.kv_heads * fp4_tile_bytes(D);
        s = { static_cast<const uint8_t*>(p.keys) + layer * layer_bytes,
              static_cast<const uint8_t*>(p.values) + layer * layer_bytes, md.table + w.table, 0,
              (uint32_t)__builtin_ctz(p.block_size / fp4_tile), p.kv_heads, w.kvh };
    } else {
        const uint64_t first = (uint64_t)(w.row0 - w.pos0) * x.kv_stride + w.kvh * D;
        s = { static_cast<const uint8_t*>(x.keys) + sizeof(T) * first, static_cast<const uint8_t*>(x.values) + sizeof(T) * first,
              nullptr, sizeof(T) * x.kv_stride, 0, 0, 0 };
    }
    // eight elements, from any alignment of them
    using eight = eight_of<F32>;
    auto gather = [](const void* from) {
        const T* e = static_cast<const T*>(from);
        eight x;
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x.w[i / 4][i % 4] = __float_as_uint(e[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                x.w[0][i] = e[2 * i] | (uint32_t)e[2 * i + 1] << 16;
        }
        return x;
    };
    auto read = [](const void* from) {
        eight x;
        x.w[0] = static_cast<const u32x4_t*>(from)[0];
        if constexpr (F32)
            x.w[1] = static_cast<const u32x4_t*>(from)[1];
        return x;
    };
    // and as an operand's words, a term each
    auto operands = [](const eight& x, auto& to) {
        if constexpr (F32) {
            const u32x4_t a = x.w[0], b = x.w[1];
            const float f[8] = { __uint_as_float(a[0]), __uint_as_float(a[1]), __uint_as_float(a[2]), __uint_as_float(a[3]),
                                 __uint_as_float(b[0]), __uint_as_float(b[1]), __uint_as_float(b[2]), __uint_as_float(b[3]) };
            terms_of<3>(f, to);
        } else {
            to[0] = __builtin_bit_cast(uint4, x.w[0]);
        }
    };
    const T* q_row = static_cast<const T*>(x.queries)
        + (uint64_t)(w.row0 + min(row, w.nrows - 1)) * x.q_stride + (uint64_t)head * D;
    uint4 qr[KS][TQ];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        eight v {};
        if (valid) {
            const T* at = q_row + ks * 16 + g * 8;
            v = x.vectors ? read(at) : gather(at);
        }
        // a negative scale turns the queries' sign, a scale of 0 leaves nothing of them
#pragma unroll
        for (int i = 0; i < (F32 ? 2 : 1); ++i)
            v.w[i] = (v.w[i] & q_and) ^ q_xor;
        operands(v, qr[ks]);
    }

    using held = staged<D, FP4, F32>;
    // Blocks on their way: 4-bit ones three ahead of the one that is stored (a block takes less
    // than a load from HBM), rows one.
    constexpr uint32_t ahead = FP4 ? 3 : 1;
    held flight[ahead];
    // where a lane's codes and scales are in a tile
    const bool v_wave = wave >= 2;
    const uint32_t code_at = v_wave ? lane * 16 : lane / 4 * (D / 2) + lane % 4 * 16;
    const uint32_t code_part = v_wave ? 1024 : 64;
    const uint32_t scale_at = 8 * D
        + (v_wave ? (D == 64 ? lane % 16 / 8 : lane % 16 / 4) * 16 + lane / 16 * 4
                  : lane / 4 * (D / 32) + (D == 64 ? lane % 4 / 2 : lane % 4));
    const uint32_t scale_part = v_wave ? 64 : 4, k_shift = scale_at % 4 * 8;
    // block kb's words of this thread into registers
    auto load = [&](uint32_t kb, held& next) __attribute__((always_inline)) {
        const uint32_t key0 = kb * block_keys;
        if constexpr (FP4) {
            // waves 0 and 1 take K of the block's two tiles, 2 and 3 V. Of K, lane 4t + i takes
            // part i of token t; of V, lane 16q + c features from c on of tokens 4q .. 4q + 3.
            const uint32_t tile = min(2 * kb + (wave & 1), w.pos_last / fp4_tile);
            const uint8_t* base = uniform_ptr((wave < 2 ? s.keys : s.values) + tile_offset<D>(s, tile));
            if constexpr (D == 64) {
                const uint2 r = *reinterpret_cast<const uint2*>(base + lane * 8);
                next.code[0] = r.x;
                next.code[1] = r.y;
            } else {
#pragma unroll
                for (uint32_t i = 0; i < held::words / 4; ++i) {
                    const uint4 r = *reinterpret_cast<const uint4*>(base + code_at + i * code_part);
                    next.code[4 * i] = r.x;
                    next.code[4 * i + 1] = r.y;
                    next.code[4 * i + 2] = r.z;
                    next.code[4 * i + 3] = r.w;
                }
            }
            // (a K lane's byte is the lowest of its word: one load for both)
#pragma unroll
            for (uint32_t i = 0; i < (D == 256 ? 2 : 1); ++i)
                next.scale[i] = *reinterpret_cast<const uint32_t*>(base + (scale_at & ~3u) + i * scale_part);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < held::per; ++i) {
                const uint32_t word = i * n_threads + tid, key = key0 + word / (D / 8), f = word % (D / 8) * 8;
                const uint64_t at = min(key, w.pos_last) * s.stride + sizeof(T) * f;
                if constexpr (SRC == FROM_WORDS) {
                    next.k[i] = read(s.keys + at);
                    next.v[i] = read(s.values + at);
                } else {
                    next.k[i] = gather(s.keys + at);
                    next.v[i] = gather(s.values + at);
                }
            }
        }
    };
    auto put_k = [&](uint8_t* st, uint32_t key, uint32_t chunk, uint4 v) {
        *reinterpret_cast<uint4*>(st + chunk * k_chunk + key_row(key) * 16) = v;
    };
    auto v_at = [&](uint8_t* st, uint32_t key) {
        return st + k_bytes + (key % 4 + 4 * (key / 16)) * v_group + key / 4 % 4 * v_row;
    };
    // and from there into its stage, zeros past the tile's last position
    auto store_keys = [&](uint32_t kb, const held& next, uint8_t* st, auto all) __attribute__((always_inline)) {
        constexpr bool ALL = decltype(all)::value;
        const uint32_t key0 = kb * block_keys;
        if constexpr (FP4) {
            const uint32_t token0 = (wave & 1) * fp4_tile;
            if (!v_wave) {
                const uint32_t key = token0 + lane / 4;
                const bool there = ALL || key0 + key <= w.pos_last;
#pragma unroll
                for (uint32_t i = 0; i < held::words; ++i) {
                    const float scale = there ? fp4_scale(next.scale[i / 4] >> k_shift & 255) : 1.0f;
                    const uint32_t chunk = D == 64 ? lane % 4 * 2 + i : i / 4 * 16 + lane % 4 * 4 + i % 4;
                    put_k(st, key, chunk, fp4_eight<F16>(there ? next.code[i] : 0, scale));
                }
            } else {
                const uint32_t quad = token0 + lane / 16 * 4, cc = lane % 16;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const bool there = ALL || key0 + quad + i <= w.pos_last;
                    uint8_t* to = v_at(st, quad + i);
#pragma unroll
                    for (uint32_t part = 0; part < (D == 256 ? 2 : 1); ++part) {
                        const float scale = there ? fp4_scale(next.scale[part] >> (8 * i) & 255) : 1.0f;
                        if constexpr (D == 64) {
                            const uint32_t codes = there ? next.code[i / 2] >> (16 * (i % 2)) : 0;
                            *reinterpret_cast<uint2*>(to + cc * 8) =
                                make_uint2(fp4_pair<0, F16>(codes, scale), fp4_pair<1, F16>(codes, scale));
                        } else {
                            *reinterpret_cast<uint4*>(to + part * 256 + cc * 16) =
                                fp4_eight<F16>(there ? next.code[4 * part + i] : 0, scale);
                        }
                    }
                }
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < held::per; ++i) {
                const uint32_t word = i * n_threads + tid, key = word / (D / 8), chunk = word % (D / 8);
                uint4 k[TK], v[TK];
                operands(next.k[i], k);
                operands(next.v[i], v);
                const bool there = ALL || key0 + key <= w.pos_last;
#pragma unroll
                for (int t = 0; t < TK; ++t) {
                    if (!there)
                        k[t] = v[t] = make_uint4(0, 0, 0, 0);
                    put_k(st + t * plane, key, chunk, k[t]);
                    *reinterpret_cast<uint4*>(v_at(st + t * plane, key) + chunk * 16) = v[t];
                }
            }
        }
    };
    auto store = [&](uint32_t kb, const held& next, uint8_t* st) __attribute__((always_inline)) {
        if (kb * block_keys + block_keys - 1 <= w.pos_last)
            store_keys(kb, next, st, std::true_type {});
        else
            store_keys(kb, next, st, std::false_type {});
    };

    f32x16_t o[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
        o[mt] = f32x16_t {};
    float m = -__builtin_inff(), l = 0.0f, m_limit = -__builtin_inff(), mx = 0.0f;
    const float rescale_raw = rescale_log2 / c;
    f32x16_t sc, sp;
    auto read_k = [&](const uint8_t* st, uint4 (&ka)[KS]) __attribute__((always_inline)) {
        const uint8_t* kl = st + g * k_chunk + n * 16;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
            ka[ks] = *reinterpret_cast<const uint4*>(kl + ks * 2 * k_chunk);
    };
    // products of terms i and j of their operands with i + j < TQ: what is left out is under
    // 2^-24 of the whole
    auto scores = [&](const uint8_t* st, const uint4 (&first)[KS]) __attribute__((always_inline)) {
        sc = f32x16_t {};
#pragma unroll
        for (int t = 0; t < TK; ++t) {
            uint4 ka[KS];
            if (t) {
                __builtin_amdgcn_sched_barrier(0); // one plane's registers at a time
                read_k(st + t * plane, ka);
            } else {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
                    ka[ks] = first[ks];
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int j = 0; j < TQ - t; ++j)
                    sc = mfma<F16>(ka[ks], qr[ks][j], sc);
        }
    };
    auto probabilities = [&](uint4 (&pt)[2][TQ]) __attribute__((always_inline)) {
        // a range of the keys may hold none that a row attends: its maximum stays -inf
        const float mc = m == -__builtin_inff() ? 0.0f : m * c;
        float sum[4];
#pragma unroll
        for (int r = 0; r < 16; ++r)
            sp[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sp[r], c, -mc));
#pragma unroll
        for (int i = 0; i < 4; ++i)
            sum[i] = (sp[4 * i] + sp[4 * i + 1]) + (sp[4 * i + 2] + sp[4 * i + 3]);
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (F32) {
                const float f[8] = { sp[8 * h], sp[8 * h + 1], sp[8 * h + 2], sp[8 * h + 3],
                                     sp[8 * h + 4], sp[8 * h + 5], sp[8 * h + 6], sp[8 * h + 7] };
                terms_of<TQ>(f, pt[h]);
            } else {
                pt[h][0] = make_uint4(pack2<F16>(sp[8 * h], sp[8 * h + 1]), pack2<F16>(sp[8 * h + 2], sp[8 * h + 3]),
                                      pack2<F16>(sp[8 * h + 4], sp[8 * h + 5]), pack2<F16>(sp[8 * h + 6], sp[8 * h + 7]));
            }
        }
    };
    const uint32_t vr_off = ((lane & 15) >> 2) * v_group + (lane >> 5) * 2 * v_row + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
    auto values = [&](const uint8_t* st, const uint4 (&pt)[2][TQ]) __attribute__((always_inline)) {
        uint32_t vaddr = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) uint8_t*)(const_cast<uint8_t*>(st) + k_bytes)) + vr_off;
        asm volatile("" : "+v"(vaddr));
        auto* vb = (__attribute__((address_space(3))) uint8_t*)(uintptr_t)vaddr;
#pragma unroll
        for (int t = 0; t < TK; ++t) {
            if (t)
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    auto* at = vb + t * plane + 4 * h * v_group + 64 * mt;
                    const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)at);
                    const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) i16x4_t*)(at + v_row));
                    const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
#pragma unroll
                    for (int j = 0; j < TQ - t; ++j)
                        o[mt] = mfma<F16>(make_uint4(l2.x, l2.y, h2.x, h2.y), pt[h][j], o[mt]);
                }
        }
    };
    auto stats = [&](uint32_t kb) __attribute__((always_inline)) {
        const uint32_t key0 = kb * block_keys;
        if (key0 + block_keys - 1 > pos_lo) { // the diagonal crosses this block
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (key0 + 16 * (r >> 3) + 8 * g + (r & 7) > qpos)
                    sc[r] = -__builtin_inff();
        }
        sp = sc;
        mx = lane_max(sp);
        if (__any(mx > m_limit)) {
            const float m_new = fmaxf(m, pair_max(mx));
            const float alpha = m_new == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((m - m_new) * c);
            l *= alpha;
            m = m_new;
            m_limit = m_new + rescale_raw;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
                o[mt] *= alpha;
        }
    };

    // Iteration kb finishes block kb - 1 and scores block kb; it stages block kb + 1, whose
    // stage was block kb - 2's, last read in iteration kb - 1. The loop goes round the stages,
    // and the registers of the blocks in flight, in turn: iteration kb_begin + 3i + S.
    static_assert(n_stages % ahead == 0);
#pragma unroll
    for (uint32_t i = 0; i < ahead; ++i)
        if (w.kb_begin + i < w.kb_end)
            load(w.kb_begin + i, flight[i]);
    store(w.kb_begin, flight[0], lds);
    if (w.kb_begin + ahead < w.kb_end)
        load(w.kb_begin + ahead, flight[0]);
    __syncthreads();
    auto iteration = [&](uint32_t kb, auto turn, auto is_first) __attribute__((always_inline)) {
        constexpr uint32_t S = decltype(turn)::value;
        constexpr bool FIRST = decltype(is_first)::value;
        uint4 ka[KS], pt[2][TQ];
        read_k(lds + S * stage_bytes, ka);
        held& next = flight[(S + 1) % ahead];
        if (kb + 1 < w.kb_end)
            store(kb + 1, next, lds + (S + 1) % n_stages * stage_bytes);
        if (kb + 1 + ahead < w.kb_end)
            load(kb + 1 + ahead, next);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!FIRST)
            probabilities(pt);
        scores(lds + S * stage_bytes, ka);
        if constexpr (!FIRST)
            values(lds + (S + 2) % n_stages * stage_bytes, pt);
        stats(kb);
        __syncthreads();
    };
    uint32_t kb = w.kb_begin;
    uint32_t last = 0; // the stage of the last block
    iteration(kb, std::integral_constant<uint32_t, 0> {}, std::true_type {});
    while (++kb < w.kb_end) {
        iteration(kb, std::integral_constant<uint32_t, 1> {}, std::false_type {});
        last = 1;
        if (++kb >= w.kb_end)
            break;
        iteration(kb, std::integral_constant<uint32_t, 2> {}, std::false_type {});
        last = 2;
        if (++kb >= w.kb_end)
            break;
        iteration(kb, std::integral_constant<uint32_t, 0> {}, std::false_type {});
        last = 0;
    }
    {
        uint4 pt[2][TQ];
        probabilities(pt);
        values(lds + last * stage_bytes, pt);
    }

    float lt = l + __shfl_xor(l, 32);
    if (w.n_parts > 1) {
        if (!fold_ranges<D>(split, w, wave * 32 + n, g, tid, c, m, lt, o, reinterpret_cast<uint32_t*>(lds)))
            return;
    }
    const float inv = 1.0f / lt;
    float odd = inv * 0.0f; // 0 unless some result of the query is infinite or NaN
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < 16; ++r)
            odd = __builtin_fmaf(o[mt][r], 0.0f, odd);
    const uint64_t odd_lanes = __ballot(valid && odd != 0.0f);
    uint32_t alone = (uint32_t)odd_lanes | (uint32_t)(odd_lanes >> 32);
    __syncthreads(); // every wave is past its LDS reads
    float* tile_out = reinterpret_cast<float*>(lds) + wave * (32 * row_floats<D>);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int quad = 0; quad < 4; ++quad) {
            const f32x16_t& acc = o[mt];
            *reinterpret_cast<float4*>(tile_out + n * row_floats<D> + 32 * mt + 8 * quad + 4 * g) =
                make_float4(acc[4 * quad] * inv, acc[4 * quad + 1] * inv, acc[4 * quad + 2] * inv, acc[4 * quad + 3] * inv);
        }
    const uint32_t there = rb * 32 < w.nrows ? min(w.nrows - rb * 32, 32u) : 0;
    const size_t o_stride = (size_t)q_heads * D;
    const size_t first = (size_t)(w.row0 + rb * 32) * o_stride + (size_t)head * D;
    if (x.out_vectors) {
        store_rows<D, DT>(tile_out, lane, there, alone, out + first, o_stride, gate ? gate + first : nullptr);
    } else {
        for (uint32_t r = 0; r < there; ++r)
            for (uint32_t f = lane; f < D; f += 64)
                if (!(alone >> r & 1)) {
                    float y = tile_out[r * row_floats<D> + f];
                    const size_t at = first + r * o_stride + f;
                    if constexpr (F32) {
                        out[at] = gate ? y * sigmoid(gate[at]) : y;
                    } else {
                        if (gate)
                            y *= sigmoid(half_value<F16>(gate[at]));
                        out[at] = (uint16_t)pack2<F16>(y, 0.0f);
                    }
                }
    }
    const float cs = q_and ? (q_xor ? -c : c) : 0.0f; // the scale in log2 units
    while (__builtin_expect(alone != 0, 0)) {
        const uint32_t r = __builtin_ctz(alone);
        alone &= alone - 1;
        const size_t at = first + r * o_stride;
        attend_row<D, DT, FP4>(s, pos_lo + r, static_cast<const T*>(x.queries) + (uint64_t)(w.row0 + rb * 32 + r) * x.q_stride + (uint64_t)head * D,
                               cs, gate ? gate + at : nullptr, out + at, lane);
    }
}

// Float rows of 256-wide heads, whose terms' planes LDS has no room for: S^T and O^T on
// v_mfma_f32_32x32x2, 128 and 128 products a block, which are 85 % of its time (8.2 us; 56 to
// 60 bytes a lane spill beside them). The
// contraction over features pairs 8i + e with 8i + 4 + e, so that a lane's operands are
// 16-byte words; that over keys pairs the two keys of an accumulator element, so that a
// probability is an operand where it was computed. Two LDS stages of whole rows.
template <int GH, source SRC>
__global__ __launch_bounds__(n_threads, 1) void prompt_f32_kernel(
    pool_view p, meta_view md, uint32_t layer, prompt_rows x, float* __restrict__ out, uint32_t q_heads,
    float c, float q_sign, const float* __restrict__ gate, prefill_split split)
{
    constexpr int D = 256, MT = D / 32, K4 = D / 8;
    constexpr uint32_t pitch = D + 4, stage_floats = 2 * block_keys * pitch;
    __shared__ __attribute__((aligned(16))) float lds[2 * stage_floats];
    static_assert(n_waves * 32 * row_floats<D> <= 2 * stage_floats);
    const uint32_t group = q_heads / p.kv_heads;
    const tile_part w = part_of(md, p.kv_heads, group / GH);
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t n = lane & 31, g = lane >> 5;
    const uint32_t head = w.kvh * group + w.pass * GH + wave % GH, rb = wave / GH;
    const uint32_t row = rb * 32 + n;
    const bool valid = row < w.nrows;
    const uint32_t qpos = w.pos0 + min(row, w.nrows - 1);
    const uint32_t pos_lo = w.pos0 + rb * 32;
    const uint64_t row_first = (uint64_t)(w.row0 - w.pos0) * x.kv_stride + w.kvh * D;
    const key_source s { static_cast<const uint8_t*>(x.keys) + 4 * row_first,
                         static_cast<const uint8_t*>(x.values) + 4 * row_first, nullptr, 4 * x.kv_stride, 0, 0, 0 };
    const float* q_row = static_cast<const float*>(x.queries)
        + (uint64_t)(w.row0 + min(row, w.nrows - 1)) * x.q_stride + (uint64_t)head * D;
    float4 qr[K4];
#pragma unroll
    for (int i = 0; i < K4; ++i) {
        float4 v = make_float4(0, 0, 0, 0);
        if (valid) {
            const float* at = q_row + 8 * i + 4 * g;
            v = x.vectors ? *reinterpret_cast<const float4*>(at) : make_float4(at[0], at[1], at[2], at[3]);
        }
        qr[i] = q_sign == 0.0f ? make_float4(0, 0, 0, 0)
                               : make_float4(v.x * q_sign, v.y * q_sign, v.z * q_sign, v.w * q_sign);
    }
    constexpr uint32_t per = D / 32; // 16-byte words
    float4 next_k[per], next_v[per];
    auto load = [&](uint32_t kb) {
#pragma unroll
        for (uint32_t i = 0; i < per; ++i) {
            const uint32_t word = i * n_threads + tid;
            const uint32_t key = min(kb * block_keys + word / (D / 4), w.pos_last), f = word % (D / 4) * 4;
            const float* k = reinterpret_cast<const float*>(s.keys + key * s.stride) + f;
            const float* v = reinterpret_cast<const float*>(s.values + key * s.stride) + f;
            if constexpr (SRC == FROM_WORDS) {
                next_k[i] = *reinterpret_cast<const float4*>(k);
                next_v[i] = *reinterpret_cast<const float4*>(v);
            } else {
                next_k[i] = make_float4(k[0], k[1], k[2], k[3]);
                next_v[i] = make_float4(v[0], v[1], v[2], v[3]);
            }
        }
    };
    auto store = [&](uint32_t kb) {
        float* st = lds + kb % 2 * stage_floats;
#pragma unroll
        for (uint32_t i = 0; i < per; ++i) {
            const uint32_t word = i * n_threads + tid, key = word / (D / 4), f = word % (D / 4) * 4;
            float4 k = next_k[i], v = next_v[i];
            if (kb * block_keys + key > w.pos_last)
                k = v = make_float4(0, 0, 0, 0);
            *reinterpret_cast<float4*>(st + key * pitch + f) = k;
            *reinterpret_cast<float4*>(st + (block_keys + key) * pitch + f) = v;
        }
    };

    f32x16_t o[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
        o[mt] = f32x16_t {};
    float m = -__builtin_inff(), l = 0.0f, m_limit = -__builtin_inff();
    const float rescale_raw = rescale_log2 / c;
    load(w.kb_begin);
    store(w.kb_begin);
    __syncthreads();
    for (uint32_t kb = w.kb_begin; kb < w.kb_end; ++kb) {
        if (kb + 1 < w.kb_end)
            load(kb + 1);
        const float* st = lds + kb % 2 * stage_floats;
        const uint32_t key0 = kb * block_keys;
        f32x16_t sc {};
#pragma unroll
        for (int i = 0; i < K4; ++i) {
            const float4 a = *reinterpret_cast<const float4*>(st + n * pitch + 8 * i + 4 * g);
            sc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x, qr[i].x, sc, 0, 0, 0);
            sc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.y, qr[i].y, sc, 0, 0, 0);
            sc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.z, qr[i].z, sc, 0, 0, 0);
            sc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.w, qr[i].w, sc, 0, 0, 0);
        }
        if (key0 + block_keys - 1 > pos_lo) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (key0 + 8 * (r >> 2) + 4 * g + (r & 3) > qpos)
                    sc[r] = -__builtin_inff();
        }
        const float mx = lane_max(sc);
        if (__any(mx > m_limit)) {
            const float m_new = fmaxf(m, pair_max(mx));
            const float alpha = m_new == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((m - m_new) * c);
            l *= alpha;
            m = m_new;
            m_limit = m_new + rescale_raw;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
                o[mt] *= alpha;
        }
        const float mc = m == -__builtin_inff() ? 0.0f : m * c;
        float sum[4] = {};
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            sc[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], c, -mc));
            sum[r & 3] += sc[r];
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float* v = st + (block_keys + 8 * (r >> 2) + 4 * g + (r & 3)) * pitch + n;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
                o[mt] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[32 * mt], sc[r], o[mt], 0, 0, 0);
        }
        if (kb + 1 < w.kb_end)
            store(kb + 1); // block kb - 1's stage, last read before the barrier
        __syncthreads();
    }
    float lt = l + __shfl_xor(l, 32);
    if (w.n_parts > 1) {
        if (!fold_ranges<D>(split, w, wave * 32 + n, g, tid, c, m, lt, o, reinterpret_cast<uint32_t*>(lds)))
            return;
        __syncthreads(); // the flag is read
    }
    const float inv = 1.0f / lt;
    float odd = inv * 0.0f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < 16; ++r)
            odd = __builtin_fmaf(o[mt][r], 0.0f, odd);
    const uint64_t odd_lanes = __ballot(valid && odd != 0.0f);
    uint32_t alone = (uint32_t)odd_lanes | (uint32_t)(odd_lanes >> 32);
    float* tile_out = lds + wave * (32 * row_floats<D>);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int quad = 0; quad < 4; ++quad) {
            const f32x16_t& acc = o[mt];
            *reinterpret_cast<float4*>(tile_out + n * row_floats<D> + 32 * mt + 8 * quad + 4 * g) =
                make_float4(acc[4 * quad] * inv, acc[4 * quad + 1] * inv, acc[4 * quad + 2] * inv, acc[4 * quad + 3] * inv);
        }
    const uint32_t there = rb * 32 < w.nrows ? min(w.nrows - rb * 32, 32u) : 0;
    const size_t o_stride = (size_t)q_heads * D;
    const size_t first = (size_t)(w.row0 + rb * 32) * o_stride + (size_t)head * D;
    if (x.out_vectors) {
        store_rows<D, CKV_F32>(tile_out, lane, there, alone, out + first, o_stride, gate ? gate + first : nullptr);
    } else {
        for (uint32_t r = 0; r < there; ++r)
            for (uint32_t f = lane; f < D; f += 64)
                if (!(alone >> r & 1)) {
                    float y = tile_out[r * row_floats<D> + f];
                    if (gate)
                        y *= sigmoid(gate[first + r * o_stride + f]);
                    out[first + r * o_stride + f] = y;
                }
    }
    while (__builtin_expect(alone != 0, 0)) {
        const uint32_t r = __builtin_ctz(alone);
        alone &= alone - 1;
        const size_t at = first + r * o_stride;
        attend_row<D, CKV_F32, false>(s, pos_lo + r, static_cast<const float*>(x.queries) + (uint64_t)(w.row0 + rb * 32 + r) * x.q_stride + (uint64_t)head * D,
                                    c * q_sign, gate ? gate + at : nullptr, out + at, lane);
    }
}

bool aligned16(const void* ptr)
{
    return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0;
}

template <int D, int GH, source SRC>
hipError_t launch_gh(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer, const prompt_rows& x,
                     uint32_t q_heads, float scale, void* out, const void* gate, const prefill_split& split)
{
    const uint64_t grid = (uint64_t)m.n_tiles * (q_heads / GH);
    if (!grid)
        return hipSuccess;
    if (grid > 0x7FFFFFFFull)
        return hipErrorInvalidValue;
    const float c = scale == 0.0f ? log2e : __builtin_fabsf(scale) * log2e;
    const dim3 blocks((uint32_t)grid), threads(n_threads);
    if constexpr (D == 256 && SRC != FROM_FP4)
        if (p.dtype == CKV_F32) {
            prompt_f32_kernel<GH, SRC><<<blocks, threads, 0, s>>>(
                p, m, layer, x, static_cast<float*>(out), q_heads, c, scale == 0.0f ? 0.0f : scale < 0.0f ? -1.0f : 1.0f,
                static_cast<const float*>(gate), split);
            return hipGetLastError();
        }
    auto* kernel = p.dtype == CKV_F16 ? prompt_kernel<D, GH, CKV_F16, SRC> : prompt_kernel<D, GH, CKV_BF16, SRC>;
    if constexpr (D != 256 || SRC == FROM_FP4)
        if (p.dtype == CKV_F32)
            kernel = prompt_kernel<D, GH, CKV_F32, SRC>;
    const uint32_t turned = p.dtype == CKV_F32 ? 0x80000000u : 0x80008000u;
    kernel<<<blocks, threads, 0, s>>>(p, m, layer, x, out, q_heads, c, scale == 0.0f ? 0u : ~0u,
                                      scale < 0.0f ? turned : 0u, gate, split);
    return hipGetLastError();
}

template <int D, source SRC, class... Args>
hipError_t launch_group(uint32_t heads, const Args&... args)
{
    return heads == 4 ? launch_gh<D, 4, SRC>(args...) : heads == 2 ? launch_gh<D, 2, SRC>(args...)
                                                                  : launch_gh<D, 1, SRC>(args...);
}

template <source SRC, class... Args>
hipError_t launch_dim(uint32_t head_dim, uint32_t heads, const Args&... args)
{
    return head_dim == 64 ? launch_group<64, SRC>(heads, args...)
        : head_dim == 128 ? launch_group<128, SRC>(heads, args...)
                          : launch_group<256, SRC>(heads, args...);
}

// Heads of a GQA group that share a workgroup's key blocks.
uint32_t heads_of(const pool_view& p, uint32_t q_heads)
{
    const uint32_t group = q_heads / p.kv_heads;
    return group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
}

} // namespace

namespace {

// Whether rows are read and written in 16-byte words.
void set_vectors(const pool_view& p, prompt_rows& x, const void* out, const void* gate, bool fp4)
{
    const uint32_t each = 16 / p.elem_size;
    x.vectors = aligned16(x.queries) && x.q_stride % each == 0
        && (fp4 || (aligned16(x.keys) && aligned16(x.values) && x.kv_stride % each == 0));
    x.out_vectors = aligned16(out) && aligned16(gate);
}

} // namespace

prompt_form prompt_form_of(const pool_view& p, const meta_view& m, const prompt_rows& rows, uint32_t q_heads,
                           float scale, const void* out, const void* gate, bool fp4, int cu_count)
{
    prompt_rows x = rows;
    set_vectors(p, x, out, gate, fp4);
    prompt_form form { n_waves, heads_of(p, q_heads), false, fp4 };
    form.paged_kernel = !fp4 && p.head_dim == 128 && p.dtype != CKV_F32 && x.vectors && x.out_vectors
        && scale > 0.0f && x.kv_stride <= 1u << 26; // (its offsets within 16 rows are 32 bits)
    if (!form.paged_kernel)
        return form;
    const uint32_t eight = form.heads == 4 ? m.row_blocks[1] : form.heads == 2 ? m.row_blocks[2] : m.n_tiles;
    if ((uint64_t)eight * (q_heads / form.heads) >= 2 * (uint64_t)std::max(cu_count, 1))
        form.waves = 8;
    if (const char* forced = std::getenv("CKV_PREFILL_WAVES"))
        form.waves = std::strtol(forced, nullptr, 10) == 8 ? 8 : 4;
    return form;
}

namespace {

// What a launch's time is estimated from, us: a key block of a workgroup alone on its compute
// unit (two there: `shared` of that more for each), what comes before and after the blocks,
// in blocks, and of a tile that is cut the handoff and each record. Fitted to times of 20
// batches in 1 to 16 ranges; the ranges it chooses are the fastest measured or within 8 % of
// that. Uncut and as chosen, us back to back: 512 rows behind 6000 tokens of 4 bits 164 and 49,
// 4 x 256 behind 2000 61 and 35, 900 rows of one prompt 21 and 17, five short float prompts 35
// and 15.5; 8 x 1024 behind 3000 stays uncut (242, in two ranges 277). The list is made at a
// batch's first call, which all layers share: 5 to 13 us more of the host's time than a later
// call, 7 to 17 us to the end of the launch (one chunk of 512 rows, nine prompts, 100 prompts).
struct prompt_cost {
    double block, shared, ends, handoff, record;
    uint32_t per_cu;
};

prompt_cost cost_of(const pool_view& p, const prompt_form& form)
{
    if (p.dtype == CKV_F32 && form.fp4)
        return p.head_dim == 64 ? prompt_cost { 0.62, 0.07, 4.8, 3.8, 2.3, 2 }
            : p.head_dim == 128 ? prompt_cost { 1.3, 0.0, 2.2, 3.1, 0.8, 1 }
                                : prompt_cost { 2.9, 0.0, 5.5, 7.6, 2.3, 1 };
    if (p.dtype == CKV_F32)
        return p.head_dim == 64 ? prompt_cost { 1.6, 0.72, 0.1, 4.5, 0.4, 2 }
            : p.head_dim == 128 ? prompt_cost { 1.9, 0.0, 5.8, 0.3, 2.4, 1 }
                                : prompt_cost { 8.2, 0.0, 2.6, 5.9, 0.14, 1 };
    if (p.head_dim == 256)
        return { 1.2, 0.62, 7.8, 6.6, 1.8, 1 };
    if (p.head_dim == 64)
        return { 0.42, 0.27, 0.25, 2.8, 1.8, 2 };
    if (form.paged_kernel)
        return { 0.67, 0.0, 5.2, 6.3, 0.2, 2 };
    return { 0.82, 0.24, 1.4, 0.1, 1.5, 2 };
}

} // namespace

void write_prompt_list(const pool_view& p, const std::vector<uint32_t>& tiles, const prompt_form& form,
                       uint32_t q_heads, int cu_count, prompt_list& list)
{
    struct tile_rows {
        uint32_t blocks, row, rows, first, table;
    };
    const uint32_t rows = form.tile_rows(), units = q_heads / form.heads;
    std::vector<tile_rows> parts;
    uint32_t longest = 0;
    for (size_t t = 0; t < tiles.size(); t += tile_entry_words)
        for (uint32_t r = 0; r < tiles[t + 1]; r += rows) {
            const uint32_t n = std::min(rows, tiles[t + 1] - r), first = tiles[t + 2] + r;
            parts.push_back({ (first + n - 1) / block_keys + 1, tiles[t] + r, n, first, tiles[t + 3] });
            longest = std::max(longest, parts.back().blocks);
        }
    const prompt_cost cost = cost_of(p, form);
    const double cus = std::max(cu_count, 1);
    // the longest range of least time
    const auto ranges_of = [](uint32_t blocks, uint32_t most) { return (blocks + most - 1) / most; };
    const auto time_of = [&](uint32_t most) {
        double work = 0, workgroups = 0, records = 0;
        uint32_t longest_range = 0, most_ranges = 1;
        for (const tile_rows& t : parts) {
            const uint32_t n = ranges_of(t.blocks, most);
            work += units * (t.blocks + n * cost.ends);
            workgroups += (double)units * n;
            records += n > 1 ? (double)units * n : 0;
            longest_range = std::max(longest_range, (t.blocks + n - 1) / n);
            most_ranges = std::max(most_ranges, n);
        }
        const bool shared = cost.per_cu == 2 && workgroups > cus;
        const double block = cost.block * (shared ? 1 + cost.shared : 1);
        const double us = std::max((longest_range + cost.ends) * block, work * block / (cus * (shared ? 2 : 1)));
        // records are written and read, out of the caches, at about 8 bytes a picosecond
        return us + (most_ranges > 1 ? cost.handoff + most_ranges * cost.record
                             + records * 128 * (p.head_dim + 4) * 8 / 8e6 : 0.0);
    };
    uint32_t most = std::max(longest, 1u);
    if (form.waves == n_waves) {
        const auto length_of = [&](uint32_t n) { return std::max(ranges_of(longest, n), 1u); };
        double best = time_of(most);
        for (uint32_t n = 2; n <= prompt_most_ranges; ++n)
            if (const double us = time_of(length_of(n)); us < best) {
                best = us;
                most = length_of(n);
            }
        if (const char* forced = std::getenv("CKV_PREFILL_SPLIT"))
            most = length_of((uint32_t)std::clamp(std::strtol(forced, nullptr, 10), 1L, (long)prompt_most_ranges));
    }
    struct entry {
        uint32_t blocks;
        std::array<uint32_t, prompt_entry_words> words;
    };
    std::vector<entry> entries;
    list.n_records = list.n_cut = 0;
    for (const tile_rows& t : parts) {
        const uint32_t n = ranges_of(t.blocks, most);
        for (uint32_t i = 0; i < n; ++i)
            entries.push_back({ (t.blocks + n - 1) / n, { t.row, t.rows, t.first, t.table, i, n, list.n_records, list.n_cut } });
        if (n > 1) {
            list.n_records += n;
            ++list.n_cut;
        }
    }
    std::stable_sort(entries.begin(), entries.end(), [](const entry& a, const entry& b) { return a.blocks > b.blocks; });
    list.words.clear();
    for (const entry& e : entries)
        list.words.insert(list.words.end(), e.words.begin(), e.words.end());
}

hipError_t launch_prompt(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                         const prompt_rows& rows, const prompt_form& form, uint32_t q_heads, float scale,
                         void* out, const void* gate, bool fp4, const prefill_split& split)
{
    if (form.paged_kernel)
        return launch_prefill_rows(s, p, m, rows, q_heads, scale, out, gate, form.heads, form.waves, split);
    prompt_rows x = rows;
    set_vectors(p, x, out, gate, fp4);
    const auto launch = [&](auto src) {
        return launch_dim<decltype(src)::value>(p.head_dim, form.heads, s, p, m, layer, x, q_heads, scale, out, gate,
                                                split);
    };
    return fp4        ? launch(std::integral_constant<source, FROM_FP4> {})
        : x.vectors ? launch(std::integral_constant<source, FROM_WORDS> {})
                    : launch(std::integral_constant<source, FROM_ROWS> {});
}

} // namespace ckv
