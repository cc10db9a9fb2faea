// Paged GQA decode attention over keys and values held in 4 bits (fp4.h), on gfx950's
// matrix cores.
//
// One workgroup per (plan workgroup, kv head, pass): its waves share a segment of a row (the
// plan of kernels_decode.hip) two tiles of 16 tokens a step, each wave's next two in flight.
// Per two tiles, with v_mfma_f32_16x16x32_bf16:
//   S^T[token][column] = K . Q^T      D/32 a tile, A = K from its codes, B = the queries
//   O^T[feature][column] += V^T . P^T  D/16 for both, A = V from its codes
// The accumulator layout (lane (c, g): rows 4g .. 4g + 3 of column c) is the order in which
// the layout keeps V's tokens, so probabilities are operands where they were computed.
// A decode step has few queries, a column holds one of a query's terms: eight queries in two
// bf16 terms each (f32 pools: four in four), columns c and c + 8, whose products are added.
// So queries and probabilities keep 16 bits or more (f32: all) in products that would cost
// the same without: bf16 queries are their first term, f16 ones the sum of two, exactly.
//
// Bound by the vector ALU's conversions beside HBM: 17 bytes of a block become 32 operands
// by 16 conversions (V: and 16 permutes that pair a feature's tokens).
// Registers are at the bound of the waves that share a SIMD: bf16 forms of 128- and 256-wide heads
// spill 12 bytes a lane, float ones 20 and 16, outside the loop over tokens.
#include "decode_wg.h"
#include "fp4.h"

namespace ckv {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4_t mfma16(uint4 a, uint4 b, f32x4_t c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b)
{
    const f32x2_t v = { a, b };
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
}

// A value and those of the columns that hold its other terms, summed in each of them.
template <int TERMS>
__device__ __forceinline__ float terms_sum(float v)
{
    v += dpp<0x128>(v); // row_ror:8
    if constexpr (TERMS == 4)
        v += dpp<0x124>(v); // row_ror:4
    return v;
}

// A tile's codes and scales as a lane holds them.
template <int D>
struct fp4_lane {
    static constexpr uint32_t words = D / 32, parts = D == 256 ? 2 : 1;
    uint32_t k[words], v[words];
    uint32_t ks[parts], vs[parts];
};

// Waves of a workgroup, at most.
constexpr uint32_t fp4_waves_of(int head_dim)
{
    return head_dim == 256 ? 4 : 8;
}

// QT: the queries' type, the rows' or float (rotated and not rounded since).
template <int D, int DT, int QT>
__global__ __launch_bounds__(64 * fp4_waves_of(D), D == 256 ? 3 : 4) void fp4_decode_kernel(
    pool_view p, meta_view m, uint32_t layer, const void* __restrict__ q, uint32_t q_heads, float scale_log2,
    float q_sign, void* __restrict__ out, const void* __restrict__ gate, split_scratch split, uint32_t passes)
{
    constexpr bool SUMMED = QT != CKV_BF16; // bf16 queries stand whole in the columns of all terms
    constexpr int TERMS = DT == CKV_F32 ? 4 : 2, GQ = 16 / TERMS;
    constexpr uint32_t KS = D / 32, MT = D / 16, RF = D + 4;
    using tile_t = fp4_lane<D>;
    extern __shared__ float lds[];
    const uint32_t W = blockDim.x >> 6;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const uint32_t H = p.kv_heads, group = q_heads / H;
    const uint32_t kv_head = blockIdx.x % H, pass = blockIdx.x / H % passes;
    const uint32_t qh0 = kv_head * group + pass * GQ, nq = min((uint32_t)GQ, group - pass * GQ);
    const uint32_t page_log = __builtin_ctz(p.block_size / fp4_tile); // a page's tiles
    constexpr uint32_t tile_bytes = fp4_tile_bytes(D);
    const uint64_t layer_bytes = ((uint64_t)p.blocks * H << page_log) * tile_bytes;
    const uint8_t* kl = static_cast<const uint8_t*>(p.keys) + layer * layer_bytes;
    const uint8_t* vl = static_cast<const uint8_t*>(p.values) + layer * layer_bytes;
    const float slack = 8.0f / scale_log2;
    const bool q_vectors = (reinterpret_cast<uintptr_t>(q) & 15) == 0;
    // a term takes what the terms before it left: bits of each earlier rounding to subtract
    const uint32_t query = c % GQ, term = c / GQ;
    const uint32_t minus1 = term >= 1 ? ~0u : 0, minus2 = term >= 2 ? ~0u : 0, minus3 = term >= 3 ? ~0u : 0;
    // two floats' terms as a packed pair
    auto split_terms = [&](float a, float b) {
        uint32_t w = pack_bf16(a, b);
        auto left = [&](uint32_t mask) {
            a -= __builtin_bit_cast(float, w << 16 & mask);
            b -= __builtin_bit_cast(float, w & 0xFFFF0000u & mask);
            w = pack_bf16(a, b);
        };
        left(minus1);
        if constexpr (TERMS == 4) {
            left(minus2);
            left(minus3);
        }
        return w;
    };

    auto segment = [&](const uint4 e0, const uint4 e1) {
        const uint32_t row = e0.x, chunk = e0.y, position = e0.z, n_chunks = e1.z;
        const uint32_t u_first = e1.x << page_log, u_last = position / fp4_tile;
        const uint32_t u_end = min(e1.y << page_log, u_last + 1);
        const uint32_t* tbl = m.table + (e0.w - e1.x); // the row's table

        // step s of the contraction: features 128i + 32g + 8w of s = 4i + w (64-wide: 16g + 8s)
        // (256-wide heads keep them in LDS behind the records: 32 registers fewer let three
        // waves run on a SIMD in place of two)
        constexpr bool Q_LDS = D == 256;
        uint4* const q_lds = reinterpret_cast<uint4*>(lds + W * GQ * RF + 4);
        uint4 qv[KS];
        auto load_query = [&](uint32_t s) {
            const uint32_t f = D == 64 ? 16 * g + 8 * s : s / 4 * 128 + 32 * g + s % 4 * 8;
            const uint64_t at = ((uint64_t)row * q_heads + qh0 + min(query, nq - 1)) * D + f;
            float x[8];
            if (q_vectors) {
                float lo[4], hi[4];
                load4<QT>(q, at, lo);
                load4<QT>(q, at + 4, hi);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = lo[i];
                    x[4 + i] = hi[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[i] = load_elem<QT>(q, at + i);
            }
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // (a negative scale turns the sign, a scale of 0 leaves nothing)
                const float u = q_sign == 0.0f ? 0.0f : x[2 * i] * q_sign;
                const float v = q_sign == 0.0f ? 0.0f : x[2 * i + 1] * q_sign;
                w[i] = SUMMED ? split_terms(u, v) : pack_bf16(u, v);
            }
            return query < nq ? make_uint4(w[0], w[1], w[2], w[3]) : make_uint4(0, 0, 0, 0);
        };
        if constexpr (Q_LDS) {
            for (uint32_t s = wave; s < KS; s += W)
                q_lds[s * 64 + lane] = load_query(s);
        } else {
#pragma unroll
            for (uint32_t s = 0; s < KS; ++s)
                qv[s] = load_query(s);
        }

        // the running maximum of the scores (unscaled), and where it has to move: states start at
        // the lowest finite one, so that a score of -inf weighs 0 also where no other came yet
        float mx = -FLT_MAX, limit = -FLT_MAX, den = 0.0f;
        f32x4_t o[MT];
#pragma unroll
        for (uint32_t t = 0; t < MT; ++t)
            o[t] = f32x4_t {};

        auto tile_base = [&](uint32_t u) {
            using c32 = const __attribute__((address_space(4))) uint32_t;
            const uint64_t page = (uint64_t)*((c32*)(uintptr_t)tbl + (u >> page_log)) * H + kv_head;
            return ((page << page_log) + (u & ((1u << page_log) - 1))) * tile_bytes;
        };
        // Of a tile past the segment's last the last is loaded again.
        auto load_keys = [&](uint64_t base, tile_t& x) {
            const uint8_t* kb = kl + base;
            if constexpr (D == 64) {
                const uint2 kk = *reinterpret_cast<const uint2*>(kb + c * 32 + g * 8);
                x.k[0] = kk.x;
                x.k[1] = kk.y;
                x.ks[0] = kb[8 * D + c * 2 + g / 2];
            } else {
#pragma unroll
                for (uint32_t i = 0; i < tile_t::parts; ++i) {
                    const uint4 kk = load_stream(kb + c * (D / 2) + i * 64 + g * 16);
                    x.k[4 * i] = kk.x;
                    x.k[4 * i + 1] = kk.y;
                    x.k[4 * i + 2] = kk.z;
                    x.k[4 * i + 3] = kk.w;
                    x.ks[i] = kb[8 * D + c * (D / 32) + 4 * i + g];
                }
            }
        };
        auto load_values = [&](uint64_t base, tile_t& x) {
            const uint8_t* vb = vl + base;
            if constexpr (D == 64) {
                const uint2 vv = *reinterpret_cast<const uint2*>(vb + lane * 8);
                x.v[0] = vv.x;
                x.v[1] = vv.y;
                x.vs[0] = *reinterpret_cast<const uint32_t*>(vb + 8 * D + c / 8 * 16 + g * 4);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < tile_t::parts; ++i) {
                    const uint4 vv = load_stream(vb + i * 1024 + lane * 16);
                    x.v[4 * i] = vv.x;
                    x.v[4 * i + 1] = vv.y;
                    x.v[4 * i + 2] = vv.z;
                    x.v[4 * i + 3] = vv.w;
                    x.vs[i] = *reinterpret_cast<const uint32_t*>(vb + 8 * D + (4 * i + c / 4) * 16 + g * 4);
                }
            }
        };
        auto scores = [&](const tile_t& x) {
            f32x4_t s {};
            uint32_t at = lane;
            if constexpr (Q_LDS)
                asm volatile("" : "+v"(at)); // read in each step, not held
#pragma unroll
            for (uint32_t i = 0; i < KS; ++i)
                s = mfma16(fp4_eight<false>(x.k[i], fp4_scale(x.ks[i / 4])), Q_LDS ? q_lds[i * 64 + at] : qv[i], s);
            return s;
        };
        // the two operand words of a feature's four tokens: features 8c + 2j and + 1 of part i
        auto scale_of = [](uint32_t bytes, int t) {
            return __builtin_bit_cast(float, (t == 3 ? bytes >> 1 : bytes << (23 - 8 * t)) & 0x7F800000u);
        };
        auto value_pairs = [&](const tile_t& x, uint32_t i, int j, uint32_t (&even)[2], uint32_t (&odd)[2]) {
            uint32_t cv[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const float scale = scale_of(x.vs[i], t);
                if constexpr (D == 64) {
                    const uint32_t w = x.v[t / 2];
                    cv[t] = t % 2 ? (j ? fp4_bf16_pair<3>(w, scale) : fp4_bf16_pair<2>(w, scale))
                                  : (j ? fp4_bf16_pair<1>(w, scale) : fp4_bf16_pair<0>(w, scale));
                } else {
                    const uint32_t w = x.v[4 * i + t];
                    cv[t] = j == 0 ? fp4_bf16_pair<0>(w, scale) : j == 1 ? fp4_bf16_pair<1>(w, scale)
                        : j == 2   ? fp4_bf16_pair<2>(w, scale)
                                   : fp4_bf16_pair<3>(w, scale);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                even[h] = __builtin_amdgcn_perm(cv[2 * h + 1], cv[2 * h], 0x05040100);
                odd[h] = __builtin_amdgcn_perm(cv[2 * h + 1], cv[2 * h], 0x07060302);
            }
        };
        // A wave has one step's tiles in its registers: the next one's keys are on their way once
        // the scores are taken, its values once these are (two sets of registers would leave
        // a compute unit half its waves, which cover more of the latency).
        tile_t a, b;
        uint32_t u = u_first + 2 * wave;
        uint64_t base_a = 0, base_b = 0;
        auto find = [&](uint32_t at) {
            base_a = tile_base(at);
            base_b = tile_base(min(at + 1, u_end - 1));
        };
        if (u < u_end) {
            find(u);
            load_keys(base_a, a);
            load_keys(base_b, b);
            load_values(base_a, a);
            load_values(base_b, b);
        }
        if constexpr (Q_LDS)
            __syncthreads();
        while (u < u_end) {
            const uint32_t next = u + 2 * W;
            const bool two = u + 1 < u_end;
            const f32x4_t sa = scores(a), sb = scores(b);
            if (next < u_end) {
                find(next);
                load_keys(base_a, a);
                load_keys(base_b, b);
            }
            float t[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                t[i] = SUMMED ? terms_sum<TERMS>(sa[i]) : sa[i];
                t[4 + i] = SUMMED ? terms_sum<TERMS>(sb[i]) : sb[i];
            }
            if (!two || u + 1 >= u_last) { // the row's end
                const uint32_t first = u * fp4_tile + 4 * g; // the lane's first token
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    t[i] = first + i <= position ? t[i] : -INFINITY;
                    t[4 + i] = two && first + fp4_tile + i <= position ? t[4 + i] : -INFINITY;
                }
                // tokens that are not attended: finite values, whatever they hold
                auto keep = [&](uint32_t token) {
                    const uint32_t n = token <= position ? position - token + 1 : 0;
                    return n >= 4 ? ~0u : (1u << 8 * n) - 1;
                };
#pragma unroll
                for (uint32_t i = 0; i < tile_t::parts; ++i) {
                    a.vs[i] &= keep(first);
                    b.vs[i] &= two ? keep(first + fp4_tile) : 0;
                }
            }
            const float top = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])),
                                    fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
            if (__builtin_amdgcn_ballot_w64(top > limit)) {
                float nm = swap16(top, [](float x, float y) { return fmaxf(x, y); });
                nm = fmaxf(mx, swap32(nm, [](float x, float y) { return fmaxf(x, y); }));
                const float alpha = fast_exp2((mx - nm) * scale_log2);
                den *= alpha;
#pragma unroll
                for (uint32_t i = 0; i < MT; ++i)
                    o[i] *= alpha;
                mx = nm;
                limit = nm + slack; // probabilities up to 2^8 weigh as exactly
            }
            // (while every score was -inf: finite, or their weights would be NaN in place of 0)
            const float shift = fminf(-mx * scale_log2, FLT_MAX);
            float pr[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                pr[i] = fast_exp2(__builtin_fmaf(t[i], scale_log2, shift));
            den += ((pr[0] + pr[1]) + (pr[2] + pr[3])) + ((pr[4] + pr[5]) + (pr[6] + pr[7]));
            const uint4 pt = make_uint4(split_terms(pr[0], pr[1]), split_terms(pr[2], pr[3]),
                                        split_terms(pr[4], pr[5]), split_terms(pr[6], pr[7]));
#pragma unroll
            for (uint32_t i = 0; i < tile_t::parts; ++i)
#pragma unroll
                for (int j = 0; j < (D == 64 ? 2 : 4); ++j) {
                    uint32_t ae[2], ao[2], be[2], bo[2];
                    value_pairs(a, i, j, ae, ao);
                    value_pairs(b, i, j, be, bo);
                    f32x4_t& even = o[8 * i + 2 * j];
                    f32x4_t& odd = o[8 * i + 2 * j + 1];
                    even = mfma16(make_uint4(ae[0], ae[1], be[0], be[1]), pt, even);
                    odd = mfma16(make_uint4(ao[0], ao[1], bo[0], bo[1]), pt, odd);
                }
            if (next < u_end) {
                load_values(base_a, a);
                load_values(base_b, b);
            }
            u = next;
        }

        // the wave's state: a record [max, denominator, 0, 0, acc[D]] per query in LDS
        den = swap16(den, [](float x, float y) { return x + y; });
        den = swap32(den, [](float x, float y) { return x + y; });
#pragma unroll
        for (uint32_t t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o[t][i] = terms_sum<TERMS>(o[t][i]);
        if (c < nq) {
            float* dst = lds + (wave * GQ + c) * RF;
            if (g == 0)
                *reinterpret_cast<float2*>(dst) = make_float2(mx, den);
            // accumulator row 4g + i of operand t: feature 8(4g + i) + t (64-wide: 4(4g + i) + t)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                if constexpr (D == 64) {
                    *reinterpret_cast<float4*>(dst + 4 + 4 * (4 * g + i)) = make_float4(o[0][i], o[1][i], o[2][i], o[3][i]);
                } else {
#pragma unroll
                    for (uint32_t h = 0; h < MT / 4; ++h)
                        *reinterpret_cast<float4*>(dst + 4 + h / 2 * 128 + 8 * (4 * g + i) + h % 2 * 4) =
                            make_float4(o[4 * h][i], o[4 * h + 1][i], o[4 * h + 2][i], o[4 * h + 3][i]);
                }
            }
        }
        __syncthreads();
        // n records of a query, four features of theirs, folded online (what is at r >= n is
        // read, in bounds, but not used)
        auto fold = [&](auto&& head_at, auto&& acc_at, uint32_t n, float& M, float& d, float (&x)[4]) {
            M = -FLT_MAX;
            d = 0.0f;
            x[0] = x[1] = x[2] = x[3] = 0.0f;
            for (uint32_t r0 = 0; r0 < n; r0 += 4) {
                float2 h[4];
                float4 v[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    h[i] = head_at(r0 + i);
                    v[i] = acc_at(r0 + i);
                    if (r0 + i >= n) { // (weights of 0 would make NaN of an infinity)
                        h[i] = make_float2(-FLT_MAX, 0.0f);
                        v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
                }
                const float nm = fmaxf(fmaxf(M, fmaxf(h[0].x, h[1].x)), fmaxf(h[2].x, h[3].x));
                const float keep = fast_exp2((M - nm) * scale_log2);
                M = nm;
                d *= keep;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[e] *= keep;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const float weight = fast_exp2((h[i].x - nm) * scale_log2);
                    d += h[i].y * weight;
                    x[0] += v[i].x * weight;
                    x[1] += v[i].y * weight;
                    x[2] += v[i].z * weight;
                    x[3] += v[i].w * weight;
                }
            }
        };
        // the first n records in LDS (the waves', or the slices' below)
        auto states = [&](uint32_t n, uint32_t j, uint32_t f, float& M, float& d, float (&x)[4]) {
            const auto record = [&](uint32_t r) { return lds + (min(r, n - 1) * GQ + j) * RF; };
            fold([&](uint32_t r) { return *reinterpret_cast<const float2*>(record(r)); },
                 [&](uint32_t r) { return *reinterpret_cast<const float4*>(record(r) + 4 + f); }, n, M, d, x);
        };
        const uint64_t out_row = ((uint64_t)row * q_heads + qh0) * D;
        auto emit = [&](uint32_t t, const float (&x)[4], float d) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] = x[e] / d;
                if (gate)
                    y[e] *= sigmoid(load_elem<DT>(gate, out_row + 4 * t + e));
            }
            if ((reinterpret_cast<uintptr_t>(out) & (DT == CKV_F32 ? 15 : 7)) == 0) {
                store4<DT>(out, out_row + 4 * t, y);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    store_elem<DT>(out, out_row + 4 * t + e, y[e]);
            }
        };
        const uint32_t T4 = nq * (D / 4); // four features of a query each
        if (n_chunks == 1) {
            for (uint32_t t = tid; t < T4; t += blockDim.x) {
                float M, d, x[4];
                states(W, t / (D / 4), 4 * t % D, M, d, x);
                emit(t, x, d);
            }
            return;
        }
        // a chunk of a cut row: its record, counted in; the last folds them (decode_wg.h)
        const uint32_t record_stride = q_heads * RF;
        float* const records = split.records + ((uint64_t)m.split_first[row] * q_heads + qh0) * RF;
        {
            const __amdgpu_buffer_rsrc_t rec = record_rsrc(records + (uint64_t)chunk * record_stride, nq * RF * 4);
            for (uint32_t t = tid; t < T4; t += blockDim.x) {
                const uint32_t j = t / (D / 4), f = 4 * t % D;
                float M, d, x[4];
                states(W, j, f, M, d, x);
                agent_store4(rec, (j * RF + 4 + f) * 4, x[0], x[1], x[2], x[3]);
                if (f == 0)
                    agent_store4(rec, j * RF * 4, M, d, 0.0f, 0.0f);
            }
        }
        wait_vector_memory();
        __syncthreads();
        uint32_t* const arrivals = split.arrivals + ((uint64_t)m.split_first[row] * H + kv_head) * passes + pass;
        uint32_t* const last_flag = reinterpret_cast<uint32_t*>(lds + W * GQ * RF);
        if (tid == 0) {
            const uint32_t before = __hip_atomic_fetch_add(arrivals, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            const uint32_t last = before == n_chunks - 1;
            if (last)
                __hip_atomic_store(arrivals, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            *last_flag = last;
        }
        __syncthreads();
        if (!*last_flag)
            return;
        // Thread (slice, j, f) folds records slice, slice + S, ... of query j; the slices are
        // folded through LDS. Slices enough for four records each, W of them fit.
        const uint32_t S = max(1u, min(min(blockDim.x / T4, W), (n_chunks + 3) / 4));
        for (uint32_t t = tid; t < S * T4; t += blockDim.x) {
            const uint32_t slice = t / T4, j = t % T4 / (D / 4), f = 4 * t % D;
            const uint32_t n = (n_chunks - slice + S - 1) / S;
            float M, d, x[4];
            // records r S .. r S + S - 1, those past the row's last out of the descriptor's range: 0
            auto at = [&](uint32_t r, uint32_t off) {
                const uint32_t first = r * S, left = first < n_chunks ? min(S, n_chunks - first) : 0;
                const __amdgpu_buffer_rsrc_t rec =
                    record_rsrc(records + (uint64_t)first * record_stride,
                                left ? ((left - 1) * record_stride + nq * RF) * 4 : 0);
                return agent_load4(rec, (slice * record_stride + j * RF + off) * 4);
            };
            fold(
                [&](uint32_t r) {
                    const u32x4_t h = at(r, 0);
                    return make_float2(__uint_as_float(h[0]), __uint_as_float(h[1]));
                },
                [&](uint32_t r) {
                    const u32x4_t v = at(r, 4 + f);
                    return make_float4(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]), __uint_as_float(v[3]));
                },
                n, M, d, x);
            if (S == 1) {
                emit(t, x, d);
                continue;
            }
            float* dst = lds + (slice * GQ + j) * RF;
            *reinterpret_cast<float4*>(dst + 4 + f) = make_float4(x[0], x[1], x[2], x[3]);
            if (f == 0)
                *reinterpret_cast<float2*>(dst) = make_float2(M, d);
        }
        if (S == 1)
            return;
        __syncthreads();
        for (uint32_t t = tid; t < T4; t += blockDim.x) {
            float M, d, x[4];
            states(S, t / (D / 4), 4 * t % D, M, d, x);
            emit(t, x, d);
        }
    };

    uint32_t at = blockIdx.x / H / passes;
    for (;;) {
        using c4 = const __attribute__((address_space(4))) u32x4_t;
        const auto* e = (c4*)(uintptr_t)(m.plan + plan_entry_words * at);
        const u32x4_t a = e[0], b = e[1];
        segment(make_uint4(a.x, a.y, a.z, a.w), make_uint4(b.x, b.y, b.z, b.w));
        at = b.w;
        if (at == plan_last)
            break;
        __syncthreads(); // the next segment's states reuse the LDS
    }
}

} // namespace

// Two workgroups a compute unit, chunks of 16 pages (one step of eight waves) at least, at
// most 32 of a row; a row up to 47 pages past its share stays whole: a segment costs a
// workgroup 3.5 us beside its pages, as much as 60 of them. As planned, in chunks of 16, 32
// and 64 pages, and whole, us: 48 rows of 900 to 12,000 tokens 69.5, 148, 102, 81 and 84; 128
// of 3,000 to 8,000 138, 327, 226, 179 and 137; 24 of 200 to 9,000 of 256-wide heads 23.2,
// 26.0, 21.9, 22.2 and 113; 4 of 60 to 1,900 8.7, 8.6, 9.0, 11.3 and 12.8; one of 16,000 12.8,
// 15.7, 12.5, 12.7 and 73; 8 of 4,000 13.1, 19.8, 14.0, 12.4 and 23.8.
decode_form fp4_decode_form()
{
    return { 2, 16, 32, 47, false };
}

// A pass reads the cache again. 48 rows of 900 to 12,000 tokens, 8 KV heads, us: groups of 1, 2, 4
// and 8 query heads 72, 74, 75 and 77, of 9 and 16 (two passes) 124 and 127, of 32 (four) 205;
// float rows, groups of 1, 2 and 4 81, 82 and 85, of 8 (two) 133, of 16 (four) 238.
uint32_t fp4_decode_passes(const pool_view& p, uint32_t q_heads)
{
    const uint32_t each = p.dtype == CKV_F32 ? 4 : 8, group = q_heads / p.kv_heads;
    return (group + each - 1) / each;
}

hipError_t launch_fp4_decode(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer, const void* q,
                             bool float_queries, uint32_t q_heads, float scale, void* out, const void* gate,
                             split_scratch split)
{
    if (!m.plan || (m.n_cut && (!split.records || !split.arrivals)))
        return hipErrorInvalidValue;
    const uint32_t passes = fp4_decode_passes(p, q_heads);
    const uint64_t grid = (uint64_t)m.n_plan * p.kv_heads * passes;
    if (!grid)
        return hipSuccess;
    if (grid > 0x7FFFFFFFull)
        return hipErrorInvalidValue;
    const uint32_t waves = fp4_waves_of(p.head_dim), queries = p.dtype == CKV_F32 ? 4 : 8;
    const size_t lds = ((size_t)waves * queries * (p.head_dim + 4) + 4) * sizeof(float)
        + (p.head_dim == 256 ? 8192 : 0);
    const float scale_log2 = scale == 0.0f ? log2e : std::fabs(scale) * log2e;
    const float sign = scale == 0.0f ? 0.0f : scale < 0.0f ? -1.0f : 1.0f;
    auto launch = [&](auto* kernel) {
        kernel<<<(uint32_t)grid, 64 * waves, lds, s>>>(p, m, layer, q, q_heads, scale_log2, sign, out, gate, split, passes);
        return hipGetLastError();
    };
    auto typed = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        if (p.dtype == CKV_F32)
            return launch(fp4_decode_kernel<D, CKV_F32, CKV_F32>);
        if (p.dtype == CKV_BF16)
            return float_queries ? launch(fp4_decode_kernel<D, CKV_BF16, CKV_F32>)
                                 : launch(fp4_decode_kernel<D, CKV_BF16, CKV_BF16>);
        return float_queries ? launch(fp4_decode_kernel<D, CKV_F16, CKV_F32>)
                             : launch(fp4_decode_kernel<D, CKV_F16, CKV_F16>);
    };
    return p.head_dim == 64 ? typed(std::integral_constant<int, 64> {})
        : p.head_dim == 128 ? typed(std::integral_constant<int, 128> {})
                            : typed(std::integral_constant<int, 256> {});
}

} // namespace ckv
