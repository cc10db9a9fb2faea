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

constexpr uint32_t fp4_lane_waves = 8;

template <int D, int DT>
__global__ __launch_bounds__(64 * fp4_lane_waves, 2) void fp4_decode_kernel(
    pool_view p, meta_view m, uint32_t layer, const void* __restrict__ q, uint32_t q_heads, float scale_log2,
    void* __restrict__ out, const void* __restrict__ gate, split_scratch split, uint32_t passes)
{
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
    const uint32_t tiles_per_page = p.block_size / fp4_tile;
    constexpr uint32_t tile_bytes = fp4_tile_bytes(D);
    const uint64_t layer_bytes = (uint64_t)p.blocks * tiles_per_page * H * tile_bytes;
    const uint8_t* kl = static_cast<const uint8_t*>(p.keys) + layer * layer_bytes;
    const uint8_t* vl = static_cast<const uint8_t*>(p.values) + layer * layer_bytes;
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
        const uint32_t u_first = e1.x * tiles_per_page, u_last = position / fp4_tile;
        const uint32_t u_end = min(e1.y * tiles_per_page, u_last + 1);
        const uint32_t* tbl = m.table + (e0.w - e1.x); // the row's table

        // step s of the contraction: features 128i + 32g + 8w of s = 4i + w (64-wide: 16g + 8s)
        uint4 qv[KS];
#pragma unroll
        for (uint32_t s = 0; s < KS; ++s) {
            const uint32_t f = D == 64 ? 16 * g + 8 * s : s / 4 * 128 + 32 * g + s % 4 * 8;
            const uint64_t at = ((uint64_t)row * q_heads + qh0 + min(query, nq - 1)) * D + f;
            uint32_t w[4] = {};
            if (query < nq) {
                if constexpr (DT == CKV_BF16) {
                    if (term == 0)
                        for (int i = 0; i < 4; ++i) {
                            const uint16_t* e = static_cast<const uint16_t*>(q) + at + 2 * i;
                            w[i] = e[0] | (uint32_t)e[1] << 16;
                        }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        w[i] = split_terms(load_elem<DT>(q, at + 2 * i), load_elem<DT>(q, at + 2 * i + 1));
                }
            }
            qv[s] = make_uint4(w[0], w[1], w[2], w[3]);
        }

        float mx = -FLT_MAX, limit = -FLT_MAX, den = 0.0f;
        f32x4_t o[MT];
#pragma unroll
        for (uint32_t t = 0; t < MT; ++t)
            o[t] = f32x4_t {};

        auto load_tile = [&](uint32_t u, tile_t& x) {
            const uint64_t at = ((uint64_t)tbl[u / tiles_per_page] * H + kv_head) * tiles_per_page + u % tiles_per_page;
            const uint8_t* kb = kl + at * tile_bytes;
            const uint8_t* vb = vl + at * tile_bytes;
            if constexpr (D == 64) {
                const uint2 kk = *reinterpret_cast<const uint2*>(kb + c * 32 + g * 8);
                const uint2 vv = *reinterpret_cast<const uint2*>(vb + lane * 8);
                x.k[0] = kk.x;
                x.k[1] = kk.y;
                x.v[0] = vv.x;
                x.v[1] = vv.y;
                x.ks[0] = kb[8 * D + c * 2 + g / 2];
                x.vs[0] = *reinterpret_cast<const uint32_t*>(vb + 8 * D + c / 8 * 16 + g * 4);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < tile_t::parts; ++i) {
                    const uint4 kk = load_stream(kb + c * (D / 2) + i * 64 + g * 16);
                    const uint4 vv = load_stream(vb + i * 1024 + lane * 16);
                    x.k[4 * i] = kk.x;
                    x.k[4 * i + 1] = kk.y;
                    x.k[4 * i + 2] = kk.z;
                    x.k[4 * i + 3] = kk.w;
                    x.v[4 * i] = vv.x;
                    x.v[4 * i + 1] = vv.y;
                    x.v[4 * i + 2] = vv.z;
                    x.v[4 * i + 3] = vv.w;
                    x.ks[i] = kb[8 * D + c * (D / 32) + 4 * i + g];
                    x.vs[i] = *reinterpret_cast<const uint32_t*>(vb + 8 * D + (4 * i + c / 4) * 16 + g * 4);
                }
            }
        };
        // A tile past the segment's last: its tokens weigh nothing, its values are zeros.
        auto no_tile = [&](tile_t& x) {
#pragma unroll
            for (uint32_t i = 0; i < tile_t::words; ++i)
                x.k[i] = x.v[i] = 0;
#pragma unroll
            for (uint32_t i = 0; i < tile_t::parts; ++i)
                x.ks[i] = x.vs[i] = 0;
        };
        auto scores = [&](const tile_t& x) {
            f32x4_t s {};
#pragma unroll
            for (uint32_t i = 0; i < KS; ++i)
                s = mfma16(fp4_eight<false>(x.k[i], fp4_scale(x.ks[i / 4])), qv[i], s);
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
        auto process = [&](tile_t& a, tile_t& b, uint32_t u) {
            const bool two = u + 1 < u_end;
            f32x4_t sa = scores(a), sb = scores(b);
            float t[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                t[i] = terms_sum<TERMS>(sa[i]) * scale_log2;
                t[4 + i] = terms_sum<TERMS>(sb[i]) * scale_log2;
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
                const float alpha = fast_exp2(mx - nm);
                den *= alpha;
#pragma unroll
                for (uint32_t i = 0; i < MT; ++i)
                    o[i] *= alpha;
                mx = nm;
                limit = nm + 8.0f; // probabilities up to 2^8 weigh as exactly
            }
            float pr[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                pr[i] = fast_exp2(t[i] - mx);
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
        };
        auto load_two = [&](uint32_t u, tile_t& a, tile_t& b) {
            load_tile(u, a);
            if (u + 1 < u_end)
                load_tile(u + 1, b);
            else
                no_tile(b);
        };
        tile_t a0, b0, a1, b1;
        uint32_t u = u_first + 2 * wave;
        if (u < u_end)
            load_two(u, a0, b0);
        while (u < u_end) {
            uint32_t next = u + 2 * W;
            if (next < u_end)
                load_two(next, a1, b1);
            process(a0, b0, u);
            u = next;
            if (u >= u_end)
                break;
            next = u + 2 * W;
            if (next < u_end)
                load_two(next, a0, b0);
            process(a1, b1, u);
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
        // n records of query j, features f .. f + 3, `stride` floats apart, folded online
        auto fold = [&](auto&& head_at, auto&& acc_at, uint32_t n, float& M, float& d, float (&x)[4]) {
            M = -FLT_MAX;
            d = 0.0f;
            x[0] = x[1] = x[2] = x[3] = 0.0f;
            for (uint32_t r0 = 0; r0 < n; r0 += 4) {
                float2 h[4];
                float4 v[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    h[i] = head_at(min(r0 + i, n - 1));
                    v[i] = acc_at(min(r0 + i, n - 1));
                    if (r0 + i >= n) { // (weights of 0 would make NaN of an infinity)
                        h[i] = make_float2(-FLT_MAX, 0.0f);
                        v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
                }
                const float nm = fmaxf(fmaxf(M, fmaxf(h[0].x, h[1].x)), fmaxf(h[2].x, h[3].x));
                const float keep = fast_exp2(M - nm);
                M = nm;
                d *= keep;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[e] *= keep;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const float weight = fast_exp2(h[i].x - nm);
                    d += h[i].y * weight;
                    x[0] += v[i].x * weight;
                    x[1] += v[i].y * weight;
                    x[2] += v[i].z * weight;
                    x[3] += v[i].w * weight;
                }
            }
        };
        auto waves_state = [&](uint32_t j, uint32_t f, float& M, float& d, float (&x)[4]) {
            fold([&](uint32_t r) { return *reinterpret_cast<const float2*>(lds + (r * GQ + j) * RF); },
                 [&](uint32_t r) { return *reinterpret_cast<const float4*>(lds + (r * GQ + j) * RF + 4 + f); }, W, M, d, x);
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
                waves_state(t / (D / 4), 4 * t % D, M, d, x);
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
                waves_state(j, f, M, d, x);
                agent_store4(rec, (j * RF + 4 + f) * 4, x[0], x[1], x[2], x[3]);
                if (f == 0)
                    agent_store4(rec, j * RF * 4, M, d, 0.0f, 0.0f);
            }
        }
        wait_vector_memory();
        __syncthreads();
        uint32_t* const arrivals = split.arrivals + ((uint64_t)m.split_first[row] * H + kv_head) * passes + pass;
        uint32_t* const last_flag = reinterpret_cast<uint32_t*>(lds);
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
        for (uint32_t t = tid; t < T4; t += blockDim.x) {
            const uint32_t j = t / (D / 4), f = 4 * t % D;
            float M, d, x[4];
            // (a descriptor for each record: a row's may span more than 4 GiB)
            auto at = [&](uint32_t r, uint32_t off) {
                return agent_load4(record_rsrc(records + (uint64_t)r * record_stride, nq * RF * 4), (j * RF + off) * 4);
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
                n_chunks, M, d, x);
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

decode_form fp4_decode_form()
{
    return { 2, 16, 32, 47, false };
}

uint32_t fp4_decode_passes(const pool_view& p, uint32_t q_heads)
{
    const uint32_t each = p.dtype == CKV_F32 ? 4 : 8, group = q_heads / p.kv_heads;
    return (group + each - 1) / each;
}

hipError_t launch_fp4_decode(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer, const void* q,
                             uint32_t q_heads, float scale, void* out, const void* gate, split_scratch split)
{
    if (!m.plan || (m.n_cut && (!split.records || !split.arrivals)))
        return hipErrorInvalidValue;
    const uint32_t passes = fp4_decode_passes(p, q_heads);
    const uint64_t grid = (uint64_t)m.n_plan * p.kv_heads * passes;
    if (!grid)
        return hipSuccess;
    if (grid > 0x7FFFFFFFull)
        return hipErrorInvalidValue;
    const uint32_t waves = fp4_lane_waves, queries = p.dtype == CKV_F32 ? 4 : 8;
    const size_t lds = (size_t)waves * queries * (p.head_dim + 4) * sizeof(float);
    auto launch = [&](auto* kernel) {
        kernel<<<(uint32_t)grid, 64 * waves, lds, s>>>(p, m, layer, q, q_heads, scale * log2e, out, gate, split, passes);
        return hipGetLastError();
    };
    auto typed = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        return p.dtype == CKV_F32 ? launch(fp4_decode_kernel<D, CKV_F32>)
            : p.dtype == CKV_BF16 ? launch(fp4_decode_kernel<D, CKV_BF16>)
                                  : launch(fp4_decode_kernel<D, CKV_F16>);
    };
    return p.head_dim == 64 ? typed(std::integral_constant<int, 64> {})
        : p.head_dim == 128 ? typed(std::integral_constant<int, 128> {})
                            : typed(std::integral_constant<int, 256> {});
}

} // namespace ckv
