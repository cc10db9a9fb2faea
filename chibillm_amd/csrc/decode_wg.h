// The fast paged GQA decode (kernels_decode.hip, kernels_decode_window.hip): the
// kernel, its waves and its launch. HIP device code.
#pragma once

#include "ckv_internal.h"
#include "prefill_records.h"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdlib>
#include <type_traits>

namespace ckv {
namespace {

constexpr float log2e = 1.4426950408889634f;

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// K/V pages are read once per decode step: nontemporal loads stream them
// past the caches (measured on MI355X: plain 16-byte streaming reads top out
// near 6.4 TB/s, nontemporal ones near 6.9 TB/s).
__device__ __forceinline__ uint4 load_stream(const void* p)
{
    const u32x4_t t = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p));
    return make_uint4(t.x, t.y, t.z, t.w);
}

// The eight elements of one K, V or query head row (D features) a lane of the
// fast decode holds: lane part p (of D / 8) takes the 16 bytes at 16p, features
// 8p..8p+7 of a 16-bit row; of an f32 row (the reference's storage,
// src/metal/metal_kv_cache.cc:57-69) also the 16 bytes at 2D + 16p, so its
// features are 4p..4p+3 and D/2+4p..D/2+4p+3. Either way each 16-byte load
// instruction of D / 8 lanes reads 2D contiguous bytes of the row.
template <int DT, int D>
struct lane8 {
    static constexpr int dtype = DT;
    static constexpr uint32_t words = DT == CKV_F32 ? 2 : 1;
    static constexpr uint32_t elem = DT == CKV_F32 ? 4 : 2; // bytes per element
    static constexpr uint32_t stride = 2 * D;               // bytes between the words
    uint4 w[words];
    // the head feature of the lane's element i (of 8), for lane part p
    static __device__ __forceinline__ uint32_t feature(uint32_t p, uint32_t i)
    {
        return DT == CKV_F32 ? (i < 4 ? 4 * p + i : D / 2 + 4 * p + (i - 4)) : 8 * p + i;
    }
};

template <class Row>
__device__ __forceinline__ Row load8_stream(const char* p)
{
    Row x;
#pragma unroll
    for (uint32_t i = 0; i < Row::words; ++i)
        x.w[i] = load_stream(p + Row::stride * i);
    return x;
}

template <class Row>
__device__ __forceinline__ Row load8(const char* p)
{
    Row x;
#pragma unroll
    for (uint32_t i = 0; i < Row::words; ++i)
        x.w[i] = *reinterpret_cast<const uint4*>(p + Row::stride * i);
    return x;
}

template <class Row>
__device__ __forceinline__ void store8(char* p, const Row& x)
{
#pragma unroll
    for (uint32_t i = 0; i < Row::words; ++i)
        *reinterpret_cast<uint4*>(p + Row::stride * i) = x.w[i];
}

__device__ __forceinline__ float fast_exp2(float x)
{
    return __builtin_amdgcn_exp2f(x);
}

// The split-K handoff between workgroups (a cut row's chunks store partial
// records, count themselves in, and the last to arrive merges) is a protocol
// of this target's memory system, not a release/acquire pair of the HIP
// memory model:
//   - records are written and read 16 bytes at a time with the sc1 cache policy
//     (prefill_records.h): what relaxed agent-scope atomic accesses carry on
//     gfx950 (the GFX942 rows of LLVM's AMDGPU memory model), which write
//     through and bypass any L2 line that could be stale, so every XCD sees
//     them in memory without an L2 writeback;
//   - each writer waits with s_waitcnt vmcnt(0) for its stores to complete
//     (on GFX9-family parts vmcnt counts stores too) before one thread's
//     relaxed agent-scope fetch-add counts the chunk in; the last arriver's
//     loads are issued after that RMW returns.
// A model-level handoff costs far more here: an agent-scope release lowers to
// buffer_wbl2 sc1, a writeback of the XCD's L2 (a release RMW +27 % and an
// acq_rel RMW +29 % on config 2's decode; a separate merge launch +1.3 %;
// an acquire fence in the last arriver alone +1.5 %). The guard below keeps
// the protocol off targets where the vmcnt wait would not cover stores
// (GFX10+, which count them with vscnt) or where sc1 means something else.
#if defined(__HIP_DEVICE_COMPILE__) && !defined(__gfx950__)
#error "kernels_decode.hip's split-K handoff relies on gfx950's memory system; build for gfx950"
#endif

// f32 -> bf16 round to nearest even, NaN quieted (src/tensor/types.h:60-75).
__device__ __forceinline__ uint32_t bf16_bits(float x)
{
    uint32_t b = __builtin_bit_cast(uint32_t, x);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u)
        return (b >> 16) | 0x40u;
    b += 0x7FFFu + ((b >> 16) & 1u);
    return b >> 16;
}

__device__ __forceinline__ uint32_t f16_bits(float x)
{
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
}

// 1 / (1 + e^-g) in float, the gate of silu_mul_f32 with sigmoid_only
// (src/metal/kernels/tensor_ops.metal:108-124): 0 and 1 at the extremes.
__device__ __forceinline__ float sigmoid(float g)
{
    return 1.0f / (1.0f + fast_exp2(-g * log2e));
}

template <bool F16>
__device__ __forceinline__ float half_value(uint16_t bits)
{
    if constexpr (F16)
        return static_cast<float>(__builtin_bit_cast(_Float16, bits));
    else
        return __builtin_bit_cast(float, static_cast<uint32_t>(bits) << 16);
}

template <bool F16>
struct half2_ops;

template <>
struct half2_ops<false> { // bf16
    static __device__ __forceinline__ float lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
    static __device__ __forceinline__ float hi(uint32_t w)
    {
        return __builtin_bit_cast(float, w & 0xFFFF0000u);
    }
    static __device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c)
    {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, a),
                                               __builtin_bit_cast(bf16x2_t, b), c, false);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        return bf16_bits(a) | (bf16_bits(b) << 16);
    }
};

template <>
struct half2_ops<true> { // fp16
    static __device__ __forceinline__ float lo(uint32_t w)
    {
        return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w)));
    }
    static __device__ __forceinline__ float hi(uint32_t w)
    {
        return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w >> 16)));
    }
    static __device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c)
    {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, a),
                                      __builtin_bit_cast(f16x2_t, b), c, false);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        return f16_bits(a) | (f16_bits(b) << 16);
    }
};

template <int CTRL>
__device__ __forceinline__ float dpp(float v)
{
    return __builtin_amdgcn_update_dpp(0.0f, v, CTRL, 0xF, 0xF, false);
}

// Sum over each row of 16 lanes, result in every lane of the row.
__device__ __forceinline__ float row16_sum(float v)
{
    v += dpp<0xB1>(v);  // quad_perm [1,0,3,2]
    v += dpp<0x4E>(v);  // quad_perm [2,3,0,1]
    v += dpp<0x141>(v); // row_half_mirror
    v += dpp<0x140>(v); // row_mirror
    return v;
}

// A value combined with the one 32 (16) lanes away, in every lane.
template <class Op>
__device__ __forceinline__ float swap32(float v, Op op)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto sw = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return op(__builtin_bit_cast(float, (uint32_t)sw[0]), __builtin_bit_cast(float, (uint32_t)sw[1]));
}

template <class Op>
__device__ __forceinline__ float swap16(float v, Op op)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto sw = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    return op(__builtin_bit_cast(float, (uint32_t)sw[0]), __builtin_bit_cast(float, (uint32_t)sw[1]));
}

// Sum over each group of LANES lanes (16 or 32), result in every lane of it.
template <uint32_t LANES>
__device__ __forceinline__ float lanes_sum(float v)
{
    static_assert(LANES == 16 || LANES == 32);
    v = row16_sum(v);
    if constexpr (LANES == 32)
        v = swap16(v, [](float a, float b) { return a + b; });
    return v;
}

// Of two values the sums over lanes l and l ^ 32: a's in lanes 0..31, b's in
// lanes 32..63 (the swap exchanges a's upper half with b's lower one); and
// over lanes l and l ^ 16: a's in the even rows of 16 lanes, b's in the odd.
__device__ __forceinline__ float scatter32(float a, float b)
{
    const auto sw = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a),
                                                     __builtin_bit_cast(uint32_t, b), false, false);
    return __builtin_bit_cast(float, (uint32_t)sw[0]) + __builtin_bit_cast(float, (uint32_t)sw[1]);
}

__device__ __forceinline__ float scatter16(float a, float b)
{
    const auto sw = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, a),
                                                     __builtin_bit_cast(uint32_t, b), false, false);
    return __builtin_bit_cast(float, (uint32_t)sw[0]) + __builtin_bit_cast(float, (uint32_t)sw[1]);
}

// Partial record per (work item, q head): [max, denominator, 0, 0, acc[D]].
__host__ __device__ constexpr uint32_t record_floats(uint32_t head_dim)
{
    return head_dim + 4;
}

// Workgroups whose lanes need more than 128 registers (more than two q heads
// per KV head, or f32 pages, whose double-buffered K/V words alone take 128)
// run at most 8 waves, two per SIMD, with up to 256 registers a lane.
__host__ __device__ constexpr bool wide_lanes(uint32_t group, int dtype)
{
    return group > 2 || dtype == CKV_F32;
}

// Eight q heads of f32 pages do not fit 256 registers a lane (the kernel
// would spill): such pools run the four-head kernel twice (launch_fast<8>).
__host__ __device__ constexpr bool fast_fits(uint32_t group, int dtype)
{
    return !(group == 8 && dtype == CKV_F32);
}

// q . k over a lane's eight elements (16-bit pairs by v_dot2 with fp32
// accumulation; f32 by fused multiply-adds), and a V row widened to floats.
template <class Row>
__device__ __forceinline__ float dot8(const Row& q, const Row& k)
{
    constexpr int DT = Row::dtype;
    if constexpr (DT == CKV_F32) {
        float d = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            d = __builtin_fmaf(__builtin_bit_cast(float, q.w[i].x), __builtin_bit_cast(float, k.w[i].x), d);
            d = __builtin_fmaf(__builtin_bit_cast(float, q.w[i].y), __builtin_bit_cast(float, k.w[i].y), d);
            d = __builtin_fmaf(__builtin_bit_cast(float, q.w[i].z), __builtin_bit_cast(float, k.w[i].z), d);
            d = __builtin_fmaf(__builtin_bit_cast(float, q.w[i].w), __builtin_bit_cast(float, k.w[i].w), d);
        }
        return d;
    } else {
        using ops = half2_ops<DT == CKV_F16>;
        float d = ops::dot2(q.w[0].x, k.w[0].x, 0.0f);
        d = ops::dot2(q.w[0].y, k.w[0].y, d);
        d = ops::dot2(q.w[0].z, k.w[0].z, d);
        return ops::dot2(q.w[0].w, k.w[0].w, d);
    }
}

template <class Row>
__device__ __forceinline__ void widen8(const Row& v, float (&f)[8])
{
    constexpr int DT = Row::dtype;
    if constexpr (DT == CKV_F32) {
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            f[4 * i + 0] = __builtin_bit_cast(float, v.w[i].x);
            f[4 * i + 1] = __builtin_bit_cast(float, v.w[i].y);
            f[4 * i + 2] = __builtin_bit_cast(float, v.w[i].z);
            f[4 * i + 3] = __builtin_bit_cast(float, v.w[i].w);
        }
    } else {
        using ops = half2_ops<DT == CKV_F16>;
        const uint4 w = v.w[0];
        f[0] = ops::lo(w.x); f[1] = ops::hi(w.x); f[2] = ops::lo(w.y); f[3] = ops::hi(w.y);
        f[4] = ops::lo(w.z); f[5] = ops::hi(w.z); f[6] = ops::lo(w.w); f[7] = ops::hi(w.w);
    }
}

// One element of a pool-dtype row (gate, output, generic-path operands) as
// float, and back (one rounding, to nearest even).
template <int DT>
__device__ __forceinline__ float load_elem(const void* base, uint64_t i)
{
    if constexpr (DT == CKV_F32)
        return static_cast<const float*>(base)[i];
    else if constexpr (DT == CKV_BF16)
        return __builtin_bit_cast(float, (uint32_t)static_cast<const uint16_t*>(base)[i] << 16);
    else
        return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<const uint16_t*>(base)[i]));
}

// Four consecutive elements, 4-element aligned.
template <int DT>
__device__ __forceinline__ void load4(const void* base, uint64_t i, float (&x)[4])
{
    if constexpr (DT == CKV_F32) {
        const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
        x[0] = v.x;
        x[1] = v.y;
        x[2] = v.z;
        x[3] = v.w;
    } else {
        using ops = half2_ops<DT == CKV_F16>;
        const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + i);
        x[0] = ops::lo(v.x);
        x[1] = ops::hi(v.x);
        x[2] = ops::lo(v.y);
        x[3] = ops::hi(v.y);
    }
}

template <int DT>
__device__ __forceinline__ void store4(void* base, uint64_t i, const float (&x)[4])
{
    if constexpr (DT == CKV_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(base) + i) =
            make_float4(x[0], x[1], x[2], x[3]);
    } else {
        using ops = half2_ops<DT == CKV_F16>;
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + i) =
            make_uint2(ops::pack(x[0], x[1]), ops::pack(x[2], x[3]));
    }
}

template <int DT>
__device__ __forceinline__ void store_elem(void* base, uint64_t i, float x)
{
    if constexpr (DT == CKV_F32)
        static_cast<float*>(base)[i] = x;
    else if constexpr (DT == CKV_BF16)
        static_cast<uint16_t*>(base)[i] = static_cast<uint16_t>(bf16_bits(x));
    else
        static_cast<uint16_t*>(base)[i] = static_cast<uint16_t>(f16_bits(x));
}

// Fast path, one workgroup per (plan workgroup, kv_head), W waves. A
// workgroup runs its plan segments one after another: each a row, or a piece
// (a run of pages) of a row that the plan cuts (the split-K of
// paged_attention_partial_f32 / paged_attention_reduce_f32,
// src/metal/kernels/attention.metal:446-615, for any row). With FUSED, the
// row's new token (position = the row's last) is taken from k_in/v_in rows
// instead of the cache and stored into its slot by the wave that owns the
// last page: the append of store_kv and the attention in one pass. Wave w
// walks pages first+w, first+w+W, ... of its segment (16-token pages, one
// scalar table read per page); the next page's K/V loads are issued before the
// current page is processed. Lane 16*group + part reads features 8*part..8*part+7 of token
// 4j + group of the page (j = 0..3): four 1 KiB wave loads per page for K and
// four for V (256-wide heads: lane 32*group + part, token 2j + group of half a
// page; pages below stand for these units). The wave's row-group softmax states
// are reduced and scattered by lane swaps, the W wave states merged through
// LDS, and the workgroup writes the normalised output of the group's q heads.
// GATED multiplies it by sigmoid(gate) first; the gate values are loaded after
// the last page, into its registers, so that their latency hides behind the
// merge. A chunk of a cut row writes its unnormalised state instead (a partial
// record per q head) with 16-byte write-through stores (prefill_records.h) and
// counts itself in; the chunk that arrives last merges
// the row's records in the same launch. (An agent-scope release fence per
// workgroup would write back the XCD's whole L2, measured at about 1.9 us per
// workgroup per XCD; stores that are coherent on their own need only a wait
// for completion before the count.) ROPE (with FUSED) rotates the
// queries and the new token's key by the row's position first, as rope_f32
// (src/metal/kernels/tensor_ops.metal:158-195) would: feature f < rotary/2
// pairs with f + rotary/2, which sits in the lane part ^ (rotary/16) of the
// same row's lanes, so one lane exchange per register rotates a head. WINDOW: the
// row's pages are those with a key it attends (key_window); the plan counts them
// without the gap between its sinks and its window, and so do the units below,
// except where their tokens are read or compared. Keys of the pages at the gap's
// edges that the row does not attend are masked as those past its end are: a
// score of -inf, and a value of 0 in place of whatever they hold.
template <int D, int G, int DT, bool FUSED, bool GATED, bool ROPE, bool WINDOW>
__global__ __launch_bounds__(wide_lanes(G, DT) ? 512 : 1024, wide_lanes(G, DT) ? 2 : 4) void decode_wg_kernel(
    pool_view p, meta_view m, uint32_t layer, const char* __restrict__ q, uint32_t q_heads,
    float scale_log2, void* __restrict__ out, const char* __restrict__ k_in,
    const char* __restrict__ v_in, const void* __restrict__ gate, rope_pairs<D / 2> freq,
    uint32_t rotary, split_scratch split, uint32_t group_stride, uint32_t head_base)
{
    static_assert(!(ROPE && DT == CKV_F32), "the fused rotation works on 16-bit pairs");
    constexpr bool F16 = DT == CKV_F16;
    using ops = half2_ops<F16>;
    using row8 = lane8<DT, D>;
    constexpr uint32_t ES = row8::elem;
    constexpr uint32_t BS = 16;
    // A wave reads ROWS token rows of LANES lanes per load instruction, and a
    // unit of UT tokens (a page, or half of one of 256-wide heads) with four.
    constexpr uint32_t LANES = D / 8, ROWS = 64 / LANES;
    constexpr uint32_t UT = 4 * ROWS, UPP = BS / UT; // units per page
    static_assert(UT * UPP == BS);
    extern __shared__ float lds[];
    const uint32_t W = blockDim.x >> 6;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); // a scalar
    const uint32_t H = p.kv_heads;
    const uint32_t kv_head = blockIdx.x % H;
    // the workgroup's q heads: qh0 .. qh0 + G - 1 (group_stride = G and
    // head_base = 0, or one of the passes over half of a larger group)
    const uint32_t qh0 = kv_head * group_stride + head_base;
    const uint32_t row_bytes = p.features * ES;
    const uint64_t page_bytes = (uint64_t)BS * row_bytes;
    const char* kl = static_cast<const char*>(p.keys) + (uint64_t)layer * p.layer_elems * ES;
    const char* vl = static_cast<const char*>(p.values) + (uint64_t)layer * p.layer_elems * ES;
    // the layer's bases and the table are known from the arguments alone: load
    // them now, beside the plan entry, not after it
    asm volatile("" ::"s"(kl), "s"(vl), "s"(m.table), "s"(row_bytes), "s"(q));

    // a gate aligned for vector loads (only the pool, queries and output need be)
    const bool gate_vectors = GATED && (reinterpret_cast<uintptr_t>(gate) & (4 * ES - 1)) == 0;

    // One segment: pages [pg_first, pg_end) of a row, chunk `chunk` of the
    // row's n_chunks (e0 = row, chunk, the row's position, the flat table
    // index of page pg_first; e1 = pg_first, pg_end, n_chunks, next entry).
    auto segment = [&](const uint4 e0, const uint4 e1) {
        // The lane's index, computed anew in each segment (a volatile asm, so it
        // is not held in a register across the segment loop), and the thread's.
        uint32_t lane;
        asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
        const uint32_t tid = wave * 64 + lane;
        const uint32_t group = lane / LANES;
        const uint32_t part = lane % LANES;
        const uint32_t head_off = kv_head * (D * ES) + part * 16u; // the lane's first word
        const uint32_t row = e0.x;
        const uint32_t chunk = e0.y;
        const uint32_t position = e0.z;
        // the window's first key, and the units from u_kept on that are left out
        const uint32_t low = WINDOW ? window_low(position, m.window) : 0;
        const window_gap gap = WINDOW ? window_gap_of(low, m.window.sinks, BS) : window_gap {};
        const uint32_t u_kept = gap.kept * UPP, u_skip = gap.skip * UPP;
        const uint32_t u_last = position / UT - u_skip; // the row's last unit
        auto in_table = [&](uint32_t u) { return WINDOW && u >= u_kept ? u + u_skip : u; };
        const uint32_t last_in_unit = position % UT;
        const uint32_t pg_first = e1.x;
        const uint32_t u_end = UPP == 1 ? e1.y : min(e1.y * UPP, u_last + 1);
        const uint32_t n_chunks = e1.z;
        const uint32_t* tbl = m.table + (e0.w - pg_first); // the row's table

        row8 qv[G];
#pragma unroll
        for (int g = 0; g < G; ++g)
            qv[g] = load8<row8>(q + ((uint64_t)row * q_heads + qh0 + g) * D * ES + part * 16);

        // ROPE: this lane's 8 features (pairs j0 .. j0 + 7) and their rotation;
        // every lane of the wave takes part in the exchanges. The queries and the
        // new token's key share the row's position: both are rotated while the
        // wave's first page loads, and the rotated key (this lane's 16 bytes of
        // it) takes the new token's place when the last page is processed. The
        // row's rotary/2 angles are computed once, by wave 0 (and 1), into LDS past
        // the merge area.
        const uint32_t rot_mask = ROPE ? rotary / 16 : 1; // lane parts per half of the rotary width
        const bool rot_on = ROPE && part < 2 * rot_mask;
        const bool rot_first = part < rot_mask;
        auto angles = [&](float (&rc)[8], float (&rs)[8]) {
            float* table = lds + W * G * (D + 2); // (cos, sin) per pair
            auto angle = [&](uint32_t j) {
                float sn, cs;
                sincosf(static_cast<float>(position) * freq.inv_freq[j], &sn, &cs);
                table[2 * j] = cs;
                table[2 * j + 1] = sn;
            };
            if (wave == 0 && lane < rotary / 2)
                angle(lane);
            if (D > 128 && wave == (W > 1) && 64 + lane < rotary / 2)
                angle(64 + lane);
            __syncthreads();
            const uint32_t j0 = 8 * (part & (rot_mask - 1));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                rc[e] = rot_on ? table[2 * (j0 + e)] : 1.0f;
                rs[e] = rot_on ? table[2 * (j0 + e) + 1] : 0.0f;
            }
        };
        auto rotate = [&](const uint4& w, const float (&rc)[8], const float (&rs)[8]) {
            const uint32_t in[4] = { w.x, w.y, w.z, w.w };
            uint32_t r[4];
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const uint32_t pw = __shfl_xor(in[d], (int)rot_mask);
                const float own[2] = { ops::lo(in[d]), ops::hi(in[d]) };
                const float par[2] = { ops::lo(pw), ops::hi(pw) };
                float x[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float ra, rb;
                    rope_pair(rot_first ? own[h] : par[h], rot_first ? par[h] : own[h],
                              rc[2 * d + h], rs[2 * d + h], ra, rb);
                    x[h] = rot_first ? ra : rb;
                }
                r[d] = rot_on ? ops::pack(x[0], x[1]) : in[d];
            }
            return make_uint4(r[0], r[1], r[2], r[3]);
        };
        const uint64_t in_row = (uint64_t)row * row_bytes + head_off;
        uint4 k_new = make_uint4(0, 0, 0, 0); // ROPE: the new token's key, rotated once loaded
        if constexpr (ROPE)
            k_new = load8<row8>(k_in + in_row).w[0];

        // A state starts at the lowest finite maximum, so that a score of -inf weighs
        // 2^-inf = 0 also where no other came yet (from -inf it would be NaN), and an
        // empty state, whose sums are 0, needs no test where states are merged.
        float mx[G], den[G], acc[G][8];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            mx[g] = -FLT_MAX;
            den[g] = 0.0f;
#pragma unroll
            for (int f = 0; f < 8; ++f)
                acc[g][f] = 0.0f;
        }

        // rows past the row's last token re-read that token (in bounds, written)
        auto load_unit = [&](uint32_t u, row8* k, row8* v) {
            const uint64_t base = (uint64_t)tbl[in_table(u) / UPP] * page_bytes;
            const uint32_t t0 = u % UPP * UT; // the unit's first token in its page
            const char* kb = kl + base;
            const char* vb = vl + base;
            const bool last_unit = u == u_last;
            const uint32_t last = last_unit ? last_in_unit : UT - 1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t r = min(ROWS * j + group, last);
                const uint32_t off = (t0 + r) * row_bytes + head_off;
                const bool fresh = FUSED && last_unit && r == last_in_unit;
                // ROPE: the new token's slot is read too and replaced in process
                k[j] = load8_stream<row8>(fresh && !ROPE ? k_in + in_row : kb + off);
                v[j] = load8_stream<row8>(fresh ? v_in + in_row : vb + off);
            }
        };

        auto process = [&](row8* k, const row8* v, uint32_t u) {
            const uint32_t valid = u == u_last ? last_in_unit + 1 : UT;
            if (FUSED && u == u_last) {
                if constexpr (ROPE) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (ROWS * j + group == last_in_unit)
                            k[j].w[0] = k_new;
                }
                // append: the lanes holding the new token write it into its slot
                const uint64_t base = (uint64_t)tbl[in_table(u) / UPP] * page_bytes;
                const uint32_t off = (u % UPP * UT + last_in_unit) * row_bytes + head_off;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (ROWS * j + group == last_in_unit) {
                        store8(const_cast<char*>(kl) + base + off, k[j]);
                        store8(const_cast<char*>(vl) + base + off, v[j]);
                    }
                }
            }
            bool ok[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                ok[j] = ROWS * j + group < valid;
            if constexpr (WINDOW) {
                // the unit's tokens from `from` on are in the window, those before
                // `held` are sinks
                const uint32_t t0 = in_table(u) * UT;
                const uint32_t from = low > t0 ? low - t0 : 0;
                const uint32_t held = m.window.sinks > t0 ? m.window.sinks - t0 : 0;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    ok[j] = ok[j] && (ROWS * j + group >= from || ROWS * j + group < held);
            }
            float pw[G][4];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float s[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float r = lanes_sum<LANES>(dot8(qv[g], k[j])) * scale_log2;
                    s[j] = ok[j] ? r : -INFINITY;
                }
                const float nm = fmaxf(mx[g], fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
                // rescale only when some lane's running max grew (alpha is 1 elsewhere)
                if (__builtin_amdgcn_ballot_w64(nm > mx[g])) {
                    const float alpha = fast_exp2(mx[g] - nm);
                    den[g] *= alpha;
#pragma unroll
                    for (int f = 0; f < 8; ++f)
                        acc[g][f] *= alpha;
                    mx[g] = nm;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    pw[g][j] = fast_exp2(s[j] - mx[g]);
                den[g] += (pw[g][0] + pw[g][1]) + (pw[g][2] + pw[g][3]);
            }
            // token by token: widen the V row once, accumulate it into every q head
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // A lane past the row's end re-read the last token: at weight 0 an
                // infinite value of it would become NaN, so it takes 0. (Selects
                // in every unit, at most 1.5 % of a launch: selects in a branch for
                // the last unit cost 256-wide rows 2.3 % in register copies, a
                // source of zeros 5.5 % and one long row 6 % in addresses, a copy
                // of the unit's code spills. f32 words are selected once widened; before,
                // they spill.)
                float vf[8];
                row8 vj = v[j];
                if constexpr (DT != CKV_F32) {
#pragma unroll
                    for (uint32_t i = 0; i < row8::words; ++i)
                        vj.w[i] = ok[j] ? vj.w[i] : make_uint4(0, 0, 0, 0);
                }
                widen8(vj, vf);
                if constexpr (DT == CKV_F32) {
#pragma unroll
                    for (int f = 0; f < 8; ++f)
                        vf[f] = ok[j] ? vf[f] : 0.0f;
                }
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int f = 0; f < 8; ++f)
                        acc[g][f] += pw[g][j] * vf[f];
            }
        };

        row8 ka[4], va[4], kb[4], vb[4];
        uint32_t u = pg_first * UPP + wave;
        if (u < u_end)
            load_unit(u, ka, va);
        // ROPE: rotate the queries and the new key while the first page loads
        if constexpr (ROPE) {
            float rc[8], rs[8];
            angles(rc, rs);
#pragma unroll
            for (int g = 0; g < G; ++g)
                qv[g].w[0] = rotate(qv[g].w[0], rc, rs);
            k_new = rotate(k_new, rc, rs);
        }
        // Issue arbitration favours older waves: with a fixed priority the
        // workgroup's youngest waves finish their pages last while the others
        // wait (in config 3's workgroups, 13.6 us median between wave 0's last
        // page and the workgroup's end). Each wave steps through the four
        // priority levels page by page, starting at its own index, so every
        // wave takes its turn at the top (5.1 us; launches 1.2-2 % shorter).
        // The pages each wave reads, and so the results, do not change.
        uint32_t turn = wave;
        auto rotate_priority = [&]() {
            switch (turn++ & 3) {
            case 0:
                __builtin_amdgcn_s_setprio(0);
                break;
            case 1:
                __builtin_amdgcn_s_setprio(1);
                break;
            case 2:
                __builtin_amdgcn_s_setprio(2);
                break;
            default:
                __builtin_amdgcn_s_setprio(3);
                break;
            }
        };
        while (u < u_end) {
            uint32_t next = u + W;
            rotate_priority();
            if (next < u_end)
                load_unit(next, kb, vb);
            process(ka, va, u);
            u = next;
            if (u >= u_end)
                break;
            next = u + W;
            rotate_priority();
            if (next < u_end)
                load_unit(next, ka, va);
            process(kb, vb, u);
            u = next;
        }
        __builtin_amdgcn_s_setprio(0); // the merge at the default priority

        // Four features of the workgroup's result per thread from here on
        constexpr uint32_t T4 = G * D / 4;
        const uint64_t out_row = ((uint64_t)row * q_heads + qh0) * D;
        // the gate's values, loaded now so that their latency hides behind the
        // merge (the pages' registers are free)
        float gate4[4];
        auto load_gate = [&](uint32_t t) {
            if (gate_vectors) {
                load4<DT>(gate, out_row + 4 * t, gate4);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    gate4[e] = load_elem<DT>(gate, out_row + 4 * t + e);
            }
        };
        if constexpr (GATED)
            if (tid < T4)
                load_gate(tid);

        // What follows bounds small batches: a launch over six rows of up to
        // 1,500 tokens has its last page scored after 5.5 us and ended at
        // 10.9, waiting on one LDS or memory round trip after another. With
        // the swaps below, the reads of the merges four at a time and 16 bytes
        // per access a layer of that batch takes 11.6 us instead of 12.9, four
        // rows of U[64, 512] 9.0 instead of 10.4, one 32K row 29.7 instead of
        // 31.3 (launch gaps included, rotated).
        // Merge the wave's row-group states. The maxima and denominators are
        // reduced into every lane; the accumulators are reduced and scattered,
        // each swap halving what a lane holds: of its features 0..7 a lane of
        // half h keeps 4h..4h+3 after the 32-lane swap, and with four groups
        // the two at 2 * (group % 2) of those after the 16-lane one.
        constexpr uint32_t KEEP = ROWS == 4 ? 2 : 4;
        const uint32_t kept = 4 * (lane >> 5) + (ROWS == 4 ? 2 * (group & 1) : 0);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float M = swap32(mx[g], [](float a, float b) { return fmaxf(a, b); });
            if constexpr (ROWS == 4)
                M = swap16(M, [](float a, float b) { return fmaxf(a, b); });
            const float w = fast_exp2(mx[g] - M);
            float d = swap32(den[g] * w, [](float a, float b) { return a + b; });
            if constexpr (ROWS == 4)
                d = swap16(d, [](float a, float b) { return a + b; });
#pragma unroll
            for (int f = 0; f < 4; ++f)
                acc[g][f] = scatter32(acc[g][f] * w, acc[g][f + 4] * w);
            if constexpr (ROWS == 4) {
                acc[g][0] = scatter16(acc[g][0], acc[g][2]);
                acc[g][1] = scatter16(acc[g][1], acc[g][3]);
            }
            den[g] = d;
            mx[g] = M;
        }
        // LDS: acc [W][G][D], then (max, denominator) [W][G][2]
        float* lds_acc = lds;
        float* lds_ml = lds + W * G * D;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float* dst = lds_acc + (wave * G + g) * D + row8::feature(part, kept);
            if constexpr (KEEP == 2)
                *reinterpret_cast<float2*>(dst) = make_float2(acc[g][0], acc[g][1]);
            else
                *reinterpret_cast<float4*>(dst) =
                    make_float4(acc[g][0], acc[g][1], acc[g][2], acc[g][3]);
            if (lane == 0)
                *reinterpret_cast<float2*>(lds_ml + (wave * G + g) * 2) =
                    make_float2(mx[g], den[g]);
        }
        __syncthreads();
        // The workgroup's state of q head g, features f .. f + 3: the n states in
        // LDS (the waves', or the slices' below) merged online, four at a time
        // so that their reads are in flight together (one after another they
        // took half a microsecond).
        auto wg_state = [&](uint32_t n, uint32_t g, uint32_t f, float& M, float& d, float (&a)[4]) {
            M = -FLT_MAX;
            d = 0.0f;
            a[0] = a[1] = a[2] = a[3] = 0.0f;
            for (uint32_t w0 = 0; w0 < n; w0 += 4) {
                float2 ml[4];
                float4 av[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t at = min(w0 + i, n - 1) * G + g;
                    ml[i] = *reinterpret_cast<const float2*>(lds_ml + at * 2);
                    av[i] = *reinterpret_cast<const float4*>(lds_acc + at * D + f);
                }
                if (w0 + 4 > n) {
                    // past the last state: nothing. (Its accumulator may hold an
                    // infinity, which a weight of 0 would turn into NaN. A branch, so
                    // that whole fours, 8 waves' among them, pay no selects: with
                    // them the 28-layer step below takes 327.3 us instead of 325.4,
                    // with a branch around each state's sums 329.8.)
                    asm volatile("");
#pragma unroll
                    for (uint32_t i = 1; i < 4; ++i)
                        if (w0 + i >= n) {
                            ml[i] = make_float2(-FLT_MAX, 0.0f);
                            av[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        }
                }
                const float nm = fmaxf(fmaxf(M, fmaxf(ml[0].x, ml[1].x)), fmaxf(ml[2].x, ml[3].x));
                const float keep = fast_exp2(M - nm);
                d *= keep;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    a[e] *= keep;
                M = nm;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const float weight = fast_exp2(ml[i].x - nm);
                    d += ml[i].y * weight;
                    a[0] += av[i].x * weight;
                    a[1] += av[i].y * weight;
                    a[2] += av[i].z * weight;
                    a[3] += av[i].w * weight;
                }
            }
        };
        // thread t's four features, divided by the denominator, gated, rounded once
        auto emit = [&](uint32_t t, const float (&a)[4], float d) {
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                o[e] = a[e] / d;
            if constexpr (GATED) {
                if (t != tid)
                    load_gate(t);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    o[e] *= sigmoid(gate4[e]);
            }
            store4<DT>(out, out_row + 4 * t, o);
        };
        if (n_chunks == 1) {
            for (uint32_t t = tid; t < T4; t += blockDim.x) {
                float M, d, a[4];
                wg_state(W, t / (D / 4), 4 * t % D, M, d, a);
                emit(t, a, d);
            }
            return;
        }
        // a chunk of a cut row: record [max, denominator, 0, 0, acc[D]] per q head,
        // stored through to where every XCD reads it, 16 bytes per thread
        constexpr uint32_t RF = D + 4;
        const uint32_t record_stride = q_heads * RF; // between a row's chunks, in floats
        float* const records = split.records
            + ((uint64_t)m.split_first[row] * q_heads + qh0) * RF;
        {
            const __amdgpu_buffer_rsrc_t rec =
                record_rsrc(records + (uint64_t)chunk * record_stride, G * RF * 4);
            for (uint32_t t = tid; t < T4; t += blockDim.x) {
                const uint32_t g = t / (D / 4), f = 4 * t % D;
                float M, d, a[4];
                wg_state(W, g, f, M, d, a);
                agent_store4(rec, (g * RF + 4 + f) * 4, a[0], a[1], a[2], a[3]);
                if (f == 0)
                    agent_store4(rec, g * RF * 4, M, d, 0.0f, 0.0f);
            }
        }
        // Arrival: every wave waits until its record stores are complete, then
        // one thread counts the chunk in. The chunk that arrives last resets the
        // counter and merges the row's records (their loads miss any cache line
        // that could be stale); the others are done.
        wait_vector_memory();
        __syncthreads();
        uint32_t* const arrivals = split.arrivals + (uint64_t)m.split_first[row] * H + kv_head;
        uint32_t* const last_flag =
            reinterpret_cast<uint32_t*>(lds_ml + W * G * 2 + (ROPE ? rotary : 0));
        if (tid == 0) {
            const uint32_t before =
                __hip_atomic_fetch_add(arrivals, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            const uint32_t last = before == n_chunks - 1;
            if (last)
                __hip_atomic_store(arrivals, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            *last_flag = last;
        }
        __syncthreads();
        if (!*last_flag)
            return;
        // Thread (slice, g, f) folds chunks slice, slice + S, ... of q head g with
        // weights 2^(m_c - M) (paged_attention_reduce_f32,
        // src/metal/kernels/attention.metal:567-615, done online), as many
        // records per round trip as a slice has, up to four; the S slices are
        // folded through LDS. The loads go to memory, past the caches: a record
        // past the row's last is not read.
        // (slices enough for four records each; W of them fit the wave states' LDS)
        const uint32_t S = max(1u, min(min(blockDim.x / T4, W), (n_chunks + 3) / 4));
        auto fold = [&](auto width) {
            constexpr uint32_t U = decltype(width)::value;
            for (uint32_t t = tid; t < S * T4; t += blockDim.x) {
                const uint32_t slice = t / T4, g = t % T4 / (D / 4), f = 4 * t % D;
                float M = -FLT_MAX, d = 0.0f, a[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
                for (uint32_t c0 = 0; c0 < n_chunks; c0 += U * S) {
                    const uint32_t left = n_chunks - c0; // records from here
                    const __amdgpu_buffer_rsrc_t rec =
                        record_rsrc(records + (uint64_t)c0 * record_stride,
                                    (min(left, U * S) - 1) * record_stride * 4 + G * RF * 4);
                    u32x4_t head[U], part4[U];
#pragma unroll
                    for (uint32_t i = 0; i < U; ++i) {
                        // out of the descriptor's range for a record past the last: reads 0
                        const uint32_t at = ((slice + i * S) * record_stride + g * RF) * 4;
                        head[i] = agent_load4(rec, at);
                        part4[i] = agent_load4(rec, at + (4 + f) * 4);
                    }
                    float mc[U], nm = M;
#pragma unroll
                    for (uint32_t i = 0; i < U; ++i) {
                        mc[i] = slice + i * S < left ? __uint_as_float(head[i][0]) : -FLT_MAX;
                        nm = fmaxf(nm, mc[i]);
                    }
                    const float keep = fast_exp2(M - nm);
                    d *= keep;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        a[e] *= keep;
                    M = nm;
#pragma unroll
                    for (uint32_t i = 0; i < U; ++i) {
                        const float take = fast_exp2(mc[i] - nm);
                        d += __uint_as_float(head[i][1]) * take;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            a[e] += __uint_as_float(part4[i][e]) * take;
                    }
                }
                if (S == 1) {
                    emit(t, a, d);
                    continue;
                }
                *reinterpret_cast<float4*>(lds_acc + (slice * G + g) * D + f) =
                    make_float4(a[0], a[1], a[2], a[3]);
                if (f == 0)
                    *reinterpret_cast<float2*>(lds_ml + (slice * G + g) * 2) = make_float2(M, d);
            }
        };
        if (n_chunks <= 2 * S)
            fold(std::integral_constant<uint32_t, 2> {});
        else
            fold(std::integral_constant<uint32_t, 4> {});
        if (S == 1)
            return;
        __syncthreads();
        for (uint32_t t = tid; t < T4; t += blockDim.x) {
            float M, d, a[4];
            wg_state(S, t / (D / 4), 4 * t % D, M, d, a);
            emit(t, a, d);
        }
    };

    // Workgroup blockIdx.x / H starts at that plan entry and follows the
    // entries' links through its segments.
    uint32_t at = blockIdx.x / H;
    for (;;) {
        // scalar loads (the plan is constant during the launch)
        using c4 = const __attribute__((address_space(4))) u32x4_t;
        const auto* e = (c4*)(uintptr_t)(m.plan + plan_entry_words * at);
        const u32x4_t a = e[0], b = e[1];
        const uint4 e0 = make_uint4(a.x, a.y, a.z, a.w);
        const uint4 e1 = make_uint4(b.x, b.y, b.z, b.w);
        segment(e0, e1);
        at = e1.w;
        if (at == plan_last)
            break;
        __syncthreads(); // the next segment's merge reuses the LDS
    }
}

constexpr uint32_t split_waves = 8;
// Waves per workgroup of a cut plan whose workgroups fit one per compute unit
// and hold at least split_alone_min_pages pages each (one long row's pieces):
// each wave holds one page in flight, and more waves per compute unit read
// faster (one 32K-token row, 64 pages per workgroup, 2.1-2.3 % faster than
// at 8 waves, a 64K-token row 1.3-2.4 %; 16 waves no faster than 8; at 32
// pages per workgroup even, at 16 pages 1.6-2.1 % slower)
constexpr uint32_t split_waves_alone = 12;
constexpr uint32_t split_alone_min_pages = 48;

// Waves per workgroup of the fast path. With one or two q heads per KV head
// and at least one (row, kv head) unit per compute unit: 10 waves (one
// workgroup per CU), except for batches of at least 6 units per CU whose rows
// average under 256 pages, which take 8 (two workgroups per CU, so one's
// start and merge overlap the other's page reads). Measured on MI355X (one
// layer): with 6-16 units per CU, 8 waves is 0.6-9.5 % faster for mean rows
// of 50-160 pages, the two tie at 256 pages and 10 is 2.7 % faster at 288
// (config 3); with 1-2 units per CU, 8 waves is 7-16 % slower. A smaller
// batch takes the maximum (16, or 8 for wide lanes) so each row streams
// as fast as one CU allows. Chunks of cut rows take split_waves (a chunk is
// short, and several of them share a CU), or split_waves_alone when the
// plan's workgroups fit one per CU with enough pages each. f32 pages take 4 waves, two
// workgroups per CU at their two waves per SIMD: on config 2's shape 4, 6 and
// 8 waves measured 90.9, 97.9 and 96.6 us per launch, on config 3's 770, 768
// and 779 us (one box).
// CKV_DECODE_WAVES overrides.
uint32_t fast_waves(uint32_t group, int dtype, uint32_t units, int cu_count,
                    uint32_t mean_pages, uint32_t split_pages)
{
    const uint32_t limit = wide_lanes(group, dtype) ? 8u : 16u;
    if (const char* forced = std::getenv("CKV_DECODE_WAVES")) {
        const long v = std::strtol(forced, nullptr, 10);
        if (v >= 1 && v <= (long)limit)
            return (uint32_t)v;
    }
    if (dtype == CKV_F32)
        return 4;
    if (split_pages) {
        const bool alone = units <= (uint32_t)std::max(cu_count, 1)
            && split_pages >= split_alone_min_pages;
        return std::min(limit, alone ? split_waves_alone : split_waves);
    }
    if (limit > 10 && cu_count > 0 && units >= (uint32_t)cu_count)
        return units / (uint32_t)cu_count >= 6 && mean_pages < 256 ? 8 : 10;
    return limit;
}

// The same for rows behind a window, which are short and mostly equally long: 8 waves,
// two workgroups to a compute unit, for one or two q heads per KV head; 4 waves where
// the units or the chunks of halved rows (shape_window_plan) are more than two for each,
// and for more q heads, whose lanes let one workgroup of 8 waves or two of 4 reside
// (8 q heads: while all units reside at once). 128-wide heads, whole rows, us at 10, 8 and
// 4 waves: 48 rows behind 1,024 tokens 45.3, 41.9 and 43.4; 64 50.8, 49.4 and 48.3; 80 69.0,
// 67.0 and 62.6; 4 q heads per KV head, at 8 and 4 waves: 80 rows behind 256 30.7 and
// 22.2, 64 behind 1,024 54.4 and 50.3; 8: 64 behind 1,024 75.2 and 68.2, 80 109 and 115.
// Pieces of 4 pages, at 8 and 4 waves: 4 rows behind 512 6.8 and 6.4, 1 behind 256 6.2
// and 6.0.
[[maybe_unused]] uint32_t window_waves(uint32_t head_dim, uint32_t group, int dtype, uint32_t units, int cu_count,
                      uint32_t mean_pages, uint32_t split_pages)
{
    const uint32_t waves = fast_waves(group, dtype, units, cu_count, mean_pages, split_pages);
    const uint32_t cus = (uint32_t)std::max(cu_count, 1);
    if (std::getenv("CKV_DECODE_WAVES") || dtype == CKV_F32)
        return waves;
    if (head_dim == 128 && split_pages && split_pages <= 4) // a page for each wave
        return std::min(waves, 4u);
    if (units < cus)
        return waves;
    const bool many = units > 2 * cus;
    if (split_pages)
        return many && group <= 4 ? 4 : waves;
    if (head_dim != 128)
        return waves;
    if (group > 2)
        return group == 8 && many ? waves : 4;
    return units >= 2 * cus ? 4 : 8;
}

template <bool WINDOW, int D, int G>
hipError_t launch_fast(hipStream_t s, const pool_view& p, const meta_view& m, uint32_t layer,
                       const void* q, uint32_t q_heads, float scale_log2, void* out, int dt,
                       const void* k_in, const void* v_in, const void* gate, int cu_count,
                       split_scratch split, const rope_table* rope = nullptr,
                       uint32_t rotary = 0, uint32_t group_stride = G, uint32_t head_base = 0)
{
    if (!m.plan || (m.n_cut && (!split.records || !split.arrivals)))
        return hipErrorInvalidValue;
    if constexpr (G == 8) {
        // f32 pages at 8 q heads per kv head: two passes over 4 heads each (one
        // pass holds twice the registers its 512-lane workgroups allow); each
        // reads the K/V once more, the fused append writes the same token twice
        if (dt == CKV_F32) {
            hipError_t e = launch_fast<WINDOW, D, 4>(s, p, m, layer, q, q_heads, scale_log2, out, dt, k_in,
                                          v_in, gate, cu_count, split, rope, rotary, 8, 0);
            if (e == hipSuccess)
                e = launch_fast<WINDOW, D, 4>(s, p, m, layer, q, q_heads, scale_log2, out, dt, k_in, v_in,
                                   gate, cu_count, split, rope, rotary, 8, 4);
            return e;
        }
    }
    const uint32_t units = m.n_plan * p.kv_heads;
    const uint32_t waves = WINDOW
        ? window_waves(D, G, dt, units, cu_count, m.mean_pages, m.split_pages)
        : fast_waves(G, dt, units, cu_count, m.mean_pages, m.split_pages);
    const dim3 grid(units), block(64 * waves);
    // the merge's (acc, max, denominator) per wave, the rope angle table, a flag
    const size_t lds = ((size_t)waves * G * (D + 2) + (rope ? rotary : 0) + 1) * sizeof(float);
    const auto qq = static_cast<const char*>(q);
    const auto ki = static_cast<const char*>(k_in);
    const auto vi = static_cast<const char*>(v_in);
    rope_pairs<D / 2> freq = {};
    if (rope)
        for (uint32_t j = 0; j < rotary / 2; ++j)
            freq.inv_freq[j] = rope->inv_freq[j];
    // one instantiation per (dtype, fused, gated, rope); rope only when fused
    // and on 16-bit pages
    const int variant = (rope ? 16 : 0) | (dt << 2) | (k_in ? 2 : 0) | (gate ? 1 : 0);
    switch (variant) {
#define CKV_FAST_CASE(DT_, FUSED_, GATED_, ROPE_)                                              \
    case (ROPE_ ? 16 : 0) | (DT_ << 2) | (FUSED_ ? 2 : 0) | (GATED_ ? 1 : 0):                  \
        if constexpr (fast_fits(G, DT_))                                                       \
            decode_wg_kernel<D, G, DT_, FUSED_, GATED_, ROPE_, WINDOW><<<grid, block, lds, s>>>(       \
                p, m, layer, qq, q_heads, scale_log2, out, ki, vi, gate, freq, rotary, split,  \
                group_stride, head_base);                                                      \
        else                                                                                   \
            return hipErrorInvalidValue;                                                       \
        break;
        CKV_FAST_CASE(CKV_F32, false, false, false)
        CKV_FAST_CASE(CKV_F32, false, true, false)
        CKV_FAST_CASE(CKV_F32, true, false, false)
        CKV_FAST_CASE(CKV_F32, true, true, false)
        CKV_FAST_CASE(CKV_BF16, false, false, false)
        CKV_FAST_CASE(CKV_BF16, false, true, false)
        CKV_FAST_CASE(CKV_BF16, true, false, false)
        CKV_FAST_CASE(CKV_BF16, true, true, false)
        CKV_FAST_CASE(CKV_F16, false, false, false)
        CKV_FAST_CASE(CKV_F16, false, true, false)
        CKV_FAST_CASE(CKV_F16, true, false, false)
        CKV_FAST_CASE(CKV_F16, true, true, false)
        CKV_FAST_CASE(CKV_BF16, true, false, true)
        CKV_FAST_CASE(CKV_BF16, true, true, true)
        CKV_FAST_CASE(CKV_F16, true, false, true)
        CKV_FAST_CASE(CKV_F16, true, true, true)
#undef CKV_FAST_CASE
    default:
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

// The instantiation for a head width and a GQA group that decode_uses_fast_path admits.
template <bool WINDOW, int D, class... Args>
hipError_t launch_group(uint32_t group, const Args&... args)
{
    switch (group) {
    case 1:
        return launch_fast<WINDOW, D, 1>(args...);
    case 2:
        return launch_fast<WINDOW, D, 2>(args...);
    case 4:
        return launch_fast<WINDOW, D, 4>(args...);
    default:
        return launch_fast<WINDOW, D, 8>(args...);
    }
}

template <bool WINDOW, class... Args>
hipError_t launch_width(uint32_t head_dim, uint32_t group, const Args&... args)
{
    return head_dim == 256 ? launch_group<WINDOW, 256>(group, args...)
                           : launch_group<WINDOW, 128>(group, args...);
}

} // namespace
} // namespace ckv
