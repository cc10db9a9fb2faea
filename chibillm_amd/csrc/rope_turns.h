// Rotary angles from turn_table's fixed-point turns. HIP device code only.
//
// A position's angle on a pair, modulo a whole turn, is the low 64 bits of
// position * step: the product wraps where the angle does, so no position is too
// far (in float, position * frequency is off by 0.004 radians at position 10^5), and
// a negative shift's two's complement wraps the same way. The 64 bits are rounded
// to 32, 7e-10 radians at most, and their top two (after half an octant's rounding)
// give the quadrant, exactly; what is left, an eighth of a turn at most, goes through
// the Taylor series of sine (to x^9) and cosine (to x^10), cut off below 2e-9.
#pragma once

#include "ckv_internal.h"

namespace ckv {
namespace {

__device__ __forceinline__ void sincos_turn(uint64_t step, uint64_t position, float& s, float& c)
{
    const uint32_t turn = (uint32_t)((step * position + 0x80000000u) >> 32); // of 2^32
    const uint32_t quadrant = (turn + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(turn - (quadrant << 30)) * 1.4629180792671596e-9f; // 2 pi / 2^32
    const float z = x * x;
    float ps = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f); // 1/9!, -1/7!
    ps = __builtin_fmaf(z, ps, 8.3333333e-3f);                   // 1/5!
    ps = __builtin_fmaf(z, ps, -1.6666667e-1f);                  // -1/3!
    ps = __builtin_fmaf(x * z, ps, x);
    float pc = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f); // -1/10!, 1/8!
    pc = __builtin_fmaf(z, pc, -1.3888889e-3f);                  // -1/6!
    pc = __builtin_fmaf(z, pc, 4.1666667e-2f);                   // 1/4!
    pc = __builtin_fmaf(z, pc, -0.5f);
    pc = __builtin_fmaf(z, pc, 1.0f);
    const float a = quadrant & 1 ? pc : ps, b = quadrant & 1 ? ps : pc;
    s = quadrant & 2 ? -a : a;
    c = (quadrant + 1) & 2 ? -b : b;
}

// One element of a row of the pool's type as float, and back (round to nearest
// even, NaN quieted).
template <int DT>
struct turn_element {
    using type = uint16_t;
    static __device__ __forceinline__ float load(type v)
    {
        if constexpr (DT == CKV_F16)
            return static_cast<float>(__builtin_bit_cast(_Float16, v));
        else
            return __builtin_bit_cast(float, static_cast<uint32_t>(v) << 16);
    }
    static __device__ __forceinline__ type store(float v)
    {
        if constexpr (DT == CKV_F16) {
            return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
        } else {
            uint32_t b = __builtin_bit_cast(uint32_t, v);
            if ((b & 0x7FFFFFFFu) > 0x7F800000u)
                return static_cast<type>((b >> 16) | 0x40u);
            b += 0x7FFFu + ((b >> 16) & 1u);
            return static_cast<type>(b >> 16);
        }
    }
};

template <>
struct turn_element<CKV_F32> {
    using type = float;
    static __device__ __forceinline__ float load(type v) { return v; }
    static __device__ __forceinline__ type store(float v) { return v; }
};

} // namespace
} // namespace ckv
