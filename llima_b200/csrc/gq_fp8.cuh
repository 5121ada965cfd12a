// e4m3 codes and power-of-two (E8M0) block scales.
//
// A block's scale is 2^e with the smallest e >= -127 such that its largest finite magnitude
// is at most 448 * 2^e (448 = 1.75 * 2^8 is the largest e4m3 value); e = 0 for an all-zero
// block.  Dividing by a power of two is exact, so a code is its value rounded once, and
// dequantization is exact.  e4m3 keeps four significant bits whatever the scale, so a finer
// scale than a power of two would gain nothing but part of the last binade; this form is the
// one the tensor cores multiply by themselves.
#pragma once

#include "gq_device.cuh"

namespace gq {

// The kernels of this family are launched so that each may begin before the one ahead of it on
// the stream has ended.  after_previous(): waits until that one has, its memory operations
// included; every thread calls it before its first access to global memory.  let_next(): the
// next one may begin, called once this CTA holds all that it will wait for (tensor memory).
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

constexpr uint32_t kInfBits = 0x7F800000u;

// |x| bits where x is finite, else 0
__device__ __forceinline__ uint32_t finite_abs(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
    return b < kInfBits ? b : 0u;
}

// The stored scale byte e + 127 for the bit pattern of the block's largest finite |x|:
// amax = 1.f * 2^(E - 127) <= 1.75 * 2^(8 + e) <=> e >= E - 135 + (f > 0.75).
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    if (amax_bits == 0) return 127u;
    const int e = static_cast<int>(amax_bits >> 23) - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return static_cast<uint32_t>(max(e, 0));
}

// 2^-e of a scale byte (0..247), a normal number
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Values already divided by the scale to codes, round to nearest even.  The conversion
// saturates, which no finite value here needs (|x| <= 448).
// Four values to a word of four codes, the first in the low byte
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint32_t r;
    asm("{ .reg .b16 lo, hi; cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1; cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3; mov.b32 %0, {lo, hi}; }"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}

// What becomes the NaN code where a value is not finite (an infinity would saturate)
__device__ __forceinline__ float nan_unless_finite(float x) {
    return (__float_as_uint(x) & 0x7FFFFFFFu) < kInfBits ? x : __uint_as_float(0x7FFFFFFFu);
}

}  // namespace gq
