// Weights of the 4-bit microscaled formats as bf16 numbers in registers, for products with activations that are not quantised.
#pragma once

#include "tcq_microscale.cuh"

namespace tcq {

// Four codes (the low 16 bits of w) as bf16 pairs, times the scale.  Two byte permutations look the magnitudes up as the bytes of bf16 numbers,
// one spreads the signs.
__device__ __forceinline__ void four_weights(uint32_t w, __nv_bfloat162 scale, uint32_t& a, uint32_t& b) {
    const uint32_t mag = w & 0x7777u;
    const uint32_t lo = __byte_perm(0xC0800000u, 0xC0804000u, mag);                   // 0 .5 1 1.5 2 3 4 6: low bytes 00 00 80 C0 00 40 80 C0
    uint32_t hi = __byte_perm(0x3F3F3F00u, 0x40404040u, mag);                         // high bytes 00 3F 3F 3F 40 40 40 40
    uint32_t sign;
    asm("prmt.b32 %0, %1, %2, 0x9D8C;" : "=r"(sign) : "r"(w), "r"(w << 4));           // the top bit of each code, over a whole byte
    hi |= sign & 0x80808080u;
    const uint32_t p = __byte_perm(lo, hi, 0x5140), q = __byte_perm(lo, hi, 0x7362);
    const __nv_bfloat162 x = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&p), scale), y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&q), scale);
    a = *reinterpret_cast<const uint32_t*>(&x);
    b = *reinterpret_cast<const uint32_t*>(&y);
}

// The scale of 16 columns q of 64, twice, out of the four e4m3 (nvfp4) or two e8m0 (mxfp4) bytes of them; every one is a bf16 number.
template <int FMT>
__device__ __forceinline__ __nv_bfloat162 scale_of(uint32_t word, int q) {
    if constexpr (FMT == kNvfp4) {
        return __float2bfloat162_rn(e4m3_to_f32((word >> (8 * q)) & 0xFFu));
    } else {
        const uint32_t byte = (word >> (8 * (q / 2))) & 0xFFu;
        const uint32_t bits = byte == 0 ? 0x0040u : byte == 255 ? 0x7FC0u : byte << 7;
        const uint32_t two = bits << 16 | bits;
        return *reinterpret_cast<const __nv_bfloat162*>(&two);
    }
}

}  // namespace tcq
