// Weights of the 4-bit microscaled formats as bf16 numbers in registers, for products with activations that are not quantised.
#pragma once

#include "tcq_microscale.cuh"

namespace tcq {

// Eight codes as bf16 pairs in order, times the scale.  Two byte permutations look four magnitudes up as the bytes of bf16 numbers, one spreads the
// signs; these half-rate instructions are what bounds it, so what can be shared by all eight is.
__device__ __forceinline__ void eight_weights(uint32_t w, uint32_t scale, uint32_t (&out)[4]) {
    const uint32_t mag = w & 0x77777777u, up = w << 4;
    uint32_t sign[2];
    asm("prmt.b32 %0, %1, %2, 0x9D8C;" : "=r"(sign[0]) : "r"(w), "r"(up));            // the top bit of each code, over a whole byte
    asm("prmt.b32 %0, %1, %2, 0xBFAE;" : "=r"(sign[1]) : "r"(w), "r"(up));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t four = mag >> (16 * i);
        const uint32_t lo = __byte_perm(0xC0800000u, 0xC0804000u, four);              // 0 .5 1 1.5 2 3 4 6: low bytes 00 00 80 C0 00 40 80 C0
        const uint32_t hi = __byte_perm(0x3F3F3F00u, 0x40404040u, four) | (sign[i] & 0x80808080u);           // high bytes 00 3F 3F 3F 40 40 40 40
        const uint32_t p = __byte_perm(lo, hi, 0x5140), q = __byte_perm(lo, hi, 0x7362);
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(out[2 * i]) : "r"(p), "r"(scale));
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(out[2 * i + 1]) : "r"(q), "r"(scale));
    }
}

// The scales of 64 columns, each twice, by sixteens: out of four e4m3 (nvfp4) or two e8m0 (mxfp4) bytes; every one is a bf16 number.
template <int FMT>
__device__ __forceinline__ void four_scales(uint32_t word, uint32_t (&scale)[4]) {
    if constexpr (FMT == kNvfp4) {
        uint32_t h[2];
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}" : "=r"(h[0]), "=r"(h[1]) : "r"(word));
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float f = __half2float(__ushort_as_half(uint16_t(h[q / 2] >> (16 * (q & 1)))));
            asm("cvt.rn.bf16x2.f32 %0, %1, %1;" : "=r"(scale[q]) : "f"(f));
        }
    } else {
        uint32_t two;                                    // 2^-127 is a denormal number, 255 NaN
        asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(two) : "h"(uint16_t(word)));
        scale[0] = scale[1] = __byte_perm(two, two, 0x1010);
        scale[2] = scale[3] = __byte_perm(two, two, 0x3232);
    }
}

}  // namespace tcq
