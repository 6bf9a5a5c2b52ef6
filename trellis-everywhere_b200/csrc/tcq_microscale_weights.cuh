// Weights of the 4-bit microscaled formats as bf16 numbers in registers, for products with activations that are not quantised.
#pragma once

#include "tcq_microscale.cuh"

namespace tcq {

// The magnitudes 0 .5 1 1.5 2 3 4 6 as bf16 numbers: low bytes 00 00 80 C0 00 40 80 C0, high bytes 00 3F 3F 3F 40 40 40 40.  Made so that they stay in registers
// (the compiler would put each anew before every use: a third more instructions).  QUARTER: a fourth of them, high bytes 00 3E 3E 3E 3F 3F 3F 3F.
template <bool QUARTER>
struct E2m1Bytes {
    uint32_t low0, low1, high0, high1;
    __device__ __forceinline__ E2m1Bytes() {
        asm volatile("mov.b32 %0, 0xC0800000;\n\tmov.b32 %1, 0xC0804000;\n\tmov.b32 %2, %4;\n\tmov.b32 %3, %5;"
                     : "=r"(low0), "=r"(low1), "=r"(high0), "=r"(high1) : "n"(QUARTER ? 0x3E3E3E00 : 0x3F3F3F00), "n"(QUARTER ? 0x3F3F3F3F : 0x40404040));
    }
};
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t pick) {      // (__byte_perm masks what picks)
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(pick));
    return r;
}
// Eight codes as bf16 pairs in order, times the scale.  Two byte permutations look four magnitudes up as the bytes of bf16 numbers, one spreads the
// signs; these half-rate instructions are what bounds it, so what can be shared by all eight is.
template <bool QUARTER>
__device__ __forceinline__ void eight_weights(const E2m1Bytes<QUARTER>& e, uint32_t w, uint32_t scale, uint32_t (&out)[4]) {
    const uint32_t mag = w & 0x77777777u, up = w << 4;
    const uint32_t sign[2] = {prmt(w, up, 0x9D8Cu), prmt(w, up, 0xBFAEu)};            // the top bit of each code, over a whole byte
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t four = mag >> (16 * i);
        const uint32_t lo = prmt(e.low0, e.low1, four), hi = prmt(e.high0, e.high1, four) | (sign[i] & 0x80808080u);
        const uint32_t p = prmt(lo, hi, 0x5140u), q = prmt(lo, hi, 0x7362u);
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
