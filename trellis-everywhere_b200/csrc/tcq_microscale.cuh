// Shared definitions of the 4-bit microscaled formats: geometry of their storage, and the three small types as device functions.
//
// A matrix of rows x k values (value = e2m1(code) * block scale [* row scale]) is held as
//   codes      [rows][pitch] bytes, pitch = 16 * ceil(k / 32): two e2m1 codes a byte, the even column in the low half; zeros behind column k
//   scales     [ceil(rows / 128)][atoms][32][4][4] bytes: block b of row r at [r / 128][b / 4][r % 32][r % 128 / 32][b % 4].  512 bytes are
//              what one tcgen05.cp of 32 x 128 bits takes to tensor memory for 128 rows; atoms = 4 (nvfp4) or 2 (mxfp4) for every 256
//              columns begun, so that a tile of 256 columns always has all its scales.  Zeros behind column k; the places of rows
//              behind the last one are never read for a result and are left as they are.
//   row_scale  [rows] fp32 (nvfp4), none (mxfp4)
#pragma once

#include <atomic>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace tcq {

enum : int { kMxfp4 = 0, kNvfp4 = 1 };
enum : int { kF32 = 0, kF16 = 1, kBf16 = 2 };

constexpr int kMsTileK = 256;                            // columns that storage and kernels count in

template <int FMT> struct Ms;
template <> struct Ms<kMxfp4> { static constexpr int kBlock = 32, kAtoms = 2; };
template <> struct Ms<kNvfp4> { static constexpr int kBlock = 16, kAtoms = 4; };

inline long long ms_pitch(long long k) { return (k + 31) / 32 * 16; }
inline long long ms_tiles_k(long long k) { return (k + kMsTileK - 1) / kMsTileK; }
inline int ms_atoms(int fmt) { return fmt == kNvfp4 ? 4 : 2; }
inline long long ms_scale_bytes(long long rows, long long k, int fmt) { return (rows + 127) / 128 * ms_tiles_k(k) * ms_atoms(fmt) * 512; }

// Place of the scale of block b of row r, `atoms` = atoms of a row in all.
__device__ __forceinline__ long long ms_scale_at(long long r, int b, long long atoms) {
    return ((r >> 7) * atoms + (b >> 2)) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (b & 3);
}

// Nearest e2m1 codes of two values (ties to the even code, beyond 6 to 6, the sign kept); lo in the low half of the byte.
__device__ __forceinline__ uint32_t f32x2_to_e2m1x2(float lo, float hi) {
    uint32_t r;
    asm("{\n\t.reg .b8 b;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %2, %1;\n\tcvt.u32.u8 %0, b;\n\t}" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}
// Nearest e4m3 of one value (ties to even, NaN to 0x7F).
__device__ __forceinline__ uint32_t f32_to_e4m3(float v) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
    return r & 0xFFu;
}
__device__ __forceinline__ float e4m3_to_f32(uint32_t byte) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(uint16_t(byte)));
    return __half2float(__ushort_as_half(uint16_t(r)));
}
// 2^(byte - 127); 255 is NaN.  Byte 0 is a denormal number.
__device__ __forceinline__ float e8m0_to_f32(uint32_t byte) {
    return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
}
// Eight codes as four pairs of fp16 numbers, in order.
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}" : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <int FMT> __device__ __forceinline__ float ms_scale_to_f32(uint32_t byte) {
    if constexpr (FMT == kNvfp4) return e4m3_to_f32(byte);
    else return e8m0_to_f32(byte);
}

// A row scale g as power * rest: a power of two, within 2^-90 and 2^90, that goes into the products or into parts of their sum, which then are of the size of the
// result, and what the sum is multiplied by at the end (1 to 2 where g is within those bounds).
__device__ __forceinline__ float row_power(float g) {
    return fminf(fmaxf(__uint_as_float(__float_as_uint(g) & 0x7F800000u), 0x1p-90f), 0x1p90f);
}
__device__ __forceinline__ float row_rest(float g) { return g * __uint_as_float(0x7F000000u - __float_as_uint(row_power(g))); }      // exact: divided by it

// For products of both sides' scales: g as inner * outer, the inner one within 2^-60 and 2^60.  A sum of 4-bit products (2^-20 to 2^47) times one side's inner
// part, the other side's scale and then the outer part leaves the range of fp32 only where the result does; the outer part is 1 unless g is extreme.
__device__ __forceinline__ float inner_part(float g) { return g > 0x1p60f ? 0x1p60f : g < 0x1p-60f ? 0x1p-60f : g; }
__device__ __forceinline__ float outer_part(float g) { return g > 0x1p60f ? g * 0x1p-60f : g < 0x1p-60f ? g * 0x1p60f : 1.0f; }

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
// Results are rounded here and nowhere before.
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// One operand in 4 bits, as the kernels take it.
struct MsMatrix {
    const uint8_t* codes;
    const uint8_t* scales;
    const float* row_scale;      // null for mxfp4
    long long rows;
};

int ms_sm_count();             // of the current device
// How many clusters of `size` CTAs of a kernel, `ctas` (1 or 2) of which an SM holds, run at once: fewer than SMs * ctas / size, since a cluster lies within a
// group of SMs.  `kept`: this kernel's answers so far, by device and log2(size).  (Statics of calls are atomic: two threads may make their first calls at once.)
struct MostClusters { std::atomic<int> of[64][4]; };
int ms_most_clusters(MostClusters& kept, const void* kernel, int threads, size_t smem, int ctas, int size);
int report_cuda_error(cudaError_t err, const char* where);     // tcq_capi.cu

cudaError_t launch_ms_quantize(const void* x, int dtype, long long rows, long long k, long long ldx, int fmt, int rotate, const float* signs,
                               uint8_t* codes, uint8_t* scales, float* row_scale, cudaStream_t stream);
cudaError_t launch_ms_dequantize(const MsMatrix& q, long long k, int fmt, void* out, int dtype, long long ldo, cudaStream_t stream);
constexpr unsigned kMsAllLoads = 0xFFFFFFFFu;     // `loads` of the products: how many stages a CTA loads before it stops (a self-test's limit)
cudaError_t launch_ms_linear(const void* x, int dtype, long long m, long long ldx, const MsMatrix& w, long long k, int fmt, void* y,
                             long long ldy, void* ws, unsigned loads, cudaStream_t stream);
bool ms_linear_direct(const void* x, int dtype, long long m, long long ldx, int fmt);      // needs no scratch
size_t ms_linear_workspace_bytes(long long m, long long n, long long k, int dtype, int fmt);
cudaError_t launch_ms_matmul(const MsMatrix& x, const MsMatrix& w, long long k, int fmt, void* y, int dtype, long long ldy, unsigned loads, cudaStream_t stream);

}  // namespace tcq
