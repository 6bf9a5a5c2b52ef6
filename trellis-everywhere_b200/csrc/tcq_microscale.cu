// Quantisation to 4-bit microscaled formats, and back.
//
// mxfp4: block of 32, scale X = 2^(floor(log2 amax) - 2), code = e2m1(x / X).
// nvfp4: block of 16, row scale g = the least 2^j, j >= -80, with amax(row) <= 2688 g (2688 = 6 * 448, the largest values of the two small
// types), block scale s = e4m3(amax / (6 g)), code = e2m1(x / (s g)).
// Every code is the nearest of the real quotient: divisors are powers of two times at most four bits, so that an fp32 quotient, correctly
// rounded, is on a border between two codes (a number of at most four bits) only where the real one is.  (For x near t d, both on
// grids no finer than ulp(x), |x / d - t| >= ulp(x) / d, which is more than half an ulp of t.)  The same holds for amax / 6 and e4m3.
// A block with a NaN or an infinity gets the scale NaN and codes 0; its finite values count in the row's largest value.
#include <algorithm>

#include "tcq_common.cuh"
#include "tcq_microscale.cuh"

namespace tcq {

namespace {

constexpr int kRun = 16;         // consecutive values of a thread: one nvfp4 block, half an mxfp4 block

// w[i] = the four bytes from byte 4 i + bytes on, 0 <= bytes < 16, as far as they are among the N words.
template <int N>
__device__ __forceinline__ void shift_words(uint32_t (&w)[N], uint32_t bytes) {
#pragma unroll
    for (int step = 2; step >= 1; --step)
        if (bytes & (4 * step))
#pragma unroll
            for (int i = 0; i + step < N; ++i) w[i] = w[i + step];
#pragma unroll
    for (int i = 0; i + 1 < N; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 8 * (bytes & 3));
}

// The matrix in memory: from its first value to behind its last.
struct Extent { const void *from, *to; };

// kRun values at any address, by 16-byte pieces that start on 16 bytes: one more than they fill.  False where a piece would reach out of the matrix.
template <typename T>
__device__ __forceinline__ bool load_pieces(const T* at, Extent x, uint4 (&out)[sizeof(T)]) {
    constexpr int kPieces = sizeof(T);                   // of 16 bytes a run
    const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(at)) & 15u;
    const char* const base = reinterpret_cast<const char*>(at) - off;
    if (base < x.from || base + 16 * (kPieces + 1) > x.to) return false;
    uint32_t w[4 * (kPieces + 1)];
#pragma unroll
    for (int i = 0; i <= kPieces; ++i) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(base) + i);
        w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
    }
    shift_words(w, off);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) out[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    return true;
}

template <typename T>
__device__ __forceinline__ void load_run(const T* __restrict__ row, long long c0, long long k, bool wide, Extent x, float (&v)[kRun]) {
    if (c0 + kRun <= k) {
        if (wide) {
            constexpr int kPer = 16 / sizeof(T);
#pragma unroll
            for (int q = 0; q < kRun / kPer; ++q) {
                uint4 u = __ldg(reinterpret_cast<const uint4*>(row + c0) + q);
                const T* const p = reinterpret_cast<const T*>(&u);
#pragma unroll
                for (int i = 0; i < kPer; ++i) v[q * kPer + i] = to_f32<T>(p[i]);
            }
            return;
        }
        uint4 u[sizeof(T)];
        if (load_pieces<T>(row + c0, x, u)) {
#pragma unroll
            for (int i = 0; i < kRun; ++i) v[i] = to_f32<T>(reinterpret_cast<const T*>(u)[i]);
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i) v[i] = c0 + i < k ? to_f32<T>(row[c0 + i]) : 0.0f;
}

// Times 2^-7, so that no sum of 128 leaves the range of fp32 before it is multiplied by 128^(-1/2) (exact but for numbers below 2^-119).
__device__ __forceinline__ void load_signs(const float* __restrict__ signs, long long c0, long long k, bool wide, float (&v)[kRun]) {
    if (wide && c0 + kRun <= k) {
#pragma unroll
        for (int q = 0; q < kRun / 4; ++q) {
            const float4 u = __ldg(reinterpret_cast<const float4*>(signs + c0) + q);
            v[4 * q] = u.x; v[4 * q + 1] = u.y; v[4 * q + 2] = u.z; v[4 * q + 3] = u.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kRun; ++i) v[i] = c0 + i < k ? signs[c0 + i] : 1.0f;
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i) v[i] *= 0x1p-7f;
}

// One stage of the transform between lanes h apart.
__device__ __forceinline__ void rotate_lanes(float (&v)[kRun], int h) {
    const float sign = threadIdx.x & h ? -1.0f : 1.0f;
#pragma unroll
    for (int i = 0; i < kRun; ++i) v[i] = __fmaf_rn(v[i], sign, __shfl_xor_sync(0xFFFFFFFFu, v[i], h));
}
// Signs, then the transform of every b = `rotate` columns: the first four stages within the thread, the others between neighbouring lanes.
// b divides k, and all lanes of a group of b / 16 take part.
__device__ __forceinline__ void rotate_run(float (&v)[kRun], const float (&signs)[kRun], int rotate) {
#pragma unroll
    for (int i = 0; i < kRun; ++i) v[i] *= signs[i];
#pragma unroll
    for (int h = 1; h < kRun; h *= 2)
#pragma unroll
        for (int i = 0; i < kRun; ++i)
            if (!(i & h)) {
                const float a = v[i], b = v[i + h];
                v[i] = a + b;
                v[i + h] = a - b;
            }
    if (rotate >= 32) rotate_lanes(v, 1);
    if (rotate >= 64) rotate_lanes(v, 2);
    if (rotate >= 128) rotate_lanes(v, 4);
    const float scale = rotate == 16 ? 32.0f : rotate == 32 ? 0.17677669529663687f * 128 : rotate == 64 ? 16.0f : 0.08838834764831845f * 128;     // 2^7 b^(-1/2)
#pragma unroll
    for (int i = 0; i < kRun; ++i) v[i] *= scale;
}

// Largest magnitude of a run, and whether all of it is finite (bits, so that NaN counts as more than infinity).
__device__ __forceinline__ uint32_t largest_bits(const float (&v)[kRun]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kRun; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
}
// Largest finite magnitude of a run.
__device__ __forceinline__ uint32_t largest_finite_bits(const float (&v)[kRun]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
        m = max(m, b < 0x7F800000u ? b : 0u);
    }
    return m;
}

__device__ __forceinline__ float pow2(int e) {                   // -127 <= e <= 127
    return __uint_as_float(e <= -127 ? 0x00400000u : uint32_t(e + 127) << 23);
}

// The exponent j of the row scale: the least j >= -80 with amax <= 2688 * 2^j; 0 for a row of zeros.
__device__ __forceinline__ int row_exponent(uint32_t amax_bits) {
    if (amax_bits == 0) return 0;
    const int e = int(amax_bits >> 23) - 127;                     // a denormal number is far below the least j anyway
    const int j = (amax_bits & 0x7FFFFFu) <= 0x280000u ? e - 11 : e - 10;      // 2688 = 1.3125 * 2^11
    return max(j, -80);
}

__device__ __forceinline__ uint2 codes_of(const float (&q)[kRun]) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kRun; i += 2) w[i / 8] |= f32x2_to_e2m1x2(q[i], q[i + 1]) << (4 * (i % 8));
    return make_uint2(w[0], w[1]);
}

// A row's largest finite magnitude so far, as bits.
__device__ __forceinline__ uint32_t row_largest(const float (&v)[kRun]) {
    const uint32_t m = largest_bits(v);
    return m < 0x7F800000u ? m : largest_finite_bits(v);
}

// A run's codes and scale byte out of its values; j: the row scale's exponent (nvfp4).  Lanes 2 i and 2 i + 1 have the halves of an mxfp4 block.
// nvfp4's quotients, by s and by 6: one step from a product with the correctly rounded reciprocal, which gives the correctly rounded quotient
// (Markstein; checked for all mantissas of x and all eight of s, 6 = 1.5 * 4 among them).
template <int FMT>
__device__ __forceinline__ uint2 quantize_run(float (&v)[kRun], int j, uint32_t& byte) {
    uint32_t m = largest_bits(v);
    if constexpr (FMT == kNvfp4) {
        const float t = __uint_as_float(m) * pow2(-j), sixth = 0x1.555556p-3f, q6 = t * sixth;
        byte = m < 0x7F800000u ? f32_to_e4m3(__fmaf_rn(__fmaf_rn(q6, -6.0f, t), sixth, q6)) : 0x7Fu;
        const float s = e4m3_to_f32(byte), r = s > 0.0f ? __frcp_rn(s) * pow2(-j) : 0.0f, by = -s * pow2(j);
        const f32x2 r2 = pack2(r, r), by2 = pack2(by, by);
#pragma unroll
        for (int i = 0; i < kRun; i += 2) {
            const f32x2 x = pack2(v[i], v[i + 1]), q = mul2(x, r2);
            float a, b;
            unpack2(fma2(fma2(q, by2, x), r2, q), a, b);
            v[i] = __uint_as_float(__float_as_uint(a) | (__float_as_uint(v[i]) & 0x80000000u));          // (the sum of two zeros has lost a sign)
            v[i + 1] = __uint_as_float(__float_as_uint(b) | (__float_as_uint(v[i + 1]) & 0x80000000u));
        }
    } else {
        m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
        const int e = m == 0 ? -127 : max(int(m >> 23) - 127 - 2, -127);
        byte = m < 0x7F800000u ? uint32_t(e + 127) : 0xFFu;
        const float inv = e <= -127 ? 1.7014118346046923e38f : pow2(-e);
#pragma unroll
        for (int i = 0; i < kRun; ++i) v[i] *= inv;
    }
    if (m >= 0x7F800000u) {
#pragma unroll
        for (int i = 0; i < kRun; ++i) v[i] = 0.0f;
    }
    return codes_of(v);
}

// Codes and scales of the run of columns c0 ... to their places.  The scales of four blocks are one word, which the first of their lanes stores.
template <int FMT>
__device__ __forceinline__ void store_run(long long r, bool row_is, long long c0, long long k, long long span, uint2 code, uint32_t byte, uint8_t* __restrict__ codes,
                                          long long pitch, uint8_t* __restrict__ scales, long long atoms) {
    constexpr int kLanes = FMT == kNvfp4 ? 1 : 2;        // of a block
    uint32_t word = (c0 < k ? byte : 0u) << (8 * (threadIdx.x / kLanes & 3));
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, kLanes);
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2 * kLanes);
    if (!row_is) return;
    if (c0 < 2 * pitch) *reinterpret_cast<uint2*>(codes + r * pitch + c0 / 2) = code;
    if (c0 < span && threadIdx.x % (4 * kLanes) == 0) *reinterpret_cast<uint32_t*>(scales + ms_scale_at(r, int(c0 / Ms<FMT>::kBlock), atoms)) = word;
}

struct QuantizeArgs {
    long long rows, k, ldx;
    bool wide;                                           // rows of x start on 16 bytes
    int rotate;
    const float* signs;
    bool wide_signs;
    uint8_t* codes;
    long long pitch;
    uint8_t* scales;
    long long atoms;
    float* row_scale;
    int lanes;                                           // threads of a row
};

// `lanes` threads a row, RUNS runs of 16 columns each, blockDim / lanes rows a CTA at a time; a row is read once (the next one while this one is
// worked on) and stays with its threads: in registers, but for 32 to 520 bytes a thread that spill at two runs (16385 to 32768 columns).  Columns up to the next multiple of 256 are worked on as zeros, so that the storage behind column k is
// written.  The factors of a rotation are a thread's own for all its rows.  Bound by instruction issue (70 to 77 % of the slots), not by memory:
// 12288 x 4096 bf16 25.9 us (mxfp4, 5.0 TB/s of x and codes), 39 (nvfp4, for its quotients); rotated by 128 46.4 and 60.9; fp32 35.8 and 44.5.
template <typename T, int FMT, int RUNS, bool ROTATED>
__global__ void __launch_bounds__(1024) tcq_ms_quantize_kernel(const T* __restrict__ x, const __grid_constant__ QuantizeArgs p) {
    constexpr int kPieces = sizeof(T);                   // of 16 bytes a run
    __shared__ uint32_t part[2][32];
    const int slot = threadIdx.x / p.lanes, lane = threadIdx.x - slot * p.lanes, slots = blockDim.x / p.lanes;
    const long long span = (p.k + kMsTileK - 1) / kMsTileK * kMsTileK;
    float signs[ROTATED ? RUNS : 1][kRun];
    if constexpr (ROTATED)
#pragma unroll
        for (int q = 0; q < RUNS; ++q) load_signs(p.signs, ((long long)q * p.lanes + lane) * kRun, p.k, p.wide_signs, signs[q]);
    const Extent extent{x, x + (p.rows - 1) * p.ldx + p.k};
    uint4 next[RUNS][kPieces];
    auto fetch = [&](long long r) {
        const T* const row = x + (r < p.rows ? r : p.rows - 1) * p.ldx;
#pragma unroll
        for (int q = 0; q < RUNS; ++q) {
            const long long c0 = ((long long)q * p.lanes + lane) * kRun;
            if (p.wide && c0 + kRun <= p.k) {
#pragma unroll
                for (int i = 0; i < kPieces; ++i) next[q][i] = __ldg(reinterpret_cast<const uint4*>(row + c0) + i);
            } else if (ROTATED || c0 + kRun > p.k || !load_pieces<T>(row + c0, extent, next[q])) {      // (rotated rows are nearly always aligned)
                T* const v = reinterpret_cast<T*>(next[q]);
#pragma unroll
                for (int i = 0; i < kRun; ++i) v[i] = c0 + i < p.k ? row[c0 + i] : from_f32<T>(0.0f);
            }
        }
    };
    int turn = 0;
    long long r0 = (long long)blockIdx.x * slots;
    fetch(r0 + slot);
    for (; r0 < p.rows; r0 += (long long)gridDim.x * slots, turn ^= 1) {
        const long long r = r0 + slot;
        const bool row_is = r < p.rows;
        float v[RUNS][kRun];
#pragma unroll
        for (int q = 0; q < RUNS; ++q)
#pragma unroll
            for (int i = 0; i < kRun; ++i) v[q][i] = to_f32<T>(reinterpret_cast<const T*>(next[q])[i]);
        if (r0 + (long long)gridDim.x * slots < p.rows) fetch(r + (long long)gridDim.x * slots);
        if constexpr (ROTATED)
#pragma unroll
            for (int q = 0; q < RUNS; ++q) rotate_run(v[q], signs[q], p.rotate);
        int j = 0;
        if constexpr (FMT == kNvfp4) {
            uint32_t m = 0;
#pragma unroll
            for (int q = 0; q < RUNS; ++q) m = max(m, row_largest(v[q]));
            if (p.lanes >= 32) {
                m = __reduce_max_sync(0xFFFFFFFFu, m);
                if (p.lanes > 32) {
                    if ((threadIdx.x & 31) == 0) part[turn][threadIdx.x >> 5] = m;
                    __syncthreads();                     // (the other turn's parts may still be read)
                    const int from = slot * (p.lanes / 32);
                    for (int w = 0; w < p.lanes / 32; ++w) m = max(m, part[turn][from + w]);
                }
            } else {
                for (int h = 1; h < p.lanes; h *= 2) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, h));
            }
            j = row_exponent(m);
            if (lane == 0 && row_is) p.row_scale[r] = pow2(j);
        }
#pragma unroll
        for (int q = 0; q < RUNS; ++q) {
            uint32_t byte;
            const uint2 code = quantize_run<FMT>(v[q], j, byte);
            store_run<FMT>(r, row_is, ((long long)q * p.lanes + lane) * kRun, p.k, span, code, byte, p.codes, p.pitch, p.scales, p.atoms);
        }
    }
}

// Rows too long for registers: one CTA a row, nvfp4's largest value in a pass of its own, whose second reading comes from L2 (64 x 100000 fp32 25 us).
template <typename T, int FMT>
__global__ void __launch_bounds__(256) tcq_ms_quantize_long_kernel(const T* __restrict__ x, const __grid_constant__ QuantizeArgs p) {
    const long long r = blockIdx.x, span = (p.k + kMsTileK - 1) / kMsTileK * kMsTileK;
    const T* const row = x + r * p.ldx;
    const Extent extent{x, x + (p.rows - 1) * p.ldx + p.k};
    float v[kRun], signs[kRun];
    auto load = [&](long long c0) {
        load_run(row, c0, p.k, p.wide, extent, v);
        if (p.rotate) {
            load_signs(p.signs, c0, p.k, p.wide_signs, signs);
            rotate_run(v, signs, p.rotate);
        }
    };
    int j = 0;
    if constexpr (FMT == kNvfp4) {
        __shared__ uint32_t part[8];
        uint32_t m = 0;
        for (long long c = 0; c < span; c += 256 * kRun) {
            load(c + (long long)threadIdx.x * kRun);
            m = max(m, row_largest(v));
        }
        m = __reduce_max_sync(0xFFFFFFFFu, m);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
        __syncthreads();
        for (int w = 0; w < 8; ++w) m = max(m, part[w]);
        j = row_exponent(m);
        if (threadIdx.x == 0) p.row_scale[r] = pow2(j);
    }
    for (long long c = 0; c < span; c += 256 * kRun) {
        const long long c0 = c + (long long)threadIdx.x * kRun;
        load(c0);
        uint32_t byte;
        const uint2 code = quantize_run<FMT>(v, j, byte);
        store_run<FMT>(r, true, c0, p.k, span, code, byte, p.codes, p.pitch, p.scales, p.atoms);
    }
}

// `lanes` threads a row, 16 columns each: 8 bytes of codes, one scale.  (A thread for several rows, one after the other, is 20 % slower.)
// 12288 x 4096 to bf16 23.7 us (5.4 TB/s), to fp32 41 (5.6 TB/s).
template <typename T, int FMT, bool WIDE>
__global__ void __launch_bounds__(256) tcq_ms_dequantize_kernel(const uint8_t* __restrict__ codes, long long pitch, const uint8_t* __restrict__ scales,
                                                                long long atoms, const float* __restrict__ row_scale, long long rows,
                                                                long long k, T* __restrict__ out, long long ldo, int log_lanes) {
    const long long r = ((long long)blockIdx.x << (8 - log_lanes)) + (threadIdx.x >> log_lanes);
    const long long c0 = (((long long)blockIdx.y << log_lanes) + (threadIdx.x & ((1 << log_lanes) - 1))) * kRun;
    const bool is = r < rows && c0 < k;
    const long long rc = is ? r : 0, cc = is ? c0 : 0;
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(codes + rc * pitch + cc / 2));
    const float s = ms_scale_to_f32<FMT>(__ldg(scales + ms_scale_at(rc, int(cc / Ms<FMT>::kBlock), atoms)));
    float row = 1.0f;
    if constexpr (FMT == kNvfp4) row = __ldg(row_scale + rc);
    uint32_t h[8];
    e2m1x8_to_f16(u.x, reinterpret_cast<uint32_t(&)[4]>(h[0]));
    e2m1x8_to_f16(u.y, reinterpret_cast<uint32_t(&)[4]>(h[4]));
    constexpr int kPieces = sizeof(T), kWords = 4 * kPieces, kPer = 16 / sizeof(T);        // pieces of 16 bytes, words of a run; values of a piece
    uint32_t w[4 + kWords];                              // four words of the lane before, then this lane's
    T* const o = reinterpret_cast<T*>(w + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        // (the first product is exact; nvfp4's row scale, which may be any number, rounds once in fp32)
        o[2 * i] = from_f32<T>(FMT == kNvfp4 ? f.x * s * row : f.x * s);
        o[2 * i + 1] = from_f32<T>(FMT == kNvfp4 ? f.y * s * row : f.y * s);
    }
    T* const to = out + rc * ldo + cc;
    const bool full = is && c0 + kRun <= k;
    if constexpr (WIDE) {                                // rows of out start on 16 bytes
        // Two neighbours swap half of their pieces and write 32 bytes side by side instead of 16 bytes 32 or 64 apart (12288 x 4096 to bf16 26.7 -> 23.7 us,
        // to fp32 56 -> 41).
        const bool odd = threadIdx.x & 1, stored = __shfl_xor_sync(0xFFFFFFFFu, full, 1) && full && log_lanes > 0;
#pragma unroll
        for (int q = 0; q < kPieces; q += 2)             // the even lane gives its odd pieces, the odd one its even ones
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, odd ? w[4 + 4 * q + i] : w[8 + 4 * q + i], 1);
                if (stored && odd) w[4 + 4 * q + i] = got;
                if (stored && !odd) w[8 + 4 * q + i] = got;
            }
        if (stored) {                                    // E0 O0 (E2 O2) in the even lane, E1 O1 (E3 O3) in the odd one
            uint4* const both = reinterpret_cast<uint4*>(to - (odd ? kRun : 0)) + odd;
#pragma unroll
            for (int q = 0; q < kPieces; ++q) {
                const int mine = kPieces == 2 ? q : q < 2 ? 2 * q : 2 * q - 3;
                both[2 * q] = make_uint4(w[4 + 4 * mine], w[5 + 4 * mine], w[6 + 4 * mine], w[7 + 4 * mine]);
            }
        }
        if (full && !stored) {
#pragma unroll
            for (int q = 0; q < kPieces; ++q) reinterpret_cast<uint4*>(to)[q] = make_uint4(w[4 + 4 * q], w[5 + 4 * q], w[6 + 4 * q], w[7 + 4 * q]);
        } else if (is && !full) {
#pragma unroll
            for (int i = 0; i < kRun; ++i)
                if (c0 + i < k) to[i] = o[i];
        }
        return;
    }
    // Rows at any address: pieces that start on 16 bytes, the first of them with the end of the lane before (9300 x 12287 to bf16 622 -> 97 us).
    const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(to)) & 15u;
    const int lane = threadIdx.x & 31, lanes = min(32, 1 << log_lanes);
    const bool before = (lane & (lanes - 1)) != 0, after = __shfl_down_sync(0xFFFFFFFFu, full, 1) && ((lane + 1) & (lanes - 1)) != 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __shfl_up_sync(0xFFFFFFFFu, w[kWords + i], 1);
    if (!is) return;
    const int spill = int(off / sizeof(T));              // this many values at the end are in the next lane's first piece
#pragma unroll
    for (int i = 0; i < kRun; ++i)
        if (c0 + i < k && (!full || (i < kPer - spill && !before && spill) || (i >= kRun - spill && !after))) to[i] = o[i];
    if (!full) return;
    uint4* const pieces = reinterpret_cast<uint4*>(reinterpret_cast<char*>(to) - off);
    if (off == 0) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = w[4 + i];
    } else {
        shift_words(w, 16 - off);
    }
#pragma unroll
    for (int q = 0; q < kPieces; ++q)
        if (q > 0 || before || spill == 0) pieces[q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
}

template <typename T, int FMT>
cudaError_t quantize_fmt(const T* x, QuantizeArgs p, cudaStream_t stream) {
    const long long runs = ms_tiles_k(p.k) * (kMsTileK / kRun);
    if (runs > 2 * 1024) {
        tcq_ms_quantize_long_kernel<T, FMT><<<unsigned(p.rows), 256, 0, stream>>>(x, p);
        return cudaGetLastError();
    }
    // Up to 256 threads a row: a power of two of them, as many rows as make 256.  More: a CTA a row, up to 1024 threads of one run, then of two.
    const int each = runs > 1024 ? 2 : 1;
    int threads = 256;
    p.lanes = 16;
    while (p.lanes < runs && p.lanes < 256) p.lanes *= 2;
    if (runs > 256) threads = p.lanes = int((runs / each + 31) / 32 * 32);
    const long long ctas = (p.rows + threads / p.lanes - 1) / (threads / p.lanes);
    const unsigned grid = unsigned(std::min<long long>(ctas, 2048ll / threads * ms_sm_count()));
    if (each == 1 && p.rotate) tcq_ms_quantize_kernel<T, FMT, 1, true><<<grid, threads, 0, stream>>>(x, p);
    else if (each == 1) tcq_ms_quantize_kernel<T, FMT, 1, false><<<grid, threads, 0, stream>>>(x, p);
    else if (p.rotate) tcq_ms_quantize_kernel<T, FMT, 2, true><<<grid, threads, 0, stream>>>(x, p);
    else tcq_ms_quantize_kernel<T, FMT, 2, false><<<grid, threads, 0, stream>>>(x, p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t quantize_t(const void* x, long long rows, long long k, long long ldx, int fmt, int rotate, const float* signs, uint8_t* codes,
                       uint8_t* scales, float* row_scale, cudaStream_t stream) {
    const QuantizeArgs p{rows, k, ldx, reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * sizeof(T) % 16 == 0, rotate, signs,
                         reinterpret_cast<uintptr_t>(signs) % 16 == 0, codes, ms_pitch(k), scales, ms_tiles_k(k) * ms_atoms(fmt), row_scale, 256};
    const T* const from = static_cast<const T*>(x);
    return fmt == kNvfp4 ? quantize_fmt<T, kNvfp4>(from, p, stream) : quantize_fmt<T, kMxfp4>(from, p, stream);
}

template <typename T>
cudaError_t dequantize_t(const MsMatrix& q, long long k, int fmt, void* out, long long ldo, cudaStream_t stream) {
    const bool wide = reinterpret_cast<uintptr_t>(out) % 16 == 0 && ldo * sizeof(T) % 16 == 0;
    const long long atoms = ms_tiles_k(k) * ms_atoms(fmt), runs = (k + kRun - 1) / kRun;
    int log_lanes = 0;
    while ((1 << log_lanes) < runs && log_lanes < 8) ++log_lanes;
    const dim3 grid(unsigned((q.rows + (256 >> log_lanes) - 1) >> (8 - log_lanes)), unsigned((runs + (1 << log_lanes) - 1) >> log_lanes));
    T* const o = static_cast<T*>(out);
    const auto kernel = fmt == kNvfp4 ? (wide ? tcq_ms_dequantize_kernel<T, kNvfp4, true> : tcq_ms_dequantize_kernel<T, kNvfp4, false>)
                                      : (wide ? tcq_ms_dequantize_kernel<T, kMxfp4, true> : tcq_ms_dequantize_kernel<T, kMxfp4, false>);
    kernel<<<grid, 256, 0, stream>>>(q.codes, ms_pitch(k), q.scales, atoms, q.row_scale, q.rows, k, o, ldo, log_lanes);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_ms_quantize(const void* x, int dtype, long long rows, long long k, long long ldx, int fmt, int rotate, const float* signs,
                               uint8_t* codes, uint8_t* scales, float* row_scale, cudaStream_t stream) {
    switch (dtype) {
        case kF32: return quantize_t<float>(x, rows, k, ldx, fmt, rotate, signs, codes, scales, row_scale, stream);
        case kF16: return quantize_t<__half>(x, rows, k, ldx, fmt, rotate, signs, codes, scales, row_scale, stream);
        default: return quantize_t<__nv_bfloat16>(x, rows, k, ldx, fmt, rotate, signs, codes, scales, row_scale, stream);
    }
}

cudaError_t launch_ms_dequantize(const MsMatrix& q, long long k, int fmt, void* out, int dtype, long long ldo, cudaStream_t stream) {
    switch (dtype) {
        case kF32: return dequantize_t<float>(q, k, fmt, out, ldo, stream);
        case kF16: return dequantize_t<__half>(q, k, fmt, out, ldo, stream);
        default: return dequantize_t<__nv_bfloat16>(q, k, fmt, out, ldo, stream);
    }
}

}  // namespace tcq
