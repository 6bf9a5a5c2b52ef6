// Quantisation to 4-bit microscaled formats, and back.
//
// mxfp4: block of 32, scale X = 2^(floor(log2 amax) - 2), code = e2m1(x / X).
// nvfp4: block of 16, row scale g = the least 2^j, j >= -80, with amax(row) <= 2688 g (2688 = 6 * 448, the largest values of the two small
// types), block scale s = e4m3(amax / (6 g)), code = e2m1(x / (s g)).
// Every code is the nearest of the real quotient: divisors are powers of two times at most four bits, so that an fp32 quotient, correctly
// rounded, is on a border between two codes (a number of at most four bits) only where the real one is.  (For x near t d, both on
// grids no finer than ulp(x), |x / d - t| >= ulp(x) / d, which is more than half an ulp of t.)  The same holds for amax / 6 and e4m3.
// A block with a NaN or an infinity gets the scale NaN and codes 0, and counts for nothing in the row's largest value.
#include "tcq_microscale.cuh"

namespace tcq {

namespace {

constexpr int kRun = 16;         // consecutive values of a thread: one nvfp4 block, half an mxfp4 block

template <typename T>
__device__ __forceinline__ void load_run(const T* __restrict__ row, long long c0, long long k, bool wide, float (&v)[kRun]) {
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
        } else {
#pragma unroll
            for (int i = 0; i < kRun; ++i) v[i] = to_f32<T>(row[c0 + i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kRun; ++i) v[i] = c0 + i < k ? to_f32<T>(row[c0 + i]) : 0.0f;
    }
}

// Signs, then the transform of every b = `rotate` columns: the first four stages within the thread, the others between neighbouring lanes.
// b divides k, and all lanes of a group of b / 16 take part.
__device__ __forceinline__ void rotate_run(float (&v)[kRun], const float* __restrict__ signs, long long c0, long long k, int rotate) {
#pragma unroll
    for (int i = 0; i < kRun; ++i) v[i] *= c0 + i < k ? signs[c0 + i] : 1.0f;
#pragma unroll
    for (int h = 1; h < kRun; h *= 2)
#pragma unroll
        for (int i = 0; i < kRun; ++i)
            if (!(i & h)) {
                const float a = v[i], b = v[i + h];
                v[i] = a + b;
                v[i + h] = a - b;
            }
    for (int h = 1; h < rotate / kRun; h *= 2) {
        const bool upper = threadIdx.x & h;
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            const float o = __shfl_xor_sync(0xFFFFFFFFu, v[i], h);
            v[i] = upper ? o - v[i] : v[i] + o;
        }
    }
    const float scale = rotate == 16 ? 0.25f : rotate == 32 ? 0.17677669529663687f : rotate == 64 ? 0.125f : 0.08838834764831845f;
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

// One CTA a row (nvfp4 needs the row's largest value first); a thread takes 16 columns at a time.  Columns up to the next multiple of 256
// are worked on as zeros, so that the storage behind column k is written.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) tcq_ms_quantize_kernel(const T* __restrict__ x, long long k, long long ldx, bool wide, int rotate,
                                                              const float* __restrict__ signs, uint8_t* __restrict__ codes, long long pitch,
                                                              uint8_t* __restrict__ scales, long long atoms, float* __restrict__ row_scale) {
    const long long r = blockIdx.x;
    const T* const row = x + r * ldx;
    const long long span = (k + kMsTileK - 1) / kMsTileK * kMsTileK;
    int j = 0;
    float v[kRun];
    if constexpr (FMT == kNvfp4) {
        __shared__ uint32_t part[8];
        uint32_t m = 0;
        for (long long c = 0; c < span; c += 256 * kRun) {
            const long long c0 = c + (long long)threadIdx.x * kRun;
            load_run(row, c0, k, wide, v);
            if (rotate) rotate_run(v, signs, c0, k, rotate);
            if (largest_bits(v) < 0x7F800000u) m = max(m, largest_bits(v));
            else m = max(m, largest_finite_bits(v));
        }
        m = __reduce_max_sync(0xFFFFFFFFu, m);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
        __syncthreads();
        for (int w = 0; w < 8; ++w) m = max(m, part[w]);
        j = row_exponent(m);
        if (threadIdx.x == 0) row_scale[r] = pow2(j);
    }
    for (long long c = 0; c < span; c += 256 * kRun) {
        const long long c0 = c + (long long)threadIdx.x * kRun;
        load_run(row, c0, k, wide, v);
        if (rotate) rotate_run(v, signs, c0, k, rotate);
        uint32_t m = largest_bits(v), byte;
        if constexpr (FMT == kNvfp4) {
            const float inv = pow2(-j);
            byte = m < 0x7F800000u ? f32_to_e4m3(__fdiv_rn(__uint_as_float(m) * inv, 6.0f)) : 0x7Fu;
            const float s = e4m3_to_f32(byte);
#pragma unroll
            for (int i = 0; i < kRun; ++i) v[i] = s > 0.0f ? __fdiv_rn(v[i] * inv, s) : v[i] * 0.0f;
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
        if (c0 < 2 * pitch) *reinterpret_cast<uint2*>(codes + r * pitch + c0 / 2) = codes_of(v);
        if (c0 < span) {
            if constexpr (FMT == kNvfp4) scales[ms_scale_at(r, int(c0 / 16), atoms)] = uint8_t(c0 < k ? byte : 0);
            else if (!(threadIdx.x & 1)) scales[ms_scale_at(r, int(c0 / 32), atoms)] = uint8_t(c0 < k ? byte : 0);
        }
    }
}

// A thread takes 16 columns: 8 bytes of codes, one scale.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) tcq_ms_dequantize_kernel(const uint8_t* __restrict__ codes, long long pitch, const uint8_t* __restrict__ scales,
                                                                long long atoms, const float* __restrict__ row_scale, long long rows,
                                                                long long k, T* __restrict__ out, long long ldo, bool wide) {
    const long long runs = (k + kRun - 1) / kRun;
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id >= rows * runs) return;
    const long long r = id / runs, c0 = (id - r * runs) * kRun;
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(codes + r * pitch + c0 / 2));
    float s = ms_scale_to_f32<FMT>(scales[ms_scale_at(r, int(c0 / Ms<FMT>::kBlock), atoms)]);
    if constexpr (FMT == kNvfp4) s *= row_scale[r];
    T o[kRun];
#pragma unroll
    for (int i = 0; i < kRun; i += 2) {
        const uint32_t p = e2m1x2_to_f16x2(((i < 8 ? u.x : u.y) >> (4 * (i % 8))) & 0xFFu);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
        o[i] = from_f32<T>(f.x * s);
        o[i + 1] = from_f32<T>(f.y * s);
    }
    T* const to = out + r * ldo + c0;
    if (wide && c0 + kRun <= k) {
#pragma unroll
        for (int q = 0; q < int(kRun * sizeof(T) / 16); ++q) reinterpret_cast<uint4*>(to)[q] = reinterpret_cast<const uint4*>(o)[q];
    } else {
#pragma unroll
        for (int i = 0; i < kRun; ++i)
            if (c0 + i < k) to[i] = o[i];
    }
}

template <typename T>
cudaError_t quantize_t(const void* x, long long rows, long long k, long long ldx, int fmt, int rotate, const float* signs, uint8_t* codes,
                       uint8_t* scales, float* row_scale, cudaStream_t stream) {
    const bool wide = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * sizeof(T) % 16 == 0;
    const long long atoms = ms_tiles_k(k) * ms_atoms(fmt);
    const T* const p = static_cast<const T*>(x);
    if (fmt == kNvfp4) tcq_ms_quantize_kernel<T, kNvfp4><<<unsigned(rows), 256, 0, stream>>>(p, k, ldx, wide, rotate, signs, codes, ms_pitch(k), scales, atoms, row_scale);
    else tcq_ms_quantize_kernel<T, kMxfp4><<<unsigned(rows), 256, 0, stream>>>(p, k, ldx, wide, rotate, signs, codes, ms_pitch(k), scales, atoms, row_scale);
    return cudaGetLastError();
}

template <typename T>
cudaError_t dequantize_t(const MsMatrix& q, long long k, int fmt, void* out, long long ldo, cudaStream_t stream) {
    const bool wide = reinterpret_cast<uintptr_t>(out) % 16 == 0 && ldo * sizeof(T) % 16 == 0;
    const long long atoms = ms_tiles_k(k) * ms_atoms(fmt), runs = (k + kRun - 1) / kRun;
    const unsigned grid = unsigned((q.rows * runs + 255) / 256);
    T* const o = static_cast<T*>(out);
    if (fmt == kNvfp4) tcq_ms_dequantize_kernel<T, kNvfp4><<<grid, 256, 0, stream>>>(q.codes, ms_pitch(k), q.scales, atoms, q.row_scale, q.rows, k, o, ldo, wide);
    else tcq_ms_dequantize_kernel<T, kMxfp4><<<grid, 256, 0, stream>>>(q.codes, ms_pitch(k), q.scales, atoms, q.row_scale, q.rows, k, o, ldo, wide);
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
