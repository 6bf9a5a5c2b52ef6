// Products with 4-bit microscaled matrices: y[i][row] = sum_c X[i][c] * W[row][c], X in 32 or 16 bits or in 4 bits itself.
//
// 64 right-hand sides x 64 rows per CTA, 32 columns at a time as fp32 values in shared memory, 4 x 4 sums per thread; fp32
// products and sums in a fixed order.
#include <type_traits>

#include "tcq_microscale.cuh"

namespace tcq {

namespace {

constexpr int kTile = 64, kStep = 32;

// Rows r0 .. r0 + 63, columns c0 .. c0 + 31 of a 4-bit matrix as values without the row scale (zeros outside): thread t does eight columns of row t / 4.
template <int FMT>
__device__ __forceinline__ void stage_codes(const MsMatrix& q, long long r0, long long c0, long long k, long long pitch, long long atoms,
                                            float (*to)[kTile + 4]) {
    const int t = threadIdx.x, lr = t >> 2, lc = (t & 3) * 8;
    const long long r = r0 + lr, c = c0 + lc;
    uint32_t u = 0;
    float s = 0.0f;
    if (r < q.rows && c < k) {
        u = __ldg(reinterpret_cast<const uint32_t*>(q.codes + r * pitch + c / 2));
        s = ms_scale_to_f32<FMT>(q.scales[ms_scale_at(r, int(c / Ms<FMT>::kBlock), atoms)]);
    }
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint32_t p = e2m1x2_to_f16x2((u >> (4 * i)) & 0xFFu);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
        to[lc + i][lr] = f.x * s;
        to[lc + i + 1][lr] = f.y * s;
    }
}

template <typename T>
__device__ __forceinline__ void stage_values(const T* __restrict__ x, long long ldx, long long m, long long r0, long long c0, long long k,
                                             float (*to)[kTile + 4]) {
    const int t = threadIdx.x, lr = t >> 2, lc = (t & 3) * 8;
    const long long r = r0 + lr;
#pragma unroll
    for (int i = 0; i < 8; ++i) to[lc + i][lr] = r < m && c0 + lc + i < k ? to_f32<T>(x[r * ldx + c0 + lc + i]) : 0.0f;
}

// XT: the right-hand sides' type, or void for 4 bits (xq).
template <typename XT, typename YT, int FMT>
__global__ void __launch_bounds__(256) tcq_ms_product_kernel(const void* __restrict__ x, long long ldx, long long m, MsMatrix xq, MsMatrix w,
                                                             long long k, long long pitch, long long atoms, YT* __restrict__ y, long long ldy) {
    __shared__ float xs[kStep][kTile + 4], ws[kStep][kTile + 4];
    const long long r0 = (long long)blockIdx.x * kTile, i0 = (long long)blockIdx.y * kTile;
    const int tr = (threadIdx.x & 15) * 4, ti = (threadIdx.x >> 4) * 4;
    float acc[4][4] = {};
    for (long long c0 = 0; c0 < k; c0 += kStep) {
        if constexpr (std::is_void_v<XT>) stage_codes<FMT>(xq, i0, c0, k, pitch, atoms, xs);
        else stage_values(static_cast<const XT*>(x), ldx, m, i0, c0, k, xs);
        stage_codes<FMT>(w, r0, c0, k, pitch, atoms, ws);
        __syncthreads();
#pragma unroll 8
        for (int c = 0; c < kStep; ++c) {
            const float4 a = *reinterpret_cast<const float4*>(&xs[c][ti]), b = *reinterpret_cast<const float4*>(&ws[c][tr]);
            const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __fmaf_rn(av[i], bv[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const long long t = i0 + ti + i, r = r0 + tr + j;
            if (t >= m || r >= w.rows) continue;
            float v = acc[i][j];
            if constexpr (FMT == kNvfp4) {
                v *= w.row_scale[r];
                if constexpr (std::is_void_v<XT>) v *= xq.row_scale[t];
            }
            y[t * ldy + r] = from_f32<YT>(v);
        }
}

template <typename XT, typename YT>
cudaError_t launch_product(const void* x, long long ldx, long long m, const MsMatrix& xq, const MsMatrix& w, long long k, int fmt, void* y,
                           long long ldy, cudaStream_t stream) {
    const long long atoms = ms_tiles_k(k) * ms_atoms(fmt);
    const dim3 grid(unsigned((w.rows + kTile - 1) / kTile), unsigned((m + kTile - 1) / kTile));
    if (fmt == kNvfp4) tcq_ms_product_kernel<XT, YT, kNvfp4><<<grid, 256, 0, stream>>>(x, ldx, m, xq, w, k, ms_pitch(k), atoms, static_cast<YT*>(y), ldy);
    else tcq_ms_product_kernel<XT, YT, kMxfp4><<<grid, 256, 0, stream>>>(x, ldx, m, xq, w, k, ms_pitch(k), atoms, static_cast<YT*>(y), ldy);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_ms_linear(const void* x, int dtype, long long m, long long ldx, const MsMatrix& w, long long k, int fmt, void* y,
                             long long ldy, cudaStream_t stream) {
    const MsMatrix none{};
    switch (dtype) {
        case kF32: return launch_product<float, float>(x, ldx, m, none, w, k, fmt, y, ldy, stream);
        case kF16: return launch_product<__half, __half>(x, ldx, m, none, w, k, fmt, y, ldy, stream);
        default: return launch_product<__nv_bfloat16, __nv_bfloat16>(x, ldx, m, none, w, k, fmt, y, ldy, stream);
    }
}

}  // namespace tcq
