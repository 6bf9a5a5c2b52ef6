// Products of 16- and 32-bit activations with a 4-bit microscaled matrix, few tokens: y[i][r] = sum_c x[i][c] * W[r][c].
//
// Every value of W is a bf16 number (two bits of e2m1 times at most four of a scale), and an fp16 or fp32 activation is the sum of two or
// three of them (8 significant bits each, cut off, not rounded; each held times 2^8 more than the one before).  So all products are exact on the tensor cores' bf16 path, and x enters
// as m * P rows of bf16: P = 1 (bf16), 2 (fp16), 3 (fp32), the parts of a token next to each other, added up at the end.
//
// A warp takes 16 rows of W x 256 columns a step (mma.sync m16n8k16): lane (g, t) holds columns 64 t .. 64 t + 63 of two rows, which are 32
// bytes of codes and one word of scales each; the order of the columns within a product is free as long as W and x agree, so four
// consecutive codes are a lane's share of a 16-column product.  Two byte permutations look the four magnitudes up as the bytes of bf16 numbers,
// one spreads the signs, one multiplication per pair brings the scale in.
// The 16 rows are 4 x 4: rows 4 i .. 4 i + 3 of each 32 in a group of 128, whose scales are 64 neighbouring bytes.
// Warps of a CTA share the columns; partial sums meet in shared memory, in a fixed order.  Sums within a step are the tensor core's, steps are
// added in fp32 with rounding to nearest.
#include "tcq_microscale_weights.cuh"

namespace tcq {

namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;

struct LinearArgs {
    const __nv_bfloat16* x;      // [virtual tokens][ldx], zeros behind column k up to a multiple of 256; 16-byte aligned rows
    long long ldx;
    long long m;                 // tokens
    MsMatrix w;
    long long pitch, atoms;      // bytes of codes a row; atoms of scales a row group
    int k_tiles;
    void* y;
    long long ldy;
    int warps_k;                 // warps that share a row group's columns: 1, 2, 4 or 8
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// NT: groups of eight virtual tokens; P: of them per token.
template <typename YT, int FMT, int NT, int P>
__global__ void __launch_bounds__(kThreads) tcq_ms_linear_kernel(const __grid_constant__ LinearArgs p) {
    constexpr int kTokens = 8 * NT / P;                  // of a pass
    __shared__ float part[kWarps][16][8 * NT + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wk = warp % p.warps_k, local = warp / p.warps_k, groups = kWarps / p.warps_k;
    const long long token0 = (long long)blockIdx.y * kTokens;
    const long long row_groups = (p.w.rows + 127) / 128 * 8;
    const long long virt = (p.m - token0 < kTokens ? p.m - token0 : kTokens) * P;

    for (long long rg0 = (long long)blockIdx.x * groups; rg0 < row_groups; rg0 += (long long)gridDim.x * groups) {
        const long long rg = rg0 + local;
        float acc[NT][4] = {};
        if (rg < row_groups) {
            const long long group = rg >> 3;
            const int r32 = int(rg & 7) * 4 + (g & 3), q0 = g >> 2;               // row 128 group + 32 q + r32, q = q0 and q0 + 2
            const long long row[2] = {group * 128 + 32 * q0 + r32, group * 128 + 32 * (q0 + 2) + r32};
            const uint8_t* codes[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) codes[h] = p.w.codes + (row[h] < p.w.rows ? row[h] : p.w.rows - 1) * p.pitch;
            const uint8_t* const scales = p.w.scales + group * p.atoms * 512 + r32 * 16 + q0 * 4;
            for (int kt = wk; kt < p.k_tiles; kt += p.warps_k) {
                uint4 c[2][2];
                uint32_t s[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const long long at = (long long)kt * 128 + 32 * t + 16 * i;
                        c[h][i] = at < p.pitch ? __ldg(reinterpret_cast<const uint4*>(codes[h] + at)) : make_uint4(0, 0, 0, 0);
                    }
                    if constexpr (FMT == kNvfp4) s[h] = __ldg(reinterpret_cast<const uint32_t*>(scales + ((long long)kt * 4 + t) * 512 + 8 * h));
                    else s[h] = __ldg(reinterpret_cast<const uint16_t*>(scales + ((long long)kt * 2 + t / 2) * 512 + 8 * h + 2 * (t & 1)));
                }
                float sum[NT][4] = {};
#pragma unroll
                for (int q = 0; q < 4; ++q) {            // 16 columns of each lane
                    const __nv_bfloat162 s0 = scale_of<FMT>(s[0], q), s1 = scale_of<FMT>(s[1], q);
                    uint4 b[NT][2];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint4* const from = reinterpret_cast<const uint4*>(p.x + (token0 * P + 8 * n + g) * p.ldx + (long long)kt * 256 + 64 * t + 16 * q);
#pragma unroll
                        for (int i = 0; i < 2; ++i) b[n][i] = 8 * n + g < virt ? __ldg(from + i) : make_uint4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {        // four of them are a lane's share of a product
                        const int word = q % 2 * 2 + j / 2;
                        uint32_t a[4];
                        const uint4 c0 = c[0][q / 2], c1 = c[1][q / 2];
                        const uint32_t w0 = word == 0 ? c0.x : word == 1 ? c0.y : word == 2 ? c0.z : c0.w;
                        const uint32_t w1 = word == 0 ? c1.x : word == 1 ? c1.y : word == 2 ? c1.z : c1.w;
                        four_weights(j & 1 ? w0 >> 16 : w0, s0, a[0], a[2]);
                        four_weights(j & 1 ? w1 >> 16 : w1, s1, a[1], a[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const uint4 v = b[n][j / 2];
                            mma_bf16(sum[n], a, j & 1 ? v.z : v.x, j & 1 ? v.w : v.y);
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[n][i] += sum[n][i];
            }
        }
        __syncthreads();                                 // (the previous row groups' sums have been read)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[warp][g + 8 * (i >> 1)][8 * n + 2 * t + (i & 1)] = acc[n][i];
        __syncthreads();
        for (int i = threadIdx.x; i < groups * 16 * kTokens; i += kThreads) {
            const int r16 = i & 15, token = i / 16 % kTokens, lg = i / 16 / kTokens;
            const long long group_of = rg0 + lg, r = (group_of >> 3) * 128 + 32 * (r16 >> 2) + (group_of & 7) * 4 + (r16 & 3);
            if (group_of >= row_groups || r >= p.w.rows || token0 + token >= p.m) continue;
            float f = 0.0f;
#pragma unroll
            for (int q = P - 1; q >= 0; --q) {           // the smallest parts first
                float one = 0.0f;
                for (int v = 0; v < p.warps_k; ++v) one += part[lg * p.warps_k + v][r16][token * P + q];
                f += q == 2 ? one * 0x1p-16f : q == 1 ? one * 0x1p-8f : one;
            }
            if constexpr (FMT == kNvfp4) f *= p.w.row_scale[r];
            static_cast<YT*>(p.y)[(token0 + token) * p.ldy + r] = from_f32<YT>(f);
        }
    }
}

// x as m * P rows of bf16 with zeros behind column k: the parts of a token one after the other, each the next eight significant bits,
// times 2^8 more than the one before, so that the last bits of the smallest numbers are still bf16 numbers.
template <typename T, int P>
__global__ void __launch_bounds__(256) tcq_ms_parts_kernel(const T* __restrict__ x, long long m, long long k, long long ldx, __nv_bfloat16* __restrict__ out,
                                                           long long width) {
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x, runs = width / 8;
    if (id >= m * runs) return;
    const long long i = id / runs, c0 = (id - i * runs) * 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c0 + j < k ? to_f32<T>(x[i * ldx + c0 + j]) : 0.0f;
#pragma unroll
    for (int q = 0; q < P; ++q) {
        uint32_t w[4] = {};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // the top 16 bits; of a NaN, whose payload may lie below them, any NaN
            const uint32_t bits = v[j] != v[j] ? 0x7FFF0000u : __float_as_uint(v[j]) & 0xFFFF0000u;
            w[j / 2] |= j & 1 ? bits : bits >> 16;
            v[j] = (bits & 0x7F800000u) == 0x7F800000u ? 0.0f : (v[j] - __uint_as_float(bits)) * 256.0f;      // exact, and below 2 |v|
        }
        *reinterpret_cast<uint4*>(out + (i * P + q) * width + c0) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <typename YT, int FMT, int NT, int P>
cudaError_t launch(LinearArgs p, int sms, cudaStream_t stream) {
    constexpr int kTokens = 8 * NT / P;
    const long long row_groups = (p.w.rows + 127) / 128 * 8;
    p.warps_k = 8;
    while (p.warps_k > 1 && p.warps_k > p.k_tiles) p.warps_k /= 2;
    const long long want = (row_groups + kWarps / p.warps_k - 1) / (kWarps / p.warps_k);
    const dim3 grid(unsigned(want < 8ll * sms ? want : 8ll * sms), unsigned((p.m + kTokens - 1) / kTokens));
    tcq_ms_linear_kernel<YT, FMT, NT, P><<<grid, kThreads, 0, stream>>>(p);
    return cudaGetLastError();
}

template <typename YT, int P>
cudaError_t launch_fmt(const LinearArgs& p, int fmt, int sms, cudaStream_t stream) {
    return fmt == kNvfp4 ? launch<YT, kNvfp4, 1, P>(p, sms, stream) : launch<YT, kMxfp4, 1, P>(p, sms, stream);
}

template <typename T, int P>
cudaError_t split(const void* x, long long m, long long k, long long ldx, void* ws, long long width, cudaStream_t stream) {
    tcq_ms_parts_kernel<T, P><<<unsigned((m * (width / 8) + 255) / 256), 256, 0, stream>>>(static_cast<const T*>(x), m, k, ldx, static_cast<__nv_bfloat16*>(ws), width);
    return cudaGetLastError();
}

}  // namespace

// tcq_microscale_linear_many.cu: x as m * parts rows of bf16, `width` columns of them (the others zero), 16-byte aligned.
cudaError_t launch_ms_linear_many(const __nv_bfloat16* x, long long ldx, long long width, long long m, int parts, int dtype, const MsMatrix& w, long long k,
                                  int fmt, void* y, long long ldy, cudaStream_t stream);

bool ms_linear_direct(const void* x, int dtype, long long k, long long ldx) {
    return dtype == kBf16 && k % kMsTileK == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % 8 == 0;
}

size_t ms_linear_workspace_bytes(long long m, long long k, int dtype) {
    return size_t(m) * size_t(ms_tiles_k(k) * kMsTileK) * 2 * (dtype == kF32 ? 3 : dtype == kF16 ? 2 : 1);
}

cudaError_t launch_ms_linear(const void* x, int dtype, long long m, long long ldx, const MsMatrix& w, long long k, int fmt, void* y,
                             long long ldy, void* ws, cudaStream_t stream) {
    const long long width = ms_tiles_k(k) * kMsTileK;
    const int parts = dtype == kF32 ? 3 : dtype == kF16 ? 2 : 1;
    LinearArgs p{static_cast<const __nv_bfloat16*>(ws), width, m, w, ms_pitch(k), ms_tiles_k(k) * ms_atoms(fmt), int(ms_tiles_k(k)), y, ldy, 1};
    const bool few = m * parts <= 8, direct = ms_linear_direct(x, dtype, k, ldx);
    cudaError_t err = cudaSuccess;
    if (direct) { p.x = static_cast<const __nv_bfloat16*>(x); p.ldx = ldx; }
    else if (dtype == kF32) err = split<float, 3>(x, m, k, ldx, ws, width, stream);
    else if (dtype == kF16) err = split<__half, 2>(x, m, k, ldx, ws, width, stream);
    else err = split<__nv_bfloat16, 1>(x, m, k, ldx, ws, width, stream);
    if (err != cudaSuccess) return err;
    if (!few) return launch_ms_linear_many(p.x, p.ldx, direct ? k : width, m, parts, dtype, w, k, fmt, y, ldy, stream);
    const int sms = ms_sm_count();
    if (dtype == kF32) return launch_fmt<float, 3>(p, fmt, sms, stream);
    if (dtype == kF16) return launch_fmt<__half, 2>(p, fmt, sms, stream);
    return launch_fmt<__nv_bfloat16, 1>(p, fmt, sms, stream);
}

}  // namespace tcq
