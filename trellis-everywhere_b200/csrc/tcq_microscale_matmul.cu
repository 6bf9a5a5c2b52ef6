// Products of two 4-bit microscaled matrices, few tokens: y[i][r] = sum_c X[i][c] * W[r][c].
//
// tcgen05.mma (kind::mxf4nvf4, block scaled) multiplies 64 columns of 128 rows of W and NT tokens, with the block scales in tensor memory;
// codes come by TMA as they are stored, the scales by plain bulk copies, because the storage order of the scales is the one that
// tcgen05.cp wants.  fp32 sums stay in tensor memory over the whole of k.
//
// Work split: one CTA per SM goes through tiles of 128 rows of W x NT tokens.  One warp loads stages of 256 columns, one issues copies of
// scales and products, four take finished sums out of tensor memory (two buffers), scale them by the row scales, round and store.
// W is read once; where there are fewer tiles than SMs, a cluster of S CTAs shares the columns of a tile, and the S partial sums meet
// through distributed shared memory, in rank order.  Bound by the latency of one pass (few rows: one token,
// 4096 x 4096 5.4 us) or by what W's bytes take (many: 40960 x 4096 17.2 us, 5.5 TB/s; mxfp4 14.9, 6.3 TB/s).
//
// A wait that runs out (kMbarWaitCycles) makes its CTA stop, and its results from there on NaN, as those of its cluster.
#include <algorithm>

#include "tcq_microscale.cuh"
#include "tcq_tcgen05.cuh"

namespace tcq {

namespace {

constexpr int kThreads = 192;                    // loader, issuer, four warps for the results
constexpr int kRowsW = 128, kMostSplits = 8;

template <int FMT, int NT>
struct Tile {
    static constexpr int kAtoms = Ms<FMT>::kAtoms;
    static constexpr int kBytesW = kRowsW * 128, kBytesX = NT * 128, kBytesSw = kAtoms * 512, kBytesSx = kAtoms * 512;
    static constexpr int kStageBytes = (kBytesW + kBytesX + kBytesSw + kBytesSx + 1023) / 1024 * 1024;
    static constexpr int kSumColumns = NT < 32 ? 32 : NT;                     // of one of the two buffers of sums
    static constexpr int kScaleColumns = kAtoms * 4 * 2;                      // of one stage
    // as many stages as fit in 216 KB and in what the sums leave of 512 columns of tensor memory
    static constexpr int kBySmem = 216 * 1024 / kStageBytes, kByTmem = (512 - 2 * kSumColumns) / kScaleColumns;
    static constexpr int kStages = std::min(std::min(kBySmem, kByTmem), 12);
    static constexpr int kColumns = 2 * kSumColumns + kStages * kScaleColumns <= 256 ? 256 : 512;
    // over half of an SM's shared memory: two CTAs never share an SM, so that none waits for another's tensor memory
    static constexpr int kSmem = kStages * kStageBytes + 1024;
    static_assert(kSmem >= 116 * 1024 && kSmem <= 226 * 1024 && kStages >= 3 && kStages * kStageBytes >= NT * kRowsW * 4);
};

}  // namespace

// tcq_microscale_pair.cu: tiles of 256 tokens x nt rows of W on pairs of SMs.
cudaError_t launch_ms_matmul_pair(const MsMatrix& x, const MsMatrix& w, long long k, int fmt, void* y, int dtype, long long ldy, int nt, int sms, unsigned loads,
                                  cudaStream_t stream);

namespace {

struct MatmulArgs {
    const uint8_t* w_scales;
    const uint8_t* x_scales;
    const float* w_row;
    const float* x_row;
    long long n, m;
    int tiles_n, tiles_m, k_tiles;
    void* y;
    long long ldy;
    int dtype;
    bool aligned;                                // y and ldy multiples of four elements
    unsigned loads;                              // stages that a CTA loads, at most (a self-test's limit)
};

__device__ __forceinline__ void store(const MatmulArgs& p, long long at, float v) {
    if (p.dtype == kF32) static_cast<float*>(p.y)[at] = v;
    else if (p.dtype == kF16) static_cast<__half*>(p.y)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ void store4(const MatmulArgs& p, long long at, float4 v) {
    if (p.dtype == kF32) {
        *reinterpret_cast<float4*>(static_cast<float*>(p.y) + at) = v;
    } else if (p.dtype == kF16) {
        const __half2 h[2] = {__floats2half2_rn(v.x, v.y), __floats2half2_rn(v.z, v.w)};
        *reinterpret_cast<uint2*>(static_cast<__half*>(p.y) + at) = *reinterpret_cast<const uint2*>(h);
    } else {
        const __nv_bfloat162 h[2] = {__floats2bfloat162_rn(v.x, v.y), __floats2bfloat162_rn(v.z, v.w)};
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.y) + at) = *reinterpret_cast<const uint2*>(h);
    }
}

// Columns c0 .. c0 + N - 1 (tokens) of 32 rows of W, one a lane, scaled, rounded and stored: a store is 32 neighbours in y.
template <typename YT, int FMT, int N>
__device__ __forceinline__ void store_columns(const MatmulArgs& p, uint32_t (&v)[N], long long r, long long token0, float fw, float fx) {
    YT* to = static_cast<YT*>(p.y) + token0 * p.ldy + r;
    const int columns = int(min((long long)N, p.m - token0));
    if constexpr (FMT == kNvfp4) {
        const float inner = inner_part(fw), outer = outer_part(fw);
#pragma unroll
        for (int c = 0; c < N; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * inner * __shfl_sync(0xFFFFFFFFu, fx, c));
        if (__any_sync(0xFFFFFFFFu, outer != 1.0f)) {
#pragma unroll
            for (int c = 0; c < N; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * outer);
        }
    }
#pragma unroll
    for (int c = 0; c < N; ++c, to += p.ldy) {
        if (r < p.n && c < columns) *to = from_f32<YT>(__uint_as_float(v[c]));
    }
}

template <int FMT>
__device__ __forceinline__ void mma_block_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, bool add) {
    if constexpr (FMT == kNvfp4)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(uint32_t(add)) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(uint32_t(add)) : "memory");
}

template <int FMT, int NT>
__global__ void __launch_bounds__(kThreads, 1) tcq_ms_matmul_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                                                    const __grid_constant__ MatmulArgs p) {
    using T = Tile<FMT, NT>;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[T::kStages], empty[T::kStages], sum_full[2], sum_empty[2], drained;
    __shared__ uint32_t tmem_at;
    __shared__ unsigned int gave_up;
    const uint32_t smem = (smem_u32(raw) + 1023) & ~1023u;
    const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), splits = cluster_size();
    const int first = int((long long)p.k_tiles * rank / splits), last = int((long long)p.k_tiles * (rank + 1) / splits);
    const int tiles = p.tiles_n * p.tiles_m, clusters = gridDim.x / splits;
    const long long atoms = (long long)p.k_tiles * T::kAtoms;

    auto load = [&](uint32_t s, int t, int kt) {
        const int tn = t / p.tiles_m, tm = t % p.tiles_m;
        const uint32_t to = smem + s * T::kStageBytes, bar = smem_u32(&full[s]);
        mbar_expect(bar, T::kBytesW + T::kBytesX + T::kBytesSw + T::kBytesSx);
        tma_load(to, &map_w, kt * 128, tn * kRowsW, bar);
        tma_load(to + T::kBytesW, &map_x, kt * 128, tm * NT, bar);
        bulk_load(to + T::kBytesW + T::kBytesX, p.w_scales + (tn * atoms + (long long)kt * T::kAtoms) * 512, T::kBytesSw, bar);
        bulk_load(to + T::kBytesW + T::kBytesX + T::kBytesSw, p.x_scales + (tm * atoms + (long long)kt * T::kAtoms) * 512, T::kBytesSx, bar);
    };
    // The first tile's first stages are on their way before anything else: with few tokens a call is little more than its latencies.
    const int ahead = min(min(unsigned(T::kStages), unsigned(last - first)), p.loads);
    if (warp == 0) {
        if (elect_one()) {
            gave_up = 0;
            for (int s = 0; s < T::kStages; ++s) { mbar_init(smem_u32(&full[s]), 1); mbar_init(smem_u32(&empty[s]), 1); }
            for (int s = 0; s < 2; ++s) { mbar_init(smem_u32(&sum_full[s]), 1); mbar_init(smem_u32(&sum_empty[s]), 4); }
            mbar_init(smem_u32(&drained), 1);
            asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
            for (int i = 0; i < ahead; ++i) load(i, blockIdx.x / splits, first + i);
        }
        __syncwarp();
    }
    if (warp == 1) tmem_alloc(smem_u32(&tmem_at), T::kColumns);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at, tmem_scales = tmem + 2 * T::kSumColumns;

    if (warp == 0) {
        // ---- loads; the warp stays together, one lane issues
        const bool one = elect_one();
        uint32_t s = ahead % T::kStages, phase = ahead == T::kStages ? 0 : 1, loaded = ahead;    // (the first wait for a stage is for the phase before the first)
        unsigned left = p.loads - ahead;
        bool ok = true;
        int kt = first + ahead;
        for (int t = blockIdx.x / splits; t < tiles && ok; t += clusters, kt = first)
            for (; kt < last; ++kt) {
                ok = still_waits(left-- > 0, smem_u32(&empty[s]), phase, &gave_up);      // every lane has seen this phase before the next can begin
                if (!ok) break;
                if (one) load(s, t, kt);
                __syncwarp();
                if (++s == T::kStages) { s = 0; phase ^= 1; }
                if (loaded < T::kStages) ++loaded;
            }
        wait_for_loads<T::kStages>(full, s, phase, loaded);
        if (splits > 1 && gave_up)                       // a load that was late may lie over the NaN of this CTA's part
            for (int i = lane; i < NT * kRowsW; i += 32) reinterpret_cast<uint32_t*>(raw + (smem - smem_u32(raw)))[i] = 0x7FC00000u;
    } else if (warp == 1) {
        // ---- products; likewise
        constexpr uint32_t kIdesc = 1u << 7 | 1u << 10 | uint32_t(NT >> 3) << 17 | (FMT == kMxfp4 ? 1u : 0u) << 23 | 1u << 27;
        const bool one = elect_one();
        uint32_t s = 0, phase = 0;
        int n = 0;
        bool ok = true;
        for (int t = blockIdx.x / splits; t < tiles && ok; t += clusters, ++n) {
            const int buf = n & 1;
            if (n >= 2) ok = mbar_wait(smem_u32(&sum_empty[buf]), uint32_t(n / 2 - 1) & 1, &gave_up);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tmem + buf * T::kSumColumns;
            for (int kt = first; kt < last; ++kt) {
                ok = mbar_wait(smem_u32(&full[s]), phase, &gave_up);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = smem + s * T::kStageBytes, sw = tmem_scales + s * T::kScaleColumns, sx = sw + T::kAtoms * 4;
                const uint64_t dw = desc_rows128(at), dx = desc_rows128(at + T::kBytesW), ds = desc_rows16(at + T::kBytesW + T::kBytesX);
                if (one) {
#pragma unroll
                    for (int j = 0; j < T::kAtoms; ++j) {
                        tc_copy_scales(sw + 4 * j, ds + 32 * j);
                        tc_copy_scales(sx + 4 * j, ds + (T::kBytesSw >> 4) + 32 * j);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {            // 64 columns: 32 bytes of a row, one word of scales (nvfp4) or half a word (mxfp4)
                        const int atom = FMT == kNvfp4 ? j : j / 2;
                        const uint32_t id = FMT == kNvfp4 ? 0u : 2u * (j % 2);
                        mma_block_scaled<FMT>(d, dw + 2 * j, dx + 2 * j, kIdesc | id << 4 | id << 29, sw + 4 * atom, sx + 4 * atom, kt > first || j > 0);
                    }
                    tc_commit(smem_u32(&empty[s]));
                }
                __syncwarp();
                if (++s == T::kStages) { s = 0; phase ^= 1; }
            }
            if (ok && one) tc_commit(smem_u32(&sum_full[buf]));
            __syncwarp();
        }
        if (!ok) {                                           // what was issued ends before the tensor memory goes
            if (one) tc_commit(smem_u32(&drained));
            __syncwarp();
            for (long long t0 = clock64(); !mbar_try_wait(smem_u32(&drained), 0) && clock64() - t0 < kMbarWaitCycles;) {}
        }
    } else {
        // ---- results: this warp's lanes are 32 rows of W, so that a store is 32 neighbours in y
        const int quarter = warp & 3;
        constexpr int kChunk = NT < 32 ? NT : 32;
        int n = 0;
        bool ok = true;
        for (int t = blockIdx.x / splits; t < tiles; t += clusters, ++n) {
            const int buf = n & 1;
            const long long r = (long long)(t / p.tiles_m) * kRowsW + 32 * quarter + lane, i0 = (long long)(t % p.tiles_m) * NT;
            const float fw = FMT == kNvfp4 && r < p.n ? p.w_row[r] : 1.0f;
            ok = still_waits(ok, smem_u32(&sum_full[buf]), uint32_t(n / 2) & 1, &gave_up);
            tc_fence_after();
#pragma unroll 1
            for (int c0 = 0; c0 < NT; c0 += kChunk) {
                uint32_t v[kChunk];
                tmem_load<kChunk>(tmem + buf * T::kSumColumns + c0 + (uint32_t(32 * quarter) << 16), v);
                const float fx = FMT == kNvfp4 && i0 + c0 + lane < p.m ? __ldg(p.x_row + i0 + c0 + lane) : 1.0f;       // of column c0 + lane
                tmem_wait_ld();
                if (c0 + kChunk >= NT) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sum_empty[buf]));
                }
#pragma unroll
                for (int c = 0; c < kChunk; ++c)
                    if (!ok) v[c] = 0x7FC00000u;
                if (splits > 1) {
                    float* const part = reinterpret_cast<float*>(raw + (smem - smem_u32(raw))) + c0 * kRowsW + 32 * quarter + lane;
#pragma unroll
                    for (int c = 0; c < kChunk; ++c) part[c * kRowsW] = __uint_as_float(v[c]);
                } else if (p.dtype == kF32) {
                    store_columns<float, FMT>(p, v, r, i0 + c0, fw, fx);
                } else if (p.dtype == kF16) {
                    store_columns<__half, FMT>(p, v, r, i0 + c0, fw, fx);
                } else {
                    store_columns<__nv_bfloat16, FMT>(p, v, r, i0 + c0, fw, fx);
                }
            }
        }
    }
    __syncwarp();
    if (splits > 1) {                                        // one tile a cluster: add up the parts of it, four neighbours a thread
        cluster_sync();
        const int t = blockIdx.x / splits;
        const long long r0 = (long long)(t / p.tiles_m) * kRowsW, i0 = (long long)(t % p.tiles_m) * NT;
        const int columns = int(min((long long)NT, p.m - i0));
        for (int i = int(rank) * kThreads + threadIdx.x; i < kRowsW / 4 * columns; i += int(splits) * kThreads) {
            const long long r = r0 + i % (kRowsW / 4) * 4, token = i0 + i / (kRowsW / 4);
            if (r >= p.n) continue;
            float4 part[kMostSplits];
#pragma unroll
            for (uint32_t q = 0; q < kMostSplits; ++q)
                if (q < splits) part[q] = ld_cluster_f32x4(smem + 16 * i, q);
            float4 f = part[0];
#pragma unroll
            for (uint32_t q = 1; q < kMostSplits; ++q)
                if (q < splits) f = make_float4(f.x + part[q].x, f.y + part[q].y, f.z + part[q].z, f.w + part[q].w);
            float* const e = &f.x;
            if constexpr (FMT == kNvfp4) {
                const float fx = p.x_row[token];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float fw = r + j < p.n ? p.w_row[r + j] : 1.0f;
                    e[j] = e[j] * inner_part(fw) * fx * outer_part(fw);
                }
            }
            if (p.aligned && r + 4 <= p.n) {
                store4(p, token * p.ldy + r, f);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (r + j < p.n) store(p, token * p.ldy + r + j, e[j]);
            }
        }
        cluster_sync();                                      // no CTA ends while another reads its part
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free(tmem, T::kColumns);
    }
}

template <int FMT, int NT>
cudaError_t launch(const MsMatrix& x, const MsMatrix& w, long long k, void* y, int dtype, long long ldy, unsigned loads, cudaStream_t stream) {
    using T = Tile<FMT, NT>;
    static std::atomic<bool> ready[64];
    static MostClusters kept;
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev >= 64 || !ready[dev]) {
        if ((err = cudaFuncSetAttribute(tcq_ms_matmul_kernel<FMT, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem)) != cudaSuccess) return err;
        if (dev < 64) ready[dev] = true;
    }
    CUtensorMap map_w, map_x;
    const long long pitch = ms_pitch(k);
    if ((err = make_byte_map(&map_w, w.codes, pitch, w.rows, pitch, kRowsW)) != cudaSuccess) return err;
    if ((err = make_byte_map(&map_x, x.codes, pitch, x.rows, pitch, NT)) != cudaSuccess) return err;
    const size_t four = dtype == kF32 ? 16 : 8;
    const MatmulArgs p{w.scales, x.scales, w.row_scale, x.row_scale, w.rows, x.rows, int((w.rows + kRowsW - 1) / kRowsW), int((x.rows + NT - 1) / NT),
                       int(ms_tiles_k(k)), y, ldy, dtype, reinterpret_cast<uintptr_t>(y) % four == 0 && ldy % 4 == 0, loads};
    const long long tiles = (long long)p.tiles_n * p.tiles_m;
    int splits = 1;
    while (p.k_tiles >= 8 && splits < kMostSplits && splits * 4 <= p.k_tiles &&
           tiles <= ms_most_clusters(kept, reinterpret_cast<const void*>(tcq_ms_matmul_kernel<FMT, NT>), kThreads, T::kSmem, 1, splits * 2)) splits *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(splits > 1 ? tiles * splits : std::min<long long>(tiles, ms_sm_count())));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = T::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = unsigned(splits);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, tcq_ms_matmul_kernel<FMT, NT>, map_w, map_x, p);
}

// Which form.  us on a B200, nvfp4 (mxfp4 is up to 15 % faster at the same choices):
//   the columns shared by S CTAs while all run at once, at least two stages of 256 columns each, from eight stages on: one token, S = 1 / 2 / 4 / 8,
//     4096 x 4096 7.5 / 6.8 / 5.7 / 11.9 (more CTAs than SMs), 1024 x 4096 7.5 / 6.8 / 5.4 / 5.0, 4096 x 1024 4.5 / 5.1 / 4.9
//   one SM against a pair of SMs on 256 x 128 results: 64 tokens 8.8 and 10.9 (12288 x 4096), 7.8 and 7.6 (4096 x 4096); 128 tokens 10.5 and 11.5
//     (12288 x 4096, every SM busy), 12.6 and 13.6 (4096 x 12288, S = 4), but 10.2 and 8.2 (4096 x 4096), 6.7 and 6.0 (4096 x 1024);
//     256 tokens 14.9 and 11.8 (12288 x 4096)
//   pairs: a tile of 256 x 256 takes 1.8 times as long as one of 256 x 128, which decides by the rounds that either needs: 512 tokens 12288 x 4096
//     18.1 and 15.7, 2048 tokens 4096 x 12288 39.9 and 43.1
template <int FMT>
cudaError_t launch_fmt(const MsMatrix& x, const MsMatrix& w, long long k, void* y, int dtype, long long ldy, unsigned loads, cudaStream_t stream) {
    const long long m = x.rows, k_tiles = ms_tiles_k(k), tiles = (w.rows + kRowsW - 1) / kRowsW;
    const int sms = ms_sm_count();
    if (m > 128 || (m > 64 && tiles <= sms / 2 && k_tiles < 32)) {
        const long long pairs = sms / 2, tiles_m = (m + 255) / 256;
        const long long rounds128 = (tiles_m * tiles + pairs - 1) / pairs, rounds256 = (tiles_m * ((w.rows + 255) / 256) + pairs - 1) / pairs;
        return launch_ms_matmul_pair(x, w, k, FMT, y, dtype, ldy, 5 * rounds128 > 9 * rounds256 ? 256 : 128, sms, loads, stream);
    }
    if (m <= 8) return launch<FMT, 8>(x, w, k, y, dtype, ldy, loads, stream);
    if (m <= 16) return launch<FMT, 16>(x, w, k, y, dtype, ldy, loads, stream);
    if (m <= 32) return launch<FMT, 32>(x, w, k, y, dtype, ldy, loads, stream);
    if (m <= 64) return launch<FMT, 64>(x, w, k, y, dtype, ldy, loads, stream);
    return launch<FMT, 128>(x, w, k, y, dtype, ldy, loads, stream);
}

}  // namespace

int ms_sm_count() {
    static std::atomic<int> cache[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    if (dev < 64 && (n = cache[dev]) != 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    if (dev < 64) cache[dev] = n;
    return n;
}

int ms_most_clusters(MostClusters& kept, const void* kernel, int threads, size_t smem, int ctas, int size) {
    const int slot = size >= 8 ? 3 : size / 2, most = ctas * ms_sm_count() / size;
    int dev = 0, n = 0;
    if (size == 1 || cudaGetDevice(&dev) != cudaSuccess) return most;
    if (dev < 64 && (n = kept.of[dev][slot]) != 0) return n;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(size));
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = unsigned(size);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
        (void)cudaGetLastError();
        return most;
    }
    if (dev < 64) kept.of[dev][slot] = n;
    return n;
}

namespace {
cudaError_t encode_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, cuuint64_t width, cuuint64_t rows, cuuint64_t pitch, cuuint32_t box_width,
                       cuuint32_t box_rows, CUtensorMapSwizzle swizzle) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static std::atomic<Encode> kept{nullptr};
    Encode encode = kept;
    if (encode == nullptr) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found{};
        const cudaError_t err = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found);
        if (err != cudaSuccess) return err;
        if (found != cudaDriverEntryPointSuccess || fn == nullptr) return cudaErrorNotSupported;
        kept = encode = reinterpret_cast<Encode>(fn);
    }
    const cuuint64_t dims[2] = {width, rows}, strides[1] = {pitch};
    const cuuint32_t box[2] = {box_width, box_rows}, steps[2] = {1, 1};
    const CUresult rc = encode(map, type, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}
}  // namespace

cudaError_t make_byte_map(CUtensorMap* map, const void* base, long long width, long long rows, long long pitch, int box_rows) {
    return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, width, rows, pitch, 128, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

cudaError_t make_16bit_map(CUtensorMap* map, const void* base, long long width, long long rows, long long ld, int box_rows) {
    return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, base, width, rows, 2 * ld, 64, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

cudaError_t make_scale_map(CUtensorMap* map, const void* base, long long rows, int box_rows) {
    return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, base, 128, rows, 512, 128, box_rows, CU_TENSOR_MAP_SWIZZLE_NONE);
}

cudaError_t launch_ms_matmul(const MsMatrix& x, const MsMatrix& w, long long k, int fmt, void* y, int dtype, long long ldy, unsigned loads, cudaStream_t stream) {
    return fmt == kNvfp4 ? launch_fmt<kNvfp4>(x, w, k, y, dtype, ldy, loads, stream) : launch_fmt<kMxfp4>(x, w, k, y, dtype, ldy, loads, stream);
}

}  // namespace tcq
