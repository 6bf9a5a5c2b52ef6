// Products of two 4-bit microscaled matrices on the tensor cores: y[i][r] = sum_c X[i][c] * W[r][c].
//
// tcgen05.mma (kind::mxf4nvf4, block scaled) multiplies 64 columns of 128 rows of one operand ("A") and NT rows of the other ("B"), with
// the block scales in tensor memory; both operands come by TMA as they are stored, the scales by plain bulk copies, because
// the storage order of the scales is the one that tcgen05.cp wants.  fp32 sums stay in tensor memory over the whole of k.
//
// Work split: one CTA per SM goes through tiles of 128 x NT results.  One thread loads stages of 256 columns, one issues copies of
// scales and products, four warps take finished sums out of tensor memory (two buffers, where they fit), scale them by the row scales, round
// and store.  With few tokens W's rows are the 128 and the tokens the NT: the weights are read once, and a cluster of S CTAs shares the
// columns of a tile where there are fewer tiles than SMs; the S partial sums meet through distributed shared memory, in rank order.
//
// A wait that runs out (kMbarWaitCycles) makes its CTA stop, and its results NaN.
#include <algorithm>

#include "tcq_microscale.cuh"
#include "tcq_tcgen05.cuh"

namespace tcq {

namespace {

constexpr int kThreads = 192;                    // loader, issuer, four warps for the results
constexpr int kRowsA = 128;

template <int FMT, int NT>
struct Tile {
    static constexpr int kAtoms = Ms<FMT>::kAtoms;
    static constexpr int kGroups = (NT + 127) / 128;                          // 128-row groups of B's scales
    static constexpr int kBytesA = kRowsA * 128, kBytesB = NT * 128, kBytesSa = kAtoms * 512, kBytesSb = kGroups * kAtoms * 512;
    static constexpr int kStageBytes = (kBytesA + kBytesB + kBytesSa + kBytesSb + 1023) / 1024 * 1024;
    static constexpr int kSumBuffers = NT <= 128 ? 2 : 1;
    static constexpr int kSumColumns = NT < 32 ? 32 : NT;                     // of one buffer
    static constexpr int kScaleColumns = kAtoms * 4 * (1 + kGroups);          // of one stage
    // as many stages as fit in 216 KB and in what the sums leave of 512 columns of tensor memory
    static constexpr int kBySmem = 216 * 1024 / kStageBytes, kByTmem = (512 - kSumBuffers * kSumColumns) / kScaleColumns;
    static constexpr int kStages = std::min(std::min(kBySmem, kByTmem), 12);
    static constexpr int kColumns = kSumBuffers * kSumColumns + kStages * kScaleColumns <= 256 ? 256 : 512;
    // over half of an SM's shared memory: two CTAs never share an SM, so that none waits for another's tensor memory
    static constexpr int kSmem = kStages * kStageBytes + 1024;
    static_assert(kSmem > 114 * 1024 && kSmem <= 226 * 1024 && kStages >= 3);
};

}  // namespace

// tcq_microscale_pair.cu: tiles of 256 tokens x nt rows of W on pairs of SMs.
cudaError_t launch_ms_matmul_pair(const MsMatrix& x, const MsMatrix& w, long long k, int fmt, void* y, int dtype, long long ldy, int nt, int sms, cudaStream_t stream);

namespace {

struct MatmulArgs {
    const uint8_t* a_scales;
    const uint8_t* b_scales;
    const float* a_row;
    const float* b_row;
    long long a_rows, b_rows;
    int tiles_a, tiles_b, k_tiles;
    void* y;
    long long step_a, step_b;                    // elements of y between neighbouring rows of A and of B
    int dtype;
};

__device__ __forceinline__ void store(const MatmulArgs& p, long long at, float v) {
    if (p.dtype == kF32) static_cast<float*>(p.y)[at] = v;
    else if (p.dtype == kF16) static_cast<__half*>(p.y)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v);
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
__global__ void __launch_bounds__(kThreads, 1) tcq_ms_matmul_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                                    const __grid_constant__ MatmulArgs p) {
    using T = Tile<FMT, NT>;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[T::kStages], empty[T::kStages], sum_full[T::kSumBuffers], sum_empty[T::kSumBuffers], drained;
    __shared__ uint32_t tmem_at;
    __shared__ unsigned int gave_up;
    const uint32_t smem = (smem_u32(raw) + 1023) & ~1023u;
    const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), splits = cluster_size();
    const int first = int((long long)p.k_tiles * rank / splits), last = int((long long)p.k_tiles * (rank + 1) / splits);
    const int tiles = p.tiles_a * p.tiles_b, clusters = gridDim.x / splits;

    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < T::kStages; ++s) { mbar_init(smem_u32(&full[s]), 1); mbar_init(smem_u32(&empty[s]), 1); }
        for (int s = 0; s < T::kSumBuffers; ++s) { mbar_init(smem_u32(&sum_full[s]), 1); mbar_init(smem_u32(&sum_empty[s]), 4); }
        mbar_init(smem_u32(&drained), 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(smem_u32(&tmem_at), T::kColumns);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at, tmem_scales = tmem + T::kSumBuffers * T::kSumColumns;
    const long long atoms = (long long)p.k_tiles * T::kAtoms;

    if (warp == 0) {
        // ---- loads; the warp stays together, one lane issues
        const bool one = elect_one();
        uint32_t s = 0, phase = 1, loaded = 0;           // (the first wait for each stage is for the phase before the first)
        bool ok = true;
        const long long groups_b = (p.b_rows + 127) / 128;
        for (int t = blockIdx.x / splits; t < tiles && ok; t += clusters) {
            const int ta = t / p.tiles_b, tb = t % p.tiles_b;
            const uint8_t* const from_a = p.a_scales + ta * atoms * 512;
            const uint8_t* from_b[T::kGroups];
#pragma unroll
            for (int g = 0; g < T::kGroups; ++g) {
                const long long group = (long long)tb * NT / 128 + g;             // one behind the last only has rows without results
                from_b[g] = p.b_scales + (group < groups_b ? group : groups_b - 1) * atoms * 512;
            }
            for (int kt = first; kt < last; ++kt) {
                ok = mbar_wait(smem_u32(&empty[s]), phase, &gave_up);
                ok = __all_sync(0xFFFFFFFFu, ok);        // every lane has seen this phase before the next can begin
                if (!ok) break;
                if (one) {
                    const uint32_t to = smem + s * T::kStageBytes, bar = smem_u32(&full[s]);
                    mbar_expect(bar, T::kBytesA + T::kBytesB + T::kBytesSa + T::kBytesSb);
                    tma_load(to, &map_a, kt * 128, ta * kRowsA, bar);
                    tma_load(to + T::kBytesA, &map_b, kt * 128, tb * NT, bar);
                    bulk_load(to + T::kBytesA + T::kBytesB, from_a + (long long)kt * T::kBytesSa, T::kBytesSa, bar);
#pragma unroll
                    for (int g = 0; g < T::kGroups; ++g)
                        bulk_load(to + T::kBytesA + T::kBytesB + T::kBytesSa + g * T::kAtoms * 512, from_b[g] + (long long)kt * T::kAtoms * 512, T::kAtoms * 512, bar);
                }
                __syncwarp();
                if (++s == T::kStages) { s = 0; phase ^= 1; }
                if (loaded < T::kStages) ++loaded;
            }
        }
        if (gave_up)                                     // nothing may be on its way to this CTA's memory when it ends: the last loads of each stage
            for (uint32_t i = 0; i < loaded; ++i) {
                if (s == 0) phase ^= 1;
                s = s == 0 ? T::kStages - 1 : s - 1;
                for (long long t0 = clock64(); !mbar_try_wait(smem_u32(&full[s]), phase ^ 1) && clock64() - t0 < kMbarWaitCycles;) {}
            }
    } else if (warp == 1) {
        // ---- products; likewise
        constexpr uint32_t kIdesc = 1u << 7 | 1u << 10 | uint32_t(NT >> 3) << 17 | (FMT == kMxfp4 ? 1u : 0u) << 23 | 1u << 27;
        const bool one = elect_one();
        uint32_t s = 0, phase = 0;
        int n = 0;
        bool ok = true;
        for (int t = blockIdx.x / splits; t < tiles && ok; t += clusters, ++n) {
            const int buf = n % T::kSumBuffers, use = n / T::kSumBuffers;
            if (use > 0) ok = mbar_wait(smem_u32(&sum_empty[buf]), uint32_t(use - 1) & 1, &gave_up);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tmem + buf * T::kSumColumns;
            for (int kt = first; kt < last; ++kt) {
                ok = mbar_wait(smem_u32(&full[s]), phase, &gave_up);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = smem + s * T::kStageBytes, sa = tmem_scales + s * T::kScaleColumns, sb = sa + T::kAtoms * 4;
                const uint64_t da = desc_rows128(at), db = desc_rows128(at + T::kBytesA), ds = desc_rows16(at + T::kBytesA + T::kBytesB);
                if (one) {
#pragma unroll
                    for (int j = 0; j < T::kAtoms; ++j) {
                        tc_copy_scales(sa + 4 * j, ds + 32 * j);
#pragma unroll
                        for (int g = 0; g < T::kGroups; ++g)
                            tc_copy_scales(sb + 4 * (j * T::kGroups + g), ds + (T::kBytesSa >> 4) + 32 * (g * T::kAtoms + j));
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {            // 64 columns: 32 bytes of a row, one word of scales (nvfp4) or half a word (mxfp4)
                        const int atom = FMT == kNvfp4 ? j : j / 2;
                        const uint32_t id = FMT == kNvfp4 ? 0u : 2u * (j % 2);
                        mma_block_scaled<FMT>(d, da + 2 * j, db + 2 * j, kIdesc | id << 4 | id << 29, sa + 4 * atom, sb + 4 * T::kGroups * atom, kt > first || j > 0);
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
    } else if (warp >= 2) {
        // ---- results: this warp's lanes are 32 rows of A
        const int quarter = warp & 3;
        constexpr int kChunk = NT < 32 ? NT : 32;
        int n = 0;
        for (int t = blockIdx.x / splits; t < tiles; t += clusters, ++n) {
            const int buf = n % T::kSumBuffers, use = n / T::kSumBuffers;
            const bool ok = mbar_wait(smem_u32(&sum_full[buf]), uint32_t(use) & 1, &gave_up);
            __syncwarp();
            tc_fence_after();
            const long long ra = (long long)(t / p.tiles_b) * kRowsA + 32 * quarter + lane, rb0 = (long long)(t % p.tiles_b) * NT;
            const float fa = FMT == kNvfp4 && ra < p.a_rows ? p.a_row[ra] : 1.0f;
#pragma unroll 1
            for (int c0 = 0; c0 < NT; c0 += kChunk) {
                uint32_t v[kChunk];
                tmem_load<kChunk>(tmem + buf * T::kSumColumns + c0 + (uint32_t(32 * quarter) << 16), v);
                tmem_wait_ld();
                if (c0 + kChunk >= NT) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sum_empty[buf]));
                }
#pragma unroll
                for (int c = 0; c < kChunk; ++c) {
                    float f = ok ? __uint_as_float(v[c]) : __uint_as_float(0x7FC00000u);
                    const long long rb = rb0 + c0 + c;
                    if (splits > 1) {
                        reinterpret_cast<float*>(raw + (smem - smem_u32(raw)))[(c0 + c) * kRowsA + 32 * quarter + lane] = f;
                    } else if (ra < p.a_rows && rb < p.b_rows) {
                        if constexpr (FMT == kNvfp4) f = f * fa * p.b_row[rb];
                        store(p, ra * p.step_a + rb * p.step_b, f);
                    }
                }
            }
        }
    }
    __syncwarp();
    if (splits > 1) {                                        // one tile a cluster: add up the parts of it
        cluster_sync();
        const int t = blockIdx.x / splits;
        const long long ra0 = (long long)(t / p.tiles_b) * kRowsA, rb0 = (long long)(t % p.tiles_b) * NT;
        for (int i = int(rank) * kThreads + threadIdx.x; i < kRowsA * NT; i += int(splits) * kThreads) {
            const long long ra = ra0 + i % kRowsA, rb = rb0 + i / kRowsA;
            if (ra >= p.a_rows || rb >= p.b_rows) continue;
            float f = 0.0f;
            for (uint32_t q = 0; q < splits; ++q) f += ld_cluster_f32(smem + 4 * i, q);
            if constexpr (FMT == kNvfp4) f = f * p.a_row[ra] * p.b_row[rb];
            store(p, ra * p.step_a + rb * p.step_b, f);
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

int sm_count() {
    static int cache[64] = {};
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    if (dev < 64 && cache[dev]) return cache[dev];
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    if (dev < 64) cache[dev] = n;
    return n;
}

template <int FMT, int NT>
cudaError_t launch(const MsMatrix& a, const MsMatrix& b, bool tokens_a, long long k, void* y, int dtype, long long ldy, int splits, cudaStream_t stream) {
    using T = Tile<FMT, NT>;
    static bool ready[64] = {};
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev >= 64 || !ready[dev]) {
        if ((err = cudaFuncSetAttribute(tcq_ms_matmul_kernel<FMT, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem)) != cudaSuccess) return err;
        if (dev < 64) ready[dev] = true;
    }
    CUtensorMap map_a, map_b;
    const long long pitch = ms_pitch(k);
    if ((err = make_byte_map(&map_a, a.codes, pitch, a.rows, pitch, kRowsA)) != cudaSuccess) return err;
    if ((err = make_byte_map(&map_b, b.codes, pitch, b.rows, pitch, NT)) != cudaSuccess) return err;
    MatmulArgs p{a.scales, b.scales, a.row_scale, b.row_scale, a.rows, b.rows, int((a.rows + kRowsA - 1) / kRowsA), int((b.rows + NT - 1) / NT),
                 int(ms_tiles_k(k)), y, tokens_a ? ldy : 1, tokens_a ? 1 : ldy, dtype};
    const long long tiles = (long long)p.tiles_a * p.tiles_b;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(splits > 1 ? tiles * splits : std::min<long long>(tiles, sm_count())));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = T::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = unsigned(splits);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, tcq_ms_matmul_kernel<FMT, NT>, map_a, map_b, p);
}

template <int FMT>
cudaError_t launch_fmt(const MsMatrix& x, const MsMatrix& w, long long k, void* y, int dtype, long long ldy, cudaStream_t stream) {
    const long long m = x.rows;
    // Few tokens: W's rows are the 128.
    if (m <= 64) {
        const long long tiles = (w.rows + kRowsA - 1) / kRowsA;
        int splits = 1;
        while (splits < 8 && tiles * splits * 2 <= sm_count() && splits * 2 <= ms_tiles_k(k)) splits *= 2;
        if (m <= 8) return launch<FMT, 8>(w, x, false, k, y, dtype, ldy, splits, stream);
        if (m <= 16) return launch<FMT, 16>(w, x, false, k, y, dtype, ldy, splits, stream);
        if (m <= 32) return launch<FMT, 32>(w, x, false, k, y, dtype, ldy, splits, stream);
        return launch<FMT, 64>(w, x, false, k, y, dtype, ldy, splits, stream);
    }
    const long long ta = (m + kRowsA - 1) / kRowsA;
    if (m > 128) return launch_ms_matmul_pair(x, w, k, FMT, y, dtype, ldy, (m + 255) / 256 * ((w.rows + 255) / 256) * 2 >= sm_count() ? 256 : 128, sm_count(), stream);
    const long long tiles = ta * ((w.rows + 127) / 128);
    int splits = 1;
    while (splits < 8 && tiles * splits * 2 <= sm_count() && splits * 2 <= ms_tiles_k(k)) splits *= 2;
    return launch<FMT, 128>(x, w, true, k, y, dtype, ldy, splits, stream);
}

}  // namespace

namespace {
cudaError_t encode_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, cuuint64_t width, cuuint64_t rows, cuuint64_t pitch, cuuint32_t box_width,
                       cuuint32_t box_rows, CUtensorMapSwizzle swizzle) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode encode = nullptr;
    if (encode == nullptr) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found{};
        const cudaError_t err = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found);
        if (err != cudaSuccess) return err;
        if (found != cudaDriverEntryPointSuccess || fn == nullptr) return cudaErrorNotSupported;
        encode = reinterpret_cast<Encode>(fn);
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

cudaError_t make_scale_map(CUtensorMap* map, const void* base, long long rows, int box_rows) {
    return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, base, 128, rows, 512, 128, box_rows, CU_TENSOR_MAP_SWIZZLE_NONE);
}

cudaError_t launch_ms_matmul(const MsMatrix& x, const MsMatrix& w, long long k, int fmt, void* y, int dtype, long long ldy, cudaStream_t stream) {
    return fmt == kNvfp4 ? launch_fmt<kNvfp4>(x, w, k, y, dtype, ldy, stream) : launch_fmt<kMxfp4>(x, w, k, y, dtype, ldy, stream);
}

}  // namespace tcq
