// Products of two 4-bit microscaled matrices, many tokens: y[i][r] = sum_c X[i][c] * W[r][c].
//
// tcgen05.mma over a pair of SMs: 256 tokens x NT rows of W at a time, 64 columns an instruction.  Each CTA of the pair holds 128 of the
// tokens and half of W's rows (the tensor cores read the other half from the neighbour), the scales of its own tokens and of all NT
// rows; the first CTA issues for both.  Against one SM on 128 x 256 results this halves what W costs of shared memory's bandwidth, which
// that form is bound by: 24 KB written and read for 128 clocks of products at the 4-bit rate; here 16 KB.
//
// Work split: pairs go through tiles of 256 x NT.  In each CTA one thread loads stages of 256 columns (codes and scales by TMA, all
// counted by the first CTA's barrier); in the first CTA one thread issues; eight warps take the sums of their CTA's 128 tokens, each 32
// tokens x half the columns, into registers (scaled and rounded), hand the tensor memory back, and store while the next tile runs.  At
// NT = 256 there is one buffer of sums, at 128 two.
//
// Bound by power in long runs (1000 W: 1.5 to 1.7 GHz), then by the copies of scales to tensor memory, which nvfp4 has twice as many of: 8192 tokens
// through 12288 x 4096 back to back 190 us (4.3 PFLOP/s); a dozen calls at full clocks 160 to 164 (5.1), mxfp4 146 to 150 (5.6); 2048 tokens 47.4 and 42.6.
//
// A wait that runs out (kMbarWaitCycles) makes its CTA stop, and its results from there on NaN.
#include <algorithm>

#include "tcq_microscale.cuh"
#include "tcq_tcgen05.cuh"

namespace tcq {

namespace {

constexpr int kWarps = 10, kThreads = 32 * kWarps;       // loader, issuer, eight for the results

template <int FMT, int NT>
struct Tile {
    static constexpr int kAtoms = Ms<FMT>::kAtoms, kGroups = NT / 128;
    static constexpr int kBytesA = 128 * 128, kBytesB = NT / 2 * 128, kBytesSa = kAtoms * 512, kBytesSb = kGroups * kAtoms * 512;
    static constexpr int kStageBytes = (kBytesA + kBytesB + kBytesSa + kBytesSb + 1023) / 1024 * 1024;
    static constexpr int kLoaded = kBytesA + kBytesB + kBytesSa + kBytesSb;
    static constexpr int kSumBuffers = NT == 128 ? 2 : 1;
    static constexpr int kScaleColumns = kAtoms * 4 * (1 + kGroups);
    static constexpr int kTurnBytes = 8 * 32 * 36 * 4;   // 32 x 32 results a warp, for rows of y that are not aligned
    static constexpr int kBySmem = (225 * 1024 - kTurnBytes) / kStageBytes, kByTmem = (512 - kSumBuffers * NT) / kScaleColumns;
    static constexpr int kStages = std::min(kBySmem, kByTmem);
    static constexpr int kSmem = kStages * kStageBytes + kTurnBytes + 1024;
    static_assert(kSmem >= 116 * 1024 && kSmem <= 226 * 1024 && kStages >= 4);
};

struct PairArgs {
    const float* x_row;
    const float* w_row;
    long long m, n;
    int tiles_m, tiles_n, k_tiles, groups_m, groups_n;
    void* y;
    long long ldy;
    int dtype;
    bool aligned;                                        // rows of y start on 32 bytes
    unsigned loads;                                      // stages that a CTA loads, at most (a self-test's limit)
};

template <int FMT>
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, bool add) {
    if constexpr (FMT == kNvfp4)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(uint32_t(add)) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(uint32_t(add)) : "memory");
}

template <typename YT> __device__ __forceinline__ uint32_t pack(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void store32(void* to, const uint32_t* v) {       // 32 bytes, aligned
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

// What 32 tokens (one a lane) x COLS columns of results are scaled by; fetched while the products run.
template <int FMT, int COLS>
struct Factors {
    float x, outer, w[FMT == kNvfp4 ? COLS / 32 : 1];    // w: of column 32 q + lane
    __device__ __forceinline__ Factors(const PairArgs& p, long long token0, long long col0) {
        if constexpr (FMT == kNvfp4) {
            const int lane = threadIdx.x & 31;
            const float g = token0 + lane < p.m ? __ldg(p.x_row + token0 + lane) : 1.0f;
            x = inner_part(g);
            outer = outer_part(g);
#pragma unroll
            for (int q = 0; q < COLS / 32; ++q) w[q] = col0 + 32 * q + lane < p.n ? __ldg(p.w_row + col0 + 32 * q + lane) : 1.0f;
        }
    }
};

// 32 tokens x COLS columns out of tensor memory, which is handed back at once; then scaled, rounded and stored.
template <typename YT, int FMT, int COLS>
__device__ __forceinline__ void results(const PairArgs& p, uint32_t tmem, uint32_t sum_empty, bool ok, long long token0, long long col0,
                                        const Factors<FMT, COLS>& by, uint32_t* turn) {
    constexpr int kWords = sizeof(YT) == 4 ? 32 : 16;     // of 32 results
    const int lane = threadIdx.x & 31;
    const long long token = token0 + lane;
    uint32_t v[COLS / 32][32];
#pragma unroll
    for (int q = 0; q < COLS / 32; ++q) tmem_load<32>(tmem + 32 * q, v[q]);
    tmem_wait_ld();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive_cluster(sum_empty);
    YT* const y = static_cast<YT*>(p.y);
    const bool direct = p.aligned && col0 + COLS <= p.n;
#pragma unroll
    for (int q = 0; q < COLS / 32; ++q) {
        uint32_t out[kWords];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            if constexpr (FMT == kNvfp4) v[q][i] = __float_as_uint(__uint_as_float(v[q][i]) * by.x * __shfl_sync(0xFFFFFFFFu, by.w[q], i));
            if (!ok) v[q][i] = 0x7FC00000u;
        }
        if (FMT == kNvfp4 && __any_sync(0xFFFFFFFFu, by.outer != 1.0f)) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[q][i] = __float_as_uint(__uint_as_float(v[q][i]) * by.outer);
        }
        if constexpr (sizeof(YT) == 4) {
#pragma unroll
            for (int i = 0; i < 32; ++i) out[i] = v[q][i];
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) out[i] = pack<YT>(__uint_as_float(v[q][2 * i]), __uint_as_float(v[q][2 * i + 1]));
        }
        if (direct) {
            if (token < p.m) {
                uint8_t* const to = reinterpret_cast<uint8_t*>(y + token * p.ldy + col0) + q * kWords * 4;
#pragma unroll
                for (int i = 0; i < kWords; i += 8) store32(to + 4 * i, out + i);
            }
            continue;
        }
        // a row at a time, a result a lane; 32 columns through shared memory
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kWords; i += 4) *reinterpret_cast<uint4*>(turn + lane * 36 + i) = make_uint4(out[i], out[i + 1], out[i + 2], out[i + 3]);
        __syncwarp();
        const long long c = col0 + 32 * q + lane;
        if (c < p.n)
            for (int r = 0; r < 32 && token0 + r < p.m; ++r) y[(token0 + r) * p.ldy + c] = reinterpret_cast<const YT*>(turn + r * 36)[lane];
    }
}

template <int FMT, int NT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
tcq_ms_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_sx,
                   const __grid_constant__ CUtensorMap map_sw, const __grid_constant__ PairArgs p) {
    using T = Tile<FMT, NT>;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[T::kStages], empty[T::kStages], sum_full[T::kSumBuffers], sum_empty[T::kSumBuffers], drained;
    __shared__ uint32_t tmem_at;
    __shared__ unsigned int gave_up;
    const uint32_t smem = (smem_u32(raw) + 1023) & ~1023u;
    const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x) >> 5, 0);
    const int rank = int(cluster_rank()), tiles = p.tiles_m * p.tiles_n, pair = blockIdx.x / 2, pairs = gridDim.x / 2;

    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < T::kStages; ++s) { mbar_init(smem_u32(&full[s]), 1); mbar_init(smem_u32(&empty[s]), 1); }
        for (int s = 0; s < T::kSumBuffers; ++s) { mbar_init(smem_u32(&sum_full[s]), 1); mbar_init(smem_u32(&sum_empty[s]), 16); }
        mbar_init(smem_u32(&drained), 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    cluster_sync();                                      // the neighbour's barriers are there: the loads begin
    uint32_t tmem = 0;
    if (warp > 0) {
        if (warp == 1) tmem_alloc<2>(smem_u32(&tmem_at), 512);
        tc_fence_before();
        asm volatile("bar.sync 1, %0;" ::"n"(kThreads - 32) : "memory");
        tc_fence_after();
        tmem = tmem_at;
    }
    const uint32_t tmem_scales = tmem + T::kSumBuffers * NT, full_first = map_rank(smem_u32(&full[0]), 0);

    if (warp == 0) {
        // ---- loads of this CTA; the warp stays together, one lane issues
        const bool one = elect_one();
        uint32_t s = 0, phase = 1, loaded = 0;           // (the first wait for each stage is for the phase before the first)
        unsigned left = p.loads;
        bool ok = true;
        for (int t = pair; t < tiles && ok; t += pairs) {
            const int tm = t % p.tiles_m, tn = t / p.tiles_m;
            const int row_x = (2 * tm + rank) * 128, row_w = tn * NT + rank * (NT / 2);
            int row_sx = min(2 * tm + rank, p.groups_m - 1) * p.k_tiles * T::kAtoms;             // (a group behind the last holds no results)
            int row_sw[T::kGroups];
#pragma unroll
            for (int g = 0; g < T::kGroups; ++g) row_sw[g] = min(tn * T::kGroups + g, p.groups_n - 1) * p.k_tiles * T::kAtoms;
            for (int kt = 0; kt < p.k_tiles; ++kt) {
                ok = still_waits(left-- > 0, smem_u32(&empty[s]), phase, &gave_up);      // every lane has seen this phase before the next can begin
                if (!ok) break;
                if (one) {
                    const uint32_t to = smem + s * T::kStageBytes, bar = full_first + s * 8;
                    if (rank == 0) mbar_expect(smem_u32(&full[s]), 2 * T::kLoaded);
                    tma_load_pair(to, &map_x, kt * 128, row_x, bar);
                    tma_load_pair(to + T::kBytesA, &map_w, kt * 128, row_w, bar);
                    tma_load_pair(to + T::kBytesA + T::kBytesB, &map_sx, 0, row_sx + kt * T::kAtoms, bar);
#pragma unroll
                    for (int g = 0; g < T::kGroups; ++g)
                        tma_load_pair(to + T::kBytesA + T::kBytesB + T::kBytesSa + g * T::kAtoms * 512, &map_sw, 0, row_sw[g] + kt * T::kAtoms, bar);
                }
                __syncwarp();
                if (++s == T::kStages) { s = 0; phase ^= 1; }
                if (loaded < T::kStages) ++loaded;
            }
        }
        if (rank == 0) wait_for_loads<T::kStages>(full, s, phase, loaded);       // (of both CTAs)
    } else if (warp == 1 && rank == 0) {
        // ---- products of the pair; the warp stays together, one lane issues
        constexpr uint32_t kIdesc = 1u << 7 | 1u << 10 | uint32_t(NT >> 3) << 17 | (FMT == kMxfp4 ? 1u : 0u) << 23 | 2u << 27;
        constexpr uint64_t kHigh128 = uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61, kHigh16 = uint64_t(128 >> 4) << 32 | uint64_t(1) << 46;
        const bool one = elect_one();
        uint32_t s = 0, phase = 0;
        int n = 0;
        bool ok = true;
        for (int t = pair; t < tiles && ok; t += pairs, ++n) {
            const int buf = n % T::kSumBuffers, use = n / T::kSumBuffers;
            if (use > 0) ok = mbar_wait(smem_u32(&sum_empty[buf]), uint32_t(use - 1) & 1, &gave_up);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tmem + buf * NT;
            for (int kt = 0; kt < p.k_tiles; ++kt) {
                ok = mbar_wait(smem_u32(&full[s]), phase, &gave_up);
                ok = __all_sync(0xFFFFFFFFu, ok);        // every lane has seen this phase before the stage can be loaded again
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = (smem + s * T::kStageBytes) >> 4, sa = tmem_scales + s * T::kScaleColumns, sb = sa + T::kAtoms * 4;
                const uint64_t da = kHigh128 | (at | 1u << 16), db = kHigh128 | ((at + (T::kBytesA >> 4)) | 1u << 16);
                const uint64_t ds = kHigh16 | (at + ((T::kBytesA + T::kBytesB) >> 4));
                if (one) {
#pragma unroll
                    for (int j = 0; j < T::kAtoms; ++j) {
                        tc_copy_scales<2>(sa + 4 * j, ds + 32 * j);
#pragma unroll
                        for (int g = 0; g < T::kGroups; ++g)
                            tc_copy_scales<2>(sb + 4 * (j * T::kGroups + g), ds + (T::kBytesSa >> 4) + 32 * (g * T::kAtoms + j));
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int atom = FMT == kNvfp4 ? j : j / 2;
                        const uint32_t id = FMT == kNvfp4 ? 0u : 2u * (j % 2);
                        mma_pair<FMT>(d, da + 2 * j, db + 2 * j, kIdesc | id << 4 | id << 29, sa + 4 * atom, sb + 4 * T::kGroups * atom, kt > 0 || j > 0);
                    }
                    tc_commit_pair(smem_u32(&empty[s]));
                }
                __syncwarp();
                if (++s == T::kStages) { s = 0; phase ^= 1; }
            }
            if (ok && one) tc_commit_pair(smem_u32(&sum_full[buf]));
            __syncwarp();
        }
        if (!ok) {                                       // what was issued ends before the tensor memory goes
            if (one) tc_commit_pair(smem_u32(&drained));
            __syncwarp();
            for (long long t0 = clock64(); !mbar_try_wait(smem_u32(&drained), 0) && clock64() - t0 < kMbarWaitCycles;) {}
        }
    } else if (warp >= 2) {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        uint32_t* const turn = reinterpret_cast<uint32_t*>(raw + (smem - smem_u32(raw)) + T::kStages * T::kStageBytes) + (warp - 2) * 32 * 36;
        int n = 0;
        bool ok = true;
        for (int t = pair; t < tiles; t += pairs, ++n) {
            const int buf = n % T::kSumBuffers, use = n / T::kSumBuffers;
            const long long token0 = (long long)(t % p.tiles_m) * 256 + rank * 128 + 32 * quarter, col0 = (long long)(t / p.tiles_m) * NT + half * (NT / 2);
            const Factors<FMT, NT / 2> by(p, token0, col0);
            ok = still_waits(ok, smem_u32(&sum_full[buf]), uint32_t(use) & 1, &gave_up);
            tc_fence_after();
            const uint32_t from = tmem + buf * NT + half * (NT / 2) + (uint32_t(32 * quarter) << 16), free_bar = map_rank(smem_u32(&sum_empty[buf]), 0);
            if (p.dtype == kF32) results<float, FMT, NT / 2>(p, from, free_bar, ok, token0, col0, by, turn);
            else if (p.dtype == kF16) results<__half, FMT, NT / 2>(p, from, free_bar, ok, token0, col0, by, turn);
            else results<__nv_bfloat16, FMT, NT / 2>(p, from, free_bar, ok, token0, col0, by, turn);
        }
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();                                      // both are through: no more reads of the neighbour's memory, no arrivals at its barriers
    if (warp == 1) {
        tc_fence_after();
        tmem_free<2>(tmem, 512);
    }
}

template <int FMT, int NT>
cudaError_t launch(const MsMatrix& x, const MsMatrix& w, long long k, void* y, int dtype, long long ldy, int sms, unsigned loads, cudaStream_t stream) {
    using T = Tile<FMT, NT>;
    static std::atomic<bool> ready[64];
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev >= 64 || !ready[dev]) {
        if ((err = cudaFuncSetAttribute(tcq_ms_pair_kernel<FMT, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem)) != cudaSuccess) return err;
        if (dev < 64) ready[dev] = true;
    }
    const long long pitch = ms_pitch(k), k_tiles = ms_tiles_k(k), gx = (x.rows + 127) / 128, gw = (w.rows + 127) / 128;
    CUtensorMap map_x, map_w, map_sx, map_sw;
    if ((err = make_byte_map(&map_x, x.codes, pitch, x.rows, pitch, 128)) != cudaSuccess) return err;
    if ((err = make_byte_map(&map_w, w.codes, pitch, w.rows, pitch, NT / 2)) != cudaSuccess) return err;
    if ((err = make_scale_map(&map_sx, x.scales, gx * k_tiles * T::kAtoms, T::kAtoms)) != cudaSuccess) return err;
    if ((err = make_scale_map(&map_sw, w.scales, gw * k_tiles * T::kAtoms, T::kAtoms)) != cudaSuccess) return err;
    const size_t bytes = dtype == kF32 ? 4 : 2;
    const PairArgs p{x.row_scale, w.row_scale, x.rows, w.rows, int((x.rows + 255) / 256), int((w.rows + NT - 1) / NT), int(k_tiles), int(gx), int(gw),
                     y, ldy, dtype, reinterpret_cast<uintptr_t>(y) % 32 == 0 && ldy * bytes % 32 == 0, loads};
    const long long tiles = (long long)p.tiles_m * p.tiles_n;
    tcq_ms_pair_kernel<FMT, NT><<<unsigned(2 * std::min<long long>(tiles, sms / 2)), kThreads, T::kSmem, stream>>>(map_x, map_w, map_sx, map_sw, p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_ms_matmul_pair(const MsMatrix& x, const MsMatrix& w, long long k, int fmt, void* y, int dtype, long long ldy, int nt, int sms, unsigned loads,
                                  cudaStream_t stream) {
    if (fmt == kNvfp4) return nt == 256 ? launch<kNvfp4, 256>(x, w, k, y, dtype, ldy, sms, loads, stream) : launch<kNvfp4, 128>(x, w, k, y, dtype, ldy, sms, loads, stream);
    return nt == 256 ? launch<kMxfp4, 256>(x, w, k, y, dtype, ldy, sms, loads, stream) : launch<kMxfp4, 128>(x, w, k, y, dtype, ldy, sms, loads, stream);
}

}  // namespace tcq
