// Products of 16- and 32-bit activations with a 4-bit microscaled matrix, many tokens: y[i][r] = sum_c x[i][c] * W[r][c].
//
// Every value of W is a bf16 number, and x comes as m * P rows of bf16 parts (P = 1, 2, 3 for bf16, fp16, fp32, each the next eight
// significant bits), so the products are exact ones of a bf16 matrix product.  fp16 x needs one part where the weights are fp16 numbers:
// nvfp4's are; mxfp4's are, times a power of two for each row, unless a row's scales are more than 2^36 apart.  128 rows of W are the left
// operand, in tensor memory: eight warps read 64 columns of codes at a time from shared memory, make 16-bit numbers of them (a thread one
// row) and store them there, so that neither these weights nor their reading takes any of shared memory's bandwidth.  NT rows of x are the
// right operand, by TMA.
//
// Work split: one CTA per SM, or two, goes through tiles of 128 rows of W x NT rows of x.  One warp loads (codes and scales of 256 columns, x of 64),
// one issues products, eight make weights (two groups of four take turns), four take finished sums out of tensor memory.  With few tokens a
// cluster of S CTAs shares the columns of a tile; the partial sums meet through distributed shared memory, in rank order.
//
// Bound by the making of weights, beside the tensor cores (57 % busy): 1000 tokens through 12288 x 4096 81 us (1.24 PFLOP/s), mxfp4 79; fp16 75 and 90 (mxfp4 as
// called, with a scan of the scales and a form that ends at once, 105).  fp32 tokens, 21 to a tile at most: 40 through 4096 x 4096 19 us, 100 (mxfp4) 50.
//
// A wait that runs out (kMbarWaitCycles) makes its CTA stop, and its results from there on NaN, as those of its cluster.
#include <algorithm>
#include <type_traits>

#include "tcq_microscale_many.cuh"
#include "tcq_microscale_weights.cuh"
#include "tcq_tcgen05.cuh"

namespace tcq {

namespace {

// Warps: loader, issuer, four for the results, and groups of four that make weights.
constexpr int kMakers = 2;
constexpr int kThreads = 32 * (6 + 4 * kMakers);
constexpr int kRows = 128, kStepK = 64;          // rows of W; columns of a step
constexpr int kMostSplits = 8;

template <int FMT, int NT, int P>
struct Tile {
    // Up to 64 rows of x two CTAs share an SM: making weights is what takes the time, and eight warps do not fill the SM
    // (16 through 40960 x 4096 67.4 -> 54.6 us).
    static constexpr int kCtas = NT <= 64 && P != 3 ? 2 : 1;
    static constexpr int kAtoms = Ms<FMT>::kAtoms;
    static constexpr int kBytesW = kRows * 128, kBytesS = kAtoms * 512, kStageW = kBytesW + 2048, kStagesW = 3;      // 256 columns
    static constexpr int kBytesX = NT * 128;                                                                        // 64 columns
    static constexpr int kStagesX = std::min(8, ((kCtas == 2 ? 111 : 220) * 1024 - kStagesW * kStageW) / kBytesX);
    static constexpr int kSumBuffers = NT <= 128 ? 2 : 1, kSumColumns = NT < 32 ? 32 : NT;
    static constexpr int kStagesA = 4, kColumnsA = kStepK / 2;                                                      // weights in tensor memory
    static constexpr int kColumns = 512 / kCtas;
    static constexpr int kBytes = (kStagesW * kStageW + 1023) / 1024 * 1024 + kStagesX * kBytesX;
    // An SM (228 KB) holds two halves or one whole, so that no CTA waits for the tensor memory of another kernel's.
    static constexpr int kSmem = kCtas == 2 ? 112 * 1024 : std::max(kBytes + 1024, 116 * 1024);
    static_assert(kSumBuffers * kSumColumns + kStagesA * kColumnsA <= kColumns && kBytes + 1024 <= kSmem && kSmem <= 226 * 1024 && kStagesX >= 4);
    static_assert(kStagesX * kBytesX >= NT * kRows * 4 || NT == 256, "the parts of a tile");
};

struct ManyArgs {
    MsMatrix w;
    long long m;                                 // tokens
    int tiles_n, tiles_m, steps;                 // steps of 64 columns
    long long atoms;                             // of scales a row group
    void* y;
    long long ldy;
    const unsigned int* wide;                    // run only if *wide is `run_if`
    unsigned int run_if;
    const uint8_t* largest;                      // fp16, mxfp4
    unsigned loads;                              // stages of W that a CTA loads, at most (a self-test's limit)
};

__device__ __forceinline__ void mma_from_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)) : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t tmem, const uint32_t (&v)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(tmem), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                   "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
                   "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
                   "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]) : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t smem) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem));
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t smem) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(smem));
    return v;
}

// What a row's sums are multiplied by.
template <int FMT, bool FP16>
__device__ __forceinline__ float row_factor(const ManyArgs& p, long long r) {
    if (r >= p.w.rows) return 1.0f;
    if constexpr (FMT == kNvfp4) return FP16 ? p.w.row_scale[r] : row_rest(p.w.row_scale[r]);
    else if constexpr (FP16) return __uint_as_float(uint32_t(p.largest[r]) << 23 | (p.largest[r] == 0 ? 0x00400000u : 0u)) * 0x1p-13f;      // (2^-127: a denormal number)
    else return 1.0f;
}

// Weights as bf16 numbers carry the power of two of nvfp4's row scale: their sums, of activations of up to 2^128, are of the size of the results.  (fp16 activations
// are small, and take the row scale at the end.)  Where x is in three parts, of which a later one may be up to four times the first before its 2^-8 or 2^-16, weights are
// a quarter of what they are: still bf16 numbers, down to half of 2^-127.  (fp32 results below 2^-124 are then multiples of 2^-147, not of 2^-149.)
template <int P> constexpr float kWeightPower = P == 3 ? 0x1p-2f : 1.0f;

// The parts of a token, smallest first, as its sum.
template <int P>
__device__ __forceinline__ float whole_of(const float* v) {
    if constexpr (P == 1) return v[0];
    else if constexpr (P == 2) return v[1] * 0x1p-8f + v[0];
    else return v[2] * (0x1p-16f / kWeightPower<P>) + v[1] * (0x1p-8f / kWeightPower<P>) + v[0] / kWeightPower<P>;
}

// Steps whose sums stay in tensor memory.  The tensor cores cut sums off where fp32 arithmetic rounds, which over 12288 columns comes to 2.2e-6 of a
// result; where that is all the error there is (fp32 results), 256 columns at a time are added up in registers instead (1.5e-7).
template <int P> constexpr int kStepsHeld = P == 3 ? 4 : 1 << 29;

// fp16 scales of mxfp4: 2^13 over the row's largest scale (`most`, a byte), times the block's; 0 for what is too small for fp16 (blocks of zeros).
__device__ __forceinline__ uint32_t relative_scale(uint32_t byte, uint32_t most) {
    const int e = int(byte) - int(most) + 13;
    const __half h = byte == 255 ? __ushort_as_half(0x7FFF) : e < -23 ? __ushort_as_half(0) : __float2half_rn(__uint_as_float(uint32_t(e + 127) << 23));
    return uint32_t(__half_as_ushort(h)) * 0x10001u;
}

template <typename YT, int FMT, int NT, int P, bool FP16>
__global__ void __launch_bounds__(kThreads, Tile<FMT, NT, P>::kCtas) tcq_ms_linear_many_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                                                         const __grid_constant__ ManyArgs p) {
    using T = Tile<FMT, NT, P>;
    constexpr int kTokens = NT / P;                      // of a tile
    if (p.wide != nullptr && *p.wide != p.run_if) return;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t w_full[T::kStagesW], w_empty[T::kStagesW], x_full[T::kStagesX], x_empty[T::kStagesX], a_full[T::kStagesA], a_empty[T::kStagesA],
        sum_full[T::kSumBuffers], sum_empty[T::kSumBuffers], drained;
    __shared__ uint32_t tmem_at;
    __shared__ unsigned int gave_up;
    const uint32_t smem_w = (smem_u32(raw) + 1023) & ~1023u, smem_x = smem_w + (T::kStagesW * T::kStageW + 1023) / 1024 * 1024;
    const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), splits = cluster_size();
    const int all_tiles_k = (p.steps + 3) / 4;           // columns are shared in whole 256s
    const int first = 4 * int((long long)all_tiles_k * rank / splits), last = min(4 * int((long long)all_tiles_k * (rank + 1) / splits), p.steps);
    const int tiles = p.tiles_n * p.tiles_m, clusters = gridDim.x / splits;

    if (warp == 0 && elect_one()) {
        gave_up = 0;
        for (int s = 0; s < T::kStagesW; ++s) { mbar_init(smem_u32(&w_full[s]), 1); mbar_init(smem_u32(&w_empty[s]), 4 * kMakers); }
        for (int s = 0; s < T::kStagesX; ++s) { mbar_init(smem_u32(&x_full[s]), 1); mbar_init(smem_u32(&x_empty[s]), 1); }
        for (int s = 0; s < T::kStagesA; ++s) { mbar_init(smem_u32(&a_full[s]), 4); mbar_init(smem_u32(&a_empty[s]), 1); }
        for (int s = 0; s < T::kSumBuffers; ++s) { mbar_init(smem_u32(&sum_full[s]), 1); mbar_init(smem_u32(&sum_empty[s]), 4); }
        mbar_init(smem_u32(&drained), 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    if (warp == 1) tmem_alloc(smem_u32(&tmem_at), T::kColumns);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at, tmem_a = tmem + T::kSumBuffers * T::kSumColumns;

    if (warp == 0) {
        // ---- loads; the warp stays together, one lane issues
        const bool one = elect_one();
        uint32_t sw = 0, pw = 1, sx = 0, px = 1, loaded_w = 0, loaded_x = 0;      // (the first waits are for the phase before the first)
        unsigned left = p.loads;
        bool ok = true;
        for (int t = blockIdx.x / splits; t < tiles && ok; t += clusters) {
            const int tn = t / p.tiles_m, tm = t % p.tiles_m;
            for (int step = first; step < last; ++step) {
                if (step % 4 == 0) {
                    ok = still_waits(left-- > 0, smem_u32(&w_empty[sw]), pw, &gave_up) && !__any_sync(0xFFFFFFFFu, gave_up);
                    if (!ok) break;
                    if (one) {
                        const uint32_t to = smem_w + sw * T::kStageW, bar = smem_u32(&w_full[sw]);
                        mbar_expect(bar, T::kBytesW + T::kBytesS);
                        tma_load(to, &map_w, step * 32, tn * kRows, bar);
                        bulk_load(to + T::kBytesW, p.w.scales + (tn * p.atoms + (long long)(step / 4) * T::kAtoms) * 512, T::kBytesS, bar);
                    }
                    __syncwarp();
                    if (++sw == T::kStagesW) { sw = 0; pw ^= 1; }
                    if (loaded_w < T::kStagesW) ++loaded_w;
                }
                ok = still_waits(ok, smem_u32(&x_empty[sx]), px, &gave_up);
                if (!ok) break;
                if (one) {
                    mbar_expect(smem_u32(&x_full[sx]), T::kBytesX);
                    tma_load(smem_x + sx * T::kBytesX, &map_x, step * kStepK, tm * kTokens * P, smem_u32(&x_full[sx]));
                }
                __syncwarp();
                if (++sx == T::kStagesX) { sx = 0; px ^= 1; }
                if (loaded_x < T::kStagesX) ++loaded_x;
            }
        }
        wait_for_loads<T::kStagesW>(w_full, sw, pw, loaded_w);
        wait_for_loads<T::kStagesX>(x_full, sx, px, loaded_x);
        if (splits > 1 && gave_up)                       // a load that was late may lie over the NaN of this CTA's part
            for (int i = lane; i < kTokens * P * kRows; i += 32) reinterpret_cast<uint32_t*>(raw + (smem_x - smem_u32(raw)))[i] = 0x7FC00000u;
    } else if (warp == 1) {
        // ---- products; likewise
        constexpr uint32_t kIdesc = 1u << 4 | (FP16 ? 0u : 1u << 7 | 1u << 10) | uint32_t(NT >> 3) << 17 | uint32_t(kRows >> 4) << 24;      // bf16 x bf16 (or fp16 x fp16), fp32 sums
        const bool one = elect_one();
        uint32_t sx = 0, px = 0, sa = 0, pa = 0;
        int n = 0;
        bool ok = true;
        for (int t = blockIdx.x / splits; t < tiles && ok; t += clusters) {
            for (int from = first; from < last && ok; from += kStepsHeld<P>, ++n) {
                const int buf = n % T::kSumBuffers, use = n / T::kSumBuffers, to = P == 3 ? min(from + kStepsHeld<P>, last) : last;
                if (use > 0) ok = mbar_wait(smem_u32(&sum_empty[buf]), uint32_t(use - 1) & 1, &gave_up);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + buf * T::kSumColumns;
                for (int step = from; step < to; ++step) {
                    ok = mbar_wait(smem_u32(&x_full[sx]), px, &gave_up) && mbar_wait(smem_u32(&a_full[sa]), pa, &gave_up);
                    ok = __all_sync(0xFFFFFFFFu, ok);    // every lane has seen these phases before the stages can be filled again
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t db = desc_rows128(smem_x + sx * T::kBytesX);
                    const uint32_t a = tmem_a + sa * T::kColumnsA;
                    if (one) {
#pragma unroll
                        for (int j = 0; j < kStepK / 16; ++j) mma_from_tmem(d, a + 8 * j, db + 2 * j, kIdesc, step > from || j > 0);
                        tc_commit(smem_u32(&x_empty[sx]));
                        tc_commit(smem_u32(&a_empty[sa]));
                    }
                    __syncwarp();
                    if (++sx == T::kStagesX) { sx = 0; px ^= 1; }
                    if (++sa == T::kStagesA) { sa = 0; pa ^= 1; }
                }
                if (ok && one) tc_commit(smem_u32(&sum_full[buf]));
                __syncwarp();
            }
        }
        if (!ok) {                                       // what was issued ends before the tensor memory goes
            if (one) tc_commit(smem_u32(&drained));
            __syncwarp();
            for (long long t0 = clock64(); !mbar_try_wait(smem_u32(&drained), 0) && clock64() - t0 < kMbarWaitCycles;) {}
        }
    } else if (warp >= 6) {
        // ---- weights: lane = row of this warp's quarter; the groups of four warps take turns
        const int quarter = warp & 3, mine = (warp - 6) >> 2;
        const int row = 32 * quarter + lane;
        const E2m1Bytes<P == 3> bytes;
        const auto scale_of = [&](int t) {               // of this lane's row; fetched a tile ahead
            const long long r = (long long)(t / p.tiles_m) * kRows + row;
            return !FP16 && FMT == kNvfp4 && t < tiles && r < p.w.rows ? __ldg(p.w.row_scale + r) : 1.0f;
        };
        float next = scale_of(blockIdx.x / splits);
        uint32_t sw = 0, pw = 0, sa = 0, pa = 1;
        bool ok = true;
        for (int t = blockIdx.x / splits; t < tiles && ok; t += clusters) {
            uint32_t most = 0;
            const long long r = (long long)(t / p.tiles_m) * kRows + row;
            float power = 1.0f;
            if constexpr (!FP16 && FMT == kNvfp4) {
                power = row_power(next);
                next = scale_of(t + clusters);
            }
            const uint32_t power2 = (__float_as_uint(power) >> 16) * 0x10001u;               // twice, as a bf16 number
            if constexpr (FP16 && FMT == kMxfp4) most = r < p.w.rows ? p.largest[r] : 0;
            for (int step = first; step < last && ok; ++step) {
                if (step % 4 == 0) ok = __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&w_full[sw]), pw, &gave_up));
                if (step % kMakers == mine && ok) {
                    const uint32_t from = smem_w + sw * T::kStageW + row * 128, sub = step % 4;
                    uint32_t word;
                    const uint32_t scales = smem_w + sw * T::kStageW + T::kBytesW + lane * 16 + quarter * 4;
                    if constexpr (FMT == kNvfp4) word = lds32(scales + 512 * sub);
                    else word = lds32(scales + 512 * (sub / 2)) >> (16 * (sub & 1));
                    uint32_t v[32], scales16[4];
                    if constexpr (!FP16) four_scales<FMT>(word, scales16);
                    if constexpr (!FP16 && FMT == kNvfp4) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(scales16[q]) : "r"(power2));
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {        // 16 bytes: 32 columns; the swizzle has put piece c of row r at c ^ (r % 8)
                        const uint4 c = lds128(from + (((2 * sub + i) ^ (row & 7)) << 4));
                        const uint32_t cw[4] = {c.x, c.y, c.z, c.w};
                        if constexpr (FP16) {
                            uint32_t s[2];               // of the two halves
                            if constexpr (FMT == kNvfp4) {
                                uint32_t two;
                                asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(two) : "r"(word >> (16 * i)));
                                s[0] = __byte_perm(two, two, 0x1010);
                                s[1] = __byte_perm(two, two, 0x3232);
                            } else {
                                s[0] = s[1] = relative_scale((word >> (8 * i)) & 0xFFu, most);
                            }
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                uint32_t h[4];
                                e2m1x8_to_f16(cw[j], h);
#pragma unroll
                                for (int q = 0; q < 4; ++q) v[16 * i + 4 * j + q] = mul_f16x2(h[q], s[j / 2]);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                uint32_t h[4];
                                eight_weights(bytes, cw[j], scales16[2 * i + j / 2], h);
#pragma unroll
                                for (int q = 0; q < 4; ++q) v[16 * i + 4 * j + q] = h[q];
                            }
                        }
                    }
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&a_empty[sa]), pa, &gave_up));
                    if (ok) {
                        tc_fence_after();
                        tmem_store32(tmem_a + sa * T::kColumnsA + (uint32_t(32 * quarter) << 16), v);
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&a_full[sa]));
                    }
                }
                if (++sa == T::kStagesA) { sa = 0; pa ^= 1; }
                if (step % 4 == 3 || step + 1 == last) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&w_empty[sw]));
                    if (++sw == T::kStagesW) { sw = 0; pw ^= 1; }
                }
            }
        }
    } else {
        // ---- results: this warp's lanes are 32 rows of W, so that a store is 32 neighbours in y
        const int quarter = warp & 3;
        constexpr int kChunk = NT < 32 ? NT : 32, kUsed = kChunk / P * P;            // columns loaded, and columns of whole tokens
        int n = 0;
        bool ok = true;
        for (int t = blockIdx.x / splits; t < tiles; t += clusters) {
            const long long r = (long long)(t / p.tiles_m) * kRows + 32 * quarter + lane, token0 = (long long)(t % p.tiles_m) * kTokens;
            const float fw = row_factor<FMT, FP16>(p, r);
            const int here = int(min((long long)kTokens, p.m - token0));
            float* const part = reinterpret_cast<float*>(raw + (smem_x - smem_u32(raw))) + 32 * quarter + lane;
            YT* const y = static_cast<YT*>(p.y) + token0 * p.ldy + r;
            // the finished columns c0 .. c0 + N - 1
            auto finish = [&](const float* f, int c0, auto count) {
                constexpr int N = decltype(count)::value;
                if (splits > 1) {
#pragma unroll
                    for (int c = 0; c < N; ++c)
                        if (c0 + c < kTokens * P) part[(c0 + c) * kRows] = f[c];
                } else {
                    YT* to = y + c0 / P * p.ldy;
#pragma unroll
                    for (int i = 0; i < N / P; ++i, to += p.ldy) {
                        float whole = whole_of<P>(f + i * P);
                        if constexpr (FMT == kNvfp4 || FP16) whole *= fw;
                        if (r < p.w.rows && c0 / P + i < here) *to = from_f32<YT>(whole);
                    }
                }
            };
            if constexpr (P == 3) {
                float acc[NT] = {};
                for (int step = first; step < last; step += kStepsHeld<P>, ++n) {
                    const int buf = n % T::kSumBuffers;
                    ok = still_waits(ok, smem_u32(&sum_full[buf]), uint32_t(n / T::kSumBuffers) & 1, &gave_up);
                    tc_fence_after();
#pragma unroll
                    for (int c0 = 0; c0 < NT; c0 += kChunk) {
                        uint32_t v[kChunk];
                        tmem_load<kChunk>(tmem + buf * T::kSumColumns + c0 + (uint32_t(32 * quarter) << 16), v);
                        tmem_wait_ld();
#pragma unroll
                        for (int c = 0; c < kChunk; ++c) acc[c0 + c] += ok ? __uint_as_float(v[c]) : __uint_as_float(0x7FC00000u);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sum_empty[buf]));
                }
                finish(acc, 0, std::integral_constant<int, NT / P * P>{});
            } else {
                const int buf = n % T::kSumBuffers;
                ok = still_waits(ok, smem_u32(&sum_full[buf]), uint32_t(n / T::kSumBuffers) & 1, &gave_up);
                ++n;
                tc_fence_after();
#pragma unroll 1
                for (int c0 = 0; c0 < kTokens * P; c0 += kUsed) {
                    uint32_t v[kChunk];
                    tmem_load<kChunk>(tmem + buf * T::kSumColumns + c0 + (uint32_t(32 * quarter) << 16), v);
                    tmem_wait_ld();
                    float f[kChunk];
#pragma unroll
                    for (int c = 0; c < kChunk; ++c) f[c] = ok ? __uint_as_float(v[c]) : __uint_as_float(0x7FC00000u);
                    finish(f, c0, std::integral_constant<int, kUsed>{});
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sum_empty[buf]));
            }
        }
    }
    __syncwarp();
    if (splits > 1) {                                    // one tile a cluster: add up the parts of it
        cluster_sync();
        const int t = blockIdx.x / splits;
        const long long r0 = (long long)(t / p.tiles_m) * kRows, token0 = (long long)(t % p.tiles_m) * kTokens;
        const int tokens = int(min((long long)kTokens, p.m - token0));
        for (int i = int(rank) * kThreads + threadIdx.x; i < kRows / 4 * tokens; i += int(splits) * kThreads) {
            const int r4 = i % (kRows / 4), token = i / (kRows / 4);
            const long long r = r0 + 4 * r4;
            if (r >= p.w.rows) continue;
            float sum[4][P];
#pragma unroll
            for (int q = 0; q < P; ++q) {
                float4 part[kMostSplits];
#pragma unroll
                for (uint32_t s = 0; s < kMostSplits; ++s)
                    if (s < splits) part[s] = ld_cluster_f32x4(smem_x + 16 * ((token * P + q) * (kRows / 4) + r4), s);
                float4 f = part[0];
#pragma unroll
                for (uint32_t s = 1; s < kMostSplits; ++s)
                    if (s < splits) f = make_float4(f.x + part[s].x, f.y + part[s].y, f.z + part[s].z, f.w + part[s].w);
                sum[0][q] = f.x; sum[1][q] = f.y; sum[2][q] = f.z; sum[3][q] = f.w;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (r + j < p.w.rows) {
                    float whole = whole_of<P>(sum[j]);
                    if constexpr (FMT == kNvfp4 || FP16) whole *= row_factor<FMT, FP16>(p, r + j);
                    static_cast<YT*>(p.y)[(token0 + token) * p.ldy + r + j] = from_f32<YT>(whole);
                }
        }
        cluster_sync();                                  // no CTA ends while another reads its part
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free(tmem, T::kColumns);
    }
}

__global__ void __launch_bounds__(256) tcq_ms_scale_range_kernel(MsMatrix w, long long k, long long pitch, int atoms, unsigned int* wide, uint8_t* largest);

template <typename YT, int FMT, int NT, int P, bool FP16>
cudaError_t launch(const ManyCall& c, cudaStream_t stream) {
    using T = Tile<FMT, NT, P>;
    const auto kernel = tcq_ms_linear_many_kernel<YT, FMT, NT, P, FP16>;
    static std::atomic<bool> ready[64];
    static MostClusters kept;
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev >= 64 || !ready[dev]) {
        // The count of clusters that run at once takes a kernel with tensor memory to be alone on its SM: two of them are counted as another kernel's.
        if (T::kCtas == 2 && (err = cudaFuncSetAttribute(tcq_ms_scale_range_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem)) != cudaSuccess) return err;
        if ((err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem)) != cudaSuccess) return err;
        if (dev < 64) ready[dev] = true;
    }
    CUtensorMap map_w, map_x;
    const long long pitch = ms_pitch(c.k), tokens = NT / P;
    if ((err = make_byte_map(&map_w, c.w.codes, pitch, c.w.rows, pitch, kRows)) != cudaSuccess) return err;
    if ((err = make_16bit_map(&map_x, c.x, c.width, c.m * P, c.ldx, NT)) != cudaSuccess) return err;
    const ManyArgs p{c.w, c.m, int((c.w.rows + kRows - 1) / kRows), int((c.m + tokens - 1) / tokens), int((c.k + kStepK - 1) / kStepK), ms_tiles_k(c.k) * T::kAtoms, c.y, c.ldy,
                     c.wide, FP16 ? 0u : 1u, c.largest, c.loads};
    const long long tiles = (long long)p.tiles_n * p.tiles_m;
    // How many CTAs share the columns of a tile: as many as leave every CTA an SM of its own (half an SM, where each still has 1024 columns:
    // 4096 columns of 4096 rows by 8 instead of 4 costs 10.7 -> 11.7 us, 12288 of them 21.3 -> 20.2 us).
    const int k_tiles = int(ms_tiles_k(c.k)), sms = ms_sm_count();
    const auto fits = [&](int s) {
        if (T::kCtas == 2 && tiles * s > sms && k_tiles < 4 * s) return false;
        return tiles <= (T::kCtas == 2 ? ms_most_clusters(kept, reinterpret_cast<const void*>(tcq_ms_scale_range_kernel), 256, T::kSmem, 2, s)
                                       : ms_most_clusters(kept, reinterpret_cast<const void*>(kernel), kThreads, T::kSmem, 1, s));
    };
    int splits = 1;
    while (NT <= 128 && splits < kMostSplits && 2 * splits <= k_tiles && fits(2 * splits)) splits *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(splits > 1 ? tiles * splits : std::min<long long>(tiles, T::kCtas * ms_sm_count())));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = T::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = unsigned(splits);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, map_w, map_x, p);
}

// Rows of x in a tile: all of them up to 64; 128 where all tiles then run at once (100 through 4096 x 4096, its columns shared by four: 12.9 us,
// not shared 26.4, tiles of 64 16.6); else 256, which makes the weights least often.
template <typename YT, int FMT, int P, bool FP16>
cudaError_t launch_nt(const ManyCall& c, cudaStream_t stream) {
    const long long rows = c.m * P;
    constexpr bool kMany = FP16 && FMT == kMxfp4;        // called from 129 tokens on; the others from nine
    if constexpr (!kMany && P == 1)
        if (rows <= 16) return launch<YT, FMT, 16, P, FP16>(c, stream);
    if constexpr (!kMany)
        if (rows <= 32 / P * P) return launch<YT, FMT, 32, P, FP16>(c, stream);
    if constexpr (P == 3) {
        return launch<YT, FMT, 64, P, FP16>(c, stream);  // sums in registers: no more than 64 columns
    } else {
        if constexpr (!kMany)
            if (rows <= 64 / P * P) return launch<YT, FMT, 64, P, FP16>(c, stream);
        if ((c.w.rows + kRows - 1) / kRows * ((c.m + 128 / P - 1) / (128 / P)) <= ms_sm_count()) return launch<YT, FMT, 128, P, FP16>(c, stream);
        return launch<YT, FMT, 256, P, FP16>(c, stream);
    }
}

template <int FMT>
cudaError_t launch_fmt(const ManyCall& c, cudaStream_t stream) {
    if (c.dtype == kF32) return launch_nt<float, FMT, 3, false>(c, stream);
    if (c.dtype == kBf16) return launch_nt<__nv_bfloat16, FMT, 1, false>(c, stream);
    if constexpr (FMT == kMxfp4)
        if (!c.fp16) return launch_nt<__half, FMT, 2, false>(c, stream);
    return launch_nt<__half, FMT, 1, true>(c, stream);   // nvfp4's weights are fp16 numbers
}

// One CTA a group of 128 rows; a warp reads the 512 bytes of 128 columns at a time, a lane the four rows lane + 32 q.
__global__ void __launch_bounds__(256) tcq_ms_scale_range_kernel(MsMatrix w, long long k, long long pitch, int atoms, unsigned int* wide, uint8_t* largest) {
    __shared__ uint32_t part[8][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint4* const from = reinterpret_cast<const uint4*>(w.scales) + ((long long)blockIdx.x * atoms) * 32 + lane;
    const int blocks = int((k + 31) / 32);
    uint32_t most = 0;                                   // a byte a row
    for (int a = warp; a < atoms; a += 8) {
        const uint4 u = __ldg(from + a * 32);
        const uint32_t v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t m = (most >> (8 * q)) & 0xFFu;
            uint32_t b = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t s = (v[q] >> (8 * i)) & 0xFFu;
                b = max(b, s == 255u ? 0u : s);          // (NaN: no size)
            }
            if (b > m) most = (most & ~(0xFFu << (8 * q))) | b << (8 * q);
        }
    }
    part[warp][lane] = most;
    __syncthreads();
    most = part[0][lane];
    for (int i = 1; i < 8; ++i) most = __vmaxu4(most, part[i][lane]);
    if (warp < 4) {
        const long long row = (long long)blockIdx.x * 128 + 32 * warp + lane;
        if (row < w.rows) largest[row] = uint8_t(most >> (8 * warp));
    }
    bool far = false;
    for (int a = warp; a < atoms; a += 8) {
        const uint4 u = __ldg(from + a * 32);
        const uint32_t v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const long long row = (long long)blockIdx.x * 128 + 32 * q + lane;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (((v[q] >> (8 * i)) & 0xFFu) + 36 < ((most >> (8 * q)) & 0xFFu) && row < w.rows && 4 * a + i < blocks) {
                    const uint4 c = __ldg(reinterpret_cast<const uint4*>(w.codes + row * pitch) + 4 * a + i);       // 32 codes
                    far = far || ((c.x | c.y | c.z | c.w) & 0x77777777u) != 0;
                }
        }
    }
    if (far) atomicOr(wide, 1u);
}

}  // namespace

cudaError_t launch_ms_linear_many(const ManyCall& c, cudaStream_t stream) { return c.fmt == kNvfp4 ? launch_fmt<kNvfp4>(c, stream) : launch_fmt<kMxfp4>(c, stream); }

cudaError_t launch_ms_scale_range(const MsMatrix& w, long long k, unsigned int* wide, uint8_t* largest, cudaStream_t stream) {
    cudaError_t err = cudaMemsetAsync(wide, 0, sizeof(unsigned int), stream);
    if (err != cudaSuccess) return err;
    tcq_ms_scale_range_kernel<<<unsigned((w.rows + 127) / 128), 256, 0, stream>>>(w, k, ms_pitch(k), int(ms_tiles_k(k)) * 2, wide, largest);
    return cudaGetLastError();
}

}  // namespace tcq
