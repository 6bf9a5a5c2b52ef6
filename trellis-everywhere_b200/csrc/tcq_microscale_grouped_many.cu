// Rows of 16-bit activations in groups, each group times a 4-bit microscaled matrix of its own, many rows a group: y[i] = act(W[g(i)] x[i] + bias) + residual.
//
// Every value of W is a bf16 number (nvfp4's an fp16 number too), so the products are exact ones of a 16-bit matrix product.  128 rows of W are the left operand, in
// tensor memory: warps read 64 columns of codes at a time from shared memory, make 16-bit numbers of them (a thread one row) and store them there.  Up to NT rows of
// x are the right operand, by TMA; an item takes as many columns as it has rows.  Rows that are gathered are put in order first.  (TMA loads of four rows of any numbers each took twice as long
// for all.)
//
// Work split: one CTA per SM goes through items of 128 rows of a matrix x up to 256 rows of its group, of fewer where there are fewer such than SMs.  One warp loads codes and scales of
// 256 columns, another x of 64, one issues products, two groups of four make weights in turn, eight take finished sums out of tensor memory.  The sums of 128 rows are a buffer, of which there
// are three: the next item begins when the first half of the last one's sums has been taken.  x and weights of 64 columns are one stage of one ring, with one barrier that says that both are
// there and one that they are no longer needed.
//
// Measured in a graph, in short runs: 2000 rows through 12288 x 4096 nvfp4 (fp16, GELU) 168 to 173 us, 1.2 PFLOP/s, 2040 tokens to 8 of 64 experts of 2816 x 2048 228 to 232, 0.82; in long ones, at the power
// limit, and as called back to back, 192 to 204 (1.0 PFLOP/s) and 262 to 276 (0.7).  What a stage takes beside its products is waits and arrivals (0.2 to 0.3 us with neither products nor weights made; x in boxes of 64 or 128 rows, stages of half as many
// rows and twice as many of them, a third group of makers: no change; a fourth in place of takers 20 % longer).
//
// A wait that runs out (kMbarWaitCycles) makes its CTA stop, and its results from there on NaN.
#include <algorithm>

#include "tcq_microscale_grouped.cuh"
#include "tcq_microscale_weights.cuh"
#include "tcq_programmatic.cuh"
#include "tcq_tcgen05.cuh"

namespace tcq {

namespace {

constexpr int kMakers = 2, kTakers = 2;          // groups of four warps
constexpr int kFirstTaker = 2, kFirstMaker = 2 + 4 * kTakers, kLoaderW = kFirstMaker + 4 * kMakers, kThreads = 32 * (kLoaderW + 1);
constexpr int kRows = 128, kStepK = 64, kNt = 256, kHalf = 128;
constexpr int kBoxRows = 32;

template <int FMT>
struct Tile {
    static constexpr int kAtoms = Ms<FMT>::kAtoms;
    static constexpr int kBytesW = kRows * 128, kBytesS = kAtoms * 512, kStageW = kBytesW + 2048, kStagesW = 4;      // 256 columns
    static constexpr int kBytesX = kNt * 128, kStages = 4;                                                           // 64 columns
    static constexpr int kSums = 3, kColumnsA = kStepK / 2;                                                          // weights in tensor memory
    static constexpr int kColumns = 512;
    static constexpr int kSmem = (kStagesW * kStageW + 1023) / 1024 * 1024 + kStages * kBytesX + 1024;
    // A maker's wait for the stage of step u is for the products of step u - kStages, and is theirs only if those of u - 2 kStages are done: its wait before was for u - kMakers - kStages.
    static_assert(kMakers <= kStages);
    static_assert(kSums * kHalf + kStages * kColumnsA <= kColumns && kSmem + sizeof(GroupPlan) + 1024 <= 227 * 1024 && kSmem >= 116 * 1024);
};

struct ManyArgs {
    MsMatrix w;
    Groups groups;
    int tiles_n, steps;                          // steps of 64 columns
    int per;                                     // rows of x an item, at most
    long long atoms;                             // of scales a row group
    Epilogue out;
    unsigned loads;
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
// What a row's sums are multiplied by.  bf16 weights carry the power of two of nvfp4's row scale, so that sums of activations of up to 2^128 are of the size of the results;
// fp16 activations are small, and take the row scale at the end.
template <int FMT, bool FP16>
__device__ __forceinline__ float row_factor(const ManyArgs& p, long long r) {
    if constexpr (FMT == kNvfp4) return FP16 ? p.w.row_scale[r] : row_rest(p.w.row_scale[r]);
    else return 1.0f;
}

template <int FMT, bool FP16>
__global__ void __launch_bounds__(kThreads, 1) tcq_ms_grouped_many_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                                                          const __grid_constant__ ManyArgs p) {
    using T = Tile<FMT>;
    extern __shared__ uint8_t raw[];
    __shared__ GroupPlan plan;
    __shared__ uint64_t w_full[T::kStagesW], w_empty[T::kStagesW], full[T::kStages], empty[T::kStages], sum_full[T::kSums], sum_empty[T::kSums], drained;
    __shared__ uint32_t tmem_at;
    __shared__ unsigned int gave_up;
    const uint32_t smem_w = (smem_u32(raw) + 1023) & ~1023u, smem_x = smem_w + (T::kStagesW * T::kStageW + 1023) / 1024 * 1024;
    const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;

    if (warp == 0 && elect_one()) {
        gave_up = 0;
        for (int s = 0; s < T::kStagesW; ++s) { mbar_init(smem_u32(&w_full[s]), 1); mbar_init(smem_u32(&w_empty[s]), 4 * kMakers); }
        for (int s = 0; s < T::kStages; ++s) { mbar_init(smem_u32(&full[s]), 1 + 4); mbar_init(smem_u32(&empty[s]), 1); }
        for (int s = 0; s < T::kSums; ++s) { mbar_init(smem_u32(&sum_full[s]), 1); mbar_init(smem_u32(&sum_empty[s]), 4 * kTakers); }
        mbar_init(smem_u32(&drained), 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    if (warp == 1) tmem_alloc(smem_u32(&tmem_at), T::kColumns);
    wait_for_kernel_before();
    launch_dependents();
    if (warp == 2) plan_groups(p.groups, p.per, plan);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at, tmem_a = tmem + T::kSums * kHalf;
    const int items = plan.tile[p.groups.groups] * p.tiles_n;
    const auto item_of = [&](int i) { return group_item<true>(plan, p.groups.groups, p.tiles_n, p.per, i); };

    if (warp == 0) {
        // ---- loads of x; the warp stays together, one lane issues
        const bool one = elect_one();
        fence_for_bulk_loads();
        uint32_t s = 0, phase = 1, loaded = 0;           // (the first waits are for the phase before the first)
        bool ok = true;
        for (int i = blockIdx.x; i < items && ok; i += gridDim.x) {
            const GroupItem t = item_of(i);
            const int boxes = (t.rows + kBoxRows - 1) / kBoxRows;
            for (int step = 0; step < p.steps; ++step) {
                ok = still_waits(ok, smem_u32(&empty[s]), phase, &gave_up);
                if (!ok) break;
                if (one) {
                    const uint32_t to = smem_x + s * T::kBytesX, bar = smem_u32(&full[s]);
                    mbar_expect(bar, boxes * kBoxRows * 128);
                    for (int b = 0; b < boxes; ++b) tma_load(to + b * kBoxRows * 128, &map_x, step * kStepK, t.row0 + b * kBoxRows, bar);
                }
                __syncwarp();
                if (++s == T::kStages) { s = 0; phase ^= 1; }
                if (loaded < T::kStages) ++loaded;
            }
        }
        wait_for_loads<T::kStages>(full, s, phase, loaded);
    } else if (warp == kLoaderW) {
        // ---- loads of W, which are not held up by those of x: as far ahead as there is room
        const bool one = elect_one();
        fence_for_bulk_loads();
        uint32_t sw = 0, pw = 1, loaded = 0;
        unsigned left = p.loads;
        bool ok = true;
        for (int i = blockIdx.x; i < items && ok; i += gridDim.x) {
            const GroupItem t = item_of(i);
            for (int step = 0; step < p.steps; step += 4) {
                ok = still_waits(left-- > 0, smem_u32(&w_empty[sw]), pw, &gave_up) && !__any_sync(0xFFFFFFFFu, gave_up);
                if (!ok) break;
                if (one) {
                    const uint32_t to = smem_w + sw * T::kStageW, bar = smem_u32(&w_full[sw]);
                    mbar_expect(bar, T::kBytesW + T::kBytesS);
                    tma_load(to, &map_w, step * 32, int(t.group * p.w.rows + t.tn * kRows), bar);
                    bulk_load(to + T::kBytesW, p.w.scales + (((long long)t.group * p.tiles_n + t.tn) * p.atoms + (long long)(step / 4) * T::kAtoms) * 512, T::kBytesS, bar);
                }
                __syncwarp();
                if (++sw == T::kStagesW) { sw = 0; pw ^= 1; }
                if (loaded < T::kStagesW) ++loaded;
            }
        }
        wait_for_loads<T::kStagesW>(w_full, sw, pw, loaded);
    } else if (warp == 1) {
        // ---- products; likewise
        constexpr uint32_t kIdesc = 1u << 4 | (FP16 ? 0u : 1u << 7 | 1u << 10) | uint32_t(kRows >> 4) << 24;      // bf16 x bf16 (or fp16 x fp16), fp32 sums
        const bool one = elect_one();
        uint32_t s = 0, phase = 0;
        int n = 0;                                       // buffers of sums taken so far
        bool ok = true;
        for (int i = blockIdx.x; i < items && ok; i += gridDim.x) {
            const int rows = item_of(i).rows, halves = rows > kHalf ? 2 : 1;
            const auto idesc_of = [](int columns) { return kIdesc | uint32_t((columns + 15) / 16 * 2) << 17; };
            const uint32_t idesc[2] = {idesc_of(min(rows, kHalf)), idesc_of(rows - kHalf)};
            uint32_t d[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int buf = (n + h) % T::kSums, use = (n + h) / T::kSums;
                d[h] = tmem + buf * kHalf;
                if (h < halves && use > 0) ok = ok && mbar_wait(smem_u32(&sum_empty[buf]), uint32_t(use - 1) & 1, &gave_up);
            }
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            tc_fence_after();
            for (int step = 0; step < p.steps; ++step) {
                ok = mbar_wait(smem_u32(&full[s]), phase, &gave_up);
                ok = __all_sync(0xFFFFFFFFu, ok);        // every lane has seen this phase before the stage can be filled again
                if (!ok) break;
                tc_fence_after();
                const uint64_t db = desc_rows128(smem_x + s * T::kBytesX);
                const uint32_t a = tmem_a + s * T::kColumnsA;
                if (one) {
#pragma unroll
                    for (int j = 0; j < kStepK / 16; ++j) mma_from_tmem(d[0], a + 8 * j, db + 2 * j, idesc[0], step > 0 || j > 0);
                    if (halves > 1) {
#pragma unroll
                        for (int j = 0; j < kStepK / 16; ++j) mma_from_tmem(d[1], a + 8 * j, db + (kHalf * 128 >> 4) + 2 * j, idesc[1], step > 0 || j > 0);
                    }
                    tc_commit(smem_u32(&empty[s]));
                }
                __syncwarp();
                if (++s == T::kStages) { s = 0; phase ^= 1; }
            }
            if (ok && one)
                for (int h = 0; h < halves; ++h) tc_commit(smem_u32(&sum_full[(n + h) % T::kSums]));
            __syncwarp();
            n += halves;
        }
        if (!ok) {                                       // what was issued ends before the tensor memory goes
            if (one) tc_commit(smem_u32(&drained));
            __syncwarp();
            for (long long t0 = clock64(); !mbar_try_wait(smem_u32(&drained), 0) && clock64() - t0 < kMbarWaitCycles;) {}
        }
    } else if (warp >= kFirstMaker) {
        // ---- weights: lane = row of this warp's quarter; the groups of four warps take turns
        const int quarter = warp & 3, mine = (warp - kFirstMaker) >> 2;
        const int row = 32 * quarter + lane;
        const E2m1Bytes<false> bytes;
        const auto scale_of = [&](int i) {               // of this lane's row; fetched an item ahead
            if (FP16 || FMT != kNvfp4 || i >= items) return 1.0f;
            const GroupItem t = item_of(i);
            const long long r = (long long)t.tn * kRows + row;
            return r < p.w.rows ? p.w.row_scale[t.group * p.w.rows + r] : 1.0f;
        };
        float next = scale_of(blockIdx.x);
        uint32_t sw = 0, pw = 0, s = 0, phase = 1;
        int turn = 0;                                    // whose step it is
        bool ok = true;
        for (int i = blockIdx.x; i < items && ok; i += gridDim.x) {
            float power = 1.0f;
            if constexpr (!FP16 && FMT == kNvfp4) {
                power = row_power(next);
                next = scale_of(i + gridDim.x);
            }
            const uint32_t power2 = (__float_as_uint(power) >> 16) * 0x10001u;               // twice, as a bf16 number
            for (int step = 0; step < p.steps && ok; ++step) {
                if (step % 4 == 0) ok = __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&w_full[sw]), pw, &gave_up));
                if (turn == mine && ok) {
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
                    for (int h = 0; h < 2; ++h) {        // 16 bytes: 32 columns; the swizzle has put piece c of row r at c ^ (r % 8)
                        const uint4 c = lds128(from + (((2 * sub + h) ^ (row & 7)) << 4));
                        const uint32_t cw[4] = {c.x, c.y, c.z, c.w};
                        if constexpr (FP16) {
                            uint32_t two, s[2];          // of the two halves
                            asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(two) : "r"(word >> (16 * h)));
                            s[0] = __byte_perm(two, two, 0x1010);
                            s[1] = __byte_perm(two, two, 0x3232);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                uint32_t e[4];
                                e2m1x8_to_f16(cw[j], e);
#pragma unroll
                                for (int q = 0; q < 4; ++q) v[16 * h + 4 * j + q] = mul_f16x2(e[q], s[j / 2]);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                uint32_t e[4];
                                eight_weights(bytes, cw[j], scales16[2 * h + j / 2], e);
#pragma unroll
                                for (int q = 0; q < 4; ++q) v[16 * h + 4 * j + q] = e[q];
                            }
                        }
                    }
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&empty[s]), phase, &gave_up));
                    if (ok) {
                        tc_fence_after();
                        tmem_store32(tmem_a + s * T::kColumnsA + (uint32_t(32 * quarter) << 16), v);
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&full[s]));
                    }
                }
                if (++turn == kMakers) turn = 0;
                if (++s == T::kStages) { s = 0; phase ^= 1; }
                if (step % 4 == 3 || step + 1 == p.steps) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&w_empty[sw]));
                    if (++sw == T::kStagesW) { sw = 0; pw ^= 1; }
                }
            }
        }
    } else {
        // ---- results: this warp's lanes are 32 rows of W, so that a store is 32 neighbours in y
        const int quarter = warp & 3, mine = (warp - kFirstTaker) >> 2;
        constexpr int kChunk = 16;
        int n = 0;
        bool ok = true;
        for (int i = blockIdx.x; i < items; i += gridDim.x) {
            const GroupItem t = item_of(i);
            const long long r = (long long)t.tn * kRows + 32 * quarter + lane, column = t.group * p.w.rows + r;
            const bool there = r < p.w.rows;
            const float fw = there ? row_factor<FMT, FP16>(p, column) : 1.0f;
            const float bias = p.out.bias != nullptr && there ? load_as_f32(p.out.bias, p.out.bias_dtype, column) : 0.0f;
            for (int half = 0; half < t.rows; half += kHalf, ++n) {
                const int buf = n % T::kSums;
                ok = still_waits(ok, smem_u32(&sum_full[buf]), uint32_t(n / T::kSums) & 1, &gave_up);
                tc_fence_after();
                const float plus = ok ? bias : __uint_as_float(0x7FC00000u);
                const int columns = min(kHalf, t.rows - half), share = (columns + kTakers * kChunk - 1) / (kTakers * kChunk) * kChunk;
                const int first = mine * share, last = min(first + share, columns);          // those of the buffer that are this warp's
#pragma unroll 1
                for (int c0 = first; c0 < last; c0 += kChunk) {
                    uint32_t v[kChunk];
                    tmem_load<kChunk>(tmem + buf * kHalf + c0 + (uint32_t(32 * quarter) << 16), v);
                    tmem_wait_ld();
                    float h[kChunk];
#pragma unroll
                    for (int c = 0; c < kChunk; ++c) h[c] = FMT == kNvfp4 ? __fmaf_rn(__uint_as_float(v[c]), fw, plus) : __uint_as_float(v[c]) + plus;
                    if (c0 + kChunk >= last) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&sum_empty[buf]));
                    }
                    finish_rows(p.out, h, t.row0 + half + c0, last - c0, r, there);
                }
                if (first >= last && lane == 0) mbar_arrive(smem_u32(&sum_empty[buf]));       // fewer rows than reach this warp's columns
                __syncwarp();
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free(tmem, T::kColumns);
    }
}

// Rows of 16-bit numbers in order, zeros up to a multiple of eight columns; rows that x has not are NaN.  Threads in x: eight columns of a row each; in y: rows.
__global__ void __launch_bounds__(256) tcq_ms_grouped_rows_kernel(const uint16_t* x, long long x_rows, long long k, long long ldx, const int* tokens, int rows,
                                                                  uint4* out, int runs, bool wide) {
    wait_for_kernel_before();
    launch_dependents();
    for (long long i = (long long)blockIdx.x * blockDim.y + threadIdx.y; i < rows; i += (long long)gridDim.x * blockDim.y) {
        const long long token = tokens != nullptr ? tokens[i] : i;
        const bool there = token >= 0 && token < x_rows;
        const uint16_t* const from = x + token * ldx;
        for (int j = threadIdx.x; j < runs; j += blockDim.x) {
            const long long c0 = 8ll * j;
            uint32_t w[4] = {};
            if (wide && there) {
                const uint4 u = *reinterpret_cast<const uint4*>(from + c0);
                w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
            } else {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (c0 + q < k) w[q / 2] |= (there ? uint32_t(from[c0 + q]) : 0x7FFFu) << (16 * (q & 1));
            }
            out[i * runs + j] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

template <int FMT, bool FP16>
cudaError_t launch(const GroupedCall& c, cudaStream_t stream) {
    using T = Tile<FMT>;
    const auto kernel = tcq_ms_grouped_many_kernel<FMT, FP16>;
    static std::atomic<bool> ready[64];
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev >= 64 || !ready[dev]) {
        if ((err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem)) != cudaSuccess) return err;
        if (dev < 64) ready[dev] = true;
    }
    CUtensorMap map_w, map_x;
    const long long pitch = ms_pitch(c.k), n = c.w.rows;
    if ((err = make_byte_map(&map_w, c.w.codes, pitch, n * c.groups.groups, pitch, kRows)) != cudaSuccess) return err;
    if ((err = make_16bit_map(&map_x, c.x, c.k, c.x_rows, c.ldx, kBoxRows)) != cudaSuccess) return err;
    const ManyArgs p{c.w, c.groups, int((n + kRows - 1) / kRows), int((c.k + kStepK - 1) / kStepK), ms_grouped_many_rows(c.groups.rows, c.groups.groups, n), ms_tiles_k(c.k) * T::kAtoms, c.out, c.loads};
    const long long items = most_tiles(c.groups.rows, c.groups.groups, p.per) * p.tiles_n;
    return launch_programmatic(kernel, dim3(unsigned(std::min<long long>(items, ms_sm_count()))), dim3(kThreads), T::kSmem, 0, stream, map_w, map_x, p);
}

}  // namespace

// Rows of x an item: as few (by sixteens, as the products count, and one box of loads at least) as leave no more items than SMs; 256, for which weights are made once, where there are more.
// (1662 rows of 3 groups, 152 x 347: 32 rows an item 10.4 us, 256 16.9; 1000 rows through 1000 x 1111: 64 rows 13.7, 256 18.2.)
int ms_grouped_many_rows(long long rows, long long groups, long long n) {
    const long long filled = std::min(rows, groups), tiles = ms_sm_count() / ((n + kRows - 1) / kRows);      // of rows, that an SM each can have
    long long per = kNt;
    if (groups == 1 && tiles > 0) per = (rows + tiles - 1) / tiles;
    else if (tiles > filled) per = (rows - filled + tiles - filled - 1) / (tiles - filled);                  // most_tiles() of it is `tiles` at most
    return int(std::min<long long>(kNt, std::max<long long>(kBoxRows, (per + 15) / 16 * 16)));
}

size_t ms_grouped_many_workspace_bytes(long long rows, long long k) { return size_t(rows) * size_t((k + 7) / 8 * 16); }

cudaError_t launch_ms_grouped_many(const GroupedCall& call, void* ws, cudaStream_t stream) {
    GroupedCall c = call;
    if (c.tokens != nullptr || !ms_rows_aligned(c.x, c.ldx)) {      // in order, where TMA loads can start
        const long long runs = (c.k + 7) / 8;
        dim3 block(32, 8);
        while (block.x < 256 && block.x < runs) { block.x *= 2; block.y /= 2; }
        const unsigned grid = unsigned(std::min<long long>((c.groups.rows + block.y - 1) / block.y, 1 << 20));
        const cudaError_t err = launch_programmatic(tcq_ms_grouped_rows_kernel, dim3(grid), block, 0, 0, stream, static_cast<const uint16_t*>(c.x), c.x_rows, c.k, c.ldx, c.tokens,
                                                    c.groups.rows, static_cast<uint4*>(ws), int(runs), c.k % 8 == 0 && ms_rows_aligned(c.x, c.ldx));
        if (err != cudaSuccess) return err;
        c.x = ws;
        c.x_rows = c.groups.rows;
        c.ldx = 8 * runs;
    }
    if (c.fmt == kNvfp4) {
        if (c.dtype == kF16) return launch<kNvfp4, true>(c, stream);
        return launch<kNvfp4, false>(c, stream);
    }
    return launch<kMxfp4, false>(c, stream);
}

}  // namespace tcq
