// Rows of 16-bit activations in groups, each group times a 4-bit microscaled matrix of its own, few rows a group: y[i] = act(W[g(i)] x[i] + bias) + residual.
//
// The tensor cores multiply 4-bit numbers as they lie in memory, so that a weight costs nothing but its bytes; it is x that is cut up.  With s = 2^(floor(log2
// amax) - 1) of a block of 16 (nvfp4) or 32 (mxfp4) columns, x / s is below 4 in magnitude; the nearest e2m1 number is off by half at most, and what is left, times
// eight, is below 4 again.  So x = s (q0 + q1 / 8 + q2 / 64 + ...), each part a row of 4-bit numbers with block scales s, s / 8, s / 64 ..., and the product is that of
// tcgen05.mma with kPartsX columns for each row of x, added up at the end.  Six parts hold every bit of bf16 numbers down to 2^-10 of their block's
// largest (fp16: 2^-7) and are off by 2^-18 of that at most elsewhere; nvfp4's scales, of a token as of a matrix, end 2^-17 below the token's largest one (2^-20 of its largest number).
//
// Work split: one small kernel finds each row's group and place, cuts it up and leaves it as the stages that the products load (codes swizzled as the tensor cores
// read them, scales in the order of tcgen05.cp).  The other goes through items of 128 rows of a matrix x NT / kPartsX rows of its group, one CTA per SM, and begins
// with the loads of W while the first still runs.  With few items a cluster of S CTAs shares the columns of one, and the partial sums meet through
// distributed shared memory, in rank order.  Where groups begin is read on the GPU; the host knows how many rows there are, and chooses by their mean.
//
// A wait that runs out (kMbarWaitCycles) makes its CTA stop, and its results from there on NaN, as those of its cluster.
#include <algorithm>

#include "tcq_microscale_grouped.cuh"
#include "tcq_tcgen05.cuh"

namespace tcq {

namespace {

constexpr int kPartsX = 6;
constexpr int kThreads = 192;                    // loader, issuer, four warps for the results
constexpr int kRowsW = 128, kMostSplits = 8;

__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_kernel_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// What a stage of a tile holds of x: block scales of up to 128 columns (parts of rows), then a row of 128 bytes of codes a column.
template <int FMT> constexpr int kBytesScales = Ms<FMT>::kAtoms * 512;
inline size_t record_bytes(int fmt, int nt) { return size_t(ms_atoms(fmt)) * 512 + size_t(nt) * 128; }

struct PartsArgs {
    const void* x;
    long long x_rows, ldx;
    const int* tokens;
    Groups groups;
    long long k;
    int k_tiles, per;                            // rows of x a tile
    long long record;
    bool wide;                                   // x in pieces of 16 bytes
    uint8_t* out;                                // [tiles][k_tiles][record]
    float* row_scale;                            // nvfp4: [tiles][per]
};

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }      // -126 <= e <= 127

// 32 columns of x from c0 on, zeros behind the last.
template <typename T>
__device__ __forceinline__ void load32(const T* row, long long c0, long long k, bool wide, float (&v)[32]) {
    if (wide && c0 + 32 <= k) {
        uint4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __ldg(reinterpret_cast<const uint4*>(row + c0) + i);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = to_f32<T>(reinterpret_cast<const T*>(u)[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = c0 + i < k ? to_f32<T>(row[c0 + i]) : 0.0f;
    }
}

// Bits of the largest magnitude of v[from .. from + N - 1]; a NaN or an infinity counts as 0x7F800000 and more.
template <int N>
__device__ __forceinline__ uint32_t largest(const float* v) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
}

// The exponent of a block's first scale: floor(log2 amax) - 1, no lower than leaves the last part a scale of its own.
__device__ __forceinline__ int first_exponent(uint32_t amax_bits) { return max(int(amax_bits >> 23) - 128, -127 + 3 * (kPartsX - 1)); }

// One CTA takes rows blockIdx.x, blockIdx.x + gridDim.x ...; a thread 32 columns at a time.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) tcq_ms_row_parts_kernel(const __grid_constant__ PartsArgs p) {
    __shared__ GroupPlan plan;
    __shared__ uint32_t most[8];
    launch_dependents();
    const int chunks = p.k_tiles * 8;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    bool planned = false;
    for (int i = blockIdx.x; i < p.groups.rows; i += gridDim.x) {
        const int token = p.tokens != nullptr ? __ldg(p.tokens + i) : i;
        const bool inside = token >= 0 && token < p.x_rows;
        const T* const row = static_cast<const T*>(p.x) + (inside ? token : 0) * p.ldx;
        float v[32];
        const bool mine = int(threadIdx.x) < chunks;
        if (mine && inside) load32(row, 32ll * threadIdx.x, p.k, p.wide, v);     // on their way while the groups are counted
        if (!planned) {
            if (warp == 0) plan_groups(p.groups, p.per, plan);
            __syncthreads();
            planned = true;
        }
        if (i < plan.begin[0] || i >= plan.begin[p.groups.groups]) continue;     // no group's
        const int g = last_not_above(plan.begin, p.groups.groups, i), at = i - plan.begin[g];
        const int tile = plan.tile[g] + at / p.per, place = at % p.per;
        int base = 0;                                    // nvfp4: exponent of the token's row scale
        if constexpr (FMT == kNvfp4) {
            uint32_t m = 0;
            for (int j = threadIdx.x; j < chunks && inside; j += blockDim.x) {
                float w[32];
                if (j == int(threadIdx.x)) {
#pragma unroll
                    for (int q = 0; q < 32; ++q) w[q] = v[q];
                } else {
                    load32(row, 32ll * j, p.k, p.wide, w);
                }
#pragma unroll
                for (int q = 0; q < 32; ++q) {
                    const uint32_t b = __float_as_uint(w[q]) & 0x7FFFFFFFu;
                    m = max(m, b < 0x7F800000u ? b : 0u);
                }
            }
            m = __reduce_max_sync(0xFFFFFFFFu, m);
            __syncthreads();                             // the row before has been read from `most`
            if (lane == 0) most[warp] = m;
            __syncthreads();
            for (int q = 0; q < int(blockDim.x) / 32; ++q) m = max(m, most[q]);
            base = max(first_exponent(m) - 8, -126);     // the largest block's scale is 2^8
            if (threadIdx.x == 0) p.row_scale[(long long)tile * p.per + place] = pow2f(base);
        }
        for (int j = threadIdx.x; j < chunks; j += blockDim.x) {
            if (j != int(threadIdx.x) && inside) load32(row, 32ll * j, p.k, p.wide, v);
            constexpr int kBlocks = 32 / Ms<FMT>::kBlock, kBlock = Ms<FMT>::kBlock;
            int e[kBlocks];
            bool nan[kBlocks];
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const uint32_t m = largest<kBlock>(v + b * kBlock);
                nan[b] = !inside || m >= 0x7F800000u;
                e[b] = first_exponent(m);
                const float down0 = pow2f(-(e[b] / 2)), down1 = pow2f(e[b] / 2 - e[b]);      // in two steps: -112 <= e <= 126
#pragma unroll
                for (int q = 0; q < kBlock; ++q) v[b * kBlock + q] = nan[b] ? 0.0f : v[b * kBlock + q] * down0 * down1;
            }
            uint8_t* const record = p.out + ((long long)tile * p.k_tiles + j / 8) * p.record;
            const int jj = j % 8;
#pragma unroll
            for (int part = 0; part < kPartsX; ++part) {
                uint32_t words[4] = {};
                uint32_t scale = 0;
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    uint32_t byte;
                    bool gone = false;                   // nvfp4: its scale would be below the least
                    if constexpr (FMT == kNvfp4) {
                        const int to = e[b] - 3 * part - base;                    // at most 8
                        gone = to < -9;
                        byte = nan[b] ? 0x7Fu : to >= -6 ? uint32_t(to + 7) << 3 : gone ? 0u : 1u << (to + 9);
                    } else {
                        byte = nan[b] ? 0xFFu : uint32_t(e[b] - 3 * part + 127);
                    }
                    scale |= byte << (8 * b);
#pragma unroll
                    for (int q = 0; q < kBlock; q += 2) {
                        const int at2 = b * kBlock + q;
                        const uint32_t code = f32x2_to_e2m1x2(v[at2], v[at2 + 1]);
                        uint32_t h;
                        asm("{\n\t.reg .b8 b0;\n\tcvt.u8.u32 b0, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b0;\n\t}" : "=r"(h) : "r"(code));
                        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&h));
                        v[at2] = (v[at2] - back.x) * 8.0f;                        // exact
                        v[at2 + 1] = (v[at2 + 1] - back.y) * 8.0f;
                        words[at2 / 8] |= (gone ? 0u : code) << (4 * (at2 % 8));
                    }
                }
                const int c = place * kPartsX + part;    // column of the tile
                *reinterpret_cast<uint4*>(record + kBytesScales<FMT> + c * 128 + ((jj ^ (c & 7)) << 4)) = make_uint4(words[0], words[1], words[2], words[3]);
                uint8_t* const s = record + (c & 31) * 16 + (c >> 5) * 4;
                if constexpr (FMT == kNvfp4) *reinterpret_cast<uint16_t*>(s + (jj / 2) * 512 + 2 * (jj & 1)) = uint16_t(scale);
                else s[(jj / 4) * 512 + (jj & 3)] = uint8_t(scale);
            }
        }
    }
}

template <int FMT, int NT>
struct Tile {
    static constexpr int kAtoms = Ms<FMT>::kAtoms, kRowsX = NT / kPartsX;
    static constexpr int kBytesW = kRowsW * 128, kBytesS = kAtoms * 512;
    static constexpr int kStageBytes = (kBytesW + 2 * kBytesS + NT * 128 + 1023) / 1024 * 1024;
    static constexpr int kSumColumns = NT < 32 ? 32 : NT;                     // of one of the two buffers of sums
    static constexpr int kScaleColumns = kAtoms * 4 * 2;                      // of one stage
    static constexpr int kBytesSum = kRowsX * kRowsW * 4;                     // partial sums of a CTA
    // as many stages as fit in 205 KB (beside 8 KB for the groups) and in what the sums leave of 512 columns of tensor memory
    static constexpr int kBySmem = (205 * 1024 - kBytesSum) / kStageBytes, kByTmem = (512 - 2 * kSumColumns) / kScaleColumns;
    static constexpr int kStages = std::min(std::min(kBySmem, kByTmem), 12);
    static constexpr int kColumns = 2 * kSumColumns + kStages * kScaleColumns <= 256 ? 256 : 512;
    // over half of an SM's shared memory: two CTAs never share an SM, so that none waits for another's tensor memory
    static constexpr int kSmem = kStages * kStageBytes + kBytesSum + 1024;
    static_assert(kSmem >= 116 * 1024 && kSmem <= 216 * 1024 && kStages >= 4 && kBytesW % 1024 == 0 && (2 * kBytesS) % 1024 == 0);
    // rows whose columns are taken out of tensor memory together, in pieces of eight columns
    static constexpr int kTake = NT <= 8 ? 1 : NT <= 16 ? 2 : 4, kPieces = (kTake * kPartsX + 7) / 8;
    static_assert(kColumns >= 2 * kSumColumns + 8 * kPieces);                 // a piece behind the last row's lies within what is allocated
};

struct GroupedArgs {
    MsMatrix w;
    Groups groups;
    int tiles_n, k_tiles;
    const uint8_t* x;                            // records
    const float* x_row;
    Epilogue out;
    unsigned loads;
};

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
__global__ void __launch_bounds__(kThreads, 1) tcq_ms_grouped_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ GroupedArgs p) {
    using T = Tile<FMT, NT>;
    extern __shared__ uint8_t raw[];
    __shared__ GroupPlan plan;
    __shared__ uint64_t full[T::kStages], empty[T::kStages], sum_full[2], sum_empty[2], drained;
    __shared__ uint32_t tmem_at;
    __shared__ unsigned int gave_up;
    const uint32_t smem = (smem_u32(raw) + 1023) & ~1023u, smem_sum = smem + T::kStages * T::kStageBytes;
    float* const sums = reinterpret_cast<float*>(raw + (smem_sum - smem_u32(raw)));
    const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), splits = cluster_size();
    const int first = int((long long)p.k_tiles * rank / splits), last = int((long long)p.k_tiles * (rank + 1) / splits);
    const int start = blockIdx.x / splits, clusters = gridDim.x / splits;
    const long long atoms = (long long)p.k_tiles * T::kAtoms;
    constexpr long long kRecord = T::kBytesS + NT * 128;

    const auto columns_of = [](const GroupItem& t) { return (t.rows * kPartsX + 7) & ~7; };
    const auto load_w = [&](uint32_t s, const GroupItem& t, int kt) {
        const uint32_t to = smem + s * T::kStageBytes, bar = smem_u32(&full[s]);
        mbar_expect(bar, T::kBytesW + 2 * T::kBytesS + columns_of(t) * 128);
        tma_load(to, &map_w, kt * 128, int(t.group * p.w.rows + t.tn * kRowsW), bar);
        bulk_load(to + T::kBytesW, p.w.scales + (((long long)t.group * p.tiles_n + t.tn) * atoms + (long long)kt * T::kAtoms) * 512, T::kBytesS, bar);
    };
    const auto load_x = [&](uint32_t s, const GroupItem& t, int kt) {
        bulk_load(smem + s * T::kStageBytes + T::kBytesW + T::kBytesS, p.x + ((long long)t.tile * p.k_tiles + kt) * kRecord, T::kBytesS + columns_of(t) * 128, smem_u32(&full[s]));
    };
    int ahead = 0;
    if (warp == 0) {
        if (elect_one()) {
            gave_up = 0;
            for (int s = 0; s < T::kStages; ++s) { mbar_init(smem_u32(&full[s]), 1); mbar_init(smem_u32(&empty[s]), 1); }
            for (int s = 0; s < 2; ++s) { mbar_init(smem_u32(&sum_full[s]), 1); mbar_init(smem_u32(&sum_empty[s]), 4); }
            mbar_init(smem_u32(&drained), 1);
            asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        plan_groups(p.groups, T::kRowsX, plan);
        // The first item's first stages of W are on their way before x is there: with few rows a call is little more than its latencies.
        if (start < plan.tile[p.groups.groups] * p.tiles_n) {
            const GroupItem t = group_item(plan, p.groups.groups, p.tiles_n, T::kRowsX, start);
            ahead = min(min(unsigned(T::kStages), unsigned(last - first)), p.loads);
            if (elect_one())
                for (int i = 0; i < ahead; ++i) load_w(i, t, first + i);
            __syncwarp();
        }
    }
    if (warp == 1) tmem_alloc(smem_u32(&tmem_at), T::kColumns);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at, tmem_scales = tmem + 2 * T::kSumColumns;
    const int items = plan.tile[p.groups.groups] * p.tiles_n;
    const auto item_of = [&](int i) { return group_item(plan, p.groups.groups, p.tiles_n, T::kRowsX, i); };

    if (warp == 0) {
        // ---- loads; the warp stays together, one lane issues
        const bool one = elect_one();
        wait_for_kernel_before();                        // x's parts are there
        asm volatile("fence.proxy.async;" ::: "memory");
        uint32_t s = ahead % T::kStages, phase = ahead == T::kStages ? 0 : 1, loaded = ahead;    // (the first wait for a stage is for the phase before the first)
        unsigned left = p.loads - ahead;
        bool ok = true;
        for (int i = start, kt = first; i < items && ok; i += clusters, kt = first) {
            const GroupItem t = item_of(i);
            if (i == start) {
                if (one)
                    for (int q = 0; q < ahead; ++q) load_x(q, t, first + q);
                __syncwarp();
                kt = first + ahead;
            }
            for (; kt < last; ++kt) {
                ok = still_waits(left-- > 0, smem_u32(&empty[s]), phase, &gave_up);      // every lane has seen this phase before the next can begin
                if (!ok) break;
                if (one) {
                    load_w(s, t, kt);
                    load_x(s, t, kt);
                }
                __syncwarp();
                if (++s == T::kStages) { s = 0; phase ^= 1; }
                if (loaded < T::kStages) ++loaded;
            }
        }
        wait_for_loads<T::kStages>(full, s, phase, loaded);
    } else if (warp == 1) {
        // ---- products; likewise
        constexpr uint32_t kIdesc = 1u << 7 | 1u << 10 | (FMT == kMxfp4 ? 1u : 0u) << 23 | 1u << 27;
        const bool one = elect_one();
        uint32_t s = 0, phase = 0;
        int n = 0;
        bool ok = true;
        for (int i = start; i < items && ok; i += clusters, ++n) {
            const uint32_t idesc0 = kIdesc | uint32_t(columns_of(item_of(i)) >> 3) << 17;
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
                const uint64_t dw = desc_rows128(at), dx = desc_rows128(at + T::kBytesW + 2 * T::kBytesS), ds = desc_rows16(at + T::kBytesW);
                if (one) {
#pragma unroll
                    for (int j = 0; j < T::kAtoms; ++j) {
                        tc_copy_scales(sw + 4 * j, ds + 32 * j);
                        tc_copy_scales(sx + 4 * j, ds + (T::kBytesS >> 4) + 32 * j);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {            // 64 columns: 32 bytes of a row, one word of scales (nvfp4) or half a word (mxfp4)
                        const int atom = FMT == kNvfp4 ? j : j / 2;
                        const uint32_t id = FMT == kNvfp4 ? 0u : 2u * (j % 2);
                        mma_block_scaled<FMT>(d, dw + 2 * j, dx + 2 * j, idesc0 | id << 4 | id << 29, sw + 4 * atom, sx + 4 * atom, kt > first || j > 0);
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
        wait_for_kernel_before();                            // rows' scales
        int n = 0;
        bool ok = true;
        for (int i = start; i < items; i += clusters, ++n) {
            const GroupItem t = item_of(i);
            const int buf = n & 1;
            const long long r = (long long)t.tn * kRowsW + 32 * quarter + lane;
            const bool there = r < p.w.rows;
            const long long column = (long long)t.group * p.w.rows + r;
            const float fw = FMT == kNvfp4 && there ? __ldg(p.w.row_scale + column) : 1.0f;
            const float inner = inner_part(fw), outer = outer_part(fw);
            const float bias = p.out.bias != nullptr && there ? load_as_f32(p.out.bias, p.out.bias_dtype, column) : 0.0f;
            ok = still_waits(ok, smem_u32(&sum_full[buf]), uint32_t(n / 2) & 1, &gave_up);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < t.rows; c += T::kTake) {
                uint32_t v[T::kPieces][8];
#pragma unroll
                for (int q = 0; q < T::kPieces; ++q) tmem_load<8>(tmem + buf * T::kSumColumns + c * kPartsX + 8 * q + (uint32_t(32 * quarter) << 16), v[q]);
                const float fx = FMT == kNvfp4 && lane < T::kTake && c + lane < t.rows ? p.x_row[(long long)t.tile * T::kRowsX + c + lane] : 1.0f;
                tmem_wait_ld();
                if (c + T::kTake >= t.rows) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sum_empty[buf]));
                }
                float h[T::kTake];
#pragma unroll
                for (int q = 0; q < T::kTake; ++q) {
                    float sum = __uint_as_float(v[(q * kPartsX + kPartsX - 1) / 8][(q * kPartsX + kPartsX - 1) % 8]);
#pragma unroll
                    for (int part = kPartsX - 2; part >= 0; --part) sum += __uint_as_float(v[(q * kPartsX + part) / 8][(q * kPartsX + part) % 8]);      // smallest first
                    if constexpr (FMT == kNvfp4) sum = sum * inner * __shfl_sync(0xFFFFFFFFu, fx, q) * outer;
                    h[q] = ok ? sum : __uint_as_float(0x7FC00000u);
                }
                if (splits > 1) {
#pragma unroll
                    for (int q = 0; q < T::kTake; ++q)
                        if (c + q < T::kRowsX) sums[(c + q) * kRowsW + 32 * quarter + lane] = h[q];
                } else {
#pragma unroll
                    for (int q = 0; q < T::kTake; ++q) h[q] += bias;
                    finish_rows(p.out, h, t.row0 + c, t.rows - c, r, there);
                }
            }
        }
    }
    __syncwarp();
    if (splits > 1) {                                        // one item a cluster: add up the parts of it, four neighbours a thread
        cluster_sync();
        if (start < items) {
            const GroupItem t = item_of(start);
            for (int i = int(rank) * kThreads + threadIdx.x; i < kRowsW / 4 * t.rows; i += int(splits) * kThreads) {
                const long long r = (long long)t.tn * kRowsW + i % (kRowsW / 4) * 4;
                if (r >= p.w.rows) continue;
                float4 part[kMostSplits];
#pragma unroll
                for (uint32_t q = 0; q < kMostSplits; ++q)
                    if (q < splits) part[q] = ld_cluster_f32x4(smem_sum + 16 * i, q);
                float4 f = part[0];
#pragma unroll
                for (uint32_t q = 1; q < kMostSplits; ++q)
                    if (q < splits) f = make_float4(f.x + part[q].x, f.y + part[q].y, f.z + part[q].z, f.w + part[q].w);
                float h[4] = {f.x, f.y, f.z, f.w};
                if (p.out.bias != nullptr)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (r + j < p.w.rows) h[j] += load_as_f32(p.out.bias, p.out.bias_dtype, (long long)t.group * p.w.rows + r + j);
                finish_four(p.out, h, t.row0 + i / (kRowsW / 4), r, p.w.rows);
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

// Columns of sums for the rows of x of one item: what holds all rows of one group, or one and a half times the mean of the groups that may have rows.
int columns_for(long long rows, long long groups) {
    const long long filled = std::min(rows, groups);
    for (int nt : {8, 16, 32, 64})
        if (2 * (nt / kPartsX) * filled >= (groups > 1 && rows > groups ? 3 : 2) * rows) return nt;
    return 128;
}

template <typename T>
cudaError_t launch_parts(const GroupedCall& c, const PartsArgs& p, cudaStream_t stream) {
    const int threads = int(std::min<long long>(256, (p.k_tiles * 8 + 31) / 32 * 32));
    const unsigned grid = unsigned(std::min<long long>(c.groups.rows, ms_sm_count() * 8));
    if (c.fmt == kNvfp4) tcq_ms_row_parts_kernel<T, kNvfp4><<<grid, threads, 0, stream>>>(p);
    else tcq_ms_row_parts_kernel<T, kMxfp4><<<grid, threads, 0, stream>>>(p);
    return cudaGetLastError();
}

template <int FMT, int NT>
cudaError_t launch(const GroupedCall& c, void* ws, cudaStream_t stream) {
    using T = Tile<FMT, NT>;
    const auto kernel = tcq_ms_grouped_kernel<FMT, NT>;
    static std::atomic<bool> ready[64];
    static MostClusters kept;
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev >= 64 || !ready[dev]) {
        if ((err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem)) != cudaSuccess) return err;
        if (dev < 64) ready[dev] = true;
    }
    CUtensorMap map_w;
    const long long pitch = ms_pitch(c.k), n = c.w.rows;
    if ((err = make_byte_map(&map_w, c.w.codes, pitch, n * c.groups.groups, pitch, kRowsW)) != cudaSuccess) return err;
    const int k_tiles = int(ms_tiles_k(c.k));
    const long long tiles = most_tiles(c.groups.rows, c.groups.groups, T::kRowsX);
    uint8_t* const records = static_cast<uint8_t*>(ws) + (tiles * T::kRowsX * 4 + 255) / 256 * 256;
    const PartsArgs parts{c.x, c.x_rows, c.ldx, c.tokens, c.groups, c.k, k_tiles, T::kRowsX, (long long)record_bytes(FMT, NT),
                          ms_rows_aligned(c.x, c.ldx), records, static_cast<float*>(ws)};
    err = c.dtype == kF16 ? launch_parts<__half>(c, parts, stream) : launch_parts<__nv_bfloat16>(c, parts, stream);
    if (err != cudaSuccess) return err;
    const GroupedArgs p{c.w, c.groups, int((n + kRowsW - 1) / kRowsW), k_tiles, records, static_cast<const float*>(ws), c.out, c.loads};
    const long long items = tiles * p.tiles_n;
    int splits = 1;
    while (splits < kMostSplits && splits * 4 <= k_tiles &&
           items <= ms_most_clusters(kept, reinterpret_cast<const void*>(kernel), kThreads, T::kSmem, 1, splits * 2)) splits *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(splits > 1 ? items * splits : std::min<long long>(items, ms_sm_count())));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = T::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2] = {};
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = unsigned(splits);
    attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // begins beside the kernel that makes the parts, and waits for it where it needs them
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, map_w, p);
}

template <int FMT>
cudaError_t launch_nt(const GroupedCall& c, void* ws, cudaStream_t stream) {
    switch (columns_for(c.groups.rows, c.groups.groups)) {
        case 8: return launch<FMT, 8>(c, ws, stream);
        case 16: return launch<FMT, 16>(c, ws, stream);
        case 32: return launch<FMT, 32>(c, ws, stream);
        case 64: return launch<FMT, 64>(c, ws, stream);
        default: return launch<FMT, 128>(c, ws, stream);
    }
}

}  // namespace

// Whether weights as 16-bit numbers pay: they are made once for up to 256 rows, where parts of x take six columns a row.
static bool many_rows(long long rows, long long groups, int dtype, int fmt) { return rows > 90 * std::min(groups, rows) && ms_grouped_many_takes(dtype, fmt); }

size_t ms_grouped_workspace_bytes(long long rows, long long groups, long long n, long long k, int dtype, int fmt, bool in_order) {
    (void)n;
    if (many_rows(rows, groups, dtype, fmt)) return in_order ? 0 : ms_grouped_many_workspace_bytes(rows, k);
    const int nt = columns_for(rows, groups), per = nt / kPartsX;
    const long long tiles = most_tiles(rows, groups, per);
    return size_t((tiles * per * 4 + 255) / 256 * 256) + size_t(tiles) * size_t(ms_tiles_k(k)) * record_bytes(fmt, nt);
}

cudaError_t launch_ms_grouped(const GroupedCall& c, void* ws, cudaStream_t stream) {
    if (many_rows(c.groups.rows, c.groups.groups, c.dtype, c.fmt)) return launch_ms_grouped_many(c, ws, stream);
    return c.fmt == kNvfp4 ? launch_nt<kNvfp4>(c, ws, stream) : launch_nt<kMxfp4>(c, ws, stream);
}

}  // namespace tcq
