// Products of 16- and 32-bit activations with a 4-bit microscaled matrix, up to eight tokens: y[i][r] = sum_c x[i][c] * W[r][c].
//
// Codes become fp16 numbers (one conversion instruction a pair), so the products are those of mma.sync on fp16.  nvfp4: times the e4m3 scale, still an
// fp16 number.  mxfp4: scales can lie outside fp16, so the sums of 32 columns are scaled instead.  x is cut into fp16 parts, 256 columns of
// a token at a time: a power of two brings the largest magnitude under 2^15, eleven bits are cut off as fp16, and what is left is the next
// part's, until nothing is left.  fp16 and bf16 activations nearly always take one part (nothing is left of numbers within 2^-31 of the
// largest), fp32 three (2^-37); more are further rounds over the same codes.  So every product is exact.  (bf16 weights need no such care but three
// times the instructions a pair, which was the bound: 4 tokens through 151936 x 4096 136 us.)
// Sums of 32 columns (mxfp4) take the block's scale, sums of 256 (nvfp4) the power of two in the row's scale, before x's factor: what is then added up is of the
// size of the results, whatever that of x and of W alone.  (Only a block scale above 2^104, of weights above 10^31, may take a sum out of range that x would bring back.)
//
// Work split: a CTA takes 128 rows of W, eight warps 16 rows each; one more warp loads 256 columns of codes (TMA) and scales at a time into a ring
// of stages.  ldmatrix gives lane (g, t) the t-th eight codes of 32 columns of rows g and g + 8, two products' share.  x is converted
// once where all columns of a CTA fit beside the stages, else a token a warp, for the next stage while this one is multiplied.  Where there are few groups of 128 rows a
// cluster of S CTAs shares the columns, and the partial sums meet through distributed shared memory, in rank order; of many groups, so are the last ones.
//
// Bound by latency (51 to 56 % of the issue slots, 18 warps an SM; nvfp4's products of a stage are one chain of sums): one token through 40960 x 4096 26.6 us
// (3.5 TB/s), mxfp4 26.2; eight 36.8 and 32.5.  Three parts of x spill (184 bytes a thread, mxfp4 384, at the 96 registers that nine warps leave): seven fp32 tokens
// through 4096 x 12288 23.6 us, mxfp4 26.7.
//
// A wait that runs out (kMbarWaitCycles) makes its CTA's results from there on NaN, and those of its cluster.
#include <algorithm>
#include <type_traits>

#include "tcq_common.cuh"
#include "tcq_microscale.cuh"
#include "tcq_microscale_many.cuh"
#include "tcq_tcgen05.cuh"

namespace tcq {

namespace {

constexpr int kConsumers = 256, kThreads = kConsumers + 32, kRows = 128, kMostSplits = 8, kTokens = 8;

template <int FMT, int PARTS, int STAGES>
struct Tile {
    static constexpr int kAtoms = Ms<FMT>::kAtoms;
    static constexpr int kBytesW = kRows * 128, kBytesS = kAtoms * 512, kStage = kBytesW + 2048;
    static constexpr int kBytesSum = kTokens * kRows * 4;
    // A token's 256 columns: 512 bytes, for the banks either with odd tokens' pieces of 64 bytes swapped in twos or (three parts have no registers
    // for that: 1.2 times the time) another 64 bytes.  So many of them are held beside three stages, and beside two.
    static constexpr bool kSwapped = PARTS == 1;
    static constexpr int kPitchX = kSwapped ? 512 : 576, kRowsX3 = kSwapped ? 100 : 88;
    static constexpr int kRowsX = kRowsX3 + (3 - STAGES) * (kStage / kPitchX);
    static constexpr int kSmem = 3 * kStage + (kRowsX3 + 1) * kPitchX + kBytesSum + 1024;
    static_assert(kSmem <= 113 * 1024 && kRowsX3 >= 2 * PARTS * kTokens);      // two CTAs an SM; at least two times eight tokens' parts
};

struct FewArgs {
    const void* x;
    long long ldx;
    int m;
    bool wide;                                   // x in pieces of 16 bytes
    long long k;
    MsMatrix w;
    long long atoms;
    int tiles, whole, k_tiles;                   // groups of 128 rows of W; how many of them a CTA does by itself
    void* y;
    long long ldy;
    unsigned loads;                              // stages that a CTA loads, at most (a self-test's limit)
};

__device__ __forceinline__ void ldmatrix4(uint32_t smem, uint32_t (&v)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(smem) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t smem) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t smem) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(smem) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(uint32_t smem, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(smem), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two e8m0 scales as bf16 numbers (2^-127 a denormal one, 255 NaN).
__device__ __forceinline__ uint32_t e8m0x2_to_bf16x2(uint16_t v) {
    uint32_t r;
    asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(r) : "h"(v));
    return r;
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }      // -126 <= e <= 127

// The next PARTS parts of eight of a token's 256 columns (a warp has them all): fp16 numbers, times the factors given, which are 2^-11 apart; r
// becomes what is left.  BITS: significant bits of the numbers at the start.
template <int PARTS, int BITS>
__device__ __forceinline__ bool next_parts(float (&r)[8], uint32_t (&h)[PARTS][4], float (&factor)[PARTS]) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(r[i]) & 0x7FFFFFFFu);
    most = __reduce_max_sync(0xFFFFFFFFu, most);
    bool left = false;
    // 2^-103 and more (2^-90 for three parts, the last of which takes 2^22 more), and finite: all factors are normal numbers
    if (most >= uint32_t(PARTS == 1 ? 24 : 15 + 11 * (PARTS - 1)) << 23 && most < 0x7F800000u) {
        const int up = 141 - int(most >> 23);            // largest magnitude below 2^15
        if constexpr (PARTS == 1) {
            const float f = pow2f(up);
            factor[0] = pow2f(-up);
            // the last of a number's bits is 2^-24 or more unless its exponent is below this: then it has been cut
            const uint32_t least = uint32_t(127 - 24 + (BITS - 1) - up) << 23;
            bool cut = false;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(h[0][i / 2]) : "f"(r[i + 1] * f), "f"(r[i] * f));
                cut = cut || (__float_as_uint(r[i]) & 0x7FFFFFFFu) - 1u < least - 1u || (__float_as_uint(r[i + 1]) & 0x7FFFFFFFu) - 1u < least - 1u;
            }
            if (!__any_sync(0xFFFFFFFFu, cut)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) r[i] = 0.0f;   // another token may have further rounds, in which this one adds nothing
                return false;
            }
        }
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
            const float f = pow2f(up + 11 * q), g = pow2f(-up - 11 * q);
            const f32x2 f2 = pack2(f, f), minus = pack2(-g, -g);
            factor[q] = g;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                float a, b;
                unpack2(mul2(pack2(r[i], r[i + 1]), f2), a, b);
                asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(h[q][i / 2]) : "f"(b), "f"(a));
                const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&h[q][i / 2]));
                unpack2(fma2(pack2(back.x, back.y), minus, pack2(r[i], r[i + 1])), r[i], r[i + 1]);      // exact: the bits that were cut off
            }
        }
    } else {
        // nothing left, tiny numbers, infinities or NaN: part by part, factors in two steps, what is not finite once and for all
#pragma unroll 1
        for (int q = 0; q < PARTS; ++q) {
            uint32_t finite = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t b = __float_as_uint(r[i]) & 0x7FFFFFFFu;
                finite = max(finite, b < 0x7F800000u ? b : 0u);
            }
            finite = __reduce_max_sync(0xFFFFFFFFu, finite);
            const int up = finite == 0 ? 0 : 141 - max(int(finite >> 23), 1);                 // -113 <= up <= 140
            const float f0 = pow2f(up / 2), f1 = pow2f(up - up / 2), g0 = pow2f(-(up / 2)), g1 = pow2f(up / 2 - up);
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(w[i / 2]) : "f"(r[i + 1] * f0 * f1), "f"(r[i] * f0 * f1));
                const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&w[i / 2]));
                r[i] = (__float_as_uint(r[i]) & 0x7F800000u) != 0x7F800000u ? r[i] - back.x * g0 * g1 : 0.0f;
                r[i + 1] = (__float_as_uint(r[i + 1]) & 0x7F800000u) != 0x7F800000u ? r[i + 1] - back.y * g0 * g1 : 0.0f;
            }
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                if (p == q) {
                    factor[p] = g0 * g1;
#pragma unroll
                    for (int i = 0; i < 4; ++i) h[p][i] = w[i];
                }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) left = left || r[i] != 0.0f;
    return left;
}

// Whether any of the 256 threads says so; all of them have arrived.
__device__ __forceinline__ bool any_of_consumers(bool mine) {
    uint32_t r;
    __syncwarp();
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.aligned.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"(uint32_t(mine)), "n"(kConsumers) : "memory");
    return r != 0;
}

// PARTS of x held at a time.
template <typename T, int FMT, int PARTS, int STAGES>
__global__ void __launch_bounds__(kThreads, 2) tcq_ms_linear_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ FewArgs p) {
    using G = Tile<FMT, PARTS, STAGES>;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[STAGES], empty[STAGES];
    __shared__ float factor[G::kRowsX];
    __shared__ unsigned int gave_up;
    const uint32_t smem = (smem_u32(raw) + 1023) & ~1023u, smem_x = smem + STAGES * G::kStage, zeros = smem_x + G::kRowsX * G::kPitchX, smem_sum = zeros + G::kPitchX;
    float* const sums = reinterpret_cast<float*>(raw + (smem_sum - smem_u32(raw)));
    const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), splits = cluster_size();
    // What this CTA does: groups of rows blockIdx.x, blockIdx.x + gridDim.x ... of the first `whole`, and with its cluster, columns share .. until, one of the others.
    const int share = int((long long)p.k_tiles * rank / splits), until = int((long long)p.k_tiles * (rank + 1) / splits);
    const int together = p.whole + blockIdx.x / splits;
    const int ends = p.whole + (splits > 1 && together < p.tiles ? int(gridDim.x) : 0);

    auto load = [&](uint32_t s, int t, int kt) {
        const uint32_t to = smem + s * G::kStage, bar = smem_u32(&full[s]);
        mbar_expect(bar, G::kBytesW + G::kBytesS);
        tma_load(to, &map_w, kt * 128, t * kRows, bar);
        bulk_load(to + G::kBytesW, p.w.scales + (t * p.atoms + (long long)kt * G::kAtoms) * 512, G::kBytesS, bar);
    };
    // The first stages are on their way before anything else: a small call is little more than its latencies.
    const int ahead = min(min(unsigned(STAGES), unsigned(p.whole ? p.k_tiles : until - share)), p.loads);
    if (warp == 8) {
        if (elect_one()) {
            gave_up = 0;
            for (int s = 0; s < STAGES; ++s) { mbar_init(smem_u32(&full[s]), 1); mbar_init(smem_u32(&empty[s]), 8); }
            asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
            for (int i = 0; i < ahead; ++i) load(i, p.whole ? blockIdx.x : together, (p.whole ? 0 : share) + i);
        }
        __syncwarp();
    }
    __syncthreads();

    if (warp == 8) {
        // ---- loads; the warp stays together, one lane issues
        const bool one = elect_one();
        uint32_t s = ahead == STAGES ? 0 : ahead, phase = ahead == STAGES ? 0 : 1, loaded = ahead;    // (the first wait for a stage is for the phase before the first)
        unsigned left = p.loads - ahead;
        bool ok = true;
        for (int t = blockIdx.x, skip = ahead; t < ends && ok; t += gridDim.x, skip = 0)
            for (int kt = (t < p.whole ? 0 : share) + skip; kt < (t < p.whole ? p.k_tiles : until); ++kt) {
                ok = still_waits(left-- > 0, smem_u32(&empty[s]), phase, &gave_up) && !__any_sync(0xFFFFFFFFu, gave_up);      // (who gave up arrives all the same)
                if (!ok) break;
                if (one) load(s, t < p.whole ? t : together, kt);
                __syncwarp();
                if (++s == STAGES) { s = 0; phase ^= 1; }
                if (loaded < STAGES) ++loaded;
            }
        wait_for_loads<STAGES>(full, s, phase, loaded);
    } else {
        const int g = lane >> 2, t4 = lane & 3;
        const uint32_t odd = G::kSwapped ? 64 * (g & 1) : 0;
        const bool converts = warp < p.m;                // a warp converts a token's columns, eight a lane
        float next[8], r[8];
        auto fetch = [&](int kt, int token) {
            if (token >= p.m) return;
            const T* const x = static_cast<const T*>(p.x) + token * p.ldx;
            const long long c = (long long)kt * kMsTileK + 8 * lane;
            if (p.wide && c + 8 <= p.k) {
                uint4 u[sizeof(T) / 2];
#pragma unroll
                for (int i = 0; i < int(sizeof(T) / 2); ++i) u[i] = __ldg(reinterpret_cast<const uint4*>(x + c) + i);
                const T* const v = reinterpret_cast<const T*>(u);
#pragma unroll
                for (int i = 0; i < 8; ++i) next[i] = to_f32<T>(v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) next[i] = c + i < p.k ? to_f32<T>(x[c + i]) : 0.0f;
            }
        };
        // The rows of x: part q of token i of the n-th 256 columns held is row (n * PARTS + q) * m + i.  PARTS more parts of r into the n-th; whether
        // something is left.
        auto convert_one = [&](int n, int token) {
            uint32_t h[PARTS][4];
            float f[PARTS];
            constexpr int kBits = std::is_same_v<T, float> ? 24 : std::is_same_v<T, __half> ? 11 : 8;
            const bool left = next_parts<PARTS, kBits>(r, h, f);
#pragma unroll
            for (int q = 0; q < PARTS; ++q) {
                const int row = (n * PARTS + q) * p.m + token;
                sts128(smem_x + row * G::kPitchX + ((16 * lane) ^ (G::kSwapped ? 64 * (token & 1) : 0)), h[q]);
                if (lane == 0) factor[row] = f[q];
            }
            return left;
        };
        auto convert = [&](int n) { return any_of_consumers(converts && convert_one(n, warp)); };
        // tokens that there are not: zeros
        if (threadIdx.x < 32) {
            const uint32_t zero[4] = {};
            sts128(zeros + 16 * lane, zero);
        }
        uint32_t s = 0, phase = 0;
        // ldmatrix: lane l gives the address of row l % 16 of this warp's, piece l / 16 of two
        const int lrow = 16 * warp + (lane & 15);
        const uint32_t from_w = lrow * 128, piece = lane >> 4, swizzle = lrow & 7;
        const int srow = 16 * warp + g;                  // rows whose scales this lane needs: srow, srow + 8
        const uint32_t from_s = G::kBytesW + (srow & 31) * 16 + (srow >> 5) * 4;
        float g2[2] = {1.0f, 1.0f};                      // nvfp4: these rows' scales; the first ones are on their way while x is converted
        auto fetch_scales = [&](int t) {
            if constexpr (FMT == kNvfp4) {
                const long long row = (long long)(t < p.whole ? t : together) * kRows + srow;
#pragma unroll
                for (int h = 0; h < 2; ++h) g2[h] = row + 8 * h < p.w.rows ? __ldg(p.w.row_scale + row + 8 * h) : 1.0f;
            }
        };
        fetch_scales(blockIdx.x);

        // Where all of this CTA's columns fit, they are converted once, by all warps; unless that leaves something, which takes further rounds.
        const int base = p.whole ? 0 : share, span = p.whole ? p.k_tiles : until - share;
        bool held = span * PARTS * p.m <= G::kRowsX;
        if (held) {
            bool left = false;
            for (int i = warp; i < span * p.m; i += 8) {
                fetch(base + i / p.m, i % p.m);
#pragma unroll
                for (int j = 0; j < 8; ++j) r[j] = next[j];
                left = convert_one(i / p.m, i % p.m) || left;
            }
            held = !any_of_consumers(left);
        }

        for (int t = blockIdx.x; t < ends; t += gridDim.x) {
            const int first = t < p.whole ? 0 : share, last = t < p.whole ? p.k_tiles : until;
            if (t != int(blockIdx.x)) fetch_scales(t);
            float acc[4] = {}, low[4] = {};              // rows g (0, 1) and g + 8, tokens 2 t4 and 2 t4 + 1; what the sums' rounding left
            int buf = 0;
            bool more = false;
            if (!held) {
                fetch(first, warp);
#pragma unroll
                for (int i = 0; i < 8; ++i) r[i] = next[i];
                more = convert(0);
            }
            for (int kt = first; kt < last; ++kt) {
                if (!held && kt + 1 < last) fetch(kt + 1, warp);
                mbar_wait(smem_u32(&full[s]), phase, &gave_up);
                __syncwarp();
                const uint32_t stage = smem + s * G::kStage;
                for (;;) {
                    float sum[PARTS][4] = {};            // of 256 columns
                    f32x2 scaled[PARTS][2] = {}, by[PARTS];       // mxfp4: the same by columns of one scale; factors of this lane's two tokens
                    uint32_t from_x[PARTS];
#pragma unroll
                    for (int q = 0; q < PARTS; ++q) {
                        const int row = ((held ? kt - base : buf) * PARTS + q) * p.m;
                        by[q] = pack2(2 * t4 < p.m ? factor[row + 2 * t4] : 0.0f, 2 * t4 + 1 < p.m ? factor[row + 2 * t4 + 1] : 0.0f);
                        from_x[q] = (g < p.m ? smem_x + (row + g) * G::kPitchX : zeros) + 16 * t4;
                    }
#pragma unroll
                    for (int c = 0; c < 8; c += 2) {     // 64 columns
                        uint32_t w[4];                   // columns 32 c: rows g and g + 8; columns 32 (c + 1)
                        ldmatrix4(stage + from_w + ((c + piece) ^ swizzle) * 16, w);
                        uint32_t scale[2][2];            // [piece][row]; nvfp4: fp16 pairs, of this lane's half of 32 columns; mxfp4: fp32
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if constexpr (FMT == kNvfp4) {
                                const uint32_t word = lds32(stage + from_s + 512 * (c / 2) + 128 * h);
                                const uint32_t two = __byte_perm(word, 0u, t4 < 2 ? 0x4420 : 0x4431);
                                uint32_t f;
                                asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(f) : "r"(two));
                                scale[0][h] = __byte_perm(f, f, 0x1010);
                                scale[1][h] = __byte_perm(f, f, 0x3232);
                            } else {
                                const uint32_t word = lds32(stage + from_s + 512 * (c / 4) + 128 * h);
                                const uint32_t f = e8m0x2_to_bf16x2(uint16_t(c % 4 ? word >> 16 : word));
                                scale[0][h] = f << 16;
                                scale[1][h] = f & 0xFFFF0000u;
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            uint32_t a0[4], a1[4];
                            e2m1x8_to_f16(w[2 * i], a0);
                            e2m1x8_to_f16(w[2 * i + 1], a1);
                            if constexpr (FMT == kNvfp4) {
#pragma unroll
                                for (int j = 0; j < 4; ++j) { a0[j] = mul_f16x2(a0[j], scale[i][0]); a1[j] = mul_f16x2(a1[j], scale[i][1]); }
                            }
                            const uint32_t lo[4] = {a0[0], a1[0], a0[1], a1[1]}, hi[4] = {a0[2], a1[2], a0[3], a1[3]};
#pragma unroll
                            for (int q = 0; q < PARTS; ++q) {
                                const uint4 b = lds128((i ? from_x[q] - odd : from_x[q] + odd) + 64 * (c + i));
                                if constexpr (FMT == kNvfp4) {
                                    mma_f16(sum[q], lo, b.x, b.y);
                                    mma_f16(sum[q], hi, b.z, b.w);
                                } else {
                                    float d[4] = {};
                                    mma_f16(d, lo, b.x, b.y);
                                    mma_f16(d, hi, b.z, b.w);
                                    const float s0 = __uint_as_float(scale[i][0]), s1 = __uint_as_float(scale[i][1]);
                                    scaled[q][0] = fma2(mul2(pack2(d[0], d[1]), pack2(s0, s0)), by[q], scaled[q][0]);
                                    scaled[q][1] = fma2(mul2(pack2(d[2], d[3]), pack2(s1, s1)), by[q], scaled[q][1]);
                                }
                            }
                        }
                    }
                    // Parts of one number meet here: added with what each addition's rounding leaves, so that the number is whole again.
#pragma unroll
                    for (int q = 0; q < PARTS; ++q) {
                        if constexpr (FMT == kNvfp4) {
                            const float power[2] = {row_power(g2[0]), row_power(g2[1])};
                            scaled[q][0] = mul2(mul2(pack2(sum[q][0], sum[q][1]), pack2(power[0], power[0])), by[q]);
                            scaled[q][1] = mul2(mul2(pack2(sum[q][2], sum[q][3]), pack2(power[1], power[1])), by[q]);
                        }
                        float v[4];
                        unpack2(scaled[q][0], v[0], v[1]);
                        unpack2(scaled[q][1], v[2], v[3]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float total = acc[i] + v[i], was = total - acc[i];
                            low[i] += (acc[i] - (total - was)) + (v[i] - was);
                            acc[i] = total;
                        }
                    }
                    if (!more) break;
                    any_of_consumers(false);             // all have read this buffer: the next parts
                    more = convert(buf);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&empty[s]));
                if (++s == STAGES) { s = 0; phase ^= 1; }
                if (!held && kt + 1 < last) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) r[i] = next[i];
                    buf ^= 1;
                    more = convert(buf);
                }
            }
            // A wait that ran out is for good, here as well: waits for later phases of that stage may have been answered by the parity of an earlier one.
            if (*static_cast<volatile unsigned int*>(&gave_up)) acc[0] = acc[1] = acc[2] = acc[3] = __uint_as_float(0x7FC00000u);
#pragma unroll
            for (int i = 0; i < 4; ++i)                  // (an infinite or NaN sum leaves NaN behind)
                sums[(2 * t4 + (i & 1)) * kRows + 16 * warp + g + 8 * (i >> 1)] = fabsf(low[i]) < __uint_as_float(0x7F800000u) ? acc[i] + low[i] : acc[i];
            if (t < p.whole) {
                any_of_consumers(false);
                for (int i = threadIdx.x; i < p.m * kRows; i += kConsumers) {
                    const long long row = (long long)t * kRows + i % kRows;
                    if (row < p.w.rows) {
                        float f = sums[i];
                        if constexpr (FMT == kNvfp4) f *= row_rest(p.w.row_scale[row]);
                        static_cast<T*>(p.y)[i / kRows * p.ldy + row] = from_f32<T>(f);
                    }
                }
                any_of_consumers(false);                 // before the next rows' sums
            }
        }
    }
    __syncwarp();
    if (splits > 1) {                                    // one group of rows a cluster: add up the parts of it
        cluster_sync();
        const long long row0 = (long long)together * kRows;
        for (int i = int(rank) * kThreads + threadIdx.x; together < p.tiles && i < p.m * (kRows / 4); i += int(splits) * kThreads) {
            const long long row = row0 + 4 * (i % (kRows / 4));
            if (row >= p.w.rows) continue;
            float4 part[kMostSplits];
#pragma unroll
            for (uint32_t q = 0; q < kMostSplits; ++q)
                if (q < splits) part[q] = ld_cluster_f32x4(smem_sum + 16 * i, q);
            float4 f = part[0];
#pragma unroll
            for (uint32_t q = 1; q < kMostSplits; ++q)
                if (q < splits) f = make_float4(f.x + part[q].x, f.y + part[q].y, f.z + part[q].z, f.w + part[q].w);
            const float e[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (row + j < p.w.rows) {
                    float one = e[j];
                    if constexpr (FMT == kNvfp4) one *= row_rest(p.w.row_scale[row + j]);
                    static_cast<T*>(p.y)[i / (kRows / 4) * p.ldy + row + j] = from_f32<T>(one);
                }
        }
        cluster_sync();                                  // no CTA ends while another reads its part
    }
}

// x as m * P rows of bf16 with zeros behind column k: the parts of a token one after the other, each the next eight significant bits,
// times 2^8 more than the one before, so that the last bits of the smallest numbers are still bf16 numbers.
template <typename T, int P>
__global__ void __launch_bounds__(256) tcq_ms_parts_kernel(const T* __restrict__ x, long long m, long long k, long long ldx, __nv_bfloat16* __restrict__ out,
                                                           long long width, const unsigned int* __restrict__ wide) {
    if (wide != nullptr && *wide == 0) return;           // the fp16 form has run
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

// Rows of 16-bit numbers with zeros behind column k, for TMA loads that cannot start at them where they lie.
__global__ void __launch_bounds__(256) tcq_ms_pad_kernel(const uint16_t* __restrict__ x, long long m, long long k, long long ldx, uint16_t* __restrict__ out, long long width) {
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x, runs = width / 8;
    if (id >= m * runs) return;
    const long long i = id / runs, c0 = (id - i * runs) * 8;
    uint32_t w[4] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (c0 + j < k) w[j / 2] |= uint32_t(x[i * ldx + c0 + j]) << (16 * (j & 1));
    *reinterpret_cast<uint4*>(out + i * width + c0) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, int FMT, int PARTS>
cudaError_t launch(FewArgs p, cudaStream_t stream) {
    using G = Tile<FMT, PARTS, 3>;
    const auto three = tcq_ms_linear_few_kernel<T, FMT, PARTS, 3>, two = tcq_ms_linear_few_kernel<T, FMT, PARTS, 2>;
    static std::atomic<bool> ready[64];
    static MostClusters kept;
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev >= 64 || !ready[dev]) {
        for (const auto kernel : {three, two})
            if ((err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem)) != cudaSuccess) return err;
        if (dev < 64) ready[dev] = true;
    }
    CUtensorMap map_w;
    const long long pitch = ms_pitch(p.k);
    if ((err = make_byte_map(&map_w, p.w.codes, pitch, p.w.rows, pitch, kRows)) != cudaSuccess) return err;
    p.wide = reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.ldx * sizeof(T) % 16 == 0;
    p.atoms = ms_tiles_k(p.k) * G::kAtoms;
    p.tiles = int((p.w.rows + kRows - 1) / kRows);
    p.k_tiles = int(ms_tiles_k(p.k));
    // S, a power of two (clusters of three and five run 20 % longer than of two and four), while all CTAs run at once.  us, nvfp4, one token, S = 1 / 2 / 4 / 8:
    // 4096 x 4096 14.2 / 9.1 / 6.8 / 6.5, 4096 x 12288 37.5 / 20.9 / 12.5 / 10.9, 12288 x 4096 14.6 / 12.9
    // (4600 x 4096, which 8 would give more clusters than run at once: 14.6 / 9.3 / 8.8 / 10.6)
    int splits = 1;
    while (splits < kMostSplits && splits * 2 <= p.k_tiles &&
           p.tiles <= ms_most_clusters(kept, reinterpret_cast<const void*>(three), kThreads, G::kSmem, 2, splits * 2)) splits *= 2;
    // One stage less where that makes room for all of x: eight tokens through 40960 x 4096 48.0 -> 41.4 us, 151936 x 4096 132 -> 91.5.
    // More groups of rows than that: all of them whole, in turns of which the last may be a short one; or the last ones shared by clusters again, at once.
    // The cost is counted in turns; a CTA alone on its SM takes 0.55 of one, an
    // exchange 0.15.  (One token: 40960 x 4096 31.2 -> 27.2 us, 40960 x 12288 86.2 -> 72.3.)
    int grid = splits > 1 ? p.tiles * splits : std::min(p.tiles, 2 * ms_sm_count());
    p.whole = splits > 1 ? 0 : p.tiles;
    if (splits == 1 && p.tiles > grid) {
        const auto part = [](int ctas) { return ctas == 0 ? 0.0 : ctas <= ms_sm_count() ? 0.55 : 1.0; };
        double least = p.tiles / grid + part(p.tiles % grid);
        for (int share = 2; share <= 4 && share <= p.k_tiles; share *= 2) {
            const int clusters = ms_most_clusters(kept, reinterpret_cast<const void*>(three), kThreads, G::kSmem, 2, share), ctas = clusters * share;
            const int left = p.tiles % ctas;
            const double cost = p.tiles / ctas + part(left * share) / share + 0.15;
            if (left <= clusters && cost < least) {
                least = cost;
                splits = share;
                grid = ctas;
                p.whole = p.tiles - left;
            }
        }
    }
    const int rows_x = (p.whole ? p.k_tiles : (p.k_tiles + splits - 1) / splits) * PARTS * p.m;
    const auto kernel = rows_x > G::kRowsX && rows_x <= Tile<FMT, PARTS, 2>::kRowsX ? two : three;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(grid));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = G::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = unsigned(splits);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, map_w, p);
}

template <typename T, int PARTS>
cudaError_t launch_fmt(const FewArgs& p, int fmt, cudaStream_t stream) {
    return fmt == kNvfp4 ? launch<T, kNvfp4, PARTS>(p, stream) : launch<T, kMxfp4, PARTS>(p, stream);
}

}  // namespace

// Whether a TMA load can start at the rows of x.
static bool rows_aligned(const void* x, long long ldx) { return reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % 8 == 0; }

// Whether a call needs no scratch: few tokens, or rows that a TMA load can start at, of a type that the weights are numbers of.
bool ms_linear_direct(const void* x, int dtype, long long m, long long ldx, int fmt) {
    return m <= kTokens || (rows_aligned(x, ldx) && (dtype == kBf16 || (dtype == kF16 && fmt == kNvfp4)));
}

// Rows of x, padded or in parts; for fp16 and mxfp4 both, a word, and the largest scale of every row of W.
static size_t row_bytes(long long m, long long k) { return size_t(m) * size_t(ms_tiles_k(k) * kMsTileK) * 2; }
size_t ms_linear_workspace_bytes(long long m, long long n, long long k, int dtype, int fmt) {
    const size_t rows = row_bytes(m, k);
    if (dtype == kF16 && fmt == kMxfp4) return 3 * rows + 256 + (size_t(n) + 127) / 128 * 128;
    return dtype == kF32 ? 3 * rows : rows;
}

cudaError_t launch_ms_linear(const void* x, int dtype, long long m, long long ldx, const MsMatrix& w, long long k, int fmt, void* y,
                             long long ldy, void* ws, unsigned loads, cudaStream_t stream) {
    if (m <= kTokens) {
        const FewArgs p{x, ldx, int(m), false, k, w, 0, 0, 0, 0, y, ldy, loads};
        if (dtype == kF32) return launch_fmt<float, 3>(p, fmt, stream);
        if (dtype == kF16) return launch_fmt<__half, 1>(p, fmt, stream);
        return launch_fmt<__nv_bfloat16, 1>(p, fmt, stream);
    }
    const long long width = ms_tiles_k(k) * kMsTileK;
    const unsigned grid = unsigned((m * (width / 8) + 255) / 256);
    uint8_t* const scratch = static_cast<uint8_t*>(ws);
    ManyCall c{x, ldx, k, m, dtype, w, k, fmt, y, ldy, false, nullptr, nullptr, loads};
    cudaError_t err;
    // fp16 through mxfp4: up to 128 tokens, and while tiles of 64 leave half of the SMs free, two bf16 parts (200 through 1024 x 4096 15.4 us), else fp16
    // weights (23.4; but through 4096 x 12288 52.5 instead of 69.5, 12288 x 4096 39 instead of 53).
    const bool fp16 = dtype == kF16 && (fmt == kNvfp4 || (m > 128 && (w.rows + 127) / 128 * ((m + 63) / 64) * 2 > ms_sm_count()));
    if (dtype == kBf16 || fp16) {
        if (!rows_aligned(x, ldx)) {
            tcq_ms_pad_kernel<<<grid, 256, 0, stream>>>(static_cast<const uint16_t*>(x), m, k, ldx, static_cast<uint16_t*>(ws), width);
            if ((err = cudaGetLastError()) != cudaSuccess) return err;
            c.x = ws;
            c.ldx = c.width = width;
        }
        c.fp16 = fp16;
        if (dtype == kBf16 || fmt == kNvfp4) return launch_ms_linear_many(c, stream);
        // fp16 weights: nvfp4's always are; mxfp4's where no row's scales are further apart than fp16 reaches, which the GPU finds out by itself: one of
        // the two forms behind it runs (8 us of small launches: for many tokens; 1000 through 12288 x 4096 184 -> 88 us).
        c.wide = reinterpret_cast<unsigned int*>(scratch + 3 * row_bytes(m, k));
        c.largest = reinterpret_cast<uint8_t*>(c.wide) + 256;
        if ((err = launch_ms_scale_range(w, k, c.wide, c.largest, stream)) != cudaSuccess) return err;
        if ((err = launch_ms_linear_many(c, stream)) != cudaSuccess) return err;
        c.fp16 = false;
    }
    // x in parts of bf16 numbers
    if (dtype == kF32) {
        c.x = ws;
        tcq_ms_parts_kernel<float, 3><<<grid, 256, 0, stream>>>(static_cast<const float*>(x), m, k, ldx, static_cast<__nv_bfloat16*>(ws), width, nullptr);
    } else {
        c.x = scratch + row_bytes(m, k);
        tcq_ms_parts_kernel<__half, 2><<<grid, 256, 0, stream>>>(static_cast<const __half*>(x), m, k, ldx, reinterpret_cast<__nv_bfloat16*>(scratch + row_bytes(m, k)), width, c.wide);
    }
    if ((err = cudaGetLastError()) != cudaSuccess) return err;
    c.ldx = c.width = width;
    return launch_ms_linear_many(c, stream);
}

}  // namespace tcq
