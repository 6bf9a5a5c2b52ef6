// Rows of 16-bit activations in groups, each group times a 4-bit microscaled matrix of its own, few rows a group: y[i] = act(W[g(i)] x[i] + bias) + residual.
//
// The tensor cores multiply 4-bit numbers as they lie in memory, so that a weight costs nothing but its bytes; it is x that is cut up.  With s the power of two of the
// largest magnitude of a block of 16 (nvfp4) or 32 (mxfp4) columns, s <= amax < 2 s, x / s rounded to 21 binary places is a number of eight digits of base 8, each of -4 .. 3, all of which are e2m1
// numbers: x = s (d0 + d1 / 8 + ... + d7 / 8^7).  Each digit is a row of 4-bit numbers with the block scales s, and the product is that of tcgen05.mma with kPartsX columns for each row
// of x, added up at the end with powers of 1 / 8.  Eight digits hold every bit of bf16 numbers down to 2^-14 of their block's largest (fp16: 2^-11) and are off by 2^-22 of that at most elsewhere,
// about what sums in fp32 are.  (With six, 2^-17, 12 and 48 tokens took 1 % less, a layer of 200 6 %, 60 tokens through 12288 x 4096, which products bind, 25 %; and a channel 20000 times the others
// left 2 % of error in results that have no weight for it.)
// nvfp4's scales, of a token as of a matrix, end 2^-17 below the token's largest one: blocks below that have its digits (2^-39 of the token's largest number off at most).  mxfp4's end at 2^-106: numbers
// are off by 2^-128 at least.
//
// Work split: one small kernel finds each row's group and place, cuts it up and leaves it as the stages that the products load (codes swizzled as the tensor cores
// read them, scales in the order of tcgen05.cp).  The other goes through items of 128 rows of a matrix x NT / kPartsX rows of its group, one CTA per SM, and begins
// with the loads of W while the first still runs.  With few items a cluster of S CTAs shares the columns of one, and the partial sums meet through
// distributed shared memory, in rank order.  Where groups begin is read on the GPU; the host knows how many rows there are, and chooses by their mean.
//
// A wait that runs out (kMbarWaitCycles) makes its CTA stop, and its results from there on NaN, as those of its cluster.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "tcq_microscale_grouped.cuh"
#include "tcq_programmatic.cuh"
#include "tcq_tcgen05.cuh"

namespace tcq {

namespace {

constexpr int kPartsX = 8, kPlaces = 3 * (kPartsX - 1);      // digits, and binary places behind the first
constexpr int kThreads = 192;                    // loader, issuer, four warps for the results
constexpr int kRowsW = 128, kMostSplits = 8;

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

// Eight columns of x from c0 on as they are, zeros behind the last.
template <typename T>
__device__ __forceinline__ uint4 load8(const T* row, long long c0, long long k, bool wide) {
    if (wide && c0 + 8 <= k) return *reinterpret_cast<const uint4*>(row + c0);
    uint32_t w[4] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c0 + i < k) w[i / 2] |= uint32_t(reinterpret_cast<const uint16_t*>(row)[c0 + i]) << (16 * (i & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// Their largest magnitude, as bits of 16; a NaN or an infinity is kInfinite<T> or more.
template <typename T> constexpr uint32_t kInfinite = std::is_same_v<T, __half> ? 0x7C00u : 0x7F80u;
__device__ __forceinline__ uint32_t largest8(const uint4& u) {
    const uint32_t m = __vmaxu2(__vmaxu2(u.x & 0x7FFF7FFFu, u.y & 0x7FFF7FFFu), __vmaxu2(u.z & 0x7FFF7FFFu, u.w & 0x7FFF7FFFu));
    return max(m & 0xFFFFu, m >> 16);
}
// The same of the finite ones.
template <typename T>
__device__ __forceinline__ uint32_t largest_finite8(const uint4& u) {
    uint32_t m = largest8(u);
    if (m >= kInfinite<T>) {                             // (seldom: one by one)
        m = 0;
        for (int i = 0; i < 8; ++i) {
            const uint32_t b = (i < 2 ? u.x : i < 4 ? u.y : i < 6 ? u.z : u.w) >> (16 * (i & 1)) & 0x7FFFu;
            if (b < kInfinite<T>) m = max(m, b);
        }
    }
    return m;
}
// 16 bits of a magnitude as those of the fp32 number.
template <typename T>
__device__ __forceinline__ uint32_t as_f32_bits(uint32_t m) {
    if constexpr (std::is_same_v<T, __half>) return __float_as_uint(__half2float(__ushort_as_half(uint16_t(m))));
    else return m << 16;
}

// Bits of the largest magnitude of v[from .. from + N - 1]; a NaN or an infinity counts as 0x7F800000 and more.
template <int N>
__device__ __forceinline__ uint32_t largest(const float* v) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
}

// The exponent of a number's power of two; denormal numbers have that of the least normal one, or less.
__device__ __forceinline__ int exponent_of(uint32_t bits) { return int(bits >> 23) - 127; }

// A block's scale as an exponent over 2^base: mxfp4's no lower than what numbers can be multiplied by 2^kPlaces over, nvfp4's (base: that of the row's scale) than its least scale.
template <int FMT>
__device__ __forceinline__ int block_exponent(uint32_t amax_bits, int base) { return FMT == kMxfp4 ? max(exponent_of(amax_bits), kPlaces - 127) : max(exponent_of(amax_bits) - base, -9); }
// nvfp4: the exponent of a row's scale, with which the largest block's is 2^8.  (FAR: numbers of fp32's range.)
template <bool FAR>
__device__ __forceinline__ int row_exponent(uint32_t amax_bits) { return max(exponent_of(amax_bits) - 8, FAR ? -126 : -60); }
// Times 2^(kPlaces - e); FAR: in two steps, where e may be below kPlaces - 127 (down to -135: nvfp4, for numbers of fp32's range).
template <bool FAR>
struct Up {
    float a, b;
    __device__ __forceinline__ Up(int e) : a(pow2f(FAR ? (kPlaces - e) / 2 : kPlaces - e)), b(FAR ? pow2f(kPlaces - e - (kPlaces - e) / 2) : 1.0f) {}
    __device__ __forceinline__ float operator()(float v) const { return FAR ? v * a * b : v * a; }
};

// The eight digits of v 2^-kPlaces, |v| < 2^22, as codes: the first in nibble 7.
// An addition rounds to a whole number, another makes digits 0 .. 7 of -4 .. 3; three bits are spread to four, and all eight are looked up as functions of their bits.
__device__ __forceinline__ uint32_t digit_codes(float v) {
    constexpr uint32_t kZero = 4 * ((1u << 24) - 1) / 7;                                     // a digit 4 in every place
    const uint32_t u = __float_as_uint(v + 12582912.0f) - (0x4B400000u - kZero);             // (3 * 2^22, and its bits)
    const uint32_t two = (u & 0x00000FFFu) | ((u << 4) & 0xFFFFF000u), four = (two & 0x003F003Fu) | ((two << 2) & ~0x003F003Fu);
    const uint32_t d = (four & 0x07070707u) | ((four << 1) & ~0x07070707u);
    const uint32_t b1 = d >> 1, b2 = d >> 2;
    const uint32_t c0 = d & ~(b1 ^ b2), c1 = (b2 & ~b1 & d) | (~b2 & ~(b1 ^ d)), c2 = (b2 & b1) | (~b2 & ~(b1 & d));      // 4 3 2 1 0 -1 .. as 6 5 4 2 0 and the sign
    uint32_t r = (c0 & 0x11111111u) | ((c1 << 1) & ~0x11111111u);
    r = (r & 0x33333333u) | ((c2 << 2) & ~0x33333333u);
    return (r & 0x77777777u) | (~(d << 1) & ~0x77777777u);
}
// The codes of two columns side by side: of part 7 - 2 b in byte b of `even`, of part 6 - 2 b in byte b of `odd`.
struct TwoColumns { uint32_t even, odd; };
__device__ __forceinline__ TwoColumns two_columns(float a, float b) {
    const uint32_t x = digit_codes(a), y = digit_codes(b);
    return {(x & 0x0F0F0F0Fu) | ((y << 4) & ~0x0F0F0F0Fu), ((x >> 4) & 0x0F0F0F0Fu) | (y & ~0x0F0F0F0Fu)};
}
__device__ __forceinline__ uint32_t of_part(const TwoColumns& t, int part) { return part & 1 ? t.even : t.odd; }
__host__ __device__ constexpr int byte_of_part(int part) { return (kPartsX - 1 - part) / 2; }

// The byte of the scale of a part.  e: the block's exponent (nvfp4: over the row's scale); nan: the block is not finite.  mxfp4's are a fourth, and those of parts behind the first an eighth of that, so
// that a sum of parts is finite where the result is: a first digit is up to 1.4 times the number, the others up to four.
template <int FMT>
__device__ __forceinline__ uint32_t part_scale(int e, bool nan, int part) {
    if constexpr (FMT == kNvfp4) return nan ? 0x7Fu : f32_to_e4m3(pow2f(e));
    else return nan ? 0xFFu : uint32_t(e + 127 - (part > 0 ? 5 : 2));
}
// A result of its parts' sums, the smallest first.
template <int FMT, typename SumOf>
__device__ __forceinline__ float join_parts(SumOf sum_of) {
    float sum = sum_of(kPartsX - 1);
#pragma unroll
    for (int part = kPartsX - 2; part >= 0; --part) sum = __fmaf_rn(sum, FMT == kMxfp4 && part == 0 ? 1.0f : 0.125f, sum_of(part));
    return FMT == kMxfp4 ? 4.0f * sum : sum;
}

// One CTA takes rows blockIdx.x, blockIdx.x + gridDim.x ...; a thread eight columns at a time (32 of them take a row of 4096 three times as long, and all of many rows no less).
constexpr int kPartsThreads = 512;
template <typename T, int FMT>
__global__ void __launch_bounds__(kPartsThreads) tcq_ms_row_parts_kernel(const __grid_constant__ PartsArgs p) {
    __shared__ GroupPlan plan;
    __shared__ uint32_t most[2][kPartsThreads / 32];
    constexpr int kRun = 8, kLanes = Ms<FMT>::kBlock / kRun;       // lanes that share a block
    wait_for_kernel_before();
    launch_dependents();
    const int runs = p.k_tiles * (kMsTileK / kRun);      // whole warps of them
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    bool planned = false;
    for (int i = blockIdx.x, turn = 0; i < p.groups.rows; i += gridDim.x) {
        const int token = p.tokens != nullptr ? p.tokens[i] : i;
        const bool inside = token >= 0 && token < p.x_rows;
        const T* const row = static_cast<const T*>(p.x) + (inside ? token : 0) * p.ldx;
        uint4 u = {};
        if (int(threadIdx.x) < runs && inside) u = load8(row, (long long)kRun * threadIdx.x, p.k, p.wide);       // on their way while the groups are counted
        if (!planned) {
            if (warp == 0) plan_groups(p.groups, p.per, plan);
            __syncthreads();
            planned = true;
        }
        if (i < plan.begin[0] || i >= plan.begin[p.groups.groups]) continue;     // no group's
        const int g = last_not_above(plan.begin, p.groups.groups, i), at = i - plan.begin[g];
        const int before = at / p.per, tile = plan.tile[g] + before, place = at - before * p.per;
        int base = 0;                                    // nvfp4: exponent of the token's row scale
        if constexpr (FMT == kNvfp4) {
            uint32_t m = largest_finite8<T>(u);
            for (int j = threadIdx.x + blockDim.x; j < runs && inside; j += blockDim.x) m = max(m, largest_finite8<T>(load8(row, (long long)kRun * j, p.k, p.wide)));
            m = __reduce_max_sync(0xFFFFFFFFu, m);
            if (lane == 0) most[turn][warp] = m;         // (two turns of them: who writes these has seen that all have read the ones before)
            __syncthreads();
            for (int q = 0; q < int(blockDim.x) / 32; ++q) m = max(m, most[turn][q]);
            turn ^= 1;
            base = row_exponent<!std::is_same_v<T, __half>>(as_f32_bits<T>(m));
            if (threadIdx.x == 0) p.row_scale[(long long)tile * p.per + place] = pow2f(base);
        }
        uint8_t* const records = p.out + (long long)tile * p.k_tiles * p.record;
        const uint32_t column = place * kPartsX;         // of the tile: the first part's
        for (int j = threadIdx.x; j < runs; j += blockDim.x) {
            if (j != int(threadIdx.x) && inside) u = load8(row, (long long)kRun * j, p.k, p.wide);
            uint32_t m = inside ? largest8(u) : kInfinite<T>;
#pragma unroll
            for (int d = 1; d < kLanes; d *= 2) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
            const bool nan = m >= kInfinite<T>;
            if (nan) u = {};
            const int e = nan ? 0 : block_exponent<FMT>(as_f32_bits<T>(m), base);
            const Up<FMT == kNvfp4 && !std::is_same_v<T, __half>> up(e + base);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
            TwoColumns two[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const T* const pair = reinterpret_cast<const T*>(&w[q]);
                two[q] = two_columns(up(to_f32<T>(pair[0])), up(to_f32<T>(pair[1])));
            }
            uint8_t* const record = records + (j / 32) * p.record;
            const uint32_t jj = j % 32, block = jj / kLanes, from = kBytesScales<FMT> + column * 128 + 4 * (jj & 3);       // of the 256 columns
#pragma unroll
            for (int part = 0; part < kPartsX; ++part) {
                const uint32_t byte = byte_of_part(part), pick = byte | (4 + byte) << 4;
                *reinterpret_cast<uint32_t*>(record + (from + 128 * part + (((jj >> 2) ^ ((column + part) & 7)) << 4))) =
                    __byte_perm(__byte_perm(of_part(two[0], part), of_part(two[1], part), pick), __byte_perm(of_part(two[2], part), of_part(two[3], part), pick), 0x5410);
            }
            // the scales: some parts each of the lanes that share a block
#pragma unroll
            for (int part = lane % kLanes; part < kPartsX; part += kLanes) {
                const uint32_t c = column + part;
                record[(block / 4) * 512 + (c & 31) * 16 + (c >> 5) * 4 + (block & 3)] = uint8_t(part_scale<FMT>(e, nan, part));
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
    static constexpr int kTake = NT <= 8 ? 1 : NT <= 16 ? 2 : 4;              // rows whose columns are taken out of tensor memory together
    static_assert(kRowsX % kTake == 0);
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

// What add_up_parts reads of global memory is on its way while the parts are waited for.
__device__ __forceinline__ void prefetch_parts(const Epilogue& out, const GroupItem& t, long long n, uint32_t rank, uint32_t splits, int threads) {
    const int i = int(rank) * threads + int(threadIdx.x);
    const long long r = (long long)t.tn * kRowsW + i % (kRowsW / 4) * 4;
    if (i >= kRowsW / 4 * t.rows || r >= n) return;
    const auto prefetch = [](const void* base, int dtype, long long at) {
        asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const char*>(base) + at * (dtype == kF32 ? 4 : 2)));
    };
    if (out.bias != nullptr) prefetch(out.bias, out.bias_dtype, (long long)t.group * n + r);
    if (out.residual != nullptr) prefetch(out.residual, out.dtype, (t.row0 + i / (kRowsW / 4)) * out.ldr + (act_gated(out.act) ? r >> 1 : r));
}

// The sums of one item out of the parts that the CTAs of a cluster have in shared memory ([rows][128] at smem_sum of each), in rank order; four neighbours a thread.
__device__ __forceinline__ void add_up_parts(const Epilogue& out, const GroupItem& t, long long n, uint32_t smem_sum, uint32_t rank, uint32_t splits, int threads) {
    for (int i = int(rank) * threads + int(threadIdx.x); i < kRowsW / 4 * t.rows; i += int(splits) * threads) {
        const long long r = (long long)t.tn * kRowsW + i % (kRowsW / 4) * 4;
        if (r >= n) continue;
        float4 part[kMostSplits];
#pragma unroll
        for (uint32_t q = 0; q < kMostSplits; ++q)
            if (q < splits) part[q] = ld_cluster_f32x4(smem_sum + 16 * i, q);
        float4 f = part[0];
#pragma unroll
        for (uint32_t q = 1; q < kMostSplits; ++q)
            if (q < splits) f = make_float4(f.x + part[q].x, f.y + part[q].y, f.z + part[q].z, f.w + part[q].w);
        float h[4] = {f.x, f.y, f.z, f.w};
        if (out.bias != nullptr)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (r + j < n) h[j] += load_as_f32(out.bias, out.bias_dtype, (long long)t.group * n + r + j);
        finish_four(out, h, t.row0 + i / (kRowsW / 4), r, n);
    }
}

// N rows' sums out of tensor memory, from column `from` on: added up and scaled.  fx: the scale of row `lane`.
template <int FMT, int N>
__device__ __forceinline__ void take_rows(uint32_t from, float fx, float inner, float outer, bool ok, float (&h)[N]) {
    uint32_t v[N][kPartsX];
#pragma unroll
    for (int q = 0; q < N; ++q) tmem_load<kPartsX>(from + kPartsX * q, v[q]);
    tmem_wait_ld();
#pragma unroll
    for (int q = 0; q < N; ++q) {
        float sum = join_parts<FMT>([&](int part) { return __uint_as_float(v[q][part]); });
        if constexpr (FMT == kNvfp4) sum = sum * inner * __shfl_sync(0xFFFFFFFFu, fx, q) * outer;
        h[q] = ok ? sum : __uint_as_float(0x7FC00000u);
    }
}

// Bound by latency with few items (8 rows through 4096 x 4096 nvfp4, the kernel before it included, 9.2 us) and by L2 with many (48 tokens to 8 of 64 experts of 4096 x 1024 mxfp4 31.8, the wide
// form 30.4: 4.7 TB/s of weights).
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
    const int first = int(uint32_t(p.k_tiles) * rank / splits), last = int(uint32_t(p.k_tiles) * (rank + 1) / splits);      // (at most 2^16 times 8)
    const int start = blockIdx.x / splits, clusters = gridDim.x / splits;
    const long long atoms = (long long)p.k_tiles * T::kAtoms;
    constexpr long long kRecord = T::kBytesS + NT * 128;

    const auto columns_of = [](const GroupItem& t) { return t.rows * kPartsX; };
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
        wait_for_kernel_before();                        // x's digits are there
        // (the next kernel begins when this one has ended: its warps beside these cost 800 rows of 32 groups of 2000 x 2048 6 %)
        fence_for_bulk_loads();
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
            const float fw = FMT == kNvfp4 && there ? p.w.row_scale[column] : 1.0f;
            const float inner = inner_part(fw), outer = outer_part(fw);
            const float bias = p.out.bias != nullptr && there ? load_as_f32(p.out.bias, p.out.bias_dtype, column) : 0.0f;
            ok = still_waits(ok, smem_u32(&sum_full[buf]), uint32_t(n / 2) & 1, &gave_up);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < t.rows; c += T::kTake) {
                float h[T::kTake];
                take_rows<FMT, T::kTake>(tmem + buf * T::kSumColumns + c * kPartsX + (uint32_t(32 * quarter) << 16),
                                                     FMT == kNvfp4 && lane < T::kTake && c + lane < t.rows ? p.x_row[(long long)t.tile * T::kRowsX + c + lane] : 1.0f, inner, outer, ok, h);
                if (c + T::kTake >= t.rows) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sum_empty[buf]));
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
        if (start < items) prefetch_parts(p.out, item_of(start), p.w.rows, rank, splits, kThreads);
        cluster_sync();
        if (start < items) add_up_parts(p.out, item_of(start), p.w.rows, smem_sum, rank, splits, kThreads);
        cluster_sync_relaxed();                              // no CTA ends while another reads its part
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free(tmem, T::kColumns);
    }
}

// More rows an item than a few, and many items: 256 rows of W an item, two halves of which share a stage's digits of x.  What binds the form above there is what comes out of L2 (9 to 10 TB/s:
// 17 KB of W and as many of x for 524 clocks of products); here x is read half as often.  Of the sums' buffers there are three, a half of an item each.
// (256 tokens to 8 of 64 experts, 2816 x 2048 with SwiGLU: mxfp4 82.5 us in the form above, 70.8 in this one; nvfp4, whose x is read for 14 rows an item where the form above has 16, 86.2 and 88.4, and 64 tokens
// of 4096 x 1024 41.8 and 36.2.)
template <int FMT>
struct WideTile {
    static constexpr int kNt = FMT == kMxfp4 ? 128 : 112, kRowsX = kNt / kPartsX;      // (nvfp4's scales take twice the tensor memory)
    static constexpr int kAtoms = Ms<FMT>::kAtoms, kBytesW = kRowsW * 128, kBytesS = kAtoms * 512;
    static constexpr int kStageBytes = (2 * kBytesW + 3 * kBytesS + kNt * 128 + 1023) / 1024 * 1024, kStages = FMT == kMxfp4 ? 4 : 3;
    static constexpr int kSums = 3, kScaleColumns = kAtoms * 4 * 3;
    static constexpr int kSmem = kStages * kStageBytes + 1024;
    static_assert(kSums * kNt + kStages * kScaleColumns <= 512 && kSmem >= 116 * 1024 && kSmem + sizeof(GroupPlan) + 1024 <= 227 * 1024 && (3 * kBytesS) % 1024 == 0);
    static constexpr int kTake = 4;
    static_assert(kSums * kNt + kTake * kPartsX <= 512);                      // rows behind the last one's, which are taken too, lie within what is allocated
};
constexpr int kWideThreads = 320;                // loader, issuer, four warps for the results of each half

template <int FMT>
__global__ void __launch_bounds__(kWideThreads, 1) tcq_ms_grouped_wide_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ GroupedArgs p) {
    using T = WideTile<FMT>;
    extern __shared__ uint8_t raw[];
    __shared__ GroupPlan plan;
    __shared__ uint64_t full[T::kStages], empty[T::kStages], sum_full[2][T::kSums], sum_empty[T::kSums], drained;
    __shared__ uint32_t tmem_at;
    __shared__ unsigned int gave_up;
    const uint32_t smem = (smem_u32(raw) + 1023) & ~1023u;
    const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
    const long long atoms = (long long)p.k_tiles * T::kAtoms;
    constexpr long long kRecord = T::kBytesS + T::kNt * 128;
    const int tiles_n2 = (p.tiles_n + 1) / 2;

    const auto columns_of = [](const GroupItem& t) { return t.rows * kPartsX; };
    const auto halves_of = [&](const GroupItem& t) { return 2 * t.tn + 1 < p.tiles_n ? 2 : 1; };
    if (warp == 0) {
        if (elect_one()) {
            gave_up = 0;
            for (int s = 0; s < T::kStages; ++s) { mbar_init(smem_u32(&full[s]), 1); mbar_init(smem_u32(&empty[s]), 1); }
            for (int s = 0; s < T::kSums; ++s) { mbar_init(smem_u32(&sum_full[0][s]), 1); mbar_init(smem_u32(&sum_full[1][s]), 1); mbar_init(smem_u32(&sum_empty[s]), 4); }
            mbar_init(smem_u32(&drained), 1);
            asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        plan_groups(p.groups, T::kRowsX, plan);
    }
    if (warp == 1) tmem_alloc(smem_u32(&tmem_at), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at, tmem_scales = tmem + T::kSums * T::kNt;
    const int items = plan.tile[p.groups.groups] * tiles_n2;
    const auto item_of = [&](int i) { return group_item(plan, p.groups.groups, tiles_n2, T::kRowsX, i); };

    if (warp == 0) {
        // ---- loads; the warp stays together, one lane issues
        const bool one = elect_one();
        wait_for_kernel_before();                        // x's digits are there
        fence_for_bulk_loads();
        uint32_t s = 0, phase = 1, loaded = 0;           // (the first wait for a stage is for the phase before the first)
        unsigned left = p.loads;
        bool ok = true;
        for (int i = blockIdx.x; i < items && ok; i += gridDim.x) {
            const GroupItem t = item_of(i);
            const int halves = halves_of(t), columns = columns_of(t);
            const long long scales = ((long long)t.group * p.tiles_n + 2 * t.tn) * atoms;
            for (int kt = 0; kt < p.k_tiles; ++kt) {
                ok = still_waits(left-- > 0, smem_u32(&empty[s]), phase, &gave_up);      // every lane has seen this phase before the next can begin
                if (!ok) break;
                if (one) {
                    const uint32_t to = smem + s * T::kStageBytes, bar = smem_u32(&full[s]), row = uint32_t(t.group * p.w.rows + t.tn * 2 * kRowsW);
                    mbar_expect(bar, halves * (T::kBytesW + T::kBytesS) + T::kBytesS + columns * 128);
                    for (int h = 0; h < halves; ++h) {
                        tma_load(to + h * T::kBytesW, &map_w, kt * 128, int(row + h * kRowsW), bar);
                        bulk_load(to + 2 * T::kBytesW + h * T::kBytesS, p.w.scales + (scales + h * atoms + (long long)kt * T::kAtoms) * 512, T::kBytesS, bar);
                    }
                    bulk_load(to + 2 * T::kBytesW + 2 * T::kBytesS, p.x + ((long long)t.tile * p.k_tiles + kt) * kRecord, T::kBytesS + columns * 128, bar);
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
        int n = 0;                                           // buffers of sums taken so far: two an item, a matrix's last one too, so that each waiter sees each phase of its barriers
        bool ok = true;
        for (int i = blockIdx.x; i < items && ok; i += gridDim.x) {
            const GroupItem t = item_of(i);
            const int halves = halves_of(t);
            const uint32_t idesc0 = kIdesc | uint32_t(columns_of(t) >> 3) << 17;
            uint32_t d[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int buf = (n + h) % T::kSums, use = (n + h) / T::kSums;
                d[h] = tmem + buf * T::kNt;
                if (use > 0) ok = ok && mbar_wait(smem_u32(&sum_empty[buf]), uint32_t(use - 1) & 1, &gave_up);
            }
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            tc_fence_after();
            for (int kt = 0; kt < p.k_tiles; ++kt) {
                ok = mbar_wait(smem_u32(&full[s]), phase, &gave_up);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = smem + s * T::kStageBytes, sw = tmem_scales + s * T::kScaleColumns, sx = sw + 2 * T::kAtoms * 4;
                const uint64_t dw = desc_rows128(at), dx = desc_rows128(at + 2 * T::kBytesW + 3 * T::kBytesS), ds = desc_rows16(at + 2 * T::kBytesW);
                if (one) {
#pragma unroll
                    for (int j = 0; j < T::kAtoms; ++j) tc_copy_scales(sx + 4 * j, ds + (2 * T::kBytesS >> 4) + 32 * j);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (h >= halves) break;
#pragma unroll
                        for (int j = 0; j < T::kAtoms; ++j) tc_copy_scales(sw + h * T::kAtoms * 4 + 4 * j, ds + (h * T::kBytesS >> 4) + 32 * j);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {        // 64 columns: 32 bytes of a row, one word of scales (nvfp4) or half a word (mxfp4)
                            const int atom = FMT == kNvfp4 ? j : j / 2;
                            const uint32_t id = FMT == kNvfp4 ? 0u : 2u * (j % 2);
                            mma_block_scaled<FMT>(d[h], dw + (h * T::kBytesW >> 4) + 2 * j, dx + 2 * j, idesc0 | id << 4 | id << 29, sw + h * T::kAtoms * 4 + 4 * atom, sx + 4 * atom, kt > 0 || j > 0);
                        }
                    }
                    tc_commit(smem_u32(&empty[s]));
                }
                __syncwarp();
                if (++s == T::kStages) { s = 0; phase ^= 1; }
            }
            if (ok && one)
                for (int h = 0; h < 2; ++h) tc_commit(smem_u32(&sum_full[h][(n + h) % T::kSums]));
            __syncwarp();
            n += 2;
        }
        if (!ok) {                                           // what was issued ends before the tensor memory goes
            if (one) tc_commit(smem_u32(&drained));
            __syncwarp();
            for (long long t0 = clock64(); !mbar_try_wait(smem_u32(&drained), 0) && clock64() - t0 < kMbarWaitCycles;) {}
        }
    } else {
        // ---- results of one half: this warp's lanes are 32 rows of W, so that a store is 32 neighbours in y
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        wait_for_kernel_before();                            // rows' scales
        bool ok = true;
        for (int i = blockIdx.x, n = 0; i < items; i += gridDim.x, ++n) {
            const GroupItem t = item_of(i);
            const int buf = (2 * n + half) % T::kSums;       // (of each half, every third item: 0, 2, 1 and 1, 0, 2)
            const long long r = (2ll * t.tn + half) * kRowsW + 32 * quarter + lane, column = (long long)t.group * p.w.rows + r;
            const bool there = r < p.w.rows;
            const float fw = FMT == kNvfp4 && there ? p.w.row_scale[column] : 1.0f;
            const float inner = inner_part(fw), outer = outer_part(fw);
            const float bias = p.out.bias != nullptr && there ? load_as_f32(p.out.bias, p.out.bias_dtype, column) : 0.0f;
            ok = still_waits(ok, smem_u32(&sum_full[half][buf]), uint32_t(n / T::kSums) & 1, &gave_up);
            tc_fence_after();
            const uint32_t from = tmem + buf * T::kNt + (uint32_t(32 * quarter) << 16);
#pragma unroll 1
            for (int c = 0; c < t.rows; c += T::kTake) {
                float h[T::kTake];
                take_rows<FMT, T::kTake>(from + c * kPartsX, FMT == kNvfp4 && lane < T::kTake && c + lane < t.rows ? p.x_row[(long long)t.tile * T::kRowsX + c + lane] : 1.0f,
                                                     inner, outer, ok, h);
                if (c + T::kTake >= t.rows) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sum_empty[buf]));
                }
#pragma unroll
                for (int q = 0; q < T::kTake; ++q) h[q] += bias;
                finish_rows(p.out, h, t.row0 + c, t.rows - c, r, there);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free(tmem, 512);
    }
}

// One or two rows an item, cut up by the CTA that multiplies them: one launch, and x goes from global memory to what the tensor cores read without a way round.  What a CTA's columns of x
// become stays in shared memory while its items are of the same rows.  Bound by latency: one row through 4096 x 4096 nvfp4 7.0 us, one token to 8 of 64 experts of 2048 x 2048 7.6 (2.5 TB/s of weights).
template <int FMT, int NT>
struct FewTile {
    static constexpr int kAtoms = Ms<FMT>::kAtoms, kRowsX = NT / kPartsX;
    static constexpr int kBytesW = kRowsW * 128, kBytesS = kAtoms * 512, kStageBytes = (kBytesW + kBytesS + 1023) / 1024 * 1024, kMostStages = 10;
    static constexpr int kRecord = (kBytesS + NT * 128 + 1023) / 1024 * 1024;
    static constexpr int kSumColumns = 32, kScaleColumns = kAtoms * 4 * 2;   // scales in tensor memory: of one stage
    static constexpr int kColumns = 512;
    static constexpr int kBytesSum = kRowsX * kRowsW * 4;
    // What x leaves is stages of W, four at least: with few columns all of them are on their way at once (eight experts of 2048 x 2048, six stages 9.7 us).
    static constexpr int kSmem = 206 * 1024, kRoom = (kSmem - 1024 - kBytesSum) / 1024 * 1024, kHeld = (kRoom - 4 * kStageBytes) / kRecord;      // pieces of 256 columns of x
    static constexpr int stages(int held) { return std::min(kMostStages, (kRoom - held * kRecord) / kStageBytes); }
    static_assert(2 * kSumColumns + kMostStages * kScaleColumns <= kColumns && NT <= 16 && stages(kHeld) >= 4);
};
constexpr int kFewWarps = 10, kFewThreads = 32 * kFewWarps, kCutters = 8;        // loader, issuer, eight that cut x up, four of which take the results

struct FewArgs {
    const void* x;
    long long x_rows, ldx;
    const int* tokens;
    bool wide;                                   // x in pieces of 16 bytes
    MsMatrix w;
    Groups groups;
    long long k;
    int tiles_n, k_tiles;
    int held, stages;                            // pieces of x that a CTA has room for, and stages of W
    Epilogue out;
    unsigned loads;
};

template <typename XT, int FMT, int NT>
__global__ void __launch_bounds__(kFewThreads, 1) tcq_ms_grouped_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ FewArgs p) {
    using T = FewTile<FMT, NT>;
    extern __shared__ uint8_t raw[];
    __shared__ GroupPlan plan;
    __shared__ uint64_t full[T::kMostStages], empty[T::kMostStages], sum_full[2], sum_empty[2], x_there, drained;
    __shared__ uint32_t tmem_at, most[2][T::kRowsX][kCutters];
    __shared__ unsigned int gave_up;
    const uint32_t stages = p.stages, smem_x = (smem_u32(raw) + 1023) & ~1023u, smem = smem_x + p.held * T::kRecord, smem_sum = smem_x + T::kRoom;
    float* const sums = reinterpret_cast<float*>(raw + (smem_sum - smem_u32(raw)));
    const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), splits = cluster_size();
    const int first = int(uint32_t(p.k_tiles) * rank / splits), last = int(uint32_t(p.k_tiles) * (rank + 1) / splits);      // (at most 2^16 times 8)
    const int start = blockIdx.x / splits, clusters = gridDim.x / splits;
    const long long atoms = (long long)p.k_tiles * T::kAtoms;

    const auto load = [&](uint32_t s, const GroupItem& t, int kt) {
        const uint32_t to = smem + s * T::kStageBytes, bar = smem_u32(&full[s]);
        mbar_expect(bar, T::kBytesW + T::kBytesS);
        tma_load(to, &map_w, kt * 128, int(t.group * p.w.rows + t.tn * kRowsW), bar);
        bulk_load(to + T::kBytesW, p.w.scales + (((long long)t.group * p.tiles_n + t.tn) * atoms + (long long)kt * T::kAtoms) * 512, T::kBytesS, bar);
    };
    const int runs = (last - first) * 64;                // of four columns of a row that this CTA has: whole warps
    constexpr int kRun = 4, kRuns = 4, kApart = 32 * kCutters;                    // a thread takes four of them at a time, kApart apart: their loads are in flight together
    // Four columns of x's row `token` (one that x has not: NaN), zeros behind the last column.  Loads stay where they stand.
    const auto fetch = [&](int token, int j, float (&v)[kRun]) {
        const int q = j >= runs ? 1 : 0;
        const long long c0 = (long long)first * kMsTileK + 4 * (j - q * runs);
        const XT* const from = static_cast<const XT*>(p.x) + token * p.ldx + c0;
        if (token < 0 || token >= p.x_rows) {
            v[0] = v[1] = v[2] = v[3] = __uint_as_float(0x7FC00000u);
        } else if (p.wide && c0 + 4 <= p.k) {
            uint2 u;
            asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(u.x), "=r"(u.y) : "l"(from) : "memory");
#pragma unroll
            for (int h = 0; h < 4; ++h) v[h] = to_f32<XT>(reinterpret_cast<const XT*>(&u)[h]);
        } else {
#pragma unroll
            for (int h = 0; h < 4; ++h) v[h] = c0 + h < p.k ? to_f32<XT>(from[h]) : 0.0f;
        }
    };
    if (warp == 0 && elect_one()) {
        gave_up = 0;
        for (uint32_t s = 0; s < stages; ++s) { mbar_init(smem_u32(&full[s]), 1); mbar_init(smem_u32(&empty[s]), 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(smem_u32(&sum_full[s]), 1); mbar_init(smem_u32(&sum_empty[s]), kCutters); }
        mbar_init(smem_u32(&x_there), kCutters);
        mbar_init(smem_u32(&drained), 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    if (warp == 1) tmem_alloc(smem_u32(&tmem_at), T::kColumns);
    wait_for_kernel_before();
    launch_dependents();
    float v[kRuns][kRun];
    int token[T::kRowsX] = {}, ahead = 0;                // x's rows of the item's rows; of all rows, a lane one, where there are no more than lanes
    if (p.tokens != nullptr && lane < p.groups.rows && p.groups.rows <= 32) asm volatile("ld.global.u32 %0, [%1];" : "=r"(ahead) : "l"(p.tokens + lane) : "memory");
    const auto fetch_tokens = [&](int row0, int rows) {
#pragma unroll
        for (int q = 0; q < T::kRowsX; ++q) {
            const int known = __shfl_sync(0xFFFFFFFFu, ahead, (row0 + q) & 31);
            token[q] = p.tokens == nullptr ? row0 + q : p.groups.rows <= 32 ? known : q < rows ? p.tokens[row0 + q] : 0;
        }
    };
    const auto fetch_all = [&](int j0, int all) {
#pragma unroll
        for (int u = 0; u < kRuns; ++u)
            if (j0 + u * kApart < all) fetch(token[j0 + u * kApart >= runs ? T::kRowsX - 1 : 0], j0 + u * kApart, v[u]);
    };
    // x is on its way before it is known whose rows they are: of one group, or with one row an item and a first group that begins with the first row, the
    // item's rows are these.
    const int guess = start / p.tiles_n * T::kRowsX, guessed = p.groups.offsets == nullptr ? min(p.groups.rows, T::kRowsX) : 1;
    const bool early = (p.groups.offsets == nullptr || T::kRowsX == 1) && guess < p.groups.rows;
    if (early && warp >= 2) {
        fetch_tokens(guess, guessed);
        fetch_all(int(threadIdx.x) - 64, guessed * runs);
    }
    if (warp == 0) plan_groups(p.groups, T::kRowsX, plan);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at, tmem_scales = tmem + 2 * T::kSumColumns;
    const int items = plan.tile[p.groups.groups] * p.tiles_n;
    const auto item_of = [&](int i) { return group_item(plan, p.groups.groups, p.tiles_n, T::kRowsX, i); };

    if (warp == 0) {
        // ---- loads; the warp stays together, one lane issues
        const bool one = elect_one();
        fence_for_bulk_loads();
        uint32_t s = 0, phase = 1, loaded = 0;           // (the first wait for a stage is for the phase before the first)
        unsigned left = p.loads;
        bool ok = true;
        for (int i = start; i < items && ok; i += clusters) {
            const GroupItem t = item_of(i);
            for (int kt = first; kt < last; ++kt) {
                ok = still_waits(left-- > 0, smem_u32(&empty[s]), phase, &gave_up);      // every lane has seen this phase before the next can begin
                if (!ok) break;
                if (one) load(s, t, kt);
                __syncwarp();
                if (++s == stages) { s = 0; phase ^= 1; }
                if (loaded < stages) ++loaded;
            }
        }
        wait_for_loads(full, stages, s, phase, loaded);
    } else if (warp == 1) {
        // ---- products; likewise
        constexpr uint32_t kIdesc = 1u << 7 | 1u << 10 | (FMT == kMxfp4 ? 1u : 0u) << 23 | 1u << 27;
        const bool one = elect_one();
        uint32_t s = 0, phase = 0;
        int n = 0, tile = -1, cut = 0;                       // rows of x that are there; how often x has been cut up
        bool ok = true;
        for (int i = start; i < items && ok; i += clusters, ++n) {
            const GroupItem t = item_of(i);
            const uint32_t idesc0 = kIdesc | uint32_t(t.rows * kPartsX / 8) << 17;
            const int buf = n & 1;
            if (n >= 2) ok = mbar_wait(smem_u32(&sum_empty[buf]), uint32_t(n / 2 - 1) & 1, &gave_up);
            if (t.tile != tile) {
                ok = ok && mbar_wait(smem_u32(&x_there), uint32_t(cut) & 1, &gave_up);
                ++cut;
                tile = t.tile;
            }
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tmem + buf * T::kSumColumns;
            for (int kt = first; kt < last; ++kt) {
                ok = mbar_wait(smem_u32(&full[s]), phase, &gave_up);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = smem + s * T::kStageBytes, x = smem_x + (kt - first) * T::kRecord, sw = tmem_scales + s * T::kScaleColumns, sx = sw + T::kAtoms * 4;
                const uint64_t dw = desc_rows128(at), dx = desc_rows128(x), ds = desc_rows16(at + T::kBytesW), dsx = desc_rows16(x + NT * 128);
                if (one) {
#pragma unroll
                    for (int j = 0; j < T::kAtoms; ++j) {
                        tc_copy_scales(sw + 4 * j, ds + 32 * j);
                        tc_copy_scales(sx + 4 * j, dsx + 32 * j);
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
                if (++s == stages) { s = 0; phase ^= 1; }
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
        // ---- x, by all eight warps, four columns a thread; results, by the first four: lanes are 32 rows of W, so that a store is 32 neighbours in y
        constexpr int kLanes = Ms<FMT>::kBlock / kRun;                            // that share a block
        const int id = threadIdx.x - 64, quarter = warp & 3;
        const bool takes = warp < 6;
        float fx[T::kRowsX];
        int n = 0, tile = -1, cut = 0;
        bool ok = true;
        for (int i = start; i < items; i += clusters, ++n) {
            const GroupItem t = item_of(i);
            const int buf = n & 1;
            if (t.tile != tile) {
                tile = t.tile;                               // (every warp here has waited for the sums of the item before: its x is no longer read)
                const int all = t.rows * runs;
                int base[T::kRowsX] = {};                    // nvfp4: exponent of the scale of this CTA's columns of each row
                if (i != start || !early || t.row0 != guess) {
                    fetch_tokens(t.row0, t.rows);
                    fetch_all(id, all);
                }
                if constexpr (FMT == kNvfp4) {
                    uint32_t m[T::kRowsX] = {};              // the largest finite magnitudes
#pragma unroll 1
                    for (int j0 = id; j0 < all; j0 += kRuns * kApart) {
                        if (j0 != id) fetch_all(j0, all);
#pragma unroll
                        for (int u = 0; u < kRuns; ++u) {
                            const int j = j0 + u * kApart;
                            uint32_t r = 0;
#pragma unroll
                            for (int h = 0; h < kRun; ++h) {
                                const uint32_t b = __float_as_uint(v[u][h]) & 0x7FFFFFFFu;
                                r = max(r, b < 0x7F800000u ? b : 0u);
                            }
#pragma unroll
                            for (int q = 0; q < T::kRowsX; ++q)
                                if (j >= q * runs && j < min(all, (q + 1) * runs)) m[q] = max(m[q], r);
                        }
                    }
                    if (all > kRuns * kApart) fetch_all(id, all);
#pragma unroll
                    for (int q = 0; q < T::kRowsX; ++q) {
                        m[q] = __reduce_max_sync(0xFFFFFFFFu, m[q]);
                        if (lane == 0) most[cut & 1][q][warp - 2] = m[q];        // (two turns of them: who writes these has seen that all have read the ones before)
                    }
                    asm volatile("bar.sync 1, %0;" ::"n"(kApart) : "memory");
#pragma unroll
                    for (int q = 0; q < T::kRowsX; ++q) {
#pragma unroll
                        for (int h = 0; h < kCutters; ++h) m[q] = max(m[q], most[cut & 1][q][h]);
                        base[q] = row_exponent<!std::is_same_v<XT, __half>>(m[q]);
                        fx[q] = pow2f(base[q]);
                    }
                }
                ++cut;
                // (as little code as there may be: a small call is over before code that is run once has been fetched)
#pragma unroll 1
                for (int j0 = id; j0 < all; j0 += kRuns * kApart) {
                    if (j0 != id) fetch_all(j0, all);
#pragma unroll 1
                    for (int u = 0; u < kRuns; ++u) {
                        const int j = j0 + u * kApart, q = j >= runs ? 1 : 0, run = j - q * runs;
                        if (j >= all) break;
                        uint32_t m = largest<kRun>(v[0]);
#pragma unroll
                        for (int d = 1; d < kLanes; d *= 2) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
                        const bool nan = m >= 0x7F800000u;
                        const int of_row = q ? base[T::kRowsX - 1] : base[0], from = nan ? 0 : block_exponent<FMT>(m, of_row), block = (run & 63) / kLanes;
                        const Up<FMT == kNvfp4 && !std::is_same_v<XT, __half>> up(from + of_row);
                        const TwoColumns lo = two_columns(nan ? 0.0f : up(v[0][0]), nan ? 0.0f : up(v[0][1])), hi = two_columns(nan ? 0.0f : up(v[0][2]), nan ? 0.0f : up(v[0][3]));
                        const uint32_t record = smem_x + run / 64 * T::kRecord + q * kPartsX * 128 + 2 * (run & 7), turn = (run & 63) >> 3;
#pragma unroll
                        for (int part = 0; part < kPartsX; ++part) {
                            const int byte = byte_of_part(part);
                            const uint32_t codes = __byte_perm(of_part(lo, part), of_part(hi, part), byte | (4 + byte) << 4);
                            asm volatile("st.shared.u16 [%0], %1;" ::"r"(record + part * 128 + (((turn ^ (q * kPartsX + part)) & 7) << 4)), "h"(uint16_t(codes)) : "memory");
                        }
                        // the scales: a part or two each of the lanes that share a block
                        const uint32_t scales = smem_x + run / 64 * T::kRecord + NT * 128 + q * kPartsX * 16 + (block / 4) * 512 + (block & 3);
#pragma unroll
                        for (int part = lane % kLanes; part < kPartsX; part += kLanes)
                            asm volatile("st.shared.u8 [%0], %1;" ::"r"(scales + part * 16), "r"(part_scale<FMT>(from, nan, part)) : "memory");
#pragma unroll
                        for (int h = 0; h + 1 < kRuns; ++h)
#pragma unroll
                            for (int f = 0; f < kRun; ++f) v[h][f] = v[h + 1][f];     // the next run's
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&x_there));
            }
            if (!takes) {
                // (an arrival of its own: the phase after the next of this barrier would answer this wait like the one before it, so it may not begin before this warp has seen its own)
                ok = still_waits(ok, smem_u32(&sum_full[buf]), uint32_t(n / 2) & 1, &gave_up);
                if (lane == 0) mbar_arrive(smem_u32(&sum_empty[buf]));
                continue;
            }
            const long long r = (long long)t.tn * kRowsW + 32 * quarter + lane;
            const bool there = r < p.w.rows;
            const long long column = (long long)t.group * p.w.rows + r;
            const float fw = FMT == kNvfp4 && there ? p.w.row_scale[column] : 1.0f;
            const float bias = p.out.bias != nullptr && there ? load_as_f32(p.out.bias, p.out.bias_dtype, column) : 0.0f;
            ok = still_waits(ok, smem_u32(&sum_full[buf]), uint32_t(n / 2) & 1, &gave_up);
            tc_fence_after();
            uint32_t sum_of[NT];
            tmem_load<NT>(tmem + buf * T::kSumColumns + (uint32_t(32 * quarter) << 16), sum_of);
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sum_empty[buf]));
            float h[T::kRowsX];
#pragma unroll
            for (int q = 0; q < T::kRowsX; ++q) {
                float sum = join_parts<FMT>([&](int part) { return __uint_as_float(sum_of[q * kPartsX + part]); });
                if constexpr (FMT == kNvfp4) sum = sum * inner_part(fw) * fx[q] * outer_part(fw);
                h[q] = ok ? sum : __uint_as_float(0x7FC00000u);
                if (splits > 1) sums[q * kRowsW + 32 * quarter + lane] = h[q];
                else h[q] += bias;
            }
            if (splits == 1) finish_rows(p.out, h, t.row0, t.rows, r, there);
        }
    }
    __syncwarp();
    if (splits > 1) {                                        // one item a cluster: add up the parts of it, four neighbours a thread
        if (start < items) prefetch_parts(p.out, item_of(start), p.w.rows, rank, splits, kFewThreads);
        cluster_sync();
        if (start < items) add_up_parts(p.out, item_of(start), p.w.rows, smem_sum, rank, splits, kFewThreads);
        cluster_sync_relaxed();                              // no CTA ends while another reads its part
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free(tmem, T::kColumns);
    }
}

// Columns of sums for the rows of x of one item: what holds all rows of one group, or three times the mean of the groups that may have rows (a group that needs a second item reads its
// matrix again: 256 rows of 64 groups, 4096 x 1024 mxfp4, with one and a half times the mean 30.7 us, with three times 28.2).
int columns_for(long long rows, long long groups) {
    const long long filled = std::min(rows, groups);
    for (int nt : {8, 16, 32, 64})
        if (2 * (nt / kPartsX) * filled >= (groups > 1 && rows > groups ? 6 : 2) * rows) return nt;
    return 128;
}

// The rows' scales, then the records, in the scratch.
size_t parts_bytes(long long rows, long long groups, long long k, int fmt, int nt) {
    const int per = nt / kPartsX;
    const long long tiles = most_tiles(rows, groups, per);
    return size_t((tiles * per * 4 + 255) / 256 * 256) + size_t(tiles) * size_t(ms_tiles_k(k)) * record_bytes(fmt, nt);
}
template <int FMT>
cudaError_t launch_parts(const GroupedCall& c, int nt, void* ws, uint8_t** records, cudaStream_t stream) {
    const int per = nt / kPartsX, k_tiles = int(ms_tiles_k(c.k));
    *records = static_cast<uint8_t*>(ws) + (most_tiles(c.groups.rows, c.groups.groups, per) * per * 4 + 255) / 256 * 256;
    const PartsArgs p{c.x, c.x_rows, c.ldx, c.tokens, c.groups, c.k, k_tiles, per, (long long)record_bytes(FMT, nt), ms_rows_aligned(c.x, c.ldx), *records, static_cast<float*>(ws)};
    // Threads of a row: all of its runs at once while there are few rows; fewer where many rows fill the SMs, since what a row takes of every thread (its group and place, its largest
    // number) is as much as eight columns do (8192 rows through 128 x 2048: 256 threads 58.4 us, 64 55.5).
    const int rows = c.groups.rows, sms = ms_sm_count();
    const int threads = std::min(rows <= sms ? 512 : rows <= 4 * sms ? 256 : rows <= 16 * sms ? 128 : 64, p.k_tiles * 32);
    const unsigned grid = unsigned(std::min<long long>(rows, sms * 1536ll / threads));
    return launch_programmatic(c.dtype == kF16 ? tcq_ms_row_parts_kernel<__half, FMT> : tcq_ms_row_parts_kernel<__nv_bfloat16, FMT>, dim3(grid), dim3(threads), 0, 0, stream, p);
}

// How many CTAs share the columns of an item: as many as leave each an SM of its own, and two pieces of 256 columns or more.
int splits_for(MostClusters& kept, const void* kernel, int threads, size_t smem, long long items, int k_tiles) {
    int splits = 1;
    while (splits < kMostSplits && splits * 4 <= k_tiles && items <= ms_most_clusters(kept, kernel, threads, smem, 1, splits * 2)) splits *= 2;
    return splits;
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
    uint8_t* records;
    if ((err = launch_parts<FMT>(c, NT, ws, &records, stream)) != cudaSuccess) return err;
    const GroupedArgs p{c.w, c.groups, int((n + kRowsW - 1) / kRowsW), k_tiles, records, static_cast<const float*>(ws), c.out, c.loads};
    const long long items = tiles * p.tiles_n;
    const int splits = splits_for(kept, reinterpret_cast<const void*>(kernel), kThreads, T::kSmem, items, k_tiles);
    // (begins beside the kernel that makes the digits, and waits for it where it needs them)
    return launch_programmatic(kernel, dim3(unsigned(splits > 1 ? items * splits : std::min<long long>(items, ms_sm_count()))), dim3(kThreads), T::kSmem, splits, stream, map_w, p);
}

template <int FMT>
cudaError_t launch_wide(const GroupedCall& c, void* ws, cudaStream_t stream) {
    using T = WideTile<FMT>;
    const auto kernel = tcq_ms_grouped_wide_kernel<FMT>;
    static std::atomic<bool> ready[64];
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
    uint8_t* records;
    if ((err = launch_parts<FMT>(c, T::kNt, ws, &records, stream)) != cudaSuccess) return err;
    const GroupedArgs p{c.w, c.groups, int((n + kRowsW - 1) / kRowsW), int(ms_tiles_k(c.k)), records, static_cast<const float*>(ws), c.out, c.loads};
    const long long items = most_tiles(c.groups.rows, c.groups.groups, T::kRowsX) * ((p.tiles_n + 1) / 2);
    return launch_programmatic(kernel, dim3(unsigned(std::min<long long>(items, ms_sm_count()))), dim3(kWideThreads), T::kSmem, 0, stream, map_w, p);
}

template <typename XT, int FMT, int NT>
cudaError_t launch_few(const GroupedCall& c, cudaStream_t stream) {
    using T = FewTile<FMT, NT>;
    const auto kernel = tcq_ms_grouped_few_kernel<XT, FMT, NT>;
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
    FewArgs p{c.x, c.x_rows, c.ldx, c.tokens, ms_rows_aligned(c.x, c.ldx), c.w, c.groups, c.k, int((n + kRowsW - 1) / kRowsW), int(ms_tiles_k(c.k)), 0, 0, c.out, c.loads};
    const long long items = most_tiles(c.groups.rows, c.groups.groups, T::kRowsX) * p.tiles_n;
    const int splits = splits_for(kept, reinterpret_cast<const void*>(kernel), kFewThreads, T::kSmem, items, p.k_tiles);
    p.held = (p.k_tiles + splits - 1) / splits;
    p.stages = T::stages(p.held);
    return launch_programmatic(kernel, dim3(unsigned(splits > 1 ? items * splits : std::min<long long>(items, ms_sm_count()))), dim3(kFewThreads), T::kSmem, splits, stream, map_w, p);
}

// Whether items of 256 rows of W take fewer of the SMs' turns: one such is as long as 1.75 of 128 rows.  (200 tokens to 4 of 32 experts, 2000 x 2048 mxfp4: 640 items and 29.2 us; 1280 and
// 32.0.  60 rows through 12288 x 4096 nvfp4: 240 items of 14 rows, two turns, 22.4 us; 384 of 16 rows, three turns, 20.0.  By the rule 42 such calls were 3 % slower than the other form at most.)
bool wide_items(long long rows, long long groups, long long n, int fmt) {
    if (columns_for(rows, groups) != 128) return false;
    const long long sms = ms_sm_count(), wide_nt = fmt == kNvfp4 ? WideTile<kNvfp4>::kNt : WideTile<kMxfp4>::kNt;
    const long long wide = most_tiles(rows, groups, wide_nt / kPartsX) * ((n + 255) / 256), narrow = most_tiles(rows, groups, 128 / kPartsX) * ((n + 127) / 128);
    return 7 * ((wide + sms - 1) / sms) <= 4 * ((narrow + sms - 1) / sms);
}

// Whether x is cut up where it is multiplied: one or two rows an item, its columns held by a CTA whatever the split, and few enough items, or only those of the same rows.
bool cut_in_place(long long rows, long long groups, long long n, long long k, int fmt) {
    const int nt = columns_for(rows, groups);
    if (nt > 16) return false;
    const int per = nt / kPartsX, held = fmt == kNvfp4 ? (nt == 8 ? FewTile<kNvfp4, 8>::kHeld : FewTile<kNvfp4, 16>::kHeld) : (nt == 8 ? FewTile<kMxfp4, 8>::kHeld : FewTile<kMxfp4, 16>::kHeld);
    return ms_tiles_k(k) <= held && (rows <= per || most_tiles(rows, groups, per) * ((n + kRowsW - 1) / kRowsW) <= 2 * ms_sm_count());
}

template <int FMT>
cudaError_t launch_cut(const GroupedCall& c, cudaStream_t stream) {
    const bool eight = columns_for(c.groups.rows, c.groups.groups) == 8;
    if (c.dtype == kF16) return eight ? launch_few<__half, FMT, 8>(c, stream) : launch_few<__half, FMT, 16>(c, stream);
    return eight ? launch_few<__nv_bfloat16, FMT, 8>(c, stream) : launch_few<__nv_bfloat16, FMT, 16>(c, stream);
}

template <int FMT>
cudaError_t launch_nt(const GroupedCall& c, void* ws, cudaStream_t stream) {
    if (wide_items(c.groups.rows, c.groups.groups, c.w.rows, FMT)) return launch_wide<FMT>(c, ws, stream);
    switch (columns_for(c.groups.rows, c.groups.groups)) {
        case 8: return launch<FMT, 8>(c, ws, stream);
        case 16: return launch<FMT, 16>(c, ws, stream);
        case 32: return launch<FMT, 32>(c, ws, stream);
        case 64: return launch<FMT, 64>(c, ws, stream);
        default: return launch<FMT, 128>(c, ws, stream);
    }
}

}  // namespace

// Whether weights as 16-bit numbers pay: they are made once for up to 256 rows, where digits take eight columns a row, and are made anew for each row.  Both forms' estimated times, us, fitted to
// measured ones of 40 to 18000 rows (63 pairs, off by 15 %; the form chosen is 0.3 % slower than the faster one on average, 14 % at most): with 16-bit weights 0.35 a step of 64 columns and
// 0.025 a row of x; with digits 0.13 (mxfp4) or 0.17 a step of 256 columns, 1.9 an item and 3.2 a million numbers of x.  (50 rows a group, 2816 x 2048: 125 and 128 in nvfp4, 117 and 102 in
// mxfp4; 64 rows: 126 and 161, 122 and 125; 100 rows through 4096 x 4096 mxfp4: 23 and 13.)  A call whose rows are put in order first takes 2 longer, but the same form.
static bool many_rows(long long rows, long long groups, long long n, long long k, int dtype, int fmt) {
    if (!ms_grouped_many_takes(dtype, fmt) || rows <= 32 * std::min(groups, rows)) return false;
    const double filled = double(std::min(groups, rows)), sms = ms_sm_count(), across = double((n + kRowsW - 1) / kRowsW);
    const auto turns = [&](int per) {
        if (groups == 1) return std::ceil(double((rows + per - 1) / per) * across / sms);
        const double items = std::max(filled, double(rows) / per + 0.5 * filled) * across / sms;
        return items <= 1 ? 1.0 : items + 0.5;
    };
    const int per = ms_grouped_many_rows(rows, groups, n);
    const double many = 4.0 + turns(per) * (0.35 * double((k + 63) / 64) + 0.025 * std::min(double(per), double(rows) / filled));
    const double step = fmt == kNvfp4 ? 0.17 : wide_items(rows, groups, n, fmt) ? 0.11 : 0.13;
    const double digits = 5.5 + turns(columns_for(rows, groups) / kPartsX) * (step * double(ms_tiles_k(k)) + 1.9) + 3.2e-6 * double(rows) * double(k);
    return many < digits;
}

size_t ms_grouped_workspace_bytes(long long rows, long long groups, long long n, long long k, int dtype, int fmt, bool in_order) {
    if (many_rows(rows, groups, n, k, dtype, fmt)) return in_order ? 0 : ms_grouped_many_workspace_bytes(rows, k);
    if (cut_in_place(rows, groups, n, k, fmt)) return 0;
    const int wide = fmt == kNvfp4 ? WideTile<kNvfp4>::kNt : WideTile<kMxfp4>::kNt;
    return parts_bytes(rows, groups, k, fmt, wide_items(rows, groups, n, fmt) ? wide : columns_for(rows, groups));
}

cudaError_t launch_ms_grouped(const GroupedCall& c, void* ws, cudaStream_t stream) {
    if (many_rows(c.groups.rows, c.groups.groups, c.w.rows, c.k, c.dtype, c.fmt)) return launch_ms_grouped_many(c, ws, stream);
    if (cut_in_place(c.groups.rows, c.groups.groups, c.w.rows, c.k, c.fmt)) return c.fmt == kNvfp4 ? launch_cut<kNvfp4>(c, stream) : launch_cut<kMxfp4>(c, stream);
    return c.fmt == kNvfp4 ? launch_nt<kNvfp4>(c, ws, stream) : launch_nt<kMxfp4>(c, ws, stream);
}

}  // namespace tcq
