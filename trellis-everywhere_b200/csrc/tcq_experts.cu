// Mixtures of experts around the products: routing, and the sum of a token's results.
//
// Routing: a warp chooses a token's experts, a round of two warp reductions each: the largest logit (as an integer of the same order), then the lowest number that has it.
// The rows are put in order of experts by counting: how many tokens before, by chunks of tokens, then by warps of a chunk, then within 32 neighbours; so
// rows of one expert keep the order of their tokens, whatever runs first.  Up to kOneChunk tokens are one CTA's and one launch; more take two.
// Bound by latency: one token of 128 experts 4.1 us, 5000 of 61 9.3.
//
// The sum: a thread has eight columns of one token, and the loads of four of its rows are in flight together.  Bound by memory: 4000 tokens of four rows of 2048 columns in fp16 15.8 us, 5.2 TB/s; by
// latency where rows begin anywhere, 2035 columns 27 us: neither memory (2.1 TB/s) nor issue (53 % of its slots) is full.
#include <algorithm>
#include <type_traits>

#include "tcq_experts.cuh"
#include "tcq_programmatic.cuh"

namespace tcq {

namespace {

constexpr int kOneChunk = 32;                    // tokens of the form that is one launch: one a warp
constexpr int kMostChunks = 148;
constexpr int kWarps = 32, kThreads = 32 * kWarps;
constexpr int kFewEntries = 128;                 // that one warp puts in order in less time than all count

// Integers in the order of the numbers: -0 as 0, every NaN above infinity; 0 stands for -infinity, which is never chosen.
__device__ __forceinline__ uint32_t ordered(float v) {
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t b = __float_as_uint(v + 0.0f);
    return v == -INFINITY ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float number_of(uint32_t key) { return __uint_as_float(key == 0xFFFFFFFFu ? 0x7FC00000u : key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }
__device__ __forceinline__ float sum_of_warp(float v) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
    return v;
}

// One token by one warp; lane l has logits l, l + 32 ...; EACH: of them.
template <int EACH>
__device__ void choose(const RouteCall& c, int token) {
    const int lane = threadIdx.x & 31;
    const long long row = token * c.ld;
    uint32_t key[EACH];
    float v[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int e = lane + 32 * i;
        v[i] = e < c.experts ? load_as_f32(c.logits, c.dtype, row + e) : -INFINITY;
        key[i] = ordered(v[i]);
    }
    float value = 0.0f;                                  // lane j: the j-th chosen
    int expert = -1, found = 0;
    for (int j = 0; j < c.top; ++j) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) best = max(best, key[i]);
        best = __reduce_max_sync(0xFFFFFFFFu, best);
        if (best == 0) break;                            // nothing is left
        uint32_t at = 0xFFFFFFFFu;
#pragma unroll
        for (int i = EACH - 1; i >= 0; --i)
            if (key[i] == best) at = lane + 32 * i;
        at = __reduce_min_sync(0xFFFFFFFFu, at);
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            if (at == uint32_t(lane + 32 * i)) key[i] = 0;
        if (lane == j) {
            value = number_of(best);
            expert = int(at);
        }
        ++found;
    }
    float w;
    if (c.score == kScoreSoftmax) {
        const float most = __shfl_sync(0xFFFFFFFFu, value, 0);
        w = lane < found ? expf(value - most) : 0.0f;
        float sum = 0.0f;
        if (c.normalize) {
            sum = w;
        } else {
#pragma unroll
            for (int i = 0; i < EACH; ++i)
                if (found > 0 && v[i] != -INFINITY) sum += expf(v[i] - most);
        }
        sum = sum_of_warp(sum);
        w = lane < found ? w / sum : 0.0f;
    } else {
        // (below zero a sigmoid is e^v / (1 + e^v); where they are normalised, all of them over e^most where that is below 1, so that nothing underflows that a quotient of two would show)
        const float most = __shfl_sync(0xFFFFFFFFu, value, 0), over = c.normalize && most < 0.0f ? most : 0.0f;
        w = lane >= found ? 0.0f : (value < 0.0f ? expf(value - over) : 1.0f) / (1.0f + expf(-fabsf(value)));
        if (c.normalize) {
            const float sum = sum_of_warp(w);
            w = lane < found ? w / sum : 0.0f;
        }
    }
    if (lane < c.top) {
        c.weights[(long long)token * c.top + lane] = w;
        c.chosen[(long long)token * c.top + lane] = expert;
    }
}
__device__ __forceinline__ void choose_any(const RouteCall& c, int token) {
    if (c.experts <= 64) choose<2>(c, token);
    else if (c.experts <= 128) choose<4>(c, token);
    else if (c.experts <= 256) choose<8>(c, token);
    else choose<32>(c, token);
}

// The chunk's rows in order: `mine`, the chunk's first entry; offsets of experts and counts of the chunks before are in base[].
// hist: [kWarps][experts] in shared memory.
__device__ void place_chunk(const RouteCall& c, long long first, int entries, const int* base, int* hist) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = ((entries + kWarps - 1) / kWarps + 31) / 32 * 32, from = warp * per, to = min(entries, from + per);
    for (int i = threadIdx.x; i < kWarps * c.experts; i += kThreads) hist[i] = 0;
    __syncthreads();
    for (int i = from + lane; i < to; i += 32) {
        const int e = c.chosen[first + i];
        if (e >= 0) atomicAdd(&hist[warp * c.experts + e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < c.experts; e += kThreads) {
        int sum = base[e];
        for (int w = 0; w < kWarps; ++w) {
            const int mine = hist[w * c.experts + e];
            hist[w * c.experts + e] = sum;
            sum += mine;
        }
    }
    __syncthreads();
    for (int i = from; i < to; i += 32) {
        const int e = i + lane < to ? c.chosen[first + i + lane] : -1;
        const unsigned same = __match_any_sync(0xFFFFFFFFu, e);
        int place = -1;
        if (e >= 0) place = hist[warp * c.experts + e] + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (e >= 0 && (same & ((1u << lane) - 1)) == 0) hist[warp * c.experts + e] += __popc(same);
        __syncwarp();
        if (i + lane < to) {
            c.places[first + i + lane] = place;
            if (place >= 0) c.order[place] = int(uint32_t(first + i + lane) / uint32_t(c.top));
        }
    }
}

// The same of few entries, by one warp: base[] counts on.
__device__ void place_few(const RouteCall& c, long long first, int entries, int* base) {
    const int lane = threadIdx.x & 31;
    int all[kFewEntries / 32];                           // loads in flight together
#pragma unroll
    for (int u = 0; u < kFewEntries / 32; ++u) all[u] = 32 * u + lane < entries ? c.chosen[first + 32 * u + lane] : -1;
#pragma unroll
    for (int u = 0; u < kFewEntries / 32; ++u) {
        if (32 * u >= entries) break;
        const int e = all[u], i = 32 * u + lane;
        const unsigned same = __match_any_sync(0xFFFFFFFFu, e), before = same & ((1u << lane) - 1);
        const int place = e >= 0 ? base[e] + __popc(before) : -1;
        __syncwarp();
        if (e >= 0 && before == 0) base[e] += __popc(same);
        __syncwarp();
        if (i < entries) {
            c.places[first + i] = place;
            if (place >= 0) c.order[place] = int(uint32_t(first + i) / uint32_t(c.top));
        }
    }
}

// base[e] from counts in it to where experts begin, by one warp; the end of all.
__device__ int scan_experts(int experts, int* base) {
    const int lane = threadIdx.x & 31;
    int sum = 0;
    for (int at = 0; at < experts; at += 32) {
        const int mine = at + lane < experts ? base[at + lane] : 0;
        int v = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int other = __shfl_up_sync(0xFFFFFFFFu, v, d);
            if (lane >= d) v += other;
        }
        if (at + lane < experts) base[at + lane] = sum + v - mine;
        sum += __shfl_sync(0xFFFFFFFFu, v, 31);
    }
    return sum;
}

// All of few tokens.
__global__ void __launch_bounds__(kThreads) tcq_route_kernel(const __grid_constant__ RouteCall c) {
    extern __shared__ int hist[];
    __shared__ int base[kMostExperts];
    const int warp = threadIdx.x >> 5, entries = c.tokens * c.top;
    wait_for_kernel_before();
    launch_dependents();
    for (int e = threadIdx.x; e < c.experts; e += kThreads) base[e] = 0;
    for (int t = warp; t < c.tokens; t += kWarps) choose_any(c, t);
    __syncthreads();
    for (int i = threadIdx.x; i < entries; i += kThreads) {
        const int e = c.chosen[i];
        if (e >= 0) atomicAdd(&base[e], 1);
    }
    __syncthreads();
    if (warp == 0) {
        const int end = scan_experts(c.experts, base);
        if (threadIdx.x == 0) c.offsets[c.experts] = end;
        for (int i = end + int(threadIdx.x); i < entries; i += 32) c.order[i] = -1;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < c.experts; e += kThreads) c.offsets[e] = base[e];
    if (entries <= kFewEntries) {
        __syncthreads();                                 // offsets are read before base[] counts on
        if (warp == 0) place_few(c, 0, entries, base);
    } else {
        place_chunk(c, 0, entries, base, hist);
    }
}

// (up to 2^31 - 1 tokens, where the end of a chunk may pass what an int holds)
__device__ __forceinline__ int end_of_chunk(const RouteCall& c, int t0, int chunk) { return int(min(uint32_t(c.tokens), uint32_t(t0) + uint32_t(chunk))); }

// A chunk of many: its experts, and how many of each.
__global__ void __launch_bounds__(kThreads) tcq_route_choose_kernel(const __grid_constant__ RouteCall c, int chunk) {
    __shared__ int count[kMostExperts];
    wait_for_kernel_before();
    launch_dependents();
    const int warp = threadIdx.x >> 5, t0 = blockIdx.x * chunk, t1 = end_of_chunk(c, t0, chunk);
    for (int e = threadIdx.x; e < c.experts; e += kThreads) count[e] = 0;
    for (uint32_t t = t0 + warp; t < uint32_t(t1); t += kWarps) choose_any(c, int(t));
    __syncthreads();
    for (uint32_t i = t0 * c.top + threadIdx.x; i < uint32_t(t1 * c.top); i += kThreads) {      // (of up to 2^31 - 1)
        const int e = c.chosen[i];
        if (e >= 0) atomicAdd(&count[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < c.experts; e += kThreads) c.counts[(long long)blockIdx.x * c.experts + e] = count[e];
}

// The chunk's rows in order, from the counts of all chunks.
__global__ void __launch_bounds__(kThreads) tcq_route_place_kernel(const __grid_constant__ RouteCall c, int chunk) {
    extern __shared__ int hist[];
    __shared__ int base[kMostExperts], before[kMostExperts];
    wait_for_kernel_before();
    launch_dependents();
    const int warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e < c.experts; e += kThreads) base[e] = before[e] = 0;
    __syncthreads();
    // neighbouring threads take neighbouring experts, groups of threads a share of the chunks each
    const int wide = min(kThreads, (c.experts + 31) / 32 * 32), groups = kThreads / wide, group = threadIdx.x / wide;
    for (int e = threadIdx.x % wide; e < c.experts && group < groups; e += wide) {
        int all = 0, lower = 0;
#pragma unroll 8
        for (int q = group; q < int(gridDim.x); q += groups) {
            const int n = c.counts[(long long)q * c.experts + e];
            all += n;
            if (q < int(blockIdx.x)) lower += n;
        }
        atomicAdd(&base[e], all);
        atomicAdd(&before[e], lower);
    }
    __syncthreads();
    if (warp == 0) {
        const int end = scan_experts(c.experts, base);
        if (blockIdx.x == 0) {
            if (threadIdx.x == 0) c.offsets[c.experts] = end;
            for (int e = threadIdx.x; e < c.experts; e += 32) c.offsets[e] = base[e];
        }
        // the rows that nobody has, a share each
        for (long long i = end + (long long)blockIdx.x * 32 + threadIdx.x; i < (long long)c.tokens * c.top; i += 32ll * gridDim.x) c.order[i] = -1;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < c.experts; e += kThreads) base[e] += before[e];
    __syncthreads();
    const int t0 = blockIdx.x * chunk, t1 = end_of_chunk(c, t0, chunk), entries = (t1 - t0) * c.top;
    if (entries > kFewEntries) place_chunk(c, (long long)t0 * c.top, entries, base, hist);
    else if (warp == 0) place_few(c, (long long)t0 * c.top, entries, base);
}

// Eight neighbouring numbers as they lie in memory.
template <typename T> struct Eight { uint4 u[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ void to_floats(const Eight<T>& e, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(reinterpret_cast<const T*>(e.u)[i]);
}
__device__ __forceinline__ void load_if(bool there, const void* p, uint4& u) {       // without a branch, so that loads behind it are in flight with it
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\t@p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
                 : "+r"(u.x), "+r"(u.y), "+r"(u.z), "+r"(u.w) : "l"(p), "r"(uint32_t(there)) : "memory");
}
template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T* p) {
    Eight<T> e;
#pragma unroll
    for (int q = 0; q < int(sizeof(T) / 2); ++q) e.u[q] = reinterpret_cast<const uint4*>(p)[q];
    return e;
}
// Eight numbers at any address: pieces of 16 bytes that start on 16 bytes, one more than they fill, and a shift; single numbers where fewer than eight exist, or in
// the first and the last row (`inner` is false), where a piece could reach out of the matrix.
template <typename T>
struct EightAt {
    static constexpr int kPieces = sizeof(T) / 2 + 1;
    const T* p;
    uint4 u[kPieces];
    bool whole;
    __device__ __forceinline__ void load(const T* at, bool some, int there, bool inner) {
        p = at;
        whole = some && there >= 8 && inner;
        const char* const base = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(at) & ~uintptr_t(15));
#pragma unroll
        for (int q = 0; q < kPieces; ++q) {
            u[q] = make_uint4(0, 0, 0, 0);
            load_if(whole, base + 16 * q, u[q]);
        }
    }
    __device__ __forceinline__ Eight<T> get(bool some, int there) const {
        Eight<T> e;
        if (whole || !some) {
            const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(p)) & 15u;
            uint32_t w[4 * kPieces];
#pragma unroll
            for (int q = 0; q < kPieces; ++q) { w[4 * q] = u[q].x; w[4 * q + 1] = u[q].y; w[4 * q + 2] = u[q].z; w[4 * q + 3] = u[q].w; }
#pragma unroll
            for (int step = 2; step >= 1; --step)
#pragma unroll
                for (int i = 0; i + step < 4 * kPieces; ++i) w[i] = off & (4 * step) ? w[i + step] : w[i];
#pragma unroll
            for (int i = 0; i + 1 < 4 * kPieces; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 8 * (off & 3));
#pragma unroll
            for (int q = 0; q + 1 < kPieces; ++q) e.u[q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(e.u)[i] = i < there ? p[i] : from_f32<T>(0.0f);
        }
        return e;
    }
};

// Y: of the rows, O: of what comes out.  Threads in x: eight columns of a token each; in y: tokens.  ALIGNED: all rows start on 16 bytes, and n is a multiple of eight.
template <typename Y, typename O, bool ALIGNED>
__global__ void __launch_bounds__(256, 3) tcq_combine_kernel(const __grid_constant__ CombineCall c) {
    __shared__ uint4 turn[ALIGNED ? 1 : 8][ALIGNED ? 1 : 32 * (sizeof(O) / 2)];      // results of a warp, which stores neighbours
    const uint32_t n = uint32_t(c.n);                    // less than 2^31, and columns of the last turn may pass that
    const int lane = threadIdx.x & 31;
    wait_for_kernel_before();
    launch_dependents();
    const long long stride = (long long)gridDim.x * blockDim.y;
    for (long long token = (long long)blockIdx.x * blockDim.y + threadIdx.y; token < c.tokens; token += stride) {
        const int* const places = c.places + token * c.top;
        const float* const weights = c.weights + token * c.top;
        for (uint32_t c0 = 8 * threadIdx.x; c0 - 8 * lane < n; c0 += 8 * blockDim.x) {     // (whole warps stay together)
            const int there = int(n - c0);
            float out[8] = {};
            const bool add = c.residual != nullptr && there > 0;
            const O* const from = static_cast<const O*>(c.residual) + token * c.ldr + c0;
            using Residual = std::conditional_t<ALIGNED, Eight<O>, EightAt<O>>;
            using Row = std::conditional_t<ALIGNED, Eight<Y>, EightAt<Y>>;
            Residual res;
            if constexpr (ALIGNED) {
                if (add) res = load_eight<O>(from);
            } else {
                res.load(from, add, there, token > 0 && token + 1 < c.tokens);
            }
            for (int j0 = 0; j0 < c.top; j0 += 4) {
                Row v[4];
                float w[4];
                int place[4];
                bool some[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) place[q] = j0 + q < c.top ? places[j0 + q] : -1;      // (before the first row: loads that stay where they stand hold up those behind them)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    some[q] = place[q] >= 0 && place[q] < c.rows && there > 0;
                    w[q] = some[q] ? weights[j0 + q] : 0.0f;
                    const Y* const row = static_cast<const Y*>(c.y) + place[q] * c.ldy + c0;
                    if constexpr (ALIGNED) {
                        v[q] = {};
                        if (some[q]) v[q] = load_eight<Y>(row);
                    } else {
                        v[q].load(row, some[q], there, place[q] > 0 && place[q] + 1 < c.rows);
                    }
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float f[8];
                    if constexpr (ALIGNED) to_floats(v[q], f);
                    else to_floats(v[q].get(some[q], there), f);
#pragma unroll
                    for (int i = 0; i < 8; ++i) out[i] = __fmaf_rn(f[i], w[q], out[i]);
                }
            }
            if (add) {
                float f[8];
                if constexpr (ALIGNED) to_floats(res, f);
                else to_floats(res.get(add, there), f);
#pragma unroll
                for (int i = 0; i < 8; ++i) out[i] += f[i];
            }
            Eight<O> r;
#pragma unroll
            for (int i = 0; i < 8; ++i) reinterpret_cast<O*>(r.u)[i] = from_f32<O>(out[i]);
            O* const to = static_cast<O*>(c.out) + token * c.ldo + c0;
            if constexpr (ALIGNED) {
                if (there > 0)
#pragma unroll
                    for (int q = 0; q < int(sizeof(O) / 2); ++q) reinterpret_cast<uint4*>(to)[q] = r.u[q];
            } else {
                uint4* const mine = turn[threadIdx.y * (blockDim.x / 32) + threadIdx.x / 32];
#pragma unroll
                for (int q = 0; q < int(sizeof(O) / 2); ++q) mine[lane * (sizeof(O) / 2) + q] = r.u[q];
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c0 - 8 * lane + lane + 32 * i < n) to[lane + 32 * i - 8 * lane] = reinterpret_cast<const O*>(mine)[lane + 32 * i];
                __syncwarp();
            }
        }
    }
}

template <typename Y, typename O>
cudaError_t combine(const CombineCall& c, cudaStream_t stream) {
    const auto rows_of_16 = [](const void* p, long long ld, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * bytes % 16 == 0; };
    const bool aligned = c.n % 8 == 0 && rows_of_16(c.y, c.ldy, sizeof(Y)) && rows_of_16(c.out, c.ldo, sizeof(O)) &&
                         (c.residual == nullptr || rows_of_16(c.residual, c.ldr, sizeof(O)));
    const long long runs = (c.n + 7) / 8;
    dim3 block(32, 8);
    while (block.x < 256 && block.x < runs) { block.x *= 2; block.y /= 2; }
    const unsigned grid = unsigned(std::min<long long>((c.tokens + block.y - 1) / block.y, 1 << 20));
    return launch_programmatic(aligned ? tcq_combine_kernel<Y, O, true> : tcq_combine_kernel<Y, O, false>, dim3(grid), block, 0, 0, stream, c);
}
template <typename Y>
cudaError_t combine_to(const CombineCall& c, cudaStream_t stream) {
    if (c.out_dtype == kF32) return combine<Y, float>(c, stream);
    return c.out_dtype == kF16 ? combine<Y, __half>(c, stream) : combine<Y, __nv_bfloat16>(c, stream);
}

__global__ void __launch_bounds__(256) tcq_epilogue_kernel(const float* h, long long rows, long long n, const __grid_constant__ Epilogue e) {
    wait_for_kernel_before();
    launch_dependents();
    const long long fours = (n + 3) / 4, id = (long long)blockIdx.x * 256 + threadIdx.x, row = id / fours, r = (id - row * fours) * 4;
    if (row >= rows) return;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = r + j < n ? h[row * n + r + j] : 0.0f;
        if (e.bias != nullptr && r + j < n) v[j] += load_as_f32(e.bias, e.bias_dtype, r + j);
    }
    finish_four(e, v, row, r, n);
}

}  // namespace

static int tokens_of_chunk(int tokens) { return std::max(32, int((tokens + (kMostChunks - 1ll)) / kMostChunks)); }
int route_chunks(int tokens) {
    if (tokens <= kOneChunk) return 1;
    const int chunk = tokens_of_chunk(tokens);
    return int((tokens + (chunk - 1ll)) / chunk);
}

cudaError_t launch_route(const RouteCall& c, cudaStream_t stream) {
    const int chunks = route_chunks(c.tokens), smem = kWarps * c.experts * int(sizeof(int));
    static std::atomic<bool> ready[64];
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev >= 64 || !ready[dev]) {
        for (const void* kernel : {reinterpret_cast<const void*>(tcq_route_kernel), reinterpret_cast<const void*>(tcq_route_place_kernel)})
            if ((err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kWarps * kMostExperts * int(sizeof(int)))) != cudaSuccess) return err;
        if (dev < 64) ready[dev] = true;
    }
    if (chunks == 1) {
        return launch_programmatic(tcq_route_kernel, dim3(1), dim3(kThreads), smem, 0, stream, c);
    }
    const int chunk = tokens_of_chunk(c.tokens);
    if ((err = launch_programmatic(tcq_route_choose_kernel, dim3(unsigned(chunks)), dim3(kThreads), 0, 0, stream, c, chunk)) != cudaSuccess) return err;
    return launch_programmatic(tcq_route_place_kernel, dim3(unsigned(chunks)), dim3(kThreads), size_t(smem), 0, stream, c, chunk);
}

cudaError_t launch_combine(const CombineCall& c, cudaStream_t stream) {
    if (c.dtype == kF32) return combine_to<float>(c, stream);
    return c.dtype == kF16 ? combine_to<__half>(c, stream) : combine_to<__nv_bfloat16>(c, stream);
}

cudaError_t launch_epilogue(const float* h, long long rows, long long n, const Epilogue& e, cudaStream_t stream) {
    const long long blocks = (rows * ((n + 3) / 4) + 255) / 256;
    if (blocks > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    return launch_programmatic(tcq_epilogue_kernel, dim3(unsigned(blocks)), dim3(256), 0, 0, stream, h, rows, n, e);
}

}  // namespace tcq
