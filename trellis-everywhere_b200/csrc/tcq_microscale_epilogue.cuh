// What follows a product before its results are rounded: bias, activation (with a gate or without), residual.
#pragma once

#include "tcq_microscale.cuh"

namespace tcq {

enum : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4, kActGeglu = 5, kActSwiglu = 6 };

// y = act(h + bias) + residual in fp32.  Gated: rows 2 j and 2 j + 1 of W are gate and value, y[j] = act(h[2 j]) * h[2 j + 1] + residual[j].
struct Epilogue {
    const void* bias;            // [groups][n], or NULL
    int bias_dtype;
    int act;
    const void* residual;        // [rows][ldr] of y's type, or NULL
    long long ldr;
    void* y;
    int dtype;
    long long ldy;
};

__host__ __device__ constexpr bool act_gated(int act) { return act >= kActGeglu; }

// A call, so that what erf and tanh take of registers and instructions is there once, beside loops that need theirs.
static __device__ __noinline__ float activate(int act, float h) {
    if (act == kActRelu) return h < 0.0f ? 0.0f : h;                              // (NaN stays)
    if (act == kActGelu || act == kActGeglu) return 0.5f * h * (1.0f + erff(h * 0.70710678118654752f));
    if (act == kActGeluTanh) {
        const float t = tanhf(0.79788456080286536f * (h + 0.044715f * h * h * h));
        return 0.5f * h * (1.0f + t);
    }
    if (act == kActSilu || act == kActSwiglu) return h / (1.0f + expf(-h));
    return h;
}

__device__ __forceinline__ float load_as_f32(const void* p, int dtype, long long at) {
    if (dtype == kF32) return __ldg(static_cast<const float*>(p) + at);
    if (dtype == kF16) return __half2float(__ldg(static_cast<const __half*>(p) + at));
    return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p) + at));
}
__device__ __forceinline__ void store_f32(void* p, int dtype, long long at, float v) {
    if (dtype == kF32) static_cast<float*>(p)[at] = v;
    else if (dtype == kF16) static_cast<__half*>(p)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(v);
}

// One result: residual and rounding.  (y may be the residual: read and written by the same thread.)
__device__ __forceinline__ void finish_one(const Epilogue& e, long long row, long long column, float v) {
    if (e.residual != nullptr) {
        const long long at = row * e.ldr + column;
        if (e.dtype == kF32) v += static_cast<const float*>(e.residual)[at];
        else if (e.dtype == kF16) v += __half2float(static_cast<const __half*>(e.residual)[at]);
        else v += __bfloat162float(static_cast<const __nv_bfloat16*>(e.residual)[at]);
    }
    store_f32(e.y, e.dtype, row * e.ldy + column, v);
}

// N rows of results of column r of h, one column a lane (lanes are 32 neighbours, lane 0 an even one); the whole warp.  h: sums with the bias in; there: whether
// column r exists; rows row0 .. row0 + rows - 1 do.
// Gated: neighbours hold gate and value of the same result, so the even lane takes every other row and the odd lane those between.
template <int N>
__device__ __forceinline__ void finish_rows(const Epilogue& e, const float (&h)[N], long long row0, int rows, long long r, bool there) {
    if (!act_gated(e.act)) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (there && i < rows) finish_one(e, row0 + i, r, e.act == kActNone ? h[i] : activate(e.act, h[i]));
    } else {
        const bool odd = r & 1;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float second = i + 1 < N ? h[i + 1 < N ? i + 1 : i] : 0.0f;
            const float got = __shfl_xor_sync(0xFFFFFFFFu, odd ? h[i] : second, 1);
            const float gate = odd ? got : h[i], value = odd ? second : got;
            const int row = i + (odd ? 1 : 0);
            if (there && row < rows && row < N) finish_one(e, row0 + row, r >> 1, activate(e.act, gate) * value);
        }
    }
}

// Four neighbouring columns r .. r + 3 of one row, sums with the bias in; r a multiple of four, `n` columns in all (an even number where gated).
__device__ __forceinline__ void finish_four(const Epilogue& e, const float (&h)[4], long long row, long long r, long long n) {
    if (!act_gated(e.act)) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (r + j < n) finish_one(e, row, r + j, e.act == kActNone ? h[j] : activate(e.act, h[j]));
    } else {
#pragma unroll
        for (int j = 0; j < 4; j += 2)
            if (r + j < n) finish_one(e, row, (r + j) >> 1, activate(e.act, h[j]) * h[j + 1]);
    }
}

}  // namespace tcq
