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

// N activations at once: one branch for all of them.  Tails keep their relative precision, down to where the results are denormal numbers: the exponential is of -|h|, so that
// what is divided by lies between 1 and 2 (where the fast quotient is within 2 ulp) and nothing overflows, and GELU takes erfc, not 1 + erf, which cancels.  What is left is the rounding of the
// functions' arguments, which grows with |h|: 2 |h| ulp of GELU's tanh form, h^2 ulp of the other.
__device__ __forceinline__ float sigmoid(float h) {
    const float t = expf(-fabsf(h));
    return __fdividef(h < 0.0f ? t : 1.0f, 1.0f + t);
}
template <int N>
__device__ __forceinline__ void activate(int act, float (&h)[N]) {
    if (act == kActRelu) {
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] = h[i] < 0.0f ? 0.0f : h[i];             // (NaN stays)
    } else if (act == kActSilu || act == kActSwiglu) {
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] *= sigmoid(h[i]);
    } else if (act == kActGeluTanh) {                                             // (1 + tanh z) / 2 = sigmoid(2 z)
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] *= sigmoid(1.5957691216057308f * __fmaf_rn(0.044715f * h[i] * h[i], h[i], h[i]));
    } else if (act == kActGelu || act == kActGeglu) {
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] *= 0.5f * erfcf(h[i] * -0.70710678118654752f);
    }
}

__device__ __forceinline__ float load_as_f32(const void* p, int dtype, long long at) {
    if (dtype == kF32) return static_cast<const float*>(p)[at];
    if (dtype == kF16) return __half2float(static_cast<const __half*>(p)[at]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
}
// N results of one column, in rows row, row + step ...: residual, rounding, stores.  (y may be the residual: read and written by the same thread.)
template <typename YT, int N>
__device__ __forceinline__ void store_rows_as(const Epilogue& e, float (&v)[N], long long row, int step, int rows, long long column) {
    YT* to = static_cast<YT*>(e.y) + row * e.ldy + column;
    const long long apart = step * e.ldy;
    if (e.residual != nullptr) {
        const YT* from = static_cast<const YT*>(e.residual) + row * e.ldr + column;
        YT r[N];
#pragma unroll
        for (int i = 0; i < N; ++i, from += step * e.ldr)
            if (i < rows) r[i] = *from;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += to_f32<YT>(r[i]);
    }
    if (rows >= N) {
#pragma unroll
        for (int i = 0; i < N; ++i, to += apart) *to = from_f32<YT>(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i, to += apart)
            if (i < rows) *to = from_f32<YT>(v[i]);
    }
}
template <int N>
__device__ __forceinline__ void store_rows(const Epilogue& e, float (&v)[N], long long row, int step, int rows, long long column) {
    if (e.dtype == kBf16) store_rows_as<__nv_bfloat16>(e, v, row, step, rows, column);
    else if (e.dtype == kF16) store_rows_as<__half>(e, v, row, step, rows, column);
    else store_rows_as<float>(e, v, row, step, rows, column);
}

// N rows of results of column r of h, one column a lane (lanes are 32 neighbours, lane 0 an even one); the whole warp.  h: sums with the bias in; there: whether
// column r exists; rows row0 .. row0 + rows - 1 do.
// Gated: neighbours hold gate and value of the same result, so the even lane takes every other row and the odd lane those between.
template <int N>
__device__ __forceinline__ void finish_rows(const Epilogue& e, float (&h)[N], long long row0, int rows, long long r, bool there) {
    if (!act_gated(e.act)) {
        activate(e.act, h);
        store_rows(e, h, row0, 1, there ? rows : 0, r);
    } else {
        constexpr int kPairs = (N + 1) / 2;
        const bool odd = r & 1;
        float gate[kPairs], value[kPairs];
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float second = i + 1 < N ? h[i + 1 < N ? i + 1 : i] : 0.0f;
            const float got = __shfl_xor_sync(0xFFFFFFFFu, odd ? h[i] : second, 1);
            gate[i / 2] = odd ? got : h[i];
            value[i / 2] = odd ? second : got;
        }
        activate(e.act, gate);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) gate[i] *= value[i];
        store_rows(e, gate, row0 + odd, 2, there ? (min(rows, N) + 1 - odd) / 2 : 0, r >> 1);
    }
}

// Four neighbouring columns r .. r + 3 of one row, sums with the bias in; r a multiple of four, `n` columns in all (an even number where gated).
__device__ __forceinline__ void finish_four(const Epilogue& e, float (&h)[4], long long row, long long r, long long n) {
    if (!act_gated(e.act)) {
        activate(e.act, h);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float one[1] = {h[j]};
            if (r + j < n) store_rows(e, one, row, 1, 1, r + j);
        }
    } else {
        float gate[2] = {h[0], h[2]};
        activate(e.act, gate);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float one[1] = {gate[j] * h[2 * j + 1]};
            if (r + 2 * j < n) store_rows(e, one, row, 1, 1, (r >> 1) + j);
        }
    }
}

}  // namespace tcq
