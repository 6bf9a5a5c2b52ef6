// Products of many tokens with a 4-bit matrix, as tcq_microscale_linear.cu asks for them.
#pragma once

#include "tcq_microscale.cuh"

namespace tcq {

struct ManyCall {
    const void* x;               // the parts of m tokens (1 for bf16, 2 for fp16, 3 for fp32) as rows of bf16, or m rows of fp16, 16-byte aligned, `width` columns of them (the others zero)
    long long ldx, width;
    long long m;
    int dtype;                   // of y
    MsMatrix w;
    long long k;
    int fmt;
    void* y;
    long long ldy;
    bool fp16;                   // x and weights as fp16 numbers; mxfp4's weights times 2^13 over the row's largest scale
    unsigned int* wide;          // mxfp4: whether some row's scales are too far apart for that, which decides on the GPU which form runs; or NULL
    uint8_t* largest;            // mxfp4, fp16: the byte of the largest scale of every row
    unsigned loads;              // stages of W that a CTA loads, at most
};

cudaError_t launch_ms_linear_many(const ManyCall& c, cudaStream_t stream);
// *wide: whether some row of an mxfp4 matrix has a block with a value other than zero whose scale is less than 2^-36 of the row's largest.
cudaError_t launch_ms_scale_range(const MsMatrix& w, long long k, unsigned int* wide, uint8_t* largest, cudaStream_t stream);

}  // namespace tcq
