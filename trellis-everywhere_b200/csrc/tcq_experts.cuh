// Mixtures of experts around the products: which experts a token goes to and in what order, its results added up; and an epilogue by itself.
#pragma once

#include "tcq_microscale_epilogue.cuh"

namespace tcq {

constexpr int kMostExperts = 1024, kMostChosen = 32;

enum : int { kScoreSoftmax = 0, kScoreSigmoid = 1 };

struct RouteCall {
    const void* logits;          // [tokens][ld] of type dtype
    int dtype;
    long long ld;
    int tokens, experts, top;
    int score;
    bool normalize;
    float* weights;              // [tokens][top]
    int* chosen;                 // [tokens][top], -1: none
    int* places;                 // [tokens][top], -1: none
    int* order;                  // [tokens * top]: the token of each row, -1 behind the last
    int* offsets;                // [experts + 1]
    int* counts;                 // scratch: [route_chunks(tokens)][experts], where there is more than one
};
int route_chunks(int tokens);
cudaError_t launch_route(const RouteCall& c, cudaStream_t stream);

struct CombineCall {
    const void* y;               // [rows][ldy] of type dtype
    int dtype;
    long long rows, ldy, n;
    const float* weights;        // [tokens][top]
    const int* places;
    long long tokens;
    int top;
    const void* residual;        // [tokens][ldr] of out's type, or NULL
    long long ldr;
    void* out;
    int out_dtype;
    long long ldo;
};
cudaError_t launch_combine(const CombineCall& c, cudaStream_t stream);

// y = act(h + bias) + residual of fp32 sums h [rows][n].
cudaError_t launch_epilogue(const float* h, long long rows, long long n, const Epilogue& e, cudaStream_t stream);

}  // namespace tcq
