// Products of rows in groups with 4-bit matrices, one matrix a group, and their epilogue.
#pragma once

#include "tcq_microscale_epilogue.cuh"
#include "tcq_microscale_groups.cuh"

namespace tcq {

struct GroupedCall {
    const void* x;               // [x_rows][ldx] of type dtype, k columns
    int dtype;
    long long x_rows, ldx;
    const int* tokens;           // row i of the product is row tokens[i] of x (one outside x: NaN); NULL: row i
    Groups groups;
    MsMatrix w;                  // rows: n of one matrix; matrix g's codes begin at row g * n, its scales at tile g * ceil(n / 128) of 128 rows
    long long k;
    int fmt;
    Epilogue out;
    unsigned loads;              // stages that a CTA loads, at most (a self-test's limit)
};

size_t ms_grouped_workspace_bytes(long long rows, long long groups, long long n, long long k, int dtype, int fmt);
cudaError_t launch_ms_grouped(const GroupedCall& c, void* ws, cudaStream_t stream);

}  // namespace tcq
