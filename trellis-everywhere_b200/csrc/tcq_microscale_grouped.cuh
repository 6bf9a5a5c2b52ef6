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

// Scratch; in_order: x is taken row by row (no tokens), aligned as ms_rows_aligned says.
size_t ms_grouped_workspace_bytes(long long rows, long long groups, long long n, long long k, int dtype, int fmt, bool in_order);
cudaError_t launch_ms_grouped(const GroupedCall& c, void* ws, cudaStream_t stream);
inline bool ms_rows_aligned(const void* x, long long ldx) { return reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % 8 == 0; }      // a TMA load can start at the rows of x

// tcq_microscale_grouped_many.cu: weights as 16-bit numbers, for many rows a group and x of a type that the weights are numbers of.  Scratch only for rows that are
// gathered, or that TMA loads cannot start at.
inline bool ms_grouped_many_takes(int dtype, int fmt) { return dtype == kBf16 || (dtype == kF16 && fmt == kNvfp4); }
int ms_grouped_many_rows(long long rows, long long groups, long long n);
size_t ms_grouped_many_workspace_bytes(long long rows, long long k);
cudaError_t launch_ms_grouped_many(const GroupedCall& c, void* ws, cudaStream_t stream);

}  // namespace tcq
