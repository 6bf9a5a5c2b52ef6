// Rows in groups, each times a matrix of its own: where groups begin, and how tiles of their rows are counted.
#pragma once

#include "tcq_microscale.cuh"

namespace tcq {

constexpr int kMostGroups = 1024;

struct Groups {
    const int* offsets;          // [groups + 1] on the device: rows offsets[g] .. offsets[g + 1] - 1 are group g's; NULL: one group of all rows
    int groups;
    int rows;                    // that there is room for; offsets are taken as far as they lie within 0 .. rows and do not fall
};

// begin[g]: the first row of group g; tile[g]: how many tiles of `per` rows the groups before it have.  Groups begin where the largest offset so far says, so that
// whatever the offsets are, no row belongs to two groups and none lies outside.
struct GroupPlan {
    int begin[kMostGroups + 1], tile[kMostGroups + 1];
};

// By one whole warp.
__device__ __forceinline__ void plan_groups(const Groups& g, int per, GroupPlan& plan) {
    const int lane = threadIdx.x & 31;
    if (g.offsets == nullptr) {
        if (lane < 2) {
            plan.begin[lane] = lane * g.rows;
            plan.tile[lane] = lane * ((g.rows + per - 1) / per);
        }
        __syncwarp();
        return;
    }
    int most = 0;                                        // of the offsets before these 32
    for (int at = 0; at <= g.groups; at += 32) {
        int v = at + lane <= g.groups ? min(max(__ldg(g.offsets + at + lane), 0), g.rows) : 0;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int other = __shfl_up_sync(0xFFFFFFFFu, v, d);
            if (lane >= d) v = max(v, other);
        }
        v = max(v, most);
        if (at + lane <= g.groups) plan.begin[at + lane] = v;
        most = __shfl_sync(0xFFFFFFFFu, v, 31);
    }
    __syncwarp();
    int sum = 0;
    for (int at = 0; at <= g.groups; at += 32) {
        const int i = at + lane;
        const int mine = i < g.groups ? (plan.begin[i + 1] - plan.begin[i] + per - 1) / per : 0;
        int v = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int other = __shfl_up_sync(0xFFFFFFFFu, v, d);
            if (lane >= d) v += other;
        }
        if (i <= g.groups) plan.tile[i] = sum + v - mine;
        sum += __shfl_sync(0xFFFFFFFFu, v, 31);
    }
    __syncwarp();
}

// The last g of 0 .. groups - 1 with at[g] <= v.
__device__ __forceinline__ int last_not_above(const int* at, int groups, int v) {
    int lo = 0, hi = groups;                             // at[lo] <= v (or lo = 0), v < at[hi] (or hi = groups)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (at[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Item i of all: 128 rows of a group's matrix times one tile of the group's rows.  The tiles of a group that share these rows of its matrix follow one another.
struct GroupItem {
    int group, tile, tn, row0, rows;                     // tile: among all tiles; tn: which 128 rows of the matrix; row0, rows: of x and y
};
__device__ __forceinline__ GroupItem group_item(const GroupPlan& plan, int groups, int tiles_n, int per, int i) {
    GroupItem t;
    t.group = last_not_above(plan.tile, groups, i / tiles_n);
    const int first = plan.tile[t.group], count = plan.tile[t.group + 1] - first, local = i - first * tiles_n;
    t.tn = local / count;
    const int turn = local - t.tn * count;
    t.tile = first + turn;
    t.row0 = plan.begin[t.group] + turn * per;
    t.rows = min(per, plan.begin[t.group + 1] - t.row0);
    return t;
}

// No more tiles than this, whatever the offsets.
inline long long most_tiles(long long rows, long long groups, int per) { return rows / per + (groups < rows ? groups : rows); }

}  // namespace tcq
