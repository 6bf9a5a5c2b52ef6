// Rows in groups, each times a matrix of its own: where groups begin, and how tiles of their rows are counted.
#pragma once

#include "tcq_microscale.cuh"
#include "tcq_programmatic.cuh"

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

// By one whole warp, which need not have waited for the kernel before where that one does not write offsets.
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
    int most = 0, sum = 0;                               // of the offsets and the tiles before these
    for (int at = 0; at <= g.groups; at += 128) {        // a lane has four neighbours, whose loads are in flight together
        const int mine = at + 4 * lane;
        int v[5];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = mine + q <= g.groups ? load_before_wait(g.offsets + mine + q) : 0;
        v[4] = at + 128 <= g.groups ? load_before_wait(g.offsets + at + 128) : 0;            // what the last lane needs of the next ones
#pragma unroll
        for (int q = 0; q < 5; ++q) v[q] = min(max(v[q], 0), g.rows);
#pragma unroll
        for (int q = 1; q < 4; ++q) v[q] = max(v[q], v[q - 1]);
        int before = v[3];
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int other = __shfl_up_sync(0xFFFFFFFFu, before, d);
            if (lane >= d) before = max(before, other);
        }
        const int last = __shfl_sync(0xFFFFFFFFu, before, 31);
        before = __shfl_up_sync(0xFFFFFFFFu, before, 1);
        before = max(lane == 0 ? 0 : before, most);
        most = max(most, last);
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = max(v[q], before);
        const int next = __shfl_down_sync(0xFFFFFFFFu, v[0], 1);
        v[4] = lane == 31 ? max(v[4], v[3]) : next;
        int tiles[4], all = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            tiles[q] = all;
            all += mine + q < g.groups ? (v[q + 1] - v[q] + per - 1) / per : 0;
        }
        int first = all;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int other = __shfl_up_sync(0xFFFFFFFFu, first, d);
            if (lane >= d) first += other;
        }
        const int end = __shfl_sync(0xFFFFFFFFu, first, 31);
        first += sum - all;
        sum += end;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (mine + q <= g.groups) {
                plan.begin[mine + q] = v[q];
                plan.tile[mine + q] = first + tiles[q];
            }
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
// EVEN: a group's rows are shared by its tiles evenly, so that items are of more equal size; else all but its last one are full.
template <bool EVEN = false>
__device__ __forceinline__ GroupItem group_item(const GroupPlan& plan, int groups, int tiles_n, int per, int i) {
    GroupItem t;
    t.group = last_not_above(plan.tile, groups, i / tiles_n);
    const int first = plan.tile[t.group], count = plan.tile[t.group + 1] - first, local = i - first * tiles_n;
    t.tn = local / count;
    const int turn = local - t.tn * count;
    t.tile = first + turn;
    const int begin = plan.begin[t.group], all = plan.begin[t.group + 1] - begin;
    if (EVEN) {
        const int share = all / count, more = all - share * count;       // the first `more` have one more (at most per, at least one)
        t.row0 = begin + turn * share + min(turn, more);
        t.rows = share + (turn < more);
    } else {
        t.row0 = begin + turn * per;
        t.rows = min(per, all - turn * per);
    }
    return t;
}

// No more tiles than this, whatever the offsets: every group that has rows may have all but one of another tile's.
inline long long most_tiles(long long rows, long long groups, int per) { return (rows + (groups < rows ? groups : rows) * (per - 1)) / per; }

}  // namespace tcq
