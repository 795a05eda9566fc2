// What a wave knows of a tree of drafted tokens: lane i holds row i's parent, its ancestors and its depth.
#pragma once

#include "shv_device.hpp"

namespace shv {

struct TreeRow {
    int n;               // rows in use of the sequence
    int parent;          // -1: the row follows the sequence's last kept token
    uint64_t ancestors;  // bit j: row j is this row or on its way to the root; 0 for a row not in use
    int depth;           // rows on that way, this one not counted
};

// Rows in use of sequence seq.
__device__ __forceinline__ int tree_rows(const int32_t *count, int seq, int rows) {
    if (!count) return rows;
    const int n = count[seq];
    return n < 0 ? 0 : n > rows ? rows : n;
}

__device__ __forceinline__ int tree_parent(const int32_t *parent, int seq, int rows, int n, int lane) {
    if (lane >= n) return -1;
    const int p = parent ? parent[static_cast<size_t>(seq) * rows + lane] : lane - 1;
    return p >= 0 && p < lane ? p : -1;
}

// The ancestors by doubling: after step k a lane holds those up to 2^k rows away, and the row 2^k away.  64 rows: six steps.
__device__ __forceinline__ TreeRow tree_row(const int32_t *parent, const int32_t *count, int seq, int rows, int lane) {
    TreeRow t;
    t.n = tree_rows(count, seq, rows);
    t.parent = tree_parent(parent, seq, rows, t.n, lane);
    uint32_t lo = lane < t.n && lane < 32 ? 1u << lane : 0, hi = lane < t.n && lane >= 32 ? 1u << (lane - 32) : 0;
    int up = t.parent;
#pragma unroll
    for (int k = 0; k < 6; k++) {
        const int from = up < 0 ? lane : up;  // a row without one that far asks itself
        lo |= __shfl(lo, from, 64);
        hi |= __shfl(hi, from, 64);
        const int next = __shfl(up, from, 64);
        up = up < 0 ? -1 : next;
    }
    t.ancestors = static_cast<uint64_t>(hi) << 32 | lo;
    t.depth = __popcll(t.ancestors) - 1;
    return t;
}

// Sum of v over a lane's row and the rows on its way to the root.
__device__ __forceinline__ float tree_sum(const TreeRow &t, float v, int lane) {
    int up = t.parent;
#pragma unroll
    for (int k = 0; k < 6; k++) {
        const int from = up < 0 ? lane : up;
        const float more = __shfl(v, from, 64);
        const int next = __shfl(up, from, 64);
        v = up < 0 ? v : v + more;
        up = up < 0 ? -1 : next;
    }
    return v;
}

}  // namespace shv
