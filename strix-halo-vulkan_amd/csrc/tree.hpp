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

// Whether a sequence has rows and they fit behind what it has kept; the others are left alone.
__device__ __forceinline__ bool tree_fits(int pos, int n, int max_cells) { return n > 0 && pos >= 0 && pos <= max_cells - n; }

// What memory says of a sequence and its tree, as words that are asked for together and branch nowhere: an absent array's word is
// read from `any`, which is readable, and not used.
struct TreeWords {
    int count, pos, slot, parent;
    __device__ __forceinline__ TreeWords(const int32_t *counts, const int32_t *positions, const int32_t *slots, const int32_t *parents, const void *any, int seq, int rows,
                                         int lane) {
        const int32_t *a = static_cast<const int32_t *>(any);
        const int at = lane < rows ? lane : rows - 1;
        parent = *(parents ? parents + static_cast<size_t>(seq) * rows + at : a);
        count = *(counts ? counts + seq : a);
        pos = *(positions ? positions + seq : a);
        slot = *(slots ? slots + seq : a);
        count = counts ? (count < 0 ? 0 : count > rows ? rows : count) : rows;
        pos = positions ? pos : 0;
        slot = slots ? slot : seq;
        parent = parents ? parent : lane - 1;
    }
};

// The ancestors by doubling: after step k a lane holds those up to 2^k rows away, and the row 2^k away.  log2(rows) steps.
__device__ __forceinline__ TreeRow tree_row(int n, int parent, int rows, int lane) {
    TreeRow t;
    t.n = n;
    t.parent = lane < n && parent >= 0 && parent < lane ? parent : -1;
    uint32_t lo = lane < n && lane < 32 ? 1u << lane : 0, hi = lane < n && lane >= 32 ? 1u << (lane - 32) : 0;
    int up = t.parent;
    for (int far = 1; far < rows; far *= 2) {
        const int from = up < 0 ? lane : up;  // a row without one that far asks itself
        const uint32_t more_lo = __shfl(lo, from, 64), more_hi = rows > 32 ? __shfl(hi, from, 64) : 0;
        const int next = __shfl(up, from, 64);
        lo |= more_lo;
        hi |= more_hi;
        up = up < 0 ? -1 : next;
    }
    t.ancestors = static_cast<uint64_t>(hi) << 32 | lo;
    t.depth = __popcll(t.ancestors) - 1;
    return t;
}

// Sum of v over a lane's row and the rows on its way to the root.
__device__ __forceinline__ double tree_sum(const TreeRow &t, double v, int rows, int lane) {
    int up = t.parent;
    for (int far = 1; far < rows; far *= 2) {
        const int from = up < 0 ? lane : up;
        const double more = __shfl(v, from, 64);
        const int next = __shfl(up, from, 64);
        v = up < 0 ? v : v + more;
        up = up < 0 ? -1 : next;
    }
    return v;
}

}  // namespace shv
