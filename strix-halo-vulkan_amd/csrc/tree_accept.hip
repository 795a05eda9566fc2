// The branch of a drafted tree that the model agrees with: the arg-max of every row's logits and the walk over them, one launch.
//
// Memory-bound on the logits, which are read once (97 rows of 151936 14.6 us where the last-level cache still holds them, 17.4 from memory, 3.4
// TB/s): a row is cut into as many pieces as fill the chip, each block leaves its piece's best, the block of a row that finishes last joins the
// row's pieces, and the row of a sequence that does walks the tree.
// (Counted by sequence alone, 64 rows of 64 pieces wait 15 ns each for one counter: 60 us, now 9.6.)  The walk
// is one wave: lane i holds row i, a step asks all lanes at once which of them follow the row it stands on with the token that row
// wants, and takes the lowest.
#include "shv_device.hpp"
#include "shv_internal.hpp"
#include "tree.hpp"

namespace {

using namespace shv;

constexpr int kBlock = 256;
// us of 5 / 64 / 192 rows of 151936, the last-level cache holding them: pieces of 1024 floats at least 6.4 / 9.7 / 21, of 2048 5.6 / 9.6 / 21 (5.6 TB/s), of 8192 6.3 / 9.7 / 21; cut for
// 4096 blocks 5.6 / 12.4 / 22.4, for 1024 5.6 / 9.6 / 20.9
constexpr int kPiece = 2048;       // floats of a row a block takes at least
constexpr int kBlocksWanted = 2048;

// By one whole wave: best_of is the lane's row's best.
__device__ __forceinline__ void walk(const shv_tree_accept_args &a, int seq, int best_of, int lane) {
    const size_t base = static_cast<size_t>(seq) * a.rows;
    int n = tree_rows(a.count, seq, a.rows);
    if (a.max_cells > 0 && !tree_fits(a.pos[seq], n, a.max_cells)) n = 0;  // no pass has looked at its rows
    const int parent = lane >= n ? -1 : a.parent ? a.parent[base + lane] : lane - 1;
    const int id = lane < n ? a.ids[base + lane] : 0;
    int kept = 0, at = 0, row_here = -1, next = -1;
    while (n > 0) {
        if (lane == kept) row_here = at;
        kept++;
        next = __builtin_amdgcn_readlane(best_of, at);
        const uint64_t follow = __ballot(lane < n && lane > at && parent == at && id == next);
        if (follow == 0) break;  // a child is a higher row than its parent: at most n steps
        at = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(follow)) - 1);
    }
    if (lane < a.rows) a.path[base + lane] = row_here;
    if (lane == 0) {
        a.n_keep[seq] = kept;
        a.next[seq] = next;
        if (a.pos) {
            const int p = a.pos[seq];
            a.base[seq] = p;
            a.pos[seq] = p + kept;
        }
    }
}

// grid: (pieces, n_seq, rows): rows that are not in use come last
__global__ __launch_bounds__(kBlock) void tree_accept_kernel(shv_tree_accept_args a, float *pval, int32_t *pidx, int32_t *counters) {
    __shared__ float sv[4];
    __shared__ int si[4];
    __shared__ int is_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int piece = blockIdx.x, nb = gridDim.x, r = blockIdx.z, seq = blockIdx.y;
    const int n = tree_rows(a.count, seq, a.rows);
    if (r >= n) {
        if (n == 0 && r == 0 && piece == 0 && wave == 0) walk(a, seq, -1, lane);
        return;
    }
    const size_t row = static_cast<size_t>(seq) * a.rows + r;
    const float *lg = a.logits + row * a.logits_stride;
    const int chunk = ((a.n + nb - 1) / nb + 3) & ~3;
    const int lo = static_cast<int>(min(static_cast<long long>(piece) * chunk, static_cast<long long>(a.n)));
    const int hi = a.n - lo < chunk ? a.n : lo + chunk;
    // "no candidate" is (-inf, n): any element that is a number beats it or, at -inf, comes before it
    float bv = -INFINITY;
    int bi = a.n;
    const auto take = [&](float v, int i) {
        if (amax_better(v, i, bv, bi)) { bv = v; bi = i; }
    };
    const int whole = (reinterpret_cast<uintptr_t>(lg) & 15) == 0 ? lo + ((hi - lo) & ~3) : lo;  // rows that do not begin on 16 bytes: one by one
#pragma unroll 4
    for (int i = lo + 4 * tid; i < whole; i += 4 * kBlock) {
        const float4 v = *reinterpret_cast<const float4 *>(lg + i);
        take(v.x, i), take(v.y, i + 1), take(v.z, i + 2), take(v.w, i + 3);
    }
    for (int i = whole + tid; i < hi; i += kBlock) take(lg[i], i);
    amax_wave(bv, bi);
    if (lane == 0) { sv[wave] = bv; si[wave] = bi; }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < 4; w++)
            if (amax_better(sv[w], si[w], bv, bi)) { bv = sv[w]; bi = si[w]; }
        store_agent(pval + row * nb + piece, bv);
        store_agent(pidx + row * nb + piece, bi);
    }
    if (!arrive_last(counters + (shv_ctx::kTreeSeqs + row) * shv_ctx::kTreeCounterStep, nb, &is_last)) return;
    bv = -INFINITY;
    bi = a.n;
    for (int b = tid; b < nb; b += kBlock) take(load_agent(pval + row * nb + b), load_agent(pidx + row * nb + b));
    amax_wave(bv, bi);
    if (lane == 0) { sv[wave] = bv; si[wave] = bi; }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < 4; w++)
            if (amax_better(sv[w], si[w], bv, bi)) { bv = sv[w]; bi = si[w]; }
        store_agent(a.best + row, bi < a.n ? bi : 0);  // nothing but NaN: 0
    }
    if (!arrive_last(counters + static_cast<size_t>(seq) * shv_ctx::kTreeCounterStep, n, &is_last)) return;
    if (wave == 0) walk(a, seq, lane < n ? load_agent(a.best + static_cast<size_t>(seq) * a.rows + lane) : -1, lane);
}

// grid: n_seq, one wave: the rows' tokens are in best already
__global__ __launch_bounds__(64) void tree_walk_kernel(shv_tree_accept_args a) {
    const int seq = blockIdx.x, lane = threadIdx.x;
    const int n = tree_rows(a.count, seq, a.rows);
    walk(a, seq, lane < n ? a.best[static_cast<size_t>(seq) * a.rows + lane] : -1, lane);
}

}  // namespace

int shv_launch_tree_accept(shv_ctx *ctx, const shv_tree_accept_args *pa) {
    const shv_tree_accept_args &a = *pa;
    SHV_REQUIRE(a.ids && a.best && a.path && a.n_keep && a.next, "tree_accept: NULL argument");
    SHV_REQUIRE(a.rows >= 1 && a.rows <= SHV_TREE_MAX_ROWS, "tree_accept: %d rows; 1..%d", a.rows, SHV_TREE_MAX_ROWS);
    SHV_REQUIRE(a.n_seq >= 1 && a.n_seq <= shv_ctx::kTreeSeqs, "tree_accept: %d sequences; 1..%d", a.n_seq, static_cast<int>(shv_ctx::kTreeSeqs));
    SHV_REQUIRE((a.pos == nullptr) == (a.base == nullptr), "tree_accept: pos and base go together");
    SHV_REQUIRE(!a.pos || a.pos != a.base, "tree_accept: pos and base are one array");
    SHV_REQUIRE(a.max_cells == 0 || (a.max_cells > 0 && a.pos), "tree_accept: max_cells %d; 0, or the cache's with pos and base", a.max_cells);
    if (!a.logits) {
        SHV_LAUNCH(ctx, tree_walk_kernel, dim3(a.n_seq), dim3(64), 0, a);
        return SHV_OK;
    }
    // (indexes along a row are 32 bits and step past its end by up to a block's stride)
    SHV_REQUIRE(a.n >= 1 && a.n <= 1 << 30 && a.logits_stride >= a.n, "tree_accept: rows of %d logits, at most %d; stride %d", a.n, 1 << 30, a.logits_stride);
    const int all = a.n_seq * a.rows;
    SHV_REQUIRE(all <= SHV_TREE_ACCEPT_MAX_ROWS, "tree_accept: %d rows; at most %d", all, SHV_TREE_ACCEPT_MAX_ROWS);
    int nb = (a.n + kPiece - 1) / kPiece;
    const int fill = kBlocksWanted / all > 1 ? kBlocksWanted / all : 1;
    if (nb > fill) nb = fill;
    SHV_LAUNCH(ctx, tree_accept_kernel, dim3(nb, a.n_seq, a.rows), dim3(kBlock), 0, a, ctx->tree_val, ctx->tree_idx, ctx->tree_counters);
    return SHV_OK;
}
