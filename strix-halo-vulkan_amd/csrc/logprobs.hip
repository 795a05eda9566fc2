// Log probabilities of given tokens, the distribution's entropy and its most likely tokens, from one pass over the logits.
//
// Of each row, with m = max x: Z = sum e^(x - m), T = sum e^(x - m) (x - m), and then
//     log p_i = (x_i - m) - log Z,    H = log Z - T / Z.
// A thread keeps (m, Z, T) of what it has read, rescaled when its maximum moves, and a wave the best tokens it has met, one a lane in falling order: what is
// no better than the last of them is passed over with a comparison, the rest is put in its place by a ballot and a shift of the lanes.
// Memory-bound on the logits, which are read once.  Few rows are cut into pieces, whose sums and best tokens the block of a row that finishes last joins.
#include "shv_device.hpp"
#include "shv_internal.hpp"

namespace {

using namespace shv;

constexpr int kBlock = 256, kWaves = kBlock / 64;
constexpr int kMaxTop = SHV_LOGPROBS_MAX_TOP;
static_assert(kMaxTop <= 64, "one token a lane");
constexpr float kLog2e = 1.44269504088896341f;
constexpr int kPiece = 4096;        // floats of a row a block takes at least
constexpr int kBlocksWanted = 1024;
constexpr int kNone = 0x7FFFFFFF;   // the place of a token that is not there: behind all others

// Sums of part of a row.
struct Sums {
    float m, z, t;
    // One more maximum and the sums beside it.
    __device__ __forceinline__ void join(float m2, float z2, float t2) {
        const float top = fmaxf(m, m2), to = top == -INFINITY ? 0.f : top;
        const float d1 = fmaxf(m - to, -200.f), d2 = fmaxf(m2 - to, -200.f);  // e^-200 is zero, and zero times -200 too
        const float f1 = __builtin_amdgcn_exp2f(d1 * kLog2e), f2 = __builtin_amdgcn_exp2f(d2 * kLog2e);
        t = f1 * fmaf(d1, z, t) + f2 * fmaf(d2, z2, t2);
        z = f1 * z + f2 * z2;
        m = top;
    }
};

// The best tokens a wave has met: lane i holds the i-th, (value, place).
struct Best {
    float v;
    int i;
    float last_v;  // the k-th, which a token has to beat
    int last_i;
    __device__ __forceinline__ void clear() { v = last_v = -INFINITY, i = last_i = kNone; }
    // Takes x of place p from the lanes where `may` says so, one after the other.
    __device__ __forceinline__ void take(float x, int p, bool may, int k, int lane) {
        uint64_t todo = __ballot(may && amax_better(x, p, last_v, last_i));
        while (todo != 0) {
            const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(todo)) - 1);
            todo &= todo - 1;
            const float nv = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l));
            const int ni = __builtin_amdgcn_readlane(p, l);
            if (!amax_better(nv, ni, last_v, last_i)) continue;
            const bool stays = amax_better(v, i, nv, ni);
            const int at = __popcll(__ballot(stays));
            const float up_v = __shfl_up(v, 1, 64);
            const int up_i = __shfl_up(i, 1, 64);
            v = stays ? v : lane == at ? nv : up_v;
            i = stays ? i : lane == at ? ni : up_i;
            last_v = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), k - 1));
            last_i = __builtin_amdgcn_readlane(i, k - 1);
        }
    }
};

// A value that k lanes' values are not below: the k-th largest of the wave's.
__device__ __forceinline__ float kth_of_wave(float v, int k, int lane) {
    int above = 0;
#pragma unroll 16
    for (int l = 0; l < 64; l++) {
        const float o = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l));
        above += o > v || (o == v && l < lane);
    }
    const uint64_t it = __ballot(above == k - 1);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), __ffsll(static_cast<unsigned long long>(it)) - 1));
}

struct Smem {
    float m[kWaves], z[kWaves], t[kWaves];
    float v[kWaves][kMaxTop];
    int i[kWaves][kMaxTop];
};

// A block's sums in every thread; its waves' best tokens to place: rank r goes to put(r, value, place).
__device__ __forceinline__ void block_sums(Sums &s, Smem &sm, int lane, int wave) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        // the lower lane's first on both sides, so that both hold the same bits
        const float m2 = __shfl_xor(s.m, off, 64), z2 = __shfl_xor(s.z, off, 64), t2 = __shfl_xor(s.t, off, 64);
        if (lane & off) {
            Sums o{m2, z2, t2};
            o.join(s.m, s.z, s.t);
            s = o;
        } else {
            s.join(m2, z2, t2);
        }
    }
    if (lane == 0) sm.m[wave] = s.m, sm.z[wave] = s.z, sm.t[wave] = s.t;
    __syncthreads();
    s = Sums{sm.m[0], sm.z[0], sm.t[0]};
#pragma unroll
    for (int w = 1; w < kWaves; w++) s.join(sm.m[w], sm.z[w], sm.t[w]);
}
template <typename Put>
__device__ __forceinline__ void block_best(const Best &b, Smem &sm, int k, int lane, int wave, Put put) {
    if (lane < k) sm.v[wave][lane] = b.v, sm.i[wave][lane] = b.i;
    __syncthreads();
    // the rank of a wave's token is its own place and how many of each other wave's stand before it
    if (lane < k) {
        int rank = lane;
#pragma unroll
        for (int o = 1; o < kWaves; o++) {
            const int w = (wave + o) & (kWaves - 1);
            int lo = 0;
            for (int hi = k; lo < hi;) {
                const int mid = (lo + hi) >> 1;
                const float ov = sm.v[w][mid];
                const int oi = sm.i[w][mid];
                // places that are not there are alike: the lower wave's first
                if (amax_better(ov, oi, b.v, b.i) || (ov == b.v && oi == b.i && w < wave)) lo = mid + 1;
                else hi = mid;
            }
            rank += lo;
        }
        if (rank < k) put(rank, b.v, b.i);
    }
}

// grid: (pieces, rows)
template <bool TOP>
__global__ __launch_bounds__(kBlock) void logprobs_kernel(shv_logprobs_args a, float *part, int32_t *counters) {
    __shared__ Smem sm;
    __shared__ int is_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int piece = blockIdx.x, nb = gridDim.x, k = a.n_top;
    const size_t row = blockIdx.y;
    const float *x = a.logits + row * a.logits_stride;
    Sums s{-INFINITY, 0.f, 0.f};
    Best best;
    best.clear();
    bool seeded = false;
    float floor_v = -INFINITY;  // k of the wave's values are not below it
    constexpr int U = 4;
    // 4 * U values of a thread, v[u] at place p + u * 4 * kBlock ..; those that are not there are -infinity at kNone
    const auto look = [&](const float (&v)[U][4], const int (&p)[U][4]) {
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) m = fmaxf(m, v[u][e]);
        if constexpr (TOP) {
            if (!seeded) {
                floor_v = kth_of_wave(m, k, lane);
                seeded = true;
            }
            if (__ballot(m >= best.last_v && m >= floor_v) != 0) {
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int e = 0; e < 4; e++) best.take(v[u][e], p[u][e], v[u][e] >= floor_v && p[u][e] != kNone, k, lane);
            }
        }
        if (m > s.m) {
            const float d = fmaxf(s.m - m, -200.f), f = __builtin_amdgcn_exp2f(d * kLog2e);
            s.t = f * fmaf(d, s.z, s.t);
            s.z *= f;
            s.m = m;
        }
        const float to = s.m == -INFINITY ? 0.f : s.m;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float d = v[u][e] - to, w = __builtin_amdgcn_exp2f(d * kLog2e);
                s.z += w;
                s.t = fmaf(w, fmaxf(d, -200.f), s.t);
            }
    };
    // the row from its first address of 16 bytes on in steps of four, what stands before and behind them by the first and the last piece
    const int head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) / 4 & 3), a.n), body = (a.n - head) / 4, tail = head + 4 * body;
    const int each = (body + nb - 1) / nb, lo = min(piece * each, body), hi = min(lo + each, body);
    const float4 *x4 = reinterpret_cast<const float4 *>(x + head);
    for (int i = lo + tid; __ballot(i < hi) != 0; i += U * kBlock) {
        float v[U][4];
        int p[U][4];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = i + u * kBlock;
            const float4 q = x4[min(j, hi - 1)];
            const bool there = j < hi;
            v[u][0] = there ? q.x : -INFINITY, v[u][1] = there ? q.y : -INFINITY, v[u][2] = there ? q.z : -INFINITY, v[u][3] = there ? q.w : -INFINITY;
#pragma unroll
            for (int e = 0; e < 4; e++) p[u][e] = there ? head + 4 * j + e : kNone;
        }
        look(v, p);
    }
    if (piece == 0 || piece == nb - 1) {
        float v[U][4];
        int p[U][4];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[u][e] = -INFINITY, p[u][e] = kNone;
        if (piece == 0 && tid < head) v[0][0] = x[tid], p[0][0] = tid;
        if (piece == nb - 1 && tid < a.n - tail) v[0][1] = x[tail + tid], p[0][1] = tail + tid;
        look(v, p);
    }
    block_sums(s, sm, lane, wave);
    if (nb > 1) {
        float *mine = part + (row * nb + piece) * shv_ctx::kLpPieceFloats;
        if (tid == 0) {
            store_agent2(mine, s.m, s.z);
            store_agent(mine + 2, s.t);
        }
        if constexpr (TOP) block_best(best, sm, k, lane, wave, [&](int r, float v, int i) { store_agent2(mine + 4 + 2 * r, v, __int_as_float(i)); });
        if (!arrive_last(counters + row * shv_ctx::kLpCounterStep, nb, &is_last)) return;
        const float *all = part + row * nb * shv_ctx::kLpPieceFloats;
        s = Sums{-INFINITY, 0.f, 0.f};
        for (int b = tid; b < nb; b += kBlock) {
            const float2 mz = load_agent2(all + static_cast<size_t>(b) * shv_ctx::kLpPieceFloats);
            s.join(mz.x, mz.y, load_agent(all + static_cast<size_t>(b) * shv_ctx::kLpPieceFloats + 2));
        }
        block_sums(s, sm, lane, wave);
        if constexpr (TOP) {
            best.clear();
            seeded = false;
            floor_v = -INFINITY;
            for (int c = tid; __ballot(c < nb * k) != 0; c += kBlock) {
                const int b = min(c, nb * k - 1) / k, r = min(c, nb * k - 1) - b * k;
                const float2 vi = load_agent2(all + static_cast<size_t>(b) * shv_ctx::kLpPieceFloats + 4 + 2 * r);
                const bool there = c < nb * k && __float_as_int(vi.y) != kNone;
                const float v = there ? vi.x : -INFINITY;
                if (!seeded) {
                    floor_v = kth_of_wave(v, k, lane);
                    seeded = true;
                }
                best.take(v, __float_as_int(vi.y), there && v >= floor_v, k, lane);
            }
        }
    }
    const float log_z = logf(s.z);
    if (tid == 0) {
        if (a.ids) {
            const int id = a.ids[row];
            a.logprob[row] = id >= 0 && id < a.n ? (x[id] - s.m) - log_z : __int_as_float(0x7fc00000);
        }
        if (a.entropy) a.entropy[row] = log_z - s.t / s.z;
    }
    if constexpr (TOP)
        block_best(best, sm, k, lane, wave, [&](int r, float v, int i) {
            a.top_ids[row * k + r] = i == kNone ? -1 : i;
            a.top_logprobs[row * k + r] = i == kNone ? -INFINITY : (v - s.m) - log_z;
        });
}

}  // namespace

int shv_launch_logprobs(shv_ctx *ctx, const shv_logprobs_args *pa) {
    const shv_logprobs_args &a = *pa;
    SHV_REQUIRE(a.logits, "logprobs: NULL logits");
    SHV_REQUIRE((a.ids == nullptr) == (a.logprob == nullptr), "logprobs: ids and logprob go together");
    SHV_REQUIRE(a.n_rows >= 1 && a.n_rows <= 65535, "logprobs: %d rows; 1..65535", a.n_rows);
    // (indexes along a row are 32 bits and step past its end by up to a block's stride)
    SHV_REQUIRE(a.n >= 1 && a.n <= 1 << 30 && a.logits_stride >= a.n, "logprobs: rows of %d logits, at most %d; stride %d", a.n, 1 << 30, a.logits_stride);
    SHV_REQUIRE(a.n_top >= 0 && a.n_top <= kMaxTop && a.n_top <= a.n, "logprobs: %d alternatives of %d; at most %d", a.n_top, a.n, kMaxTop);
    SHV_REQUIRE((a.n_top > 0) == (a.top_ids != nullptr) && (a.n_top > 0) == (a.top_logprobs != nullptr), "logprobs: top_ids and top_logprobs go with n_top %d", a.n_top);
    SHV_REQUIRE(a.ids || a.entropy || a.n_top > 0, "logprobs: nothing is asked for");
    int nb = (a.n + kPiece - 1) / kPiece;
    const int fill = kBlocksWanted / a.n_rows > 1 ? kBlocksWanted / a.n_rows : 1;
    if (nb > fill) nb = fill;
    const dim3 grid(nb, a.n_rows);
    if (a.n_top > 0) SHV_LAUNCH(ctx, logprobs_kernel<true>, grid, dim3(kBlock), 0, a, ctx->lp_part, ctx->lp_counters);
    else SHV_LAUNCH(ctx, logprobs_kernel<false>, grid, dim3(kBlock), 0, a, ctx->lp_part, ctx->lp_counters);
    return SHV_OK;
}
