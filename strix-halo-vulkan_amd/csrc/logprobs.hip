// Log probabilities of given tokens, the distribution's entropy and its most likely tokens, from one pass over the logits.
//
// Of each row, with m = max x: Z = sum e^(x - m), T = sum e^(x - m) (x - m), and then
//     log p_i = (x_i - m) - log Z,    H = log Z - T / Z.
// A thread keeps (m, Z, T) of what it has read, rescaled when its maximum moves.  The most likely tokens of a block's 8192 logits are among those of its registers that
// pass a floor: the k-th largest of a wave's 64 lanes' maxima, which a lane finds as its number of larger ones (16 reads from LDS, each for all lanes at once; by bisection
// of the bits with a ballot a step it takes 4000 cycles), is one that k logits reach, and few more do.  What passes it goes to a list in LDS, and the place of each in
// order is the number of those before it.
// Memory-bound on the logits, which are read once, where there are many rows: 1500 of 151936 take 154 us, 5.9 TB/s.  Few rows are cut into pieces, whose sums and best
// tokens the block of a row that finishes last joins: one row with 5 alternatives takes 9.5 us, of which reading 8192 logits a block is 1, finding and ordering its best 3, arriving 1.2
// and the join, the same work once more over the pieces' best, 2.5.
// Sums are float32, of a thread's at most n / 256 logits one by one and then by trees; log probabilities are (x - m) - log Z, so that what is lost is lost below m and not below x.
#include <type_traits>

#include "scan.hpp"
#include "shv_device.hpp"
#include "shv_internal.hpp"

namespace {

using namespace shv;

constexpr int kBlock = 256, kWaves = kBlock / 64;
constexpr int kMaxTop = SHV_LOGPROBS_MAX_TOP;
static_assert(kMaxTop <= 64, "a floor is one of a wave's lanes' maxima");
constexpr float kLog2e = 1.44269504088896341f;
constexpr int kQuads = 8, kSub = kQuads * 4 * kBlock;  // floats a block holds at a time: eight loads of a thread on their way
constexpr int kMaxPieces = 32, kPerPiece = kBlock / kMaxPieces;
constexpr int kBlocksWanted = 1024;  // four a unit, which its registers and LDS hold at once
constexpr int kMany = 96;           // tokens past its floor from which a wave looks for a higher one
constexpr int kList = kMaxTop + kWaves * kMany;

// Sums of part of a row.
struct Sums {
    float m, z, t;
    // The sums with a maximum that is not below m.
    __device__ __forceinline__ void rise(float top) {
        const float d = fmaxf(m - (top == -INFINITY ? 0.f : top), -200.f), f = __builtin_amdgcn_exp2f(d * kLog2e);  // e^-200 is zero, and zero times -200 too
        t = f * fmaf(d, z, t);
        z *= f;
        m = top;
    }
};

// A logit as a whole number in the order of logits (zeros of either sign alike); 0 for what is not a number, or not there.
__device__ __forceinline__ uint32_t rank_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return v == v ? b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u) : 0u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

constexpr uint32_t kLowest = 0x00800000u;  // the key of the lowest number that is not -infinity
// What a token is sorted by: its key, of equal ones the lower place first.
__device__ __forceinline__ unsigned long long token(float v, int place) { return static_cast<unsigned long long>(rank_key(v)) << 32 | ~static_cast<uint32_t>(place); }

struct Smem {
    float m[kWaves], z[kWaves], t[kWaves];
    uint32_t floor[kWaves];
    int n;              // tokens of the list
    __align__(16) unsigned long long list[kList], kept[kMaxTop];
    __align__(16) uint32_t top[kWaves][64];
};

// The largest K, but for the bits below least_bit, that at least k of the numbers which `count` counts are not below: two bits a step.
template <typename Count>
__device__ __forceinline__ uint32_t kth_key(int k, uint32_t least_bit, Count count) {
    uint32_t K = 0;
#pragma unroll 1
    for (uint32_t bit = 0x40000000u; bit >= least_bit; bit >>= 2) {
        const int one = count(K | bit), two = count(K | 2 * bit), three = count(K | 3 * bit);
        K |= three >= k ? 3 * bit : two >= k ? 2 * bit : one >= k ? bit : 0u;
    }
    return K;
}

// v[i], N a power of two: by masks, which keeps v in registers where a choice between elements would send it to memory.
template <int N, typename T>
__device__ __forceinline__ T pick(const T (&v)[N], int i) {
    uint32_t w[N];
#pragma unroll
    for (int j = 0; j < N; j++) w[j] = __builtin_bit_cast(uint32_t, v[j]);
#pragma unroll
    for (int n = N / 2; n > 0; n /= 2) {
        const uint32_t upper = i & n ? ~0u : 0u;
#pragma unroll
        for (int j = 0; j < n; j++) w[j] = (w[j + n] & upper) | (w[j] & ~upper);
    }
    return __builtin_bit_cast(T, w[0]);
}

// The best k of the list become the list, in order.  All threads take part.
__device__ __forceinline__ void settle(Smem &sm, int k, int tid) {
    __syncthreads();
    const int all = sm.n;
    for (int i = tid; i < all; i += kBlock) {
        const unsigned long long mine = sm.list[i];
        int rank = 0, j = 0;
#pragma unroll 2
        for (; j + 4 <= all; j += 4) {
            const ulonglong2 p = *reinterpret_cast<const ulonglong2 *>(sm.list + j), q = *reinterpret_cast<const ulonglong2 *>(sm.list + j + 2);
            rank += (p.x > mine) + (p.y > mine) + (q.x > mine) + (q.y > mine);
        }
        for (; j < all; j++) rank += sm.list[j] > mine;
        if (rank < k) sm.kept[rank] = mine;
    }
    __syncthreads();
    const int kept = min(all, k);
    if (tid < kept) sm.list[tid] = sm.kept[tid];
    if (tid == 0) sm.n = kept;
    __syncthreads();
}

// What a token has to reach to be among the block's best k.
struct Bar {
    float v = -INFINITY;
    bool passed = true;     // and pass: what equals it is no better, as places rise
    __device__ __forceinline__ bool by(float m) const { return passed ? m > v : m >= v; }
};

// To the list what its best k may be of what the block's threads hold, v[i] at place(i); what is -infinity or no number is left out.  m is a thread's largest.  A list of
// more than kMaxTop is cut to its best k.  All threads take part.
template <int N, typename Place>
__device__ __forceinline__ void select(const float (&v)[N], float m, Place place, Smem &sm, Bar &bar, int k, int tid, int lane, int wave) {
    // k lanes reach the floor, and so do k tokens.  (The lane's number in the lower bits makes all keys different; the floor is a little lower for it.)
    const uint32_t key = rank_key(m), mine = (key & ~63u) | (63u - lane);
    sm.top[wave][lane] = mine;
    __builtin_amdgcn_wave_barrier();
    int above_me = 0;
#pragma unroll
    for (int j = 0; j < 64; j += 4) {
        const uint4 o = *reinterpret_cast<const uint4 *>(&sm.top[wave][j]);
        above_me += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
    }
    const int kth = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(__ballot(above_me == k - 1))) - 1);
    const uint32_t floor = max(kLowest, static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(key & ~63u), kth)));
    if (lane == 0) sm.floor[wave] = floor;
    __syncthreads();
    float F = of_key(max(max(sm.floor[0], sm.floor[1]), max(sm.floor[2], sm.floor[3])));
    bar = Bar{fmaxf(bar.v, F), bar.passed && bar.v >= F};
    F = bar.v;
    uint32_t pass = 0;
#pragma unroll
    for (int i = 0; i < N; i++) pass |= v[i] >= F ? 1u << i : 0u;
    int upto = __popc(pass);
    const auto scan = [&] {
        upto = static_cast<int>(wave_upto(upto));
        return __builtin_amdgcn_readlane(upto, 63);
    };
    if (__ballot(pass != 0) != 0) {
        int n = scan();
        if (n > kMany) {
            // many in few lanes, or many that are equal: the k-th largest of all that the wave holds, those above it, which are fewer than k, and of its equals
            // the lowest places
            const auto reach = [&](uint32_t x) {
                const float f = of_key(x);
                int c = 0;
#pragma unroll
                for (int i = 0; i < N; i++) c += __popcll(__ballot(v[i] >= f));
                return c;
            };
            F = fmaxf(F, of_key(max(kLowest, kth_key(k, 1, reach))));
            int above = 0;
#pragma unroll
            for (int i = 0; i < N; i++) above += __popcll(__ballot(v[i] > F));
            const uint32_t from = kth_key(k - above, 1, [&](uint32_t x) {
                int c = 0;
#pragma unroll
                for (int i = 0; i < N; i++) c += __popcll(__ballot(v[i] == F && ~static_cast<uint32_t>(place(i)) >= x));
                return c;
            });
            pass = 0;
#pragma unroll
            for (int i = 0; i < N; i++) pass |= v[i] > F || (v[i] == F && ~static_cast<uint32_t>(place(i)) >= from) ? 1u << i : 0u;
            upto = __popc(pass);
            n = scan();
        }
        int at = 0;
        if (lane == 0) at = atomicAdd(&sm.n, n);
        at = __builtin_amdgcn_readfirstlane(at) + upto - __popc(pass);
        while (__ballot(pass != 0) != 0) {
            const int i = __ffs(pass) - 1;
            if (pass != 0) sm.list[at] = token(pick(v, i), place(i));
            at++;
            pass &= pass - 1;
        }
    }
    __syncthreads();
    if (sm.n > kMaxTop) {
        settle(sm, k, tid);
        bar = Bar{of_key(static_cast<uint32_t>(sm.list[k - 1] >> 32)), true};
    }
}

// The largest of a wave, in every lane.
__device__ __forceinline__ float wave_max_dpp(float v) {
    const auto larger = [](float a, int b) { return fmaxf(a, __int_as_float(b)); };
    v = larger(v, dpp_or_own<kDppXor1>(__float_as_int(v)));
    v = larger(v, dpp_or_own<kDppXor2>(__float_as_int(v)));
    v = larger(v, dpp_or_own<kDppHalfMirror>(__float_as_int(v)));
    v = larger(v, dpp_or_own<kDppMirror>(__float_as_int(v)));
    v = larger(v, dpp_or_own<kDppBcast15>(__float_as_int(v)));
    v = larger(v, dpp_or_own<kDppBcast31>(__float_as_int(v)));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// A block's sums in every thread.
__device__ __forceinline__ void block_sums(Sums &s, Smem &sm, int lane, int wave) {
    const float top = wave_max_dpp(s.m);
    s.rise(top);
    s.z = wave_sum_all(s.z);
    s.t = wave_sum_all(s.t);
    if (lane == 0) sm.m[wave] = s.m, sm.z[wave] = s.z, sm.t[wave] = s.t;
    __syncthreads();
    const float all = fmaxf(fmaxf(sm.m[0], sm.m[1]), fmaxf(sm.m[2], sm.m[3]));
    Sums sum{all, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        Sums o{sm.m[w], sm.z[w], sm.t[w]};
        o.rise(all);
        sum.z += o.z, sum.t += o.t;
    }
    s = sum;
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
    Bar bar;
    if (TOP && tid == 0) sm.n = 0;
    const int id = a.ids ? a.ids[row] : -1;
    const bool is_token = id >= 0 && id < a.n;
    const float given = is_token ? x[id] : 0.f;
    // Values of a thread into its sums; those that are not there are -infinity.
    const auto add = [&](const auto &v, auto n) {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < n; i++) m = fmaxf(m, v[i]);
        if (m > s.m) s.rise(m);
        const float to = s.m == -INFINITY ? 0.f : s.m;
#pragma unroll
        for (int i = 0; i < n; i++) {
            const float d = v[i] - to, w = __builtin_amdgcn_exp2f(d * kLog2e);
            s.z += w;
            s.t = fmaf(w, fmaxf(d, -200.f), s.t);
        }
        return m;
    };
    // the row from its first address of 16 bytes on in steps of four, what stands before and behind them by the first and the last piece
    const int head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) / 4 & 3), a.n), body = (a.n - head) / 4, tail = head + 4 * body;
    const int each = (body + nb - 1) / nb, lo = min(piece * each, body), hi = min(lo + each, body);
    const float4 *x4 = reinterpret_cast<const float4 *>(x + head);
    if constexpr (TOP) __syncthreads();
    for (int i0 = lo; i0 < hi; i0 += kQuads * kBlock) {
        float v[4 * kQuads];
#pragma unroll
        for (int u = 0; u < kQuads; u++) {
            const int j = i0 + u * kBlock + tid;
            const float4 q = x4[min(j, hi - 1)];
            const bool there = j < hi;
            v[4 * u] = there ? q.x : -INFINITY, v[4 * u + 1] = there ? q.y : -INFINITY, v[4 * u + 2] = there ? q.z : -INFINITY, v[4 * u + 3] = there ? q.w : -INFINITY;
        }
        const float m = add(v, std::integral_constant<int, 4 * kQuads>());
        if constexpr (TOP) {
            if (__syncthreads_or(bar.by(m))) select(v, m, [&](int i) { return head + 4 * (i0 + i / 4 * kBlock + tid) + i % 4; }, sm, bar, k, tid, lane, wave);
        }
    }
    const bool before = piece == 0 && tid < head, behind = piece == nb - 1 && tid < a.n - tail;
    if (piece == 0 || piece == nb - 1) {
        const float v[2] = {before ? x[tid] : -INFINITY, behind ? x[tail + tid] : -INFINITY};
        add(v, std::integral_constant<int, 2>());
        if constexpr (TOP) {
            // at most six; every wave has read the list's length as the last selection left it
            if (head > 0 || tail < a.n) __syncthreads();
            if (v[0] > -INFINITY) sm.list[atomicAdd(&sm.n, 1)] = token(v[0], tid);
            if (v[1] > -INFINITY) sm.list[atomicAdd(&sm.n, 1)] = token(v[1], tail + tid);
            if (head > 0 || tail < a.n) __syncthreads();
            if (sm.n > kMaxTop) settle(sm, k, tid);
        }
    }
    block_sums(s, sm, lane, wave);
    if (nb > 1) {
        float *mine = part + (row * nb + piece) * shv_ctx::kLpPieceFloats;
        const int n = TOP ? sm.n : 0;
        if (tid == 0) {
            store_agent2(mine, s.m, s.z);
            store_agent2(mine + 2, s.t, __int_as_float(n));
        }
        if (tid < n) store_agent2(mine + 4 + 2 * tid, __uint_as_float(static_cast<uint32_t>(sm.list[tid])), __uint_as_float(static_cast<uint32_t>(sm.list[tid] >> 32)));
        if (!arrive_last(counters + row * shv_ctx::kLpCounterStep, nb, &is_last)) return;
        const float *all = part + row * nb * shv_ctx::kLpPieceFloats;
        // eight threads a piece; all is asked for before any of it is used
        const int b = tid / kPerPiece, r = tid % kPerPiece;
        const float *of = all + static_cast<size_t>(min(b, nb - 1)) * shv_ctx::kLpPieceFloats;
        constexpr int kEach = kMaxTop / kPerPiece;
        const float2 mz = load_agent2(of);
        const float2 tn = load_agent2(of + 2);
        float2 best[kEach];
        if constexpr (TOP) {
#pragma unroll
            for (int i = 0; i < kEach; i++) best[i] = load_agent2(of + 4 + 2 * (r + kPerPiece * i));
        }
        s = r == 0 && b < nb ? Sums{mz.x, mz.y, tn.x} : Sums{-INFINITY, 0.f, 0.f};
        if constexpr (TOP) {
            float v[kEach], m = -INFINITY;
            int at[kEach];
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                const bool there = b < nb && r + kPerPiece * i < __float_as_int(tn.y);
                at[i] = ~__float_as_uint(best[i].x), v[i] = of_key(there ? __float_as_uint(best[i].y) : 0u);  // (a token that is not there: no number)
                m = fmaxf(m, v[i]);
            }
            if (tid == 0) sm.n = 0;
            bar = Bar{};
            select(v, m, [&](int i) { return pick(at, i); }, sm, bar, k, tid, lane, wave);
        }
        block_sums(s, sm, lane, wave);
    }
    if constexpr (TOP) {
        settle(sm, k, tid);
        // fewer than k tokens can come: the lowest places of those that cannot, in order
        for (int i0 = 0; sm.n < k && i0 < a.n; i0 += kBlock) {
            const bool is = i0 + tid < a.n && x[i0 + tid] == -INFINITY;
            const uint64_t mask = __ballot(is);
            if (lane == 0) sm.floor[wave] = __popcll(mask);
            const int kept = sm.n;
            __syncthreads();
            int at = kept, n = kept;
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                at += w < wave ? sm.floor[w] : 0;
                n += sm.floor[w];
            }
            at += static_cast<int>(__builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0)));
            if (is && at < k) sm.list[at] = token(-INFINITY, i0 + tid);
            if (tid == 0) sm.n = min(n, k);
            __syncthreads();
        }
    }
    const float log_z = logf(s.z);
    if (tid == 0) {
        if (a.ids) a.logprob[row] = is_token ? (given - s.m) - log_z : __int_as_float(0x7fc00000);
        if (a.entropy) a.entropy[row] = log_z - s.t / s.z;
    }
    if constexpr (TOP)
        if (tid < k) {
            const bool there = tid < sm.n;
            const unsigned long long best = there ? sm.list[tid] : 0ull;
            a.top_ids[row * k + tid] = there ? static_cast<int32_t>(~static_cast<uint32_t>(best)) : -1;
            a.top_logprobs[row * k + tid] = there ? (of_key(static_cast<uint32_t>(best >> 32)) - s.m) - log_z : -INFINITY;
        }
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
    int nb = (a.n + kSub - 1) / kSub;
    if (nb > kMaxPieces) nb = kMaxPieces;
    const int fill = kBlocksWanted / a.n_rows > 1 ? kBlocksWanted / a.n_rows : 1;
    if (nb > fill) nb = fill;
    const dim3 grid(nb, a.n_rows);
    if (a.n_top > 0) SHV_LAUNCH(ctx, logprobs_kernel<true>, grid, dim3(kBlock), 0, a, ctx->lp_part, ctx->lp_counters);
    else SHV_LAUNCH(ctx, logprobs_kernel<false>, grid, dim3(kBlock), 0, a, ctx->lp_part, ctx->lp_counters);
    return SHV_OK;
}
