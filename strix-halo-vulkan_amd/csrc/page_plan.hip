// The pages of a serving batch's pass: what each sequence gives back, takes and where its new rows lie, one launch.
//
// With want = ceil((pos + rows) / page): back = held - max(want, shared), need = want - held, each where above zero.  The pages given back lie behind the
// free ones, L = free | back in order, A = |L|; sequence s's j-th new page is L[A - 1 - (taken before it) - j].  All of that is two scans over the
// sequences, of (back, need, rows) and of what is granted, and lookups by bisection from there on.  Entries that come back and are no page are not in L: what comes back is looked at beside
// the second scan (two passes of 48 sequences 9.9 us and 9.0 without it, of 900 with 12007 rows 22.1 and 18.9), and where some of it is none the pages among it are laid
// on the stack first and the grants made again.
// Bound by the chain of trips to memory (a sequence's words, then pages, then the stores) and the scans' barriers, not by bytes: 48 sequences of a token each take 3.1 to 4.5 us
// of the kernel's own time, 900 with 12007 rows 9.4 to 11.4.  Every block makes the scans for itself, which costs less than a launch between them and the
// rows; a row a thread, since each is a bisection and two dependent loads (four a thread cost the 900 sequences' two passes 7 us).  The words that others
// still read (held, pos, n_free) are written by the block that arrives last.
#include "scan.hpp"
#include "shv_device.hpp"
#include "shv_internal.hpp"

namespace {

using namespace shv;

constexpr int kMaxSeqs = SHV_PAGE_MAX_SEQS;
constexpr int kMaxRows = 1 << 20;
// Pages a thread that could be given back, from which a call gets a block more.  200 sequences of up to 188 pages, a row each, two passes: 14.2 us with 16, 16.0 with 32 and 18.6 by
// one block; 4, with which a call of 48 sequences has two blocks, gains nothing there (10.3 and 10.3).
constexpr int kPagesFrom = 16;

constexpr int kOwn = 2, kAtOnce = 4;  // entries that come back: of a sequence by its own lane, and loads of a wave on their way of the others

// WAVE, up to 64 sequences: each wave makes the scans for itself and writes to LDS what the others write, without a barrier up to the last.  (48 sequences, two passes: 10.4 us, and 11.3 by a
// block's scans with two barriers each.)
template <int T, bool WAVE>
__global__ __launch_bounds__(T) void page_plan_kernel(shv_page_plan_args a, int shift, int32_t *counter) {
    constexpr int kPer = T == 1024 ? kMaxSeqs / T : 1;  // sequences a thread, side by side
    __shared__ uint32_t s_start[kPer * T], s_taken[kPer * T], s_back[kPer * T];
    __shared__ int s_held[kPer * T], s_pos[kPer * T];
    __shared__ uint32_t waves[3][T / 64];
    __shared__ int is_last, is_odd, n_many;
    const int tid = threadIdx.x;
    static_assert(!WAVE || kPer == 1, "a lane a sequence");
    const int first = WAVE ? tid & 63 : tid * kPer;
    if (!WAVE && tid == 0) is_odd = n_many = 0;
    int rows[kPer], pos[kPer], held[kPer], shared[kPer];
#pragma unroll
    for (int u = 0; u < kPer; u++) {
        const int s = min(first + u, a.n_seq - 1);
        rows[u] = a.rows[s], pos[u] = a.pos[s], held[u] = a.held[s], shared[u] = a.shared ? a.shared[s] : 0;
    }
    const uint32_t n_free = min(max(a.n_free[0], 0), a.n_pages);
    uint32_t back[kPer], need[kPer], asked[kPer];
    bool fits[kPer];
    uint32_t sums[3] = {0, 0, 0}, total[3];
#pragma unroll
    for (int u = 0; u < kPer; u++) {
        const bool there = first + u < a.n_seq, ends = rows[u] < 0;
        held[u] = min(max(held[u], 0), a.max_pages);
        shared[u] = min(max(shared[u], 0), held[u]);
        const long long upto = static_cast<long long>(pos[u]) + max(rows[u], 0);
        const long long want = ends ? 0 : (upto + a.page - 1) >> shift;
        fits[u] = there && (ends || (pos[u] >= 0 && want <= a.max_pages));
        const int w = fits[u] ? static_cast<int>(want) : held[u];
        back[u] = fits[u] ? max(held[u] - max(w, shared[u]), 0) : 0;
        need[u] = fits[u] ? max(w - held[u], 0) : 0;
        asked[u] = fits[u] ? min(static_cast<uint32_t>(max(rows[u], 0)), kFull) : 0;
        sums[0] = add_up_to(sums[0], back[u]), sums[1] = add_up_to(sums[1], need[u]), sums[2] = add_up_to(sums[2], asked[u]);
    }
    if constexpr (WAVE) wave_scan(sums, total);
    else block_scan<T, 3>(sums, total, waves);
    const uint32_t n_back = total[0];
    {
        uint32_t b = sums[0];
#pragma unroll
        for (int u = 0; u < kPer; u++) {
            s_back[first + u] = b;
            b = add_up_to(b, back[u]);
            s_held[first + u] = held[u], s_pos[first + u] = pos[u];
        }
    }
    // The r-th entry that comes back, one of sequence s.
    const auto where = [&](uint32_t r, int s) {
        const int low = s_held[s] - static_cast<int>((s + 1 < a.n_seq ? s_back[s + 1] : n_back) - s_back[s]);
        return a.table + static_cast<size_t>(s) * a.max_pages + low + (r - s_back[s]);
    };
    const auto is_page = [&](int e) { return e >= 0 && e < a.n_pages; };
    // All of them are looked at: the first few of a sequence by its lane, the others by a wave, 64 a load.  The last loads are on their way while the grants are made.
    int own[kPer][kOwn], others[kAtOnce];
    bool odd = false;
    if (n_back > 0) {
        const int lane = tid & 63;
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) others[i] = 0;
        const auto look = [&](int s, int low, int n) {
            const int32_t *of = a.table + static_cast<size_t>(s) * a.max_pages + low;
            for (int at = kOwn + lane; __ballot(at < n) != 0ull; at += 64 * kAtOnce) {
                int e[kAtOnce];
#pragma unroll
                for (int i = 0; i < kAtOnce; i++) e[i] = at + 64 * i < n ? of[at + 64 * i] : 0;
#pragma unroll
                for (int i = 0; i < kAtOnce; i++) {
                    odd |= !is_page(others[i]);
                    others[i] = e[i];
                }
            }
        };
#pragma unroll
        for (int u = 0; u < kPer; u++) {
            const int32_t *mine = a.table + static_cast<size_t>(first + u) * a.max_pages + (held[u] - back[u]);
#pragma unroll
            for (int i = 0; i < kOwn; i++) own[u][i] = i < back[u] ? mine[i] : 0;
            if (!WAVE && back[u] > kOwn) s_taken[atomicAdd(&n_many, 1)] = first + u;
        }
        if constexpr (WAVE) {
            for (uint64_t many = __ballot(back[0] > kOwn); many != 0; many &= many - 1) {
                const int l = __ffsll(static_cast<unsigned long long>(many)) - 1, n = __builtin_amdgcn_readlane(back[0], l);
                look(l, __builtin_amdgcn_readlane(held[0], l) - n, n);
            }
        } else {
            __syncthreads();
            for (int i = tid >> 6; i < n_many; i += T / 64) {
                const int s = __builtin_amdgcn_readfirstlane(s_taken[i]), n = static_cast<int>((s + 1 < a.n_seq ? s_back[s + 1] : n_back) - s_back[s]);
                look(s, s_held[s] - n, n);
            }
        }
    }
    bool stacked = false;
    uint32_t avail = n_free + n_back, n_taken, n_rows;
    uint32_t take[kPer], gets[kPer];
    for (bool again = false;; again = true) {
        uint32_t both[2] = {0, 0}, total2[2];
        {
            uint32_t n = sums[1], r = sums[2];
#pragma unroll
            for (int u = 0; u < kPer; u++) {
                n = add_up_to(n, need[u]), r = add_up_to(r, asked[u]);
                const bool granted = fits[u] && (need[u] == 0 || n <= avail) && r <= static_cast<uint32_t>(a.max_rows);
                take[u] = granted ? need[u] : 0;
                gets[u] = granted ? asked[u] : 0;
                both[0] += take[u], both[1] += gets[u];  // (at most avail and max_rows together)
            }
        }
        if constexpr (WAVE) wave_scan(both, total2);
        else block_scan<T, 2>(both, total2, waves);
        n_taken = total2[0], n_rows = total2[1];
        {
            uint32_t t = both[0], r = both[1];
#pragma unroll
            for (int u = 0; u < kPer; u++) {
                s_taken[first + u] = t, s_start[first + u] = r;
                t += take[u], r += gets[u];
            }
        }
        if (n_back > 0 && !again) {
#pragma unroll
            for (int u = 0; u < kPer; u++)
#pragma unroll
                for (int i = 0; i < kOwn; i++) odd |= !is_page(own[u][i]);
#pragma unroll
            for (int i = 0; i < kAtOnce; i++) odd |= !is_page(others[i]);
            odd = __ballot(odd) != 0ull;
            if (!WAVE && odd) is_odd = 1;
        }
        if constexpr (WAVE) {
            if (again) __syncthreads();
            else __builtin_amdgcn_wave_barrier();
        } else {
            __syncthreads();
            odd = is_odd != 0;
        }
        if (!odd || again) break;
        // what is a page among a run of them, a run a thread, goes to the stack before any is taken (by every block, the same to the same place)
        const uint32_t run = (n_back + T - 1) / T, r0 = min(tid * run, n_back), r1 = min(r0 + run, n_back);
        uint32_t v[1], all[1], at = 0, n_given = 0;
        for (bool put = false;; put = true) {
            for (uint32_t r = r0; r < r1;) {
                const int s = last_not_above(s_back, a.n_seq, r);
                const int32_t *of = where(r, s);
                const uint32_t n = min(r1, s + 1 < a.n_seq ? s_back[s + 1] : n_back) - r;
                for (uint32_t i = 0; i < n; i += kAtOnce) {
                    int e[kAtOnce];
#pragma unroll
                    for (int j = 0; j < kAtOnce; j++) e[j] = i + j < n ? of[i + j] : -1;
#pragma unroll
                    for (int j = 0; j < kAtOnce; j++)
                        if (is_page(e[j])) {
                            if (put && at < n_given) a.free_pages[n_free + at] = e[j];
                            at++;
                        }
                }
                r += n;
            }
            if (put) break;
            v[0] = at;
            block_scan<T, 1>(v, all, waves);
            at = v[0], n_given = min(all[0], a.n_pages - n_free), avail = n_free + n_given;
        }
        stacked = true;
    }
    if (blockIdx.x == 0) {
        for (int s = tid; s < a.n_seq; s += T) {
            a.start[s] = s_start[s];
            if (a.base) a.base[s] = s_pos[s];
        }
        if (tid == 0) a.start[a.n_seq] = n_rows;
    }
    const auto taken = [&](uint32_t e) {  // the e-th page from the top
        const uint32_t i = avail - 1 - e;
        return i < n_free || stacked ? a.free_pages[i] : *where(i - n_free, last_not_above(s_back, a.n_seq, i - n_free));
    };
    const uint32_t step = gridDim.x * T, me = blockIdx.x * T + tid;
    for (uint32_t t = me; t < n_rows; t += step) {
        const int s = last_not_above(s_start, a.n_seq, t);
        const int p = s_pos[s] + static_cast<int>(t - s_start[s]), at = p >> shift;
        const int page = at < s_held[s] ? a.table[static_cast<size_t>(s) * a.max_pages + at] : taken(s_taken[s] + at - s_held[s]);
        if (a.row_seq) a.row_seq[t] = s;
        a.row_pos[t] = p;
        a.row_cell[t] = page >= 0 && page < a.n_pages ? (page << shift) + (p & (a.page - 1)) : -1;
    }
    // (what is written here is read by no block: entries past a growing sequence's, and behind the free pages)
    for (uint32_t e = me; e < n_taken; e += step) {
        const int s = last_not_above(s_taken, a.n_seq, e);
        a.table[static_cast<size_t>(s) * a.max_pages + s_held[s] + (e - s_taken[s])] = taken(e);
    }
    if (!stacked)
        for (uint32_t r = me; r < n_back && n_free + r < static_cast<uint32_t>(a.n_pages); r += step) a.free_pages[n_free + r] = *where(r, last_not_above(s_back, a.n_seq, r));
    if (gridDim.x > 1) {
        if (!arrive_last(counter, gridDim.x, &is_last)) return;
    } else if (WAVE) {
        __syncthreads();  // every wave has read what is written now
    }
    if (WAVE && tid >= 64) return;
#pragma unroll
    for (int u = 0; u < kPer; u++) {
        if (!fits[u]) continue;  // left as it is, as behind the last
        a.held[first + u] = rows[u] < 0 ? 0 : held[u] - back[u] + take[u];
        if (a.base) a.pos[first + u] = rows[u] < 0 ? 0 : pos[u] + static_cast<int>(gets[u]);
    }
    if (tid == 0) a.n_free[0] = avail - n_taken;
}

}  // namespace

int shv_launch_page_plan(shv_ctx *ctx, const shv_page_plan_args *pa) {
    const shv_page_plan_args &a = *pa;
    SHV_REQUIRE(a.rows && a.pos && a.table && a.held && a.free_pages && a.n_free && a.start && a.row_pos && a.row_cell, "page_plan: NULL argument");
    SHV_REQUIRE(a.n_seq >= 1 && a.n_seq <= kMaxSeqs, "page_plan: %d sequences; 1..%d", a.n_seq, kMaxSeqs);
    SHV_REQUIRE(a.page >= 32 && a.page <= 4096 && (a.page & (a.page - 1)) == 0, "page_plan: page %d; a power of two from 32 to 4096", a.page);
    SHV_REQUIRE(a.n_pages >= 1 && static_cast<long long>(a.n_pages) * a.page < 1ll << 31, "page_plan: %d pages of %d cells; fewer than 2^31 cells", a.n_pages, a.page);
    SHV_REQUIRE(a.max_pages >= 1 && static_cast<long long>(a.max_pages) * a.page < 1ll << 31, "page_plan: max_pages %d of %d cells; fewer than 2^31 cells", a.max_pages, a.page);
    SHV_REQUIRE(a.max_rows >= 1 && a.max_rows <= kMaxRows, "page_plan: max_rows %d; 1..%d", a.max_rows, kMaxRows);
    SHV_REQUIRE(a.rows != a.pos && a.rows != a.held && a.pos != a.held && a.base != a.pos, "page_plan: rows, pos, held and base are arrays of their own");
    int shift = 0;
    while (1 << shift < a.page) shift++;
    int32_t *counter = ctx->lp_counters + shv_ctx::kLpPieces * shv_ctx::kLpCounterStep;
    // (a barrier of 4 waves costs less than one of 16)
    const int threads = a.n_seq <= 256 && a.max_rows <= 4096 ? 256 : 1024;
    const long long entries = static_cast<long long>(a.n_seq) * a.max_pages, pages = entries < a.n_pages ? entries : a.n_pages;
    const long long for_rows = (a.max_rows + threads - 1) / threads, for_pages = pages / (kPagesFrom * threads), blocks = for_rows > for_pages ? for_rows : for_pages;
    const dim3 grid(static_cast<unsigned>(blocks < 64 ? blocks : 64));
    if (threads == 256 && a.n_seq <= 64) SHV_LAUNCH(ctx, (page_plan_kernel<256, true>), grid, dim3(256), 0, a, shift, counter);
    else if (threads == 256) SHV_LAUNCH(ctx, (page_plan_kernel<256, false>), grid, dim3(256), 0, a, shift, counter);
    else SHV_LAUNCH(ctx, (page_plan_kernel<1024, false>), grid, dim3(1024), 0, a, shift, counter);
    return SHV_OK;
}
