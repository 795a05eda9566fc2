// Full attention of packed rows over a paged cache.
//
// Row r of a sequence, at position p_r, sees the sequence's cells c <= p_r that lie in a page (with a window those of them below `sinks` or above p_r - window):
//     out_r = sum over them of softmax(q_r . k_c / sqrt(d)) v_c
// q and k normed over a head and rotated at their positions.  Three launches:
//   cells  the rows' keys and values into their cells, and, in a block of its own, the plan of the next;
//   attn   a block takes one KV head and up to 64 query rows (128 of narrower heads; query row r of a sequence is head r % rep of its row r / rep), and a run of
//          their tiles of 32 cells, on v_mfma_f32_16x16x32_f16:
//              S^T = K Q^T   the cache's binary16 keys against the queries as two halves; a lane then holds eight cells of one query row, the operand
//                            of the second product
//              O  += P V     weights as two halves against values, which the cache holds by dim
//          with a running maximum and sum.  Tiles go from memory to LDS past the registers, and two blocks share a
//          unit: while one begins a piece or ends it the other's tiles keep coming;
//   join   the records of query rows whose tiles several blocks have shared.
#include <atomic>

#include "attn_rows.hpp"
#include "scan.hpp"
#include "shv_device.hpp"
#include "shv_internal.hpp"

namespace {

using namespace shv;

constexpr int kTile = 32;  // cells of a tile of V
constexpr int kMaxSeqs = SHV_PAGE_MAX_SEQS;
constexpr int kChunk = 64 * 16;
// Waves of a block: two of four share a unit, or one of eight has it (is_wide).  96 tokens in a window of 2048, 128 dims, take 170 us with two and 201 with one, 24 behind up to
// 12000 146 and 166, a chunk of 512 among 23 tokens 230 and 280, 48 tokens of 64 dims behind up to 6000 100 and 154.
constexpr int kWide = 8, kNarrow = 4;
constexpr int ring_bytes(int waves) { return waves * (16 << 10); }
// Weights are e^(s - m) 2^kLift, and m stands until a score is more than kSlack powers of two above it: up to 2^15.9, which the larger half holds, and down to
// 2^-35 of the largest with the smaller half's last place, to which it is rounded.
constexpr float kLift = 11.f, kSlack = 4.9f;
// Maxima, in powers of two, from which a weight is formed from the difference of the scores as they are: roundings of scaled scores past 2^24, which norm weights of 1500 reach with 256
// dims, would send it past binary16.  Always formed so, a chunk of 512 among 23 tokens takes 306 us for 294, and a prompt of 4096 264 for 266: 128 dims have no registers for it.
constexpr float kFar = 1024.f;
// Tiles of few query rows whose cost a block gets at least, and quarters of a tile more by every further 16 query rows, whose records cost more than what their tiles' split gains:
// one token of 256 dims behind 900 takes 18.4 us with two and 19.4 with three, 37 rows of rep 8 behind 3001 33.9 with two and 29.1 with the quarters, 64 of 128 dims behind
// 3000 38.8 and 37.0.
constexpr uint32_t kLeast = 2, kLeastMore = 3;
// Records of a query row from which a block's waves share them, at most: 200 rows of 128 dims behind 100, which have up to 9, take 35.4 us with 8 and 31.4 with 16, 8 tokens of
// 256 dims behind up to 16000, which have up to 32, 50.8 with 16 and 56.2 with 48.
constexpr int kShareFrom = 16;
// Query blocks that a plan holds: 2^20 query rows by 128, and a rest of each sequence.
constexpr int kMostBlocks = (1 << 20) / 128 + kMaxSeqs;
constexpr int kFewBlocks = 1024;  // query blocks up to which the plan is made inside the launch of the cells: a launch costs 3 us more, and more blocks more LDS than 256 threads should hold

// Groups of 16 query rows of a wave, and query rows of a block.  Of 256 dims a wave's registers hold one group; of fewer they hold two, which an operand read from LDS serves
// both.
template <int D>
constexpr int kGroups = D == 256 ? 1 : 2;
// Waves that share a group of few query rows, each with tiles of its own, so that a round in the ring is 32 KB (64 in the wide block's): 24 tokens of 128 dims behind up to
// 12000 take 146 us with two and 156 with one, 48 of 64 dims behind up to 6000 102 with two or four and 134 with one.
template <int D, int WAVES>
constexpr int kTurns = WAVES == kWide ? 2 : 256 / D;
constexpr int rows_of(int D, int waves) { return 16 * waves * (D == 256 ? 1 : 2); }

// A block's query rows of a sequence and a run of the tiles they look at.
struct Piece {
    int seq, first;     // the sequence and its first packed row
    int r0, r_end;      // the first query row, and the sequence's number of them
    int pos;            // of the sequence's first row
    int t0, t1;         // the run
    int rec;            // where its records go; -1: it is all there is
};
// What a block has: its first piece, and how many more lie from pieces[at] on; more -1: nothing.
struct Block {
    Piece piece;
    int more, at;
    int pad[6];
};
// Up to 16 query rows whose tiles several blocks share: rows r0 .. of a sequence, which are row `in` .. of their records.
struct Join {
    int first, r0, r_end, rec, n, in;
    int pad[2];
};

// Where a call's scratch lies and what it can hold; worked out by the launcher from the sizes alone.
struct Plan {
    int32_t *n_joins;
    Block *blocks;
    Piece *pieces;      // a query block's first piece, where a block has more than one
    Join *joins;
    float *sums;        // records: [record][KV head][slot_rows][D] unnormalised sums
    float2 *of;         // and their (maximum, sum)
    int slots;          // blocks a KV head that the chip holds at once
    int waves, rows, rep; // waves and query rows of a block; query heads of a KV head
    int slot_rows;      // and of a record
    int most_blocks, most_q;
    int dies, heads;    // dies that share a KV head, and KV heads of a die (place)
    int shift;          // log2 of the page
    uint32_t rep_magic; // 2^32 / rep, rounded up; 0 for rep 1
    __device__ __forceinline__ int over_rep(int r) const {  // r / rep: exact for r < 2^20 and rep <= 64, which it is off by less than 1 / 64 before it is cut
        return rep_magic == 0 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), rep_magic));
    }
};

// Which tiles of 32 cells query rows of positions lo .. hi look at: the sinks', then those the window of the first row reaches.
struct Tiles {
    int sinks, first, all;
    __device__ __forceinline__ Tiles(int window, int n_sinks, int lo, int hi) {
        const int end = hi / kTile + 1;
        sinks = first = 0;
        if (window > 0) {
            sinks = n_sinks > 0 ? min(n_sinks - 1, hi) / kTile + 1 : 0;
            first = max(sinks, max(0, lo - window + 1) / kTile);
        }
        all = sinks + max(0, end - first);
    }
    __device__ __forceinline__ int at(int i) const { return i < sinks ? i : i - sinks + first; }
};

// A sequence's rows; n 0 where it is left alone.
struct Seq {
    int first, n, pos;
    __device__ __forceinline__ Seq(const shv_attn_paged_args &a, int s) {
        first = a.start[s];
        const int to = a.start[s + 1];
        n = first >= 0 && to > first && to <= a.max_rows ? to - first : 0;
        pos = n > 0 ? a.row_pos[first] : 0;
        if (pos < 0 || static_cast<long long>(pos) + n > static_cast<long long>(a.max_pages) * a.page) n = 0;
    }
};

// ---- the plan: one block of T threads -----------------------------------------------------------
// What a block's work costs, in tenths of a microsecond of a unit: a tile of few query rows, by its block where memory has bandwidth to spare (few_least) and by memory where all units
// ask for such tiles (few); one of many query rows by its products, here of 16 groups; a piece its way in and out, and its rows' bytes.  Fitted to the times of blocks, then
// turned about on a few batches: of 128 dims a chunk of 512 among 23 tokens behind up to 12000 takes 230 us with group 21, 232 with 20, 239 with 23, 237 with 18, and with few_least 7 238,
// with 9 236; four chunks of 500 behind 3000 203 with few_beside 8, 192 with 10, 194 with 12; of 256 forty tokens behind up to 9000 105.8 with piece 90, 106.9 with 30, 104.8
// with 120.  Neighbouring values are within 4 %, and another batch may have another of them best.
struct Costs {
    int few, few_least, few_beside, group, piece, piece_group;
    __host__ __device__ __forceinline__ int tile(int groups) const { return group * groups / 16; }
    __host__ __device__ __forceinline__ int way(int groups) const { return piece + piece_group * groups / 16; }
};
__host__ __device__ constexpr Costs wide_costs(int D) { return D == 256 ? Costs{16, 12, 16, 37, 90, 128} : D == 128 ? Costs{9, 8, 10, 21, 60, 64} : Costs{5, 3, 5, 12, 60, 32}; }
// Of a block's time: two narrow ones share a unit.
__host__ __device__ __forceinline__ Costs costs_of(int D, int waves) {
    const Costs c = wide_costs(D);
    const int by = kWide / waves;
    return Costs{c.few * by, c.few_least * by, c.few_beside * by, c.group * by, c.piece, c.piece_group};
}

// The query blocks of all sequences stand in a row, each with its cost, P their running sum.  Where they fill the chip evenly each is a block's own, those with the most
// tiles first.  Otherwise block b takes what lies from b S to (b + 1) S in the row, S = all / blocks, so that all blocks have the same; a query block cut by that
// leaves a record of each piece.
constexpr uint32_t kRare = 128;  // work of other blocks, tenths of a microsecond, for each tile of few query rows; 15 to 60 where a chunk comes with a batch's tokens, 600 in chunks alone
constexpr int kSeqBits = 11, kMaxSlots = 512;  // blocks that the chip holds at once: a unit two
static_assert(kMaxSeqs <= 1 << kSeqBits, "a sequence's number");
template <int T, int SEQS, int NQ>
struct PlanSmem {
    uint32_t q0[SEQS];          // query blocks before a sequence's
    int first[SEQS], n[SEQS], pos[SEQS];
    uint32_t p[NQ], of[NQ];     // the cost before a query block; its sequence, and above kSeqBits its first piece
    int rec[NQ];                // its first record, -1: it has one piece
    uint16_t begins[kMaxSlots + 1];  // a block's first piece
    uint32_t waves[3][T / 64];
    uint32_t bucket[64];
    uint32_t most[3][T / 64];
    uint32_t first_piece[64];   // WAVE: a query block's
};
// A query block as a piece of all its tiles; what a tile of it costs, and its way in and out (which the first one's block has in any case).
struct Whole : Piece {
    uint32_t tile, way, groups;
    // What it costs but for its way; kFull, and no cut then, past 2^23 tiles, so that nothing below passes 32 bits (a tile costs less than 128).
    __device__ __forceinline__ uint32_t cost() const { return static_cast<uint32_t>(t1) > kFull / 128 ? kFull : t1 * tile; }
};
// x / d by its reciprocal: exact for x < 2^31 and quotients to 2^21, which three roundings leave off by less than 1.  (The plan is a chain; a division's is twice as long.)
struct Divisor {
    uint32_t d;
    float r;
    __device__ __forceinline__ explicit Divisor(uint32_t by) : d(by), r(__builtin_amdgcn_rcpf(static_cast<float>(by))) {}
    __device__ __forceinline__ uint32_t under(uint32_t x) const {
        const uint32_t q = static_cast<uint32_t>(static_cast<float>(x) * r);
        const int left = static_cast<int>(x - q * d);
        return left < 0 ? q - 1 : left >= static_cast<int>(d) ? q + 1 : q;
    }
};
__device__ __forceinline__ Whole whole_block(int window, int sinks, int D, int waves, int rows, uint32_t rep_magic, int seq, int first, int r_end, int pos, int r0, bool free_way, uint32_t few) {
    const auto over_rep = [&](int r) { return rep_magic == 0 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), rep_magic)); };
    const Costs costs = costs_of(D, waves);
    Whole p;
    p.seq = seq, p.first = first, p.r0 = r0, p.r_end = r_end, p.pos = pos;
    const int last = min(r0 + rows, r_end) - 1;
    p.t0 = 0, p.t1 = Tiles(window, sinks, pos + over_rep(r0), pos + over_rep(last)).all;
    p.rec = -1;
    p.groups = (last - r0) / 16 + 1;
    p.tile = max(static_cast<uint32_t>(costs.tile(p.groups)), few), p.way = free_way ? 0 : costs.way(p.groups);
    return p;
}

// The largest of a wave, in every lane.
__device__ __forceinline__ uint32_t wave_most(uint32_t v) {
    v = max(v, static_cast<uint32_t>(dpp_or_own<kDppXor1>(v)));
    v = max(v, static_cast<uint32_t>(dpp_or_own<kDppXor2>(v)));
    v = max(v, static_cast<uint32_t>(dpp_or_own<kDppHalfMirror>(v)));
    v = max(v, static_cast<uint32_t>(dpp_or_own<kDppMirror>(v)));
    v = max(v, static_cast<uint32_t>(dpp_or_own<kDppBcast15>(v)));
    v = max(v, static_cast<uint32_t>(dpp_or_own<kDppBcast31>(v)));
    return __builtin_amdgcn_readlane(static_cast<int>(v), 63);
}

// WAVE, up to 64 sequences and query blocks: each wave makes all sums for itself and writes what the others write, without a barrier between them, up to where the blocks'
// pieces are found.  (By a block's sums with two barriers each a call takes a microsecond more: 37 rows behind 3001 30.3
// us for 29.1, 8 tokens behind up to 500 20.2 for 19.1.)
template <bool WAVE, int T, int SEQS, int NQ>
__device__ __forceinline__ void make_plan(const shv_attn_paged_args &a, const Plan &plan, PlanSmem<T, SEQS, NQ> &sm) {
    const int tid = threadIdx.x, rep = plan.rep, log_rows = __builtin_ctz(plan.rows);
    constexpr int STEP = WAVE ? 64 : T;
    const int me = WAVE ? tid & 63 : tid;
    const auto sums_before = [&](auto &v, auto &all) {
        if constexpr (WAVE) wave_scan(v, all);
        else block_scan<T>(v, all, sm.waves);
    };
    const auto sync = [] {
        if constexpr (WAVE) __builtin_amdgcn_wave_barrier();
        else __syncthreads();
    };
    uint32_t nq = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += STEP) {
        const int s = s0 + me;
        uint32_t v[1] = {0}, all[1];
        if (s < a.n_seq) {
            const Seq seq(a, s);
            sm.first[s] = seq.first, sm.n[s] = seq.n, sm.pos[s] = seq.pos;
            v[0] = (static_cast<uint32_t>(seq.n) * rep + plan.rows - 1) >> log_rows;
        }
        sums_before(v, all);
        if (s < a.n_seq) sm.q0[s] = nq + v[0];
        nq += all[0];
    }
    if (tid < 64) sm.bucket[tid] = 0;
    sync();
    const Costs costs = costs_of(a.head_dim, plan.waves);
    uint32_t few = costs.few_least;
    const auto whole_of = [&](uint32_t i, int seq) {
        return whole_block(a.window, a.sinks, a.head_dim, plan.waves, plan.rows, plan.rep_magic, seq, sm.first[seq], sm.n[seq] * rep, sm.pos[seq], static_cast<int>(i - sm.q0[seq]) * plan.rows, i == 0, few);
    };
    const auto whole = [&](uint32_t i) { return whole_of(i, sm.of[i] & ((1 << kSeqBits) - 1)); };
    nq = min(nq, static_cast<uint32_t>(min(plan.most_q, NQ)));
    // Tiles of few query rows, t of them, come as fast as memory gives them, few t / slots in all, or as their blocks take them beside those of many, whose cost is c:
    // (few_least t + c) / slots.  Where the first is longer a tile costs what makes both alike.  Where they are rare, the rests of chunks, each shares its unit with a block of
    // products that was there first and is served first (few_beside).
    uint32_t both[2] = {0, 0}, sums[2];
    Whole own = {};  // query block `me`, which is all that a thread has in most calls
    for (uint32_t i = me; i < nq; i += STEP) {
        const int seq = last_not_above(sm.q0, a.n_seq, i);
        sm.of[i] = seq;
        const Whole p = whole_of(i, seq);
        if (i == me) own = p;
        const bool is_few = p.tile == few;
        both[is_few] = add_up_to(both[is_few], is_few ? min(static_cast<uint32_t>(p.t1), kFull) : p.cost());
    }
    sums_before(both, sums);
    if (sums[1] > 0) {
        const uint32_t beside = sums[0] / sums[1];
        few = beside > kRare ? costs.few_beside : max(few, costs.few - min(beside, static_cast<uint32_t>(costs.few)));
    }
    own.tile = max(own.tile, few);
    const auto mine = [&](uint32_t i) { return i == me ? own : whole(i); };
    uint32_t total = 0, most = 0, most_way = 0, most_groups = 1;
    for (uint32_t i0 = 0; i0 < nq; i0 += STEP) {
        uint32_t v[1] = {0}, all[1];
        if (i0 + me < nq) {
            const Whole p = mine(i0 + me);
            v[0] = p.way + p.cost();
            most = max(most, v[0]), most_way = max(most_way, p.way), most_groups = max(most_groups, p.groups);
        }
        if (!WAVE && i0 + T >= nq) {
            const uint32_t of_wave[3] = {wave_most(most), wave_most(most_way), wave_most(most_groups)};
            if ((tid & 63) == 0) sm.most[0][tid / 64] = of_wave[0], sm.most[1][tid / 64] = of_wave[1], sm.most[2][tid / 64] = of_wave[2];
        }
        sums_before(v, all);
        if (i0 + me < nq) sm.p[i0 + me] = add_up_to(total, v[0]);
        total = add_up_to(total, all[0]);
    }
    sync();
    if constexpr (WAVE) {
        most = wave_most(most), most_way = wave_most(most_way), most_groups = wave_most(most_groups);
    } else if (nq > 0) {
#pragma unroll
        for (int w = 0; w < T / 64; w++) most = max(most, sm.most[0][w]), most_way = max(most_way, sm.most[1][w]), most_groups = max(most_groups, sm.most[2][w]);
    }
    const uint32_t slots = plan.slots;
    const uint32_t share = max((total + slots - 1) / slots, (kLeast + (most_groups - 1) * kLeastMore / 4) * costs.few);
    // whole query blocks take as long as the longest, or as so many of the mean size one behind the other; a cut costs another way in and out, and the records' join
    const uint32_t rounds = (nq + slots - 1) / slots;
    const bool cut = total < kFull && max(most, nq > 0 ? total / nq * rounds : 0u) > share + most_way + most_way / 2;
    if (!cut) {
        __syncthreads();
        for (int pass = 0; pass < 2; pass++) {
            for (uint32_t i = tid; i < nq; i += T) {
                const Whole p = mine(i);
                const uint32_t k = 63 - min(63u, static_cast<uint32_t>(static_cast<float>(p.cost()) * (64.f / static_cast<float>(most + 1))));
                const uint32_t at = atomicAdd(&sm.bucket[k], 1u);
                if (pass == 1) plan.blocks[at] = Block{p, 0, 0, {}};
            }
            __syncthreads();
            if (pass == 0) {
                if (tid == 0) {
                    uint32_t sum = 0;
                    for (int k = 0; k < 64; k++) {
                        const uint32_t n = sm.bucket[k];
                        sm.bucket[k] = sum;
                        sum += n;
                    }
                }
                __syncthreads();
            }
        }
        for (uint32_t b = nq + tid; b < static_cast<uint32_t>(plan.most_blocks); b += T) plan.blocks[b].more = -1;
        if (tid == 0) *plan.n_joins = 0;
        return;
    }
    // Cut c of the row, at c S, falls into query block i between two of its tiles or, on its way in or behind its last tile but one, on a border of query blocks.
    // Piece k of query block i begins at its cut number first_cut + k.
    const Divisor by_share(share);
    const auto piece_of = [&](uint32_t i, Whole p, uint32_t k) {
        const uint32_t from = sm.p[i] + p.way, c = by_share.under(from) + k, all = p.t1;
        p.t0 = k == 0 ? 0 : (c * share - from + p.tile - 1) / p.tile;
        p.t1 = min(all, ((c + 1) * share - from + p.tile - 1) / p.tile);
        return p;
    };
    const uint32_t blocks = Divisor(share).under(total + share - 1);
    uint32_t before[3] = {0, 0, 0};  // pieces, records, joins
    for (uint32_t i0 = 0; i0 < nq; i0 += STEP) {
        const uint32_t i = i0 + me;
        uint32_t v[3] = {0, 0, 0}, all[3], n = 0;
        Whole p;
        if (i < nq) {
            p = mine(i);
            const uint32_t from = sm.p[i] + p.way;
            n = by_share.under(from + (p.t1 - 1) * p.tile) - by_share.under(from) + 1;
            v[0] = n, v[1] = n > 1 ? n : 0, v[2] = n > 1 ? p.groups : 0;
        }
        sums_before(v, all);
        if (i < nq) {
            const uint32_t at = before[0] + v[0], rec = before[1] + v[1];
            if constexpr (WAVE) sm.first_piece[i] = at;
            else sm.of[i] |= at << kSeqBits;
            sm.rec[i] = n > 1 ? static_cast<int>(rec) : -1;
            if (n > 1) {
                for (uint32_t g = 0; g < p.groups && (!WAVE || tid < 64); g++)
                    plan.joins[before[2] + v[2] + g] = Join{p.first, p.r0 + 16 * static_cast<int>(g), p.r_end, static_cast<int>(rec), static_cast<int>(n), 16 * static_cast<int>(g), {}};
                p = piece_of(i, p, 0);
                p.rec = rec;
            }
            if (!WAVE || tid < 64) plan.pieces[at] = p;
        }
        before[0] += all[0], before[1] += all[1], before[2] += all[2];
    }
    sync();
    // the query block and which of its pieces that begin at or behind cut c; i = nq: none
    const auto piece_at = [&](uint32_t c, uint32_t &i, uint32_t &k) {
        i = last_not_above(sm.p, nq, c * share);
        k = 0;
        Whole p = whole(i);
        const uint32_t x = c * share - sm.p[i];
        if (x <= p.way) return p;
        if (x <= p.way + (p.t1 - 1) * p.tile) {
            k = c - by_share.under(sm.p[i] + p.way);
            return p;
        }
        if (++i < nq) p = whole(i);
        return p;
    };
    constexpr int kBlocks = (kMaxSlots + T - 1) / T;  // of a thread
    uint32_t i[kBlocks], k[kBlocks];
    Whole of_block[kBlocks];
#pragma unroll
    for (int e = 0; e < kBlocks; e++) {
        const uint32_t b = e * T + tid;
        if (b >= blocks) break;
        of_block[e] = piece_at(b, i[e], k[e]);
        sm.begins[b] = i[e] < nq ? (WAVE ? sm.first_piece[i[e] & 63] : sm.of[i[e]] >> kSeqBits) + k[e] : before[0];
    }
    if (tid == 0) sm.begins[blocks] = before[0];
    __syncthreads();
    // neighbouring blocks lie on one die
    const uint32_t dies = plan.dies;  // a power of two
    const int log_dies = __builtin_ctz(dies);
    const uint32_t per = (blocks + dies - 1) >> log_dies;
    for (uint32_t slot = tid; slot < static_cast<uint32_t>(plan.most_blocks); slot += T) {
        const uint32_t row = slot >> log_dies, of = (slot & (dies - 1)) * per + row;
        if (row >= per || of >= blocks || sm.begins[of] == sm.begins[of + 1]) plan.blocks[slot].more = -1;
    }
#pragma unroll
    for (int e = 0; e < kBlocks; e++) {
        const uint32_t b = e * T + tid;
        if (b >= blocks) break;
        if (sm.begins[b] == sm.begins[b + 1]) continue;
        Whole p = piece_of(i[e], of_block[e], k[e]);
        p.rec = sm.rec[i[e]] < 0 ? -1 : sm.rec[i[e]] + static_cast<int>(k[e]);
        const uint32_t die = Divisor(per).under(b);
        plan.blocks[(b - die * per) * dies + die] = Block{p, sm.begins[b + 1] - sm.begins[b] - 1, sm.begins[b] + 1, {}};
    }
    if (tid == 0) *plan.n_joins = before[2];
}

__global__ __launch_bounds__(1024) void paged_plan_kernel(shv_attn_paged_args a, Plan plan) {
    extern __shared__ __align__(16) char raw[];
    make_plan<false>(a, plan, *reinterpret_cast<PlanSmem<1024, kMaxSeqs, kMostBlocks> *>(raw));
}

// ---- the rows' cells ----------------------------------------------------------------------------
// A wave a row's cell of a KV head; with PLAN the first block makes the plan, which takes longer than few rows' cells do: 4.5 us with one row, 7 with forty, a chain of the
// sequences' words, three sums over them, a bisection and the stores.  Many rows would be bound by the values' stores, two
// bytes in each of a cell's lines (18.2 us for 4096 rows of two heads of 256 dims, 25 MB, and 10 by columns).
// Where rows are many, blocks from values_from on take the values of eight rows by 256 columns: a thread has a column, and cells side by side in a tile are one store.
// A prompt of 2048 (two heads of 256 dims) takes 113 us with that and 115.5 without, one of 4096 (eight of 128) 303 and 314; four chunks whose cells begin anywhere 191 either
// way.
constexpr int kValuesRows = 8;
constexpr int kValuesFrom = 512;  // rows: below, the plan takes as long as the cells
__device__ __forceinline__ bool has_cell(const shv_attn_paged_args &a, const Plan &plan, int r, int p, int cell) {
    return r < a.start[a.n_seq] && p >= 0 && p < a.max_pages << plan.shift && cell >= 0 && cell < a.n_pages << plan.shift;
}
template <int D>
__device__ __forceinline__ void put_values(const shv_attn_paged_args &a, const Plan &plan, uint32_t block) {
    const uint32_t kvw = static_cast<uint32_t>(a.n_head_kv) * D, across = (kvw + 255) / 256, by = block / across;
    const int r0 = static_cast<int>(by) * kValuesRows, lane = threadIdx.x & 63;
    const uint32_t col = (block - by * across) * 256 + threadIdx.x;
    const float *src = a.qkv + static_cast<size_t>(a.n_head) * 2 * D + kvw + min(col, kvw - 1);
    float v[kValuesRows];
#pragma unroll
    for (int i = 0; i < kValuesRows; i++) v[i] = src[static_cast<size_t>(min(r0 + i, a.max_rows - 1)) * a.qkv_stride];
    const int mine = r0 + lane % kValuesRows, r = min(mine, a.max_rows - 1);
    int cell = a.row_cell[r];
    if (mine >= a.max_rows || !has_cell(a, plan, r, a.row_pos[r], cell)) cell = -1;
    const uint64_t follows = __ballot(cell >= 0 && __shfl_up(cell, 1, 64) == cell - 1 && cell % kTile != 0);  // it is in the row before's tile, behind it
    if (col >= kvw) return;
    uint16_t *const values = static_cast<uint16_t *>(a.vpages) + static_cast<size_t>(col) * kTile;
    uint16_t h[kValuesRows];
#pragma unroll
    for (int i = 0; i < kValuesRows; i++) h[i] = __half_as_ushort(__float2half_rn(v[i]));
    const auto at = [&](int i) {
        const int c = __builtin_amdgcn_readlane(cell, i);
        return values + static_cast<size_t>(c / kTile) * kvw * kTile + c % kTile;
    };
    const int c0 = __builtin_amdgcn_readlane(cell, 0);
    const bool run = c0 >= 0 && (follows & 0xFE) == 0xFE;
    if (run && c0 % 8 == 0) {
        put_bytes<16>(at(0), h);
    } else if (run && c0 % 4 == 0) {
        put_bytes<8>(at(0), h);
        put_bytes<8>(at(4), h + 4);
    } else {
#pragma unroll
        for (int i = 0; i < kValuesRows; i++)
            if (__builtin_amdgcn_readlane(cell, i) >= 0) *at(i) = h[i];
    }
}

template <int D, bool PLAN>
__global__ __launch_bounds__(256) void paged_cells_kernel(shv_attn_paged_args a, Plan plan, uint32_t values_from) {
    constexpr int VEC = D / 64;
    if constexpr (PLAN) {
        __shared__ PlanSmem<256, kFewBlocks, kFewBlocks> sm;
        if (blockIdx.x == 0) {
            if (a.n_seq <= 64 && plan.most_q <= 64) make_plan<true>(a, plan, sm);
            else make_plan<false>(a, plan, sm);
            return;
        }
    }
    if (values_from > 0 && blockIdx.x >= values_from) {
        put_values<D>(a, plan, blockIdx.x - values_from);
        return;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t item = (blockIdx.x - (PLAN ? 1 : 0)) * 4 + wave;
    const int r = static_cast<int>(item / static_cast<uint32_t>(a.n_head_kv)), head = static_cast<int>(item) - r * a.n_head_kv;
    if (r >= a.max_rows) return;
    const float *src = a.qkv + static_cast<size_t>(r) * a.qkv_stride + static_cast<size_t>(a.n_head) * 2 * D + head * D;
    Row<D> x, gamma, val;
    x.load(src, lane);
    if (values_from == 0) val.load(src + static_cast<size_t>(a.n_head_kv) * D, lane);
    gamma.load(a.k_norm, lane);
    const int p = a.row_pos[r], cell = a.row_cell[r];
    if (!has_cell(a, plan, r, p, cell)) return;
    Turn<D> turn(a.rope_dims, lane);
    if (a.rope_dims > 0) {
        turn.load(a.rope + static_cast<size_t>(p) * a.rope_dims, a.rope_dims);
        turn.settle();
    }
    uint16_t kx[VEC];
    cell_key<D>(x, gamma, turn, a.rope_dims, a.eps, kx);
    const size_t kvw = static_cast<size_t>(a.n_head_kv) * D;
    put_bytes<2 * VEC>(static_cast<uint16_t *>(a.kpages) + cell * kvw + head * D + VEC * lane, kx);
    if (values_from > 0) return;
    uint16_t *vd = static_cast<uint16_t *>(a.vpages) + (cell / kTile * kvw + static_cast<size_t>(head) * D + VEC * lane) * kTile + cell % kTile;
#pragma unroll
    for (int v = 0; v < VEC; v++) vd[v * kTile] = __half_as_ushort(__float2half_rn(val.x[v]));
}

// ---- attention ----------------------------------------------------------------------------------
// A tile in LDS, as loads of 1 KB leave it.  K cell by cell, so that a load takes whole rows of a head (3 % less, when this
// kernel came to it, for 24 tokens of 128 dims behind up to 12000 than where a load takes 64 bytes of sixteen rows); the 16-byte pieces of a cell's row lie in the order
// piece ^ turn(cell), so that the lanes of a read, (n, q) = cell 8 (n / 4) + 4 T + n % 4, piece 4 i + q, ask for different banks, whichever sixteen of them go
// together.  V chunk db behind them: lane (n, q) = dim 16 db + n, cells 8 q ...  After S^T = K Q^T lane (n, q) then holds query row n's
// scores of cells 8 q + 4 T + 0..3, T = 0, 1: the eight cells of its operand of the second product.
template <int D>
__device__ __forceinline__ int turn_of(int cell) {
    const int n = cell >> 3 << 2 | (cell & 3);
    return D == 64 ? n >> 1 : n;  // (two cells' rows of 64 dims lie in one line of banks)
}
template <int D, int WAVES>
struct AttnSmem {
    static constexpr int kStage = D / 8 * kChunk, kStages = ring_bytes(WAVES) / kStage;
    char ring[kStages][kStage];
    float p[WAVES][16 * kTile / 2];  // a wave's weights of half a tile, where its values are not all finite
};

// Waits until no more than the youngest min(rounds, N) rounds' loads of a wave, PER each, are out: they complete in order.
template <int PER, int N>
__device__ __forceinline__ void wait_but(int rounds) {
    if constexpr (N == 0) {
        wait_loads<0>();
    } else if (rounds >= N) {
        wait_loads<PER * N>();
    } else {
        wait_but<PER, N - 1>(rounds);
    }
}

// What a block is to its pieces.
struct Unit {
    int kvh, rep;
    size_t kvw;
    const uint16_t *cells;  // the KV head's keys or values, whichever the wave loads
    uint32_t from[2];       // where a lane's loads begin in a tile, of even and of odd ones
    uint32_t step;          // how far the next of the same kind is behind it
    uint32_t flip;          // and what the place of a key's pieces differs by, eight cells on
    bool keys;
};

__device__ __forceinline__ void load_8(float (&to)[8], const float *from) {
    const float4 a = *reinterpret_cast<const float4 *>(from), b = *reinterpret_cast<const float4 *>(from + 4);
    to[0] = a.x, to[1] = a.y, to[2] = a.z, to[3] = a.w, to[4] = b.x, to[5] = b.y, to[6] = b.z, to[7] = b.w;
}

__device__ __forceinline__ void store_8(float *to, const float (&from)[8]) {
    *reinterpret_cast<float4 *>(to) = make_float4(from[0], from[1], from[2], from[3]);
    *reinterpret_cast<float4 *>(to + 4) = make_float4(from[4], from[5], from[6], from[7]);
}

// Values as two halves, the large one cut off and not rounded (two in one instruction): the small one holds the rest either way, to 2^-22 of the value, and is rounded to
// nearest, so that what many cells lose cancels.
__device__ __forceinline__ void to_halves(const float (&x)[8], half8_t &hi, half8_t &lo) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const half2_t h = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(x[e], x[e + 1]));
        hi[e] = h[0], hi[e + 1] = h[1];
        lo[e] = static_cast<_Float16>(fmaf(static_cast<float>(h[0]), -1.f, x[e])), lo[e + 1] = static_cast<_Float16>(fmaf(static_cast<float>(h[1]), -1.f, x[e + 1]));
    }
}

// The rotation of a lane's dims where the two of a pair are 32 H apart, in one lane.
template <int H, int KI>
__device__ __forceinline__ void turn_in_lane(float (&x)[KI][8], const float (&c)[KI / 2][8], const float (&s)[KI / 2][8], int rope_dims) {
    if constexpr (2 * H <= KI) {
        if (rope_dims != 64 * H) return;
#pragma unroll
        for (int i = 0; i < H; i++)
#pragma unroll
            for (int t = 0; t < 8; t++) {
                const float a = x[i][t], b = x[i + H][t];
                x[i][t] = fmaf(-b, s[i][t], a * c[i][t]);
                x[i + H][t] = fmaf(a, s[i][t], b * c[i][t]);
            }
    }
}

// One piece.  A wave takes G groups of query rows; TP waves share a group, each takes every TP-th tile, and their sums are joined in LDS at the end.
template <int D, int G, int TP, int WAVES>
__device__ __forceinline__ void run_piece(const shv_attn_paged_args &a, const Plan &plan, const Piece &piece, const Unit &unit, AttnSmem<D, WAVES> &sm) {
    constexpr int KI = D / 32, DB = D / 16;
    constexpr int kPer = D / 8 / WAVES;  // chunks of a tile a wave asks for
    constexpr int kStages = AttnSmem<D, WAVES>::kStages, kRounds = kStages / TP;  // rounds of TP tiles in the ring: one is multiplied, the others are on their way
    constexpr int kBatch = 4 / G;
    static_assert(G == 1 || TP == 1, "waves that share a group have one");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, q = lane >> 4, rep = unit.rep, kvh = unit.kvh;
    const int mine_of = wave % TP;  // which tile of a round
    const int r0 = piece.r0 + 16 * G * (wave / TP), r_end = piece.r_end;
    const int last = min(piece.r0 + plan.rows, r_end) - 1;
    const bool working = r0 <= last;
    const int lo = piece.pos + plan.over_rep(piece.r0), hi = piece.pos + plan.over_rep(last);  // the block's rows' positions
    const Tiles tiles(a.window, a.sinks, lo, hi);
    const float c2 = 1.44269504088896f / sqrtf(static_cast<float>(D));
    int my_pos[G];  // (a row that is not there is the last one again, and dropped)
    // The table's entries around the tiles asked for last, one a lane.
    const int32_t *table = a.table + static_cast<size_t>(piece.seq) * a.max_pages;
    int held = 0, page0 = -64;
    uint32_t valid = 0;  // of the stages: the tile lies in a page
    const int n_tiles = piece.t1 - piece.t0, rounds = (n_tiles + TP - 1) / TP;
    const auto ask = [&](int round) {
#pragma unroll
        for (int t = 0; t < TP; t++) {
            const int j = round * TP + t, tile = tiles.at(piece.t0 + min(j, n_tiles - 1)), entry = tile >> (plan.shift - 5);
            if (static_cast<uint32_t>(entry - page0) >= 64u) {
                page0 = entry;
                held = table[min(entry + lane, a.max_pages - 1)];
            }
            const int page = __builtin_amdgcn_readlane(held, entry - page0);
            const bool is = page >= 0 && page < a.n_pages;
            const uint32_t bit = 1u << (j & (kStages - 1));
            valid = is && j < n_tiles ? valid | bit : valid & ~bit;
            const size_t cell = (static_cast<size_t>(is ? page : 0) << plan.shift) + (tile * kTile & (a.page - 1));
            const __amdgpu_buffer_rsrc_t bytes =
                __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(unit.cells + cell * unit.kvw), 0, static_cast<uint32_t>(kTile * unit.kvw) * 2, 0x00027000);
            char *to = sm.ring[j & (kStages - 1)] + (wave * kPer) * kChunk;
#pragma unroll
            for (int u = 0; u < kPer; u++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(bytes, (lds_ptr_t)(to + u * kChunk), 16, u / 2 * (1024 / D) & 8 ? unit.from[u & 1] ^ unit.flip : unit.from[u & 1], u / 2 * unit.step, 0, 0);
        }
    };
    const int cell_of = 8 * (n >> 2) + (n & 3), key_at = cell_of * 2 * D + (q ^ turn_of<D>(cell_of)) * 16;
    // ---- queries: lane (n, q) holds dims 32 i + 8 q .. of its row from the load to the operand ----
    int rope_dims = a.rope_dims, dim0 = 8 * q;
    asm volatile("" : "+s"(rope_dims), "+v"(dim0));  // (what follows from them is formed here and not once for all pieces, which registers do not hold)
    float x[G][KI][8];
    const bool by_lds = rope_dims % 64 != 0 || rope_dims == 192;  // a rotated pair's dims lie in two lanes: they meet in the ring, before any tile is asked for
    float gamma[KI][8], cosines[G][KI / 2][8], sines[G][KI / 2][8];
#pragma unroll
    for (int g = 0; g < G; g++) {
        const int mine = min(r0 + 16 * g + n, last), row = plan.over_rep(mine);
        my_pos[g] = piece.pos + row;
        const float *src = a.qkv + static_cast<size_t>(piece.first + row) * a.qkv_stride + static_cast<size_t>(kvh * rep + mine - row * rep) * 2 * D + dim0;
#pragma unroll
        for (int i = 0; i < KI; i++) load_8(x[g][i], src + 32 * i);
    }
#pragma unroll
    for (int i = 0; i < KI; i++) load_8(gamma[i], a.q_norm + 32 * i + dim0);
    if (!by_lds) {
        // (loads complete in order: all that the queries need goes out before the tiles do)
#pragma unroll
        for (int g = 0; g < G; g++) {
            const float *turn = a.rope + static_cast<size_t>(my_pos[g]) * rope_dims + dim0;
#pragma unroll
            for (int i = 0; i < KI / 2; i++)
                if (64 * i < rope_dims) {
                    load_8(cosines[g][i], turn + 32 * i);
                    load_8(sines[g][i], turn + rope_dims / 2 + 32 * i);
                }
        }
    }
    const int early = min(rounds, kRounds - 1);
    if (!by_lds)
        for (int r = 0; r < early; r++) ask(r);
#pragma unroll
    for (int g = 0; g < G; g++) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < KI; i++)
#pragma unroll
            for (int t = 0; t < 8; t++) ss = fmaf(x[g][i][t], x[g][i][t], ss);
        const float sc = __builtin_amdgcn_rsqf(fmaf(sum_over_q(ss), 1.f / static_cast<float>(D), a.eps));
#pragma unroll
        for (int i = 0; i < KI; i++) {
#pragma unroll
            for (int t = 0; t < 8; t++) x[g][i][t] *= sc * gamma[i][t];
        }
        turn_in_lane<1>(x[g], cosines[g], sines[g], rope_dims);
        turn_in_lane<2>(x[g], cosines[g], sines[g], rope_dims);
        turn_in_lane<4>(x[g], cosines[g], sines[g], rope_dims);
    }
    if (by_lds) {
        // (loops, and pairs turned where they lie: this path is for the layouts that are rare, and the instruction cache is shared with the one that is not)
        const uint32_t half = rope_dims / 2;
        float *rows = reinterpret_cast<float *>(sm.ring[0]) + wave * G * 16 * D;
        static_assert(WAVES * G * 16 * D * 4 <= ring_bytes(WAVES), "all rows in the ring");
#pragma unroll
        for (int g = 0; g < G; g++) {
            float *own = rows + (16 * g + n) * D + dim0;
#pragma unroll
            for (int i = 0; i < KI; i++) store_8(own + 32 * i, x[g][i]);
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (uint32_t k = lane; k < 16 * half; k += 64) {
                const uint32_t row = k / half, e = k - row * half;
                const float *factors = a.rope + static_cast<size_t>(__shfl(my_pos[g], static_cast<int>(row), 64)) * rope_dims;
                float *pair = rows + (16 * g + row) * D + e;
                const float c = factors[e], s = factors[half + e], u = pair[0], v = pair[half];
                pair[0] = fmaf(-v, s, u * c);
                pair[half] = fmaf(u, s, v * c);
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < KI; i++) load_8(x[g][i], own + 32 * i);
        }
        __syncthreads();
        for (int r = 0; r < early; r++) ask(r);
    }
    half8_t qh[G][KI], ql[G][KI];
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int i = 0; i < KI; i++) to_halves(x[g][i], qh[g][i], ql[g][i]);
    __builtin_amdgcn_sched_barrier(0);
    float4_t o[G][DB];
    float m_run[G], l_run[G];  // of the scores as they are, before their scale; the sums of a lane's own cells
    bool far = false;          // a maximum is past kFar
    uint32_t saw = 0;          // bit g: one of the lane's cells is one that its row sees
#pragma unroll
    for (int g = 0; g < G; g++) {
        m_run[g] = -INFINITY, l_run[g] = 0.f;
#pragma unroll
        for (int db = 0; db < DB; db++) o[g][db] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    for (int r = 0; r < rounds; r++) {
        const int j = r * TP + mine_of;
        const char *kt = sm.ring[j & (kStages - 1)];
        wait_but<kPer * TP, kRounds - 2>(rounds - 1 - r);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // everyone's: these tiles are whole, and those before have been read
        const bool is = valid >> (j & (kStages - 1)) & 1;
        if (r + kRounds - 1 < rounds) ask(r + kRounds - 1);
        if (!is || !working) continue;
        const int c0 = tiles.at(piece.t0 + j) * kTile;
        uint32_t seen[G];  // which of the lane's eight cells its query row sees
        const bool part = c0 + kTile - 1 > lo || (a.window > 0 && c0 + kTile - 1 >= a.sinks && c0 <= hi - a.window);
        int first_cell = lane;
        asm volatile("" : "+v"(first_cell));  // (here and in what follows: what is seldom needed is not formed for all tiles, which registers do not hold)
        first_cell = (first_cell >> 4) * 8;
#pragma unroll
        for (int g = 0; g < G; g++) {
            seen[g] = 0xFF;
            if (part) {
                seen[g] = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int c = c0 + first_cell + e;
                    seen[g] |= c <= my_pos[g] && (a.window == 0 || c < a.sinks || c > my_pos[g] - a.window) ? 1u << e : 0u;
                }
            }
            saw |= seen[g] != 0 ? 1u << g : 0u;
        }
        const char *vt = kt + 2 * KI * kChunk;
        // operands come from LDS eight products ahead of those that use them
        float4_t st[G][2], sl[G][2];
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
            for (int T = 0; T < 2; T++) st[g][T] = sl[g][T] = float4_t{0.f, 0.f, 0.f, 0.f};
        half8_t kb[2][kBatch];
        int key0 = key_at;
        asm volatile("" : "+v"(key0));
        const auto read_k = [&](half8_t(&to)[kBatch], int i) {
#pragma unroll
            for (int e = 0; e < kBatch; e++) {
                const int step = (kBatch * i + e) / 2;
                to[e] = *reinterpret_cast<const half8_t *>(kt + (key0 ^ (step & 3) * 64) + (e & 1) * 8 * D + step / 4 * 256);
            }
        };
        read_k(kb[0], 0);
#pragma unroll
        for (int i = 0; i < 2 * KI / kBatch; i++) {
            if (i + 1 < 2 * KI / kBatch) read_k(kb[(i + 1) & 1], i + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < kBatch; e++)
#pragma unroll
                for (int g = 0; g < G; g++) {
                    st[g][e & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb[i & 1][e], qh[g][(kBatch * i + e) / 2], st[g][e & 1], 0, 0, 0);
                    sl[g][e & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb[i & 1][e], ql[g][(kBatch * i + e) / 2], sl[g][e & 1], 0, 0, 0);
                }
        }
        float pv[G][8];
        bool by_hand = false;
#pragma unroll
        for (int g = 0; g < G; g++) {
            float mx = -INFINITY;
            float(&s)[8] = pv[g];
#pragma unroll
            for (int e = 0; e < 8; e++) s[e] = st[g][e >> 2][e & 3] + sl[g][e >> 2][e & 3];
            if (part) {
#pragma unroll
                for (int e = 0; e < 8; e++) s[e] = seen[g] >> e & 1 ? s[e] : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) mx = fmaxf(mx, s[e]);
            mx = max_over_q(mx);
            // the sums are rescaled a few times a run instead of whenever some row's maximum moves
            const bool moves = (mx - m_run[g]) * c2 > kSlack;  // (infinity less infinity: no)
            if (__ballot(moves) != 0ull) {
                const float m_new = moves ? mx : m_run[g];
                const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_run[g] - m_new) * c2);
                l_run[g] *= alpha;
                m_run[g] = m_new;
                far |= __ballot(moves && fabsf(mx) * c2 > kFar) != 0ull;
                float av[4];
                int l = lane;
                asm volatile("" : "+v"(l));
#pragma unroll
                for (int e = 0; e < 4; e++) av[e] = __shfl(alpha, (l >> 4) * 4 + e, 64);
#pragma unroll
                for (int db = 0; db < DB; db++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[g][db][e] *= av[e];
            }
        }
        if (__builtin_expect(far, 0)) {
            // (the difference first)
#pragma unroll
            for (int g = 0; g < G; g++) {
                const float m0 = m_run[g] == -INFINITY ? 0.f : m_run[g];
#pragma unroll
                for (int e = 0; e < 8; e++) pv[g][e] = __builtin_amdgcn_exp2f(fmaf(pv[g][e] - m0, c2, kLift));
            }
        } else {
#pragma unroll
            for (int g = 0; g < G; g++) {
                const float m2 = fmaf(m_run[g] == -INFINITY ? 0.f : m_run[g], c2, -kLift);
#pragma unroll
                for (int e = 0; e < 8; e++) pv[g][e] = __builtin_amdgcn_exp2f(fmaf(pv[g][e], c2, -m2));
            }
        }
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
            for (int e = 0; e < 8; e++) l_run[g] += pv[g][e];
        if (part) {
            // a value that is not finite would meet the weight 0 of rows that do not see it: such a tile is multiplied by hand
            uint32_t odd = 0;
#pragma unroll
            for (int db = 0; db < DB; db++) {
                const uint4 v = *reinterpret_cast<const uint4 *>(vt + db * kChunk + lane * 16);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; e++) odd |= ((w[e] & 0x7C007C00u) + 0x04000400u) & 0x80008000u;  // an exponent of ones carries into the sign
            }
            by_hand = __ballot(odd != 0) != 0ull;
        }
        if (by_hand) {
            float *p = sm.p[wave];
            int l = lane;
            asm volatile("" : "+v"(l));
            const int nn = l & 15, qq = l >> 4;
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll 1
                for (int half = 0; half < 2; half++) {
                    if ((qq >> 1) == half) {
#pragma unroll
                        for (int e = 0; e < 8; e++) p[nn * (kTile / 2) + 8 * (qq & 1) + e] = seen[g] >> e & 1 ? pv[g][e] : -1.f;
                    }
                    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
                    for (int i = 0; i < kTile / 2; i++) {
                        const int c = kTile / 2 * half + i;
                        float w[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) w[e] = p[(4 * qq + e) * (kTile / 2) + i];
#pragma unroll
                        for (int db = 0; db < DB; db++) {
                            const float v = static_cast<float>(*reinterpret_cast<const _Float16 *>(vt + db * kChunk + (16 * (c >> 3) + nn) * 16 + (c & 7) * 2));
#pragma unroll
                            for (int e = 0; e < 4; e++) o[g][db][e] = w[e] < 0.f ? o[g][db][e] : fmaf(w[e], v, o[g][db][e]);
                        }
                    }
                    __builtin_amdgcn_wave_barrier();
                }
            continue;
        }
        half8_t ph[G], pl[G];
#pragma unroll
        for (int g = 0; g < G; g++) to_halves(pv[g], ph[g], pl[g]);
        half8_t vb[2][kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; e++) vb[0][e] = *reinterpret_cast<const half8_t *>(vt + e * kChunk + lane * 16);
#pragma unroll
        for (int i = 0; i < DB / kBatch; i++) {
            if (i + 1 < DB / kBatch) {
#pragma unroll
                for (int e = 0; e < kBatch; e++) vb[(i + 1) & 1][e] = *reinterpret_cast<const half8_t *>(vt + (kBatch * (i + 1) + e) * kChunk + lane * 16);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int e = 0; e < kBatch; e++) o[g][kBatch * i + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[g], vb[i & 1][e], o[g][kBatch * i + e], 0, 0, 0);
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int e = 0; e < kBatch; e++) o[g][kBatch * i + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[g], vb[i & 1][e], o[g][kBatch * i + e], 0, 0, 0);
        }
    }
    bool writes = working;
    if constexpr (TP > 1) {
        // the sums of a group's other waves, by way of the ring, which is free
        constexpr int kOthers = WAVES / TP * (TP - 1);  // waves that leave theirs
        static_assert(kOthers * (DB + 1) * kChunk <= ring_bytes(WAVES), "they fit the ring");
        float4_t *slots = reinterpret_cast<float4_t *>(sm.ring[0]) + wave / TP * (TP - 1) * (DB + 1) * 64 + lane;
        __syncthreads();
        if (working && mine_of > 0) {
            float4_t *slot = slots + (mine_of - 1) * (DB + 1) * 64;
#pragma unroll
            for (int db = 0; db < DB; db++) slot[db * 64] = o[0][db];
            slot[DB * 64] = float4_t{m_run[0], l_run[0], __uint_as_float(saw), 0.f};
        }
        __syncthreads();
        writes = working && mine_of == 0;
        if (writes) {
#pragma unroll 1
            for (int k = 0; k < TP - 1; k++) {
                const float4_t *slot = slots + k * (DB + 1) * 64;
                const float4_t of = slot[DB * 64];
                const float m = fmaxf(m_run[0], of[0]);
                const float f1 = m_run[0] == m ? 1.f : __builtin_amdgcn_exp2f((m_run[0] - m) * c2), f2 = of[0] == m ? 1.f : __builtin_amdgcn_exp2f((of[0] - m) * c2);
                l_run[0] = f1 * l_run[0] + f2 * of[1];
                m_run[0] = m;
                saw |= __float_as_uint(of[2]);
                float a1[4], a2[4];
#pragma unroll
                for (int e = 0; e < 4; e++) a1[e] = __shfl(f1, 4 * q + e, 64), a2[e] = __shfl(f2, 4 * q + e, 64);
#pragma unroll
                for (int db = 0; db < DB; db++) {
                    const float4_t other = slot[db * 64];
#pragma unroll
                    for (int e = 0; e < 4; e++) o[0][db][e] = a1[e] * o[0][db][e] + a2[e] * other[e];
                }
            }
        }
    }
    if (writes) {
        int l = lane;
        asm volatile("" : "+v"(l));
        const int nn = l & 15, qq = l >> 4;
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int rg = r0 + 16 * g;
            if (rg > last) break;
            float sum = sum_over_q(l_run[g]);
            // a row whose scores are all -infinity has no weights; one that sees nothing has a sum of zero
            const uint64_t saws = __ballot(saw >> g & 1);
            if (m_run[g] == -INFINITY && ((saws >> nn) & 0x0001000100010001ull) != 0) sum = __int_as_float(0x7fc00000);
            if (piece.rec < 0) {
                float lr[4];
#pragma unroll
                for (int i = 0; i < 4; i++) lr[i] = __shfl(sum == 0.f ? 0.f : 1.f / sum, 4 * qq + i, 64);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = rg + 4 * qq + i, row = plan.over_rep(r);
                    if (r > last) continue;
                    float *dst = a.out + (static_cast<size_t>(piece.first + row) * a.n_head + kvh * rep + r - row * rep) * D;
#pragma unroll
                    for (int db = 0; db < DB; db++) dst[16 * db + nn] = o[g][db][i] * lr[i];
                }
            } else {
                const size_t base = (static_cast<size_t>(piece.rec) * a.n_head_kv + kvh) * plan.slot_rows + rg - piece.r0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (rg + 4 * qq + i > last) continue;
                    float *rec = plan.sums + (base + 4 * qq + i) * D;
#pragma unroll
                    for (int db = 0; db < DB; db++) rec[16 * db + nn] = o[g][db][i];
                }
                if (qq == 0 && rg + nn <= last) plan.of[base + nn] = make_float2(m_run[g], sum);
            }
        }
    }
    __syncthreads();  // the stages are free for the next piece
}

// Bound by memory where query rows are few (24 tokens of 128 dims behind up to 12000 read 5.5 TB/s, 40 of 256 behind up to 9000 5.0 while the kernel runs), by the
// matrix units where they are many: a chunk of 2048 behind 8000, 128 dims, runs at 1100 TFLOP/s of products, both halves counted, where a large library product reaches 1295.
//
// grid: 8 * ceil(blocks / dies) * heads.  Workgroups go to the eight dies in turn; a die's KV heads are the same ones throughout, where their number
// allows it, so that its L2 holds their cells: die x has the heads x % g, x % g + g, .. for g the power of two in their number, up to 8.
template <int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void paged_attn_kernel(shv_attn_paged_args a, Plan plan) {
    constexpr int kPer = D / 8 / WAVES;
    extern __shared__ __align__(16) char raw[];
    AttnSmem<D, WAVES> &sm = *reinterpret_cast<AttnSmem<D, WAVES> *>(raw);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, q = lane >> 4;
    const int die = blockIdx.x & 7, nth = blockIdx.x >> 3, g = 8 / plan.dies;
    const int turn = static_cast<int>(static_cast<uint32_t>(nth) / static_cast<uint32_t>(plan.heads)), slot = turn * plan.dies + die / g;
    if (slot >= plan.most_blocks) return;
    const Block *block = plan.blocks + slot;
    const int pieces = block->more + 1;
    const Piece *at = &block->piece;
    Unit unit;
    unit.kvh = die % g + g * (nth - turn * plan.heads), unit.rep = plan.rep;
    unit.kvw = static_cast<size_t>(a.n_head_kv) * D;
    unit.keys = wave < WAVES / 2;
    // loads u of the wave: of keys 1024 / 2 D cells each, of values 16 dims
    const int mine = unit.keys ? wave : wave - WAVES / 2;
    constexpr int kPieces = D / 8, kCells = 64 / kPieces;
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const int cell = (mine * kPer + u) * kCells + lane / kPieces;
        unit.from[u] = unit.keys ? static_cast<uint32_t>(cell * unit.kvw) * 2 + ((lane % kPieces) ^ turn_of<D>(cell)) * 16 : static_cast<uint32_t>((16 * (mine * kPer + u) + n) * kTile + 8 * q) * 2;
    }
    unit.step = unit.keys ? 2 * kCells * static_cast<uint32_t>(unit.kvw) * 2 : 2 * kChunk;
    unit.flip = unit.keys ? 64 : 0;
    static_assert(kPer <= 2 || (D > 64 && kPer * kCells <= 16), "eight cells on, turn_of differs by 4: 64 bytes");
    unit.cells = unit.keys ? static_cast<const uint16_t *>(a.kpages) + unit.kvh * D : static_cast<const uint16_t *>(a.vpages) + static_cast<size_t>(unit.kvh) * D * kTile;
    for (int k = 0; k < pieces; k++) {
        const Piece piece = *at;
        at = k == 0 ? plan.pieces + block->at : at + 1;
        const int groups = (min(piece.r_end - piece.r0, plan.rows) + 15) / 16;
        constexpr int kShared = kTurns<D, WAVES>;
        if constexpr (kShared > 1) {
            if (groups <= WAVES / kShared) {
                run_piece<D, 1, kShared, WAVES>(a, plan, piece, unit, sm);
                continue;
            }
        }
        run_piece<D, kGroups<D>, 1, WAVES>(a, plan, piece, unit, sm);
    }
}

// ---- the join -----------------------------------------------------------------------------------
// Weighted sums of the records: bound by the trips to memory (plan, records, sums) where there are few, 3.2 us for one token behind 900, and by their bytes from the other dies' writes
// otherwise, 4 to 25 us.  A unit is 256 / D query rows of a KV head, a lane four dims.  SHARE, where a query row has many records: a block's four waves share them, otherwise each takes a unit
// of its own.
template <int D, bool SHARE>
__global__ __launch_bounds__(256) void paged_join_kernel(shv_attn_paged_args a, Plan plan) {
    __shared__ float4_t sums[4][64];
    __shared__ float2 of[4][64];
    constexpr int kLanes = D / 4, kUnit = 64 / kLanes, kPerHead = 16 / kUnit;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rep = plan.rep;
    const float c2 = 1.44269504088896f / sqrtf(static_cast<float>(D));
    const uint32_t per = kPerHead * a.n_head_kv, units = per * *plan.n_joins;
    const uint32_t step = SHARE ? gridDim.x : gridDim.x * 4;
    for (uint32_t unit = SHARE ? blockIdx.x : blockIdx.x * 4 + wave; unit < units; unit += step) {
        const uint32_t k = unit / per, in = unit - k * per, kvh = in / kPerHead, u = in % kPerHead;
        const Join join = plan.joins[k];
        const int local = u * kUnit + lane / kLanes, r = join.r0 + local;
        const bool there = r < join.r_end;
        if (__ballot(there) == 0ull) continue;  // (the same in every wave that shares)
        const size_t row = (static_cast<size_t>(join.rec) * a.n_head_kv + kvh) * plan.slot_rows + join.in + (there ? local : 0), stride = static_cast<size_t>(a.n_head_kv) * plan.slot_rows;
        const float4_t *from = reinterpret_cast<const float4_t *>(plan.sums + row * D) + lane % kLanes;
        const float2 *from_of = plan.of + row;
        constexpr int MB = 8;
        float4_t num = {0.f, 0.f, 0.f, 0.f};
        float den = 0.f, M = -INFINITY;
        const auto fold = [&](const float4_t &v, float2 ml) {
            if (ml.x == -INFINITY && ml.y == 0.f) return;  // (sees nothing; a sum of NaN stays)
            const float Mn = fmaxf(M, ml.x);
            const float shrink = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((M - Mn) * c2), w = ml.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((ml.x - Mn) * c2);
            den = fmaf(den, M == -INFINITY ? 1.f : shrink, w * ml.y);
#pragma unroll
            for (int e = 0; e < 4; e++) num[e] = fmaf(num[e], shrink, w * v[e]);
            M = Mn;
        };
        constexpr int waves = SHARE ? 4 : 1;
        const int me = SHARE ? wave : 0;
        for (int s0 = me; s0 < join.n; s0 += waves * MB) {
            float4_t v[MB];
            float2 ml[MB];
#pragma unroll
            for (int i = 0; i < MB; i++) {
                const size_t s = s0 + waves * i < join.n ? s0 + waves * i : s0;
                v[i] = from[s * stride * kLanes];
                ml[i] = from_of[s * stride];
            }
#pragma unroll
            for (int i = 0; i < MB; i++) asm volatile("" : "+v"(v[i]));  // asked for together, not each behind the one before's test
#pragma unroll
            for (int i = 0; i < MB; i++)
                if (s0 + waves * i < join.n) fold(v[i], ml[i]);
        }
        if constexpr (SHARE) {
            __syncthreads();
            sums[wave][lane] = num;
            of[wave][lane] = make_float2(M, den);
            __syncthreads();
            if (wave != 0) continue;
#pragma unroll
            for (int w = 1; w < 4; w++) fold(sums[w][lane], of[w][lane]);
        }
        if (there) {
            float4_t y;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = den == 0.f ? 0.f : num[e] / den;
            const int t = plan.over_rep(r);
            *(reinterpret_cast<float4_t *>(a.out + (static_cast<size_t>(join.first + t) * a.n_head + kvh * rep + r - t * rep) * D) + lane % kLanes) = y;
        }
    }
}

// ---- the launcher -------------------------------------------------------------------------------
int check_sizes(const shv_attn_paged_args &a) {
    SHV_REQUIRE(a.n_seq >= 1 && a.n_seq <= SHV_PAGE_MAX_SEQS, "attn_paged: %d sequences; 1..%d", a.n_seq, SHV_PAGE_MAX_SEQS);
    SHV_REQUIRE(a.head_dim == 64 || a.head_dim == 128 || a.head_dim == 256, "attn_paged: head_dim %d; 64, 128 or 256", a.head_dim);
    SHV_REQUIRE(a.n_head_kv >= 1 && a.n_head >= 1 && a.n_head % a.n_head_kv == 0 && a.n_head / a.n_head_kv <= 64 && a.n_head <= 1024,
                "attn_paged: %d query heads over %d KV heads; 1..64 per KV head, 1024 in all", a.n_head, a.n_head_kv);
    SHV_REQUIRE(a.max_rows >= 1 && static_cast<long long>(a.max_rows) * (a.n_head / a.n_head_kv) <= 1 << 20, "attn_paged: %d rows of %d query heads per KV head; at most 2^20 together",
                a.max_rows, a.n_head / a.n_head_kv);
    // (of the cells' launch: 96 threads at most for each, fewer than 2^32 in all)
    SHV_REQUIRE(static_cast<long long>(a.max_rows) * a.n_head_kv <= 1 << 25, "attn_paged: %d rows of %d KV heads; at most 2^25 together", a.max_rows, a.n_head_kv);
    SHV_REQUIRE(a.page >= 32 && a.page <= 4096 && (a.page & (a.page - 1)) == 0, "attn_paged: page %d; a power of two from 32 to 4096", a.page);
    SHV_REQUIRE(a.n_pages >= 1 && static_cast<long long>(a.n_pages) * a.page < 1ll << 31, "attn_paged: %d pages of %d cells; fewer than 2^31 cells", a.n_pages, a.page);
    SHV_REQUIRE(a.max_pages >= 1 && static_cast<long long>(a.max_pages) * a.page < 1ll << 31, "attn_paged: max_pages %d of %d cells; fewer than 2^31 cells", a.max_pages, a.page);
    return SHV_OK;
}

// Blocks of eight waves read a tile for twice the query rows, which pays where a sequence has many of them and 256 dims: a chunk of 512 behind 7500, rep 8, takes 137 us
// with them and 146 with blocks of four, 256 behind 3000 52.7 and 55.6, 100 behind 2000 40.6 and 35.3, one token behind 900 19.8 and 18.  Of 128 dims a block of four has as many
// rows already: 2048 behind 8000 take 584 and 592, and all others are better with four.  And where blocks of four could be more than a plan holds, which those of eight never are.
constexpr int kWideFrom = 2048;  // query rows of a KV head, on average over the sequences
// Query blocks of `rows` query rows, at most: a sequence's last one may be short.
int most_query_blocks(const shv_attn_paged_args &a, int rows) { return (a.n_seq < a.max_rows ? a.n_seq : a.max_rows) + a.max_rows * (a.n_head / a.n_head_kv) / rows; }
bool is_wide(const shv_attn_paged_args &a) {
    return a.head_dim == 256 && (static_cast<long long>(a.max_rows) * (a.n_head / a.n_head_kv) >= static_cast<long long>(kWideFrom) * a.n_seq ||
                                 most_query_blocks(a, rows_of(256, kNarrow)) > kMostBlocks);
}

// The scratch of a call of these sizes, laid out from `work` on; its end is the bytes that it takes.
uintptr_t lay_out(const shv_ctx *ctx, const shv_attn_paged_args &a, Plan &plan) {
    const int rep = a.n_head / a.n_head_kv, D = a.head_dim;
    plan.waves = is_wide(a) ? kWide : kNarrow;
    plan.slots = ctx->prop.multiProcessorCount * (kWide / plan.waves) / a.n_head_kv;
    if (plan.slots < 1) plan.slots = 1;
    if (plan.slots > kMaxSlots) plan.slots = kMaxSlots;
    plan.rep_magic = rep == 1 ? 0 : static_cast<uint32_t>(((1ull << 32) + rep - 1) / rep);
    plan.rep = rep;
    const int query_rows = a.max_rows * rep;
    plan.rows = rows_of(D, plan.waves);
    plan.most_q = most_query_blocks(a, plan.rows);
    const int g = a.n_head_kv & 7 ? a.n_head_kv & -a.n_head_kv : 8;
    plan.dies = 8 / g, plan.heads = a.n_head_kv / g;
    plan.most_blocks = ((plan.most_q > plan.slots ? plan.most_q : plan.slots) + plan.dies - 1) / plan.dies * plan.dies;
    plan.slot_rows = query_rows < plan.rows ? (query_rows + 15) / 16 * 16 : plan.rows;
    plan.shift = 0;
    while (1 << plan.shift < a.page) plan.shift++;
    // a cut query block has a piece more than cuts, and there are fewer cuts than slots
    const size_t pieces = static_cast<size_t>(plan.most_q) + plan.slots, joins = plan.rows / 16 * static_cast<size_t>(plan.most_q < plan.slots ? plan.most_q : plan.slots);
    const size_t records = 2 * static_cast<size_t>(plan.slots) * a.n_head_kv * plan.slot_rows;
    uintptr_t at = reinterpret_cast<uintptr_t>(a.work);
    const auto take = [&](size_t bytes) {
        char *here = reinterpret_cast<char *>(at);
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    plan.n_joins = reinterpret_cast<int32_t *>(take(4));
    plan.blocks = reinterpret_cast<Block *>(take(plan.most_blocks * sizeof(Block)));
    plan.pieces = reinterpret_cast<Piece *>(take(pieces * sizeof(Piece)));
    plan.joins = reinterpret_cast<Join *>(take(joins * sizeof(Join)));
    plan.of = reinterpret_cast<float2 *>(take(records * 8));
    plan.sums = reinterpret_cast<float *>(take(records * D * 4));
    return at;
}

template <int D>
int launch_paged(shv_ctx *ctx, const shv_attn_paged_args &a) {
    Plan plan;
    lay_out(ctx, a, plan);
    using BigSmem = PlanSmem<1024, kMaxSeqs, kMostBlocks>;
    static std::atomic<uint64_t> raised{0};  // by device
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (!(raised.load(std::memory_order_acquire) & bit)) {
        if constexpr (D == 256)
            SHV_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(&paged_attn_kernel<D, kWide>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(AttnSmem<D, kWide>))));
        SHV_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(&paged_attn_kernel<D, kNarrow>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(AttnSmem<D, kNarrow>))));
        SHV_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(&paged_plan_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(BigSmem))));
        raised.fetch_or(bit, std::memory_order_release);
    }
    const unsigned row_blocks = static_cast<unsigned>((static_cast<long long>(a.max_rows) * a.n_head_kv + 3) / 4);
    const unsigned value_blocks = a.max_rows >= kValuesFrom ? static_cast<unsigned>((a.max_rows + kValuesRows - 1) / kValuesRows * ((a.n_head_kv * D + 255) / 256)) : 0u;
    if (plan.most_q <= kFewBlocks && a.n_seq <= kFewBlocks) {
        SHV_LAUNCH(ctx, (paged_cells_kernel<D, true>), dim3(row_blocks + 1 + value_blocks), dim3(256), 0, a, plan, value_blocks > 0 ? row_blocks + 1 : 0u);
    } else {
        SHV_LAUNCH(ctx, paged_plan_kernel, dim3(1), dim3(1024), sizeof(BigSmem), a, plan);
        SHV_LAUNCH(ctx, (paged_cells_kernel<D, false>), dim3(row_blocks + value_blocks), dim3(256), 0, a, plan, value_blocks > 0 ? row_blocks : 0u);
    }
    const dim3 blocks(plan.most_blocks / plan.dies * plan.heads * 8);
    if (plan.waves == kNarrow) {
        SHV_LAUNCH(ctx, (paged_attn_kernel<D, kNarrow>), blocks, dim3(64 * kNarrow), sizeof(AttnSmem<D, kNarrow>), a, plan);
    } else if constexpr (D == 256) {
        SHV_LAUNCH(ctx, (paged_attn_kernel<D, kWide>), blocks, dim3(64 * kWide), sizeof(AttnSmem<D, kWide>), a, plan);
    }
    const long long joins = plan.most_q < plan.slots ? plan.most_q : plan.slots, units = joins * a.n_head_kv * plan.slot_rows / (256 / D);
    const dim3 grid(static_cast<unsigned>(units < 2048 ? units : 2048));
    if (plan.slots >= kShareFrom * plan.most_q) SHV_LAUNCH(ctx, (paged_join_kernel<D, true>), grid, dim3(256), 0, a, plan);
    else SHV_LAUNCH(ctx, (paged_join_kernel<D, false>), grid, dim3(256), 0, a, plan);
    return SHV_OK;
}

}  // namespace

int shv_launch_attn_paged(shv_ctx *ctx, const shv_attn_paged_args *pa) {
    const shv_attn_paged_args &a = *pa;
    SHV_REQUIRE(a.qkv && a.q_norm && a.k_norm && a.kpages && a.vpages && a.table && a.start && a.row_pos && a.row_cell && a.work && a.out, "attn_paged: NULL argument");
    const int rc = check_sizes(a);
    if (rc != SHV_OK) return rc;
    SHV_REQUIRE(a.rope_dims >= 0 && a.rope_dims <= a.head_dim && a.rope_dims % (a.head_dim / 32) == 0,
                "attn_paged: rope_dims %d; a multiple of %d up to %d", a.rope_dims, a.head_dim / 32, a.head_dim);
    SHV_REQUIRE(a.rope || a.rope_dims == 0, "attn_paged: NULL rotary table");
    SHV_REQUIRE(a.qkv_stride >= (a.n_head + a.n_head_kv) * 2 * a.head_dim && a.qkv_stride % 4 == 0, "attn_paged: qkv_stride %d", a.qkv_stride);
    SHV_REQUIRE(a.window >= 0 && a.sinks >= 0, "attn_paged: window %d, sinks %d", a.window, a.sinks);
    SHV_REQUIRE(shv_aligned16(a.qkv) && shv_aligned16(a.q_norm) && shv_aligned16(a.k_norm) && shv_aligned16(a.rope) && shv_aligned16(a.kpages) && shv_aligned16(a.vpages) &&
                    shv_aligned16(a.work) && shv_aligned16(a.out),
                "attn_paged: qkv, norms, rotary table, pages, work and out must be 16-byte aligned");
    int64_t need = 0;
    if (shv_attn_paged_work(ctx, pa, &need) != SHV_OK) return SHV_E_INVALID;
    SHV_REQUIRE(a.work_bytes >= need, "attn_paged: %lld bytes of work; these sizes need %lld", static_cast<long long>(a.work_bytes), static_cast<long long>(need));
    if (a.head_dim == 256) return launch_paged<256>(ctx, a);
    if (a.head_dim == 128) return launch_paged<128>(ctx, a);
    return launch_paged<64>(ctx, a);
}

extern "C" int shv_attn_paged_work(shv_ctx *ctx, const shv_attn_paged_args *a, int64_t *bytes) {
    SHV_REQUIRE(ctx && a && bytes, "attn_paged_work: NULL argument");
    const int rc = check_sizes(*a);
    if (rc != SHV_OK) return rc;
    shv_attn_paged_args sizes = *a;
    sizes.work = nullptr;
    Plan plan;
    const int64_t need = static_cast<int64_t>(lay_out(ctx, sizes, plan));
    SHV_REQUIRE(plan.most_q <= kMostBlocks, "attn_paged: up to %d blocks of query rows; a plan holds %d", plan.most_q, kMostBlocks);
    *bytes = need;
    return SHV_OK;
}
