// Full attention of packed rows over a paged cache.
//
// Row r of a sequence, at position p_r, sees the sequence's cells c <= p_r that lie in a page (with a window those of them below `sinks` or above p_r - window):
//     out_r = sum over them of softmax(q_r . k_c / sqrt(d)) v_c
// q and k normed over a head and rotated at their positions.  Three launches:
//   rows   the rows' keys and values into their cells, their queries into matrix-core operands, and, in a block of its own, the plan of the next;
//   attn   a block takes one KV head and 128 query rows (query row r of a sequence is head r % rep of its row r / rep), 16 a wave, and a run of
//          their tiles of 32 cells, on v_mfma_f32_16x16x32_f16:
//              S^T = K Q^T   the cache's binary16 keys against the queries as two halves; a lane then holds eight cells of one query row, the operand
//                            of the second product
//              O  += P V     weights as two halves against values, which the cache holds by dim
//          with a running maximum and sum.  Tiles go from memory to LDS past the registers, three ahead;
//   join   the records of query rows whose tiles several blocks have shared.
#include <atomic>

#include "attn_rows.hpp"
#include "scan.hpp"
#include "shv_device.hpp"
#include "shv_internal.hpp"

namespace {

using namespace shv;

constexpr int kTile = 32;  // cells of a tile of V
constexpr int kWaves = 8, kRows = 16 * kWaves;  // waves of a block and its query rows
constexpr int kMaxSeqs = SHV_PAGE_MAX_SEQS;
constexpr int kChunk = 64 * 16;
constexpr int kStages = 4, kAhead = kStages - 1;
// Weights are e^(s - m) 2^kLift, and m stands until a score is more than kSlack powers of two above it: up to 2^15.9, which the larger half holds, and down to
// 2^-35 of the largest with the smaller half's last place, to which it is rounded.
constexpr float kLift = 11.f, kSlack = 4.9f;
constexpr int kLeast = 3;      // tiles a block gets at least
constexpr int kFewBlocks = 1024;  // query blocks up to which the plan is made inside the launch of the rows

// 128 query rows of a sequence and a run of the tiles they look at.
struct Piece {
    int seq, first;     // the sequence and its first packed row
    int r0, r_end;      // the first query row, and the sequence's number of them
    int pos;            // of the sequence's first row
    int t0, t1;         // the run
    int rec;            // where its records go; -1: it is all there is
};
struct Join {
    int first, r0, r_end, rec, n;
    int pad[3];
};
enum { kHeadBlocks = 0, kHeadCut = 1, kHeadJoins = 2, kHeadRecs = 3, kHeadWords = 16 };

// Where a call's scratch lies and what it can hold; worked out by the launcher from the sizes alone.
struct Plan {
    int32_t *head;
    int32_t *first_of;  // a block's first piece; of the last block's end too
    Piece *pieces;
    Join *joins;
    char *stage;        // queries: [KV head][packed row * rep + head of the group][large halves, small halves]
    float *sums;        // records: [record][KV head][slot_rows][D] unnormalised sums
    float2 *of;         // and their (maximum, sum)
    int slots;          // blocks a KV head that the chip holds at once
    int slot_rows;      // query rows of a record
    int most_blocks, most_q;
    int shift;          // log2 of the page
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
// The query blocks of all sequences stand in a row with the tiles each looks at, P their running sum.  With as many query blocks as fill the chip evenly
// each is a block's own, those with the most tiles first.  Otherwise block b takes the tiles b S .. (b + 1) S of the row, S = all / blocks, so that all blocks have
// the same; a query block cut by that leaves a record of each piece.
template <int T, int SEQS, int NQ>
struct PlanSmem {
    uint32_t q0[SEQS + 1];      // query blocks before a sequence's
    uint32_t p[NQ], at[NQ];     // tiles before a query block's; its first piece
    int rec[NQ];                // its first record, -1: it has one piece
    uint32_t waves[4][T / 64];
    uint32_t bucket[64];
    uint32_t most;
};
template <int T, int SEQS, int NQ>
__device__ void make_plan(const shv_attn_paged_args &a, const Plan &plan, PlanSmem<T, SEQS, NQ> &sm) {
    const int tid = threadIdx.x, rep = a.n_head / a.n_head_kv;
    uint32_t nq = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += T) {
        uint32_t v[1] = {0}, all[1];
        if (s0 + tid < a.n_seq) v[0] = (static_cast<uint32_t>(Seq(a, s0 + tid).n) * rep + kRows - 1) / kRows;
        block_scan<T, 1>(v, all, sm.waves);
        if (s0 + tid < a.n_seq) sm.q0[s0 + tid] = nq + v[0];
        nq += all[0];
    }
    if (tid == 0) sm.most = 0;
    if (tid < 64) sm.bucket[tid] = 0;
    __syncthreads();
    // query block i as a piece of all its tiles
    const auto whole = [&](uint32_t i) {
        Piece p;
        p.seq = last_not_above(sm.q0, a.n_seq, i);
        const Seq seq(a, p.seq);
        p.first = seq.first, p.pos = seq.pos, p.r_end = seq.n * rep;
        p.r0 = static_cast<int>(i - sm.q0[p.seq]) * kRows;
        const int last = min(p.r0 + kRows, p.r_end) - 1;
        p.t0 = 0, p.t1 = Tiles(a.window, a.sinks, p.pos + p.r0 / rep, p.pos + last / rep).all;
        p.rec = -1;
        return p;
    };
    nq = min(nq, static_cast<uint32_t>(min(plan.most_q, NQ)));
    uint32_t total = 0;
    for (uint32_t i0 = 0; i0 < nq; i0 += T) {
        uint32_t v[1] = {0}, all[1];
        if (i0 + tid < nq) {
            v[0] = whole(i0 + tid).t1;
            atomicMax(&sm.most, v[0]);
        }
        block_scan<T, 1>(v, all, sm.waves);
        if (i0 + tid < nq) sm.p[i0 + tid] = add_up_to(total, v[0]);
        total = add_up_to(total, all[0]);
    }
    __syncthreads();
    const uint32_t most = sm.most, slots = plan.slots;
    const uint32_t share = max((total + slots - 1) / slots, static_cast<uint32_t>(kLeast));
    const bool cut = total < kFull && !((nq >= 2 * slots && most <= share) || (nq <= slots && most * 10 <= share * 11));
    if (!cut) {
        for (int pass = 0; pass < 2; pass++) {
            for (uint32_t i = tid; i < nq; i += T) {
                const Piece p = whole(i);
                const uint32_t k = 63 - min(63u, static_cast<uint32_t>(static_cast<uint64_t>(p.t1) * 64 / (most + 1)));
                const uint32_t at = atomicAdd(&sm.bucket[k], 1u);
                if (pass == 1) {
                    plan.pieces[at] = p;
                    plan.first_of[i] = i;
                }
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
        if (tid == 0) {
            plan.first_of[nq] = nq;
            plan.head[kHeadBlocks] = nq, plan.head[kHeadCut] = 0, plan.head[kHeadJoins] = 0, plan.head[kHeadRecs] = 0;
        }
        return;
    }
    const uint32_t blocks = (total + share - 1) / share;
    uint32_t before[3] = {0, 0, 0};  // pieces, records, joins
    for (uint32_t i0 = 0; i0 < nq; i0 += T) {
        const uint32_t i = i0 + tid;
        uint32_t v[3] = {0, 0, 0}, all[3], n = 0;
        Piece p;
        if (i < nq) {
            p = whole(i);
            n = (sm.p[i] + p.t1 + share - 1) / share - sm.p[i] / share;
            v[0] = n, v[1] = n > 1 ? n : 0, v[2] = n > 1;
        }
        block_scan<T, 3>(v, all, sm.waves);
        if (i < nq) {
            const uint32_t at = before[0] + v[0], rec = before[1] + v[1];
            sm.at[i] = at;
            sm.rec[i] = n > 1 ? static_cast<int>(rec) : -1;
            if (n > 1) {
                plan.joins[before[2] + v[2]] = Join{p.first, p.r0, p.r_end, static_cast<int>(rec), static_cast<int>(n), {}};
                p.t1 = (sm.p[i] / share + 1) * share - sm.p[i];
                p.rec = rec;
            }
            plan.pieces[at] = p;
        }
        before[0] += all[0], before[1] += all[1], before[2] += all[2];
    }
    __syncthreads();
    for (uint32_t b = tid; b < blocks; b += T) {
        const uint32_t i = last_not_above(sm.p, nq, b * share), k = b - sm.p[i] / share, off = b * share - sm.p[i];
        plan.first_of[b] = sm.at[i] + (off == 0 ? 0 : k);
        if (off == 0) continue;
        Piece p = whole(i);
        p.t0 = off, p.t1 = min(static_cast<int>(off + share), p.t1), p.rec = sm.rec[i] + k;
        plan.pieces[sm.at[i] + k] = p;
    }
    if (tid == 0) {
        plan.first_of[blocks] = before[0];
        plan.head[kHeadBlocks] = blocks, plan.head[kHeadCut] = 1, plan.head[kHeadJoins] = before[2], plan.head[kHeadRecs] = before[1];
    }
}

__global__ __launch_bounds__(1024) void paged_plan_kernel(shv_attn_paged_args a, Plan plan) {
    extern __shared__ __align__(16) char raw[];
    make_plan(a, plan, *reinterpret_cast<PlanSmem<1024, kMaxSeqs, 8192 + kMaxSeqs> *>(raw));
}

// ---- the rows -----------------------------------------------------------------------------------
// A wave a query row or a row's cell of a KV head; with PLAN the first block makes the plan.
template <int D, bool PLAN>
__global__ __launch_bounds__(256) void paged_rows_kernel(shv_attn_paged_args a, Plan plan) {
    constexpr int VEC = D / 64;
    if constexpr (PLAN) {
        __shared__ PlanSmem<256, kFewBlocks, kFewBlocks> sm;
        if (blockIdx.x == 0) {
            make_plan(a, plan, sm);
            return;
        }
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rep = a.n_head / a.n_head_kv, per = a.n_head + a.n_head_kv;
    const uint32_t item = (blockIdx.x - (PLAN ? 1 : 0)) * 4 + wave;
    const int r = static_cast<int>(item / static_cast<uint32_t>(per)), h = static_cast<int>(item) - r * per;
    if (r >= a.max_rows) return;
    const bool query = h < a.n_head;
    const int head = query ? h : h - a.n_head;
    const float *src = a.qkv + static_cast<size_t>(r) * a.qkv_stride + static_cast<size_t>(query ? head : a.n_head) * 2 * D + (query ? 0 : head * D);
    Row<D> x, gamma, val;
    x.load(src, lane);
    val.load(query ? src : src + static_cast<size_t>(a.n_head_kv) * D, lane);
    gamma.load(query ? a.q_norm : a.k_norm, lane);
    const int p = a.row_pos[r], cell = a.row_cell[r];
    if (r >= a.start[a.n_seq] || p < 0 || p >= a.max_pages << plan.shift) return;
    Turn<D> turn(a.rope_dims, lane);
    if (a.rope_dims > 0) {
        turn.load(a.rope + static_cast<size_t>(p) * a.rope_dims, a.rope_dims);
        turn.settle();
    }
    if (!query) {
        if (cell < 0 || cell >= a.n_pages << plan.shift) return;
        uint16_t kx[VEC];
        cell_key<D>(x, gamma, turn, a.rope_dims, a.eps, kx);
        const size_t kvw = static_cast<size_t>(a.n_head_kv) * D;
        put_bytes<2 * VEC>(static_cast<uint16_t *>(a.kpages) + cell * kvw + head * D + VEC * lane, kx);
        uint16_t *vd = static_cast<uint16_t *>(a.vpages) + (cell / kTile * kvw + static_cast<size_t>(head) * D + VEC * lane) * kTile + cell % kTile;
#pragma unroll
        for (int v = 0; v < VEC; v++) vd[v * kTile] = __half_as_ushort(__float2half_rn(val.x[v]));
        return;
    }
    float ss = 0.f, y[VEC];
#pragma unroll
    for (int v = 0; v < VEC; v++) ss = fmaf(x.x[v], x.x[v], ss);
    const float sc = __builtin_amdgcn_rsqf(fmaf(wave_sum_all(ss), 1.f / static_cast<float>(D), a.eps));
#pragma unroll
    for (int v = 0; v < VEC; v++) {
        y[v] = x.x[v] * sc * gamma.x[v];
        if (a.rope_dims > 0) y[v] = fmaf(__shfl(y[v], turn.partner, 64), turn.s.x[v], y[v] * turn.c.x[v]);
    }
    _Float16 hi[VEC], lo[VEC];
    split_row<D>(y, hi, lo);
    const int kvh = head / rep;
    char *dst = plan.stage + ((static_cast<size_t>(kvh) * a.max_rows + r) * rep + head - kvh * rep) * D * 4 + 2 * VEC * lane;
    put_bytes<2 * VEC>(dst, hi);
    put_bytes<2 * VEC>(dst + 2 * D, lo);
}

// ---- attention ----------------------------------------------------------------------------------
// A tile in LDS: 1 KB chunks that a wave reads 16 bytes a lane.  K chunk T * (D/32) + i: lane (n, q) = cell 8 (n / 4) + 4 T + n % 4, dims
// 32 i + 8 q ..; V chunk db behind them: lane (n, q) = dim 16 db + n, cells 8 q ...  After S^T = K Q^T lane (n, q) then holds query row n's
// scores of cells 8 q + 4 T + 0..3, T = 0, 1: the eight cells of its operand of the second product.
template <int D>
struct AttnSmem {
    char ring[kStages][D / 8 * kChunk];
    float p[kWaves][16 * kTile / 2];  // a wave's weights of half a tile, where its values are not all finite
};

// Which block of the plan and KV head a workgroup has.  Workgroups go to the eight dies in turn; a die's KV heads are the same ones throughout, where their number
// allows it, so that its L2 holds their cells, and neighbouring blocks of a plan that cuts lie on one die.
struct Place {
    int block, kvh;
    __device__ __forceinline__ Place(int n_head_kv, int blocks, bool cut) {
        const int g = n_head_kv & 7 ? n_head_kv & -n_head_kv : 8;  // dies share heads g apart
        const int die = blockIdx.x & 7, nth = blockIdx.x >> 3, dies = 8 / g, heads = n_head_kv / g;
        const int k = static_cast<int>(static_cast<uint32_t>(nth) / static_cast<uint32_t>(heads)), of = die / g, per = (blocks + dies - 1) / dies;
        kvh = die % g + g * (nth - k * heads);
        block = cut ? (k < per ? of * per + k : blocks) : k * dies + of;
    }
};

// grid: 8 * ceil(blocks / dies) * heads (Place), blocks of 8 waves
template <int D>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 2 : 4) void paged_attn_kernel(shv_attn_paged_args a, Plan plan) {
    constexpr int KI = D / 32, DB = D / 16;
    constexpr int kPer = D / 8 / kWaves;  // chunks of a tile a wave asks for
    extern __shared__ __align__(16) char raw[];
    AttnSmem<D> &sm = *reinterpret_cast<AttnSmem<D> *>(raw);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, q = lane >> 4;
    const int blocks = plan.head[kHeadBlocks];
    const Place place(a.n_head_kv, blocks, plan.head[kHeadCut] != 0);
    if (place.block >= blocks) return;
    const int kvh = place.kvh, rep = a.n_head / a.n_head_kv;
    const size_t kvw = static_cast<size_t>(a.n_head_kv) * D;
    const bool keys = wave < kWaves / 2;
    const int first = (keys ? wave : wave - kWaves / 2) * kPer;  // of the wave's chunks among K's or V's
    const uint32_t from = keys ? static_cast<uint32_t>((8 * (n >> 2) + 4 * (first / KI) + (n & 3)) * kvw + 32 * (first % KI) + 8 * q) * 2
                               : static_cast<uint32_t>((16 * first + n) * kTile + 8 * q) * 2;
    const uint16_t *cells = keys ? static_cast<const uint16_t *>(a.kpages) + kvh * D : static_cast<const uint16_t *>(a.vpages) + static_cast<size_t>(kvh) * D * kTile;
    const float c2 = 1.44269504088896f / sqrtf(static_cast<float>(D));
    const int end = plan.first_of[place.block + 1];
    for (int k = plan.first_of[place.block]; k < end; k++) {
        const Piece piece = plan.pieces[k];
        const int r0 = piece.r0 + 16 * wave, r_end = piece.r_end;
        const bool working = r0 < r_end;
        const int last = min(piece.r0 + kRows, r_end) - 1;
        const int lo = piece.pos + piece.r0 / rep, hi = piece.pos + last / rep;  // the block's rows' positions
        const Tiles tiles(a.window, a.sinks, lo, hi);
        // a group that is not there is the last row again, and dropped
        const int mine = min(r0 + n, r_end - 1);
        const int my_pos = piece.pos + static_cast<int>(static_cast<uint32_t>(mine) / static_cast<uint32_t>(rep));
        const int my_first = a.window > 0 ? my_pos - a.window + 1 : 0;  // the first position it sees, but for the sinks
        // The table's entries around the tiles asked for last, one a lane.
        const int32_t *table = a.table + static_cast<size_t>(piece.seq) * a.max_pages;
        int held = 0, page0 = -64;
        uint32_t valid = 0;  // of the stages: the tile lies in a page
        const int n_tiles = piece.t1 - piece.t0;
        const auto ask = [&](int j) {
            const int tile = tiles.at(piece.t0 + j), entry = tile >> (plan.shift - 5);
            if (static_cast<uint32_t>(entry - page0) >= 64u) {
                page0 = entry;
                held = table[min(entry + lane, a.max_pages - 1)];
            }
            const int page = __builtin_amdgcn_readlane(held, entry - page0);
            const bool is = page >= 0 && page < a.n_pages;
            const uint32_t bit = 1u << (j & (kStages - 1));
            valid = is ? valid | bit : valid & ~bit;
            const size_t cell = (static_cast<size_t>(is ? page : 0) << plan.shift) + (tile * kTile & (a.page - 1));
            const __amdgpu_buffer_rsrc_t bytes = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(cells + cell * kvw), 0, static_cast<uint32_t>(kTile * kvw) * 2, 0x00027000);
            char *to = sm.ring[j & (kStages - 1)] + (wave * kPer) * kChunk;
#pragma unroll
            for (int u = 0; u < kPer; u++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(bytes, (lds_ptr_t)(to + u * kChunk), 16, from, u * (keys ? 64 : 1024), 0, 0);
        };
        half8_t qh[KI], ql[KI];
        {
            const char *src = plan.stage + ((static_cast<size_t>(kvh) * a.max_rows + piece.first) * rep + mine) * D * 4 + q * 16;
#pragma unroll
            for (int i = 0; i < KI; i++) {
                qh[i] = *reinterpret_cast<const half8_t *>(src + i * 64);
                ql[i] = *reinterpret_cast<const half8_t *>(src + 2 * D + i * 64);
            }
        }
        float4_t o[DB];
        float m_run = -INFINITY, l_run = 0.f;  // of the scores as they are, before their scale; the sums of a lane's own cells
#pragma unroll
        for (int db = 0; db < DB; db++) o[db] = float4_t{0.f, 0.f, 0.f, 0.f};
        bool saw = false;  // one of the lane's cells is one that its row sees
        for (int j = 0; j < min(n_tiles, kAhead); j++) ask(j);
        for (int j = 0; j < n_tiles; j++) {
            const char *kt = sm.ring[j & (kStages - 1)];
            // a wave's loads complete in order: this tile's have landed when no more are out than those behind it
            if (j + 2 < n_tiles) wait_loads<2 * kPer>();
            else if (j + 1 < n_tiles) wait_loads<kPer>();
            else wait_loads<0>();
            asm volatile("s_barrier" ::: "memory");  // everyone's: this tile is whole, and the stage of the one before is free
            const bool is = valid >> (j & (kStages - 1)) & 1;
            if (j + kAhead < n_tiles) ask(j + kAhead);
            if (!is || !working) continue;
            const int c0 = tiles.at(piece.t0 + j) * kTile;
            uint32_t seen = 0xFF;  // which of the lane's eight cells its query row sees
            const bool part = c0 + kTile - 1 > lo || (a.window > 0 && c0 + kTile - 1 >= a.sinks && c0 <= hi - a.window);
            if (part) {
                seen = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int c = c0 + 8 * q + e;
                    seen |= c <= my_pos && (a.window == 0 || c < a.sinks || c >= my_first) ? 1u << e : 0u;
                }
            }
            saw |= seen != 0;
            const char *vt = kt + 2 * KI * kChunk;
            // operands come from LDS four reads ahead of the products that use them
            float4_t st[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, sl[2] = {st[0], st[0]};
            half8_t kb[2][4];
            const auto read_k = [&](half8_t(&to)[4], int g) {
#pragma unroll
                for (int e = 0; e < 4; e++) to[e] = *reinterpret_cast<const half8_t *>(kt + ((e & 1) * KI + 2 * g + (e >> 1)) * kChunk + lane * 16);
            };
            read_k(kb[0], 0);
#pragma unroll
            for (int g = 0; g < KI / 2; g++) {
                if (g + 1 < KI / 2) read_k(kb[(g + 1) & 1], g + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    st[e & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb[g & 1][e], qh[2 * g + (e >> 1)], st[e & 1], 0, 0, 0);
                    sl[e & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb[g & 1][e], ql[2 * g + (e >> 1)], sl[e & 1], 0, 0, 0);
                }
            }
            float mx = -INFINITY, s[8];
#pragma unroll
            for (int e = 0; e < 8; e++) s[e] = st[e >> 2][e & 3] + sl[e >> 2][e & 3];
            if (part) {
#pragma unroll
                for (int e = 0; e < 8; e++) s[e] = seen >> e & 1 ? s[e] : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) mx = fmaxf(mx, s[e]);
            mx = max_over_q(mx);
            // the sums are rescaled a few times a run instead of whenever some row's maximum moves
            const bool moves = mx * c2 > fmaf(m_run, c2, kSlack);
            if (__ballot(moves) != 0ull) {
                const float m_new = moves ? mx : m_run;
                const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_run - m_new) * c2);
                l_run *= alpha;
                m_run = m_new;
                float av[4];
#pragma unroll
                for (int e = 0; e < 4; e++) av[e] = __shfl(alpha, 4 * q + e, 64);
#pragma unroll
                for (int db = 0; db < DB; db++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[db][e] *= av[e];
            }
            const float m2 = fmaf(m_run == -INFINITY ? 0.f : m_run, c2, -kLift);
            float pv[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                pv[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c2, -m2));
                l_run += pv[e];
            }
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
                if (__ballot(odd != 0) != 0ull) {
                    float *p = sm.p[wave];
#pragma unroll 1
                    for (int half = 0; half < 2; half++) {
                        if ((q >> 1) == half) {
#pragma unroll
                            for (int e = 0; e < 8; e++) p[n * (kTile / 2) + 8 * (q & 1) + e] = seen >> e & 1 ? pv[e] : -1.f;
                        }
                        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
                        for (int i = 0; i < kTile / 2; i++) {
                            const int c = kTile / 2 * half + i;
                            float w[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) w[e] = p[(4 * q + e) * (kTile / 2) + i];
#pragma unroll
                            for (int db = 0; db < DB; db++) {
                                const float v = static_cast<float>(*reinterpret_cast<const _Float16 *>(vt + db * kChunk + (16 * (c >> 3) + n) * 16 + (c & 7) * 2));
#pragma unroll
                                for (int e = 0; e < 4; e++) o[db][e] = w[e] < 0.f ? o[db][e] : fmaf(w[e], v, o[db][e]);
                            }
                        }
                        __builtin_amdgcn_wave_barrier();
                    }
                    continue;
                }
            }
            // weights as two halves, the large one cut off and not rounded: the small one holds the rest either way, and is rounded to nearest, so that what
            // many cells lose cancels
            half8_t ph, pl;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const half2_t h = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(pv[e], pv[e + 1]));
                const half2_t r = {static_cast<_Float16>(fmaf(static_cast<float>(h[0]), -1.f, pv[e])), static_cast<_Float16>(fmaf(static_cast<float>(h[1]), -1.f, pv[e + 1]))};
                ph[e] = h[0]; ph[e + 1] = h[1];
                pl[e] = r[0]; pl[e + 1] = r[1];
            }
            half8_t vb[2][4];
#pragma unroll
            for (int e = 0; e < 4; e++) vb[0][e] = *reinterpret_cast<const half8_t *>(vt + e * kChunk + lane * 16);
#pragma unroll
            for (int g = 0; g < DB / 4; g++) {
                if (g + 1 < DB / 4) {
#pragma unroll
                    for (int e = 0; e < 4; e++) vb[(g + 1) & 1][e] = *reinterpret_cast<const half8_t *>(vt + (4 * (g + 1) + e) * kChunk + lane * 16);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int e = 0; e < 4; e++) o[4 * g + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, vb[g & 1][e], o[4 * g + e], 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; e++) o[4 * g + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, vb[g & 1][e], o[4 * g + e], 0, 0, 0);
            }
        }
        if (working) {
            float sum = sum_over_q(l_run);
            const uint64_t saws = __ballot(saw);
            // a row whose scores are all -infinity has no weights; one that sees nothing has a sum of zero
            if (m_run == -INFINITY && ((saws >> n) & 0x0001000100010001ull) != 0) sum = __int_as_float(0x7fc00000);
            if (piece.rec < 0) {
                float lr[4];
#pragma unroll
                for (int i = 0; i < 4; i++) lr[i] = __shfl(sum, 4 * q + i, 64);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = r0 + 4 * q + i, row = static_cast<int>(static_cast<uint32_t>(r) / static_cast<uint32_t>(rep));
                    if (r >= r_end) continue;
                    float *dst = a.out + (static_cast<size_t>(piece.first + row) * a.n_head + kvh * rep + r - row * rep) * D;
#pragma unroll
                    for (int db = 0; db < DB; db++) dst[16 * db + n] = lr[i] == 0.f ? 0.f : o[db][i] / lr[i];
                }
            } else {
                const size_t base = (static_cast<size_t>(piece.rec) * a.n_head_kv + kvh) * plan.slot_rows + 16 * wave;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (r0 + 4 * q + i >= r_end) continue;
                    float *rec = plan.sums + (base + 4 * q + i) * D;
#pragma unroll
                    for (int db = 0; db < DB; db++) rec[16 * db + n] = o[db][i];
                }
                if (q == 0 && r0 + n < r_end) plan.of[base + n] = make_float2(m_run, sum);
            }
        }
        __syncthreads();  // the stages are free for the next piece
    }
}

// ---- the join -----------------------------------------------------------------------------------
// A unit is 256 / D query rows of a KV head, a lane four dims.  With many records a query row a block's four waves share them, otherwise each takes a unit of its own.
constexpr int kShareFrom = 8;  // records a query row from which the waves share them
template <int D>
__global__ __launch_bounds__(256) void paged_join_kernel(shv_attn_paged_args a, Plan plan) {
    __shared__ float4_t sums[4][64];
    __shared__ float2 of[4][64];
    constexpr int kLanes = D / 4, kUnit = 64 / kLanes;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n_joins = plan.head[kHeadJoins];
    if (n_joins == 0) return;
    const int rep = a.n_head / a.n_head_kv;
    const float c2 = 1.44269504088896f / sqrtf(static_cast<float>(D));
    const bool share = plan.head[kHeadRecs] >= kShareFrom * n_joins;
    const uint32_t per_head = (plan.slot_rows + kUnit - 1) / kUnit, per = per_head * a.n_head_kv, units = per * n_joins;
    const uint32_t step = share ? gridDim.x : gridDim.x * 4;
    for (uint32_t unit = share ? blockIdx.x : blockIdx.x * 4 + wave; unit < units; unit += step) {
        const uint32_t k = unit / per, in = unit - k * per, kvh = in / per_head, u = in - kvh * per_head;
        const Join join = plan.joins[k];
        const int local = u * kUnit + lane / kLanes, r = join.r0 + local;
        const bool there = local < plan.slot_rows && local < kRows && r < join.r_end;
        if (__ballot(there) == 0ull) continue;  // (the same in every wave that shares)
        const size_t row = (static_cast<size_t>(join.rec) * a.n_head_kv + kvh) * plan.slot_rows + (there ? local : 0), stride = static_cast<size_t>(a.n_head_kv) * plan.slot_rows;
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
        const int waves = share ? 4 : 1, me = share ? wave : 0;
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
        if (share) {
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
            const int t = r / rep;
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
    SHV_REQUIRE(a.page >= 32 && a.page <= 4096 && (a.page & (a.page - 1)) == 0, "attn_paged: page %d; a power of two from 32 to 4096", a.page);
    SHV_REQUIRE(a.n_pages >= 1 && static_cast<long long>(a.n_pages) * a.page < 1ll << 31, "attn_paged: %d pages of %d cells; fewer than 2^31 cells", a.n_pages, a.page);
    SHV_REQUIRE(a.max_pages >= 1 && static_cast<long long>(a.max_pages) * a.page < 1ll << 31, "attn_paged: max_pages %d of %d cells; fewer than 2^31 cells", a.max_pages, a.page);
    return SHV_OK;
}

// The scratch of a call of these sizes, laid out from `work` on; its end is the bytes that it takes.
uintptr_t lay_out(const shv_ctx *ctx, const shv_attn_paged_args &a, Plan &plan) {
    const int rep = a.n_head / a.n_head_kv, D = a.head_dim;
    const int per_unit = D == 256 ? 1 : 2;  // blocks a compute unit holds
    plan.slots = ctx->prop.multiProcessorCount * per_unit / a.n_head_kv;
    if (plan.slots < 1) plan.slots = 1;
    const int query_rows = a.max_rows * rep;
    plan.most_q = (a.n_seq < a.max_rows ? a.n_seq : a.max_rows) + query_rows / kRows;
    plan.most_blocks = plan.most_q > plan.slots ? plan.most_q : plan.slots;
    plan.slot_rows = query_rows < kRows ? (query_rows + 15) / 16 * 16 : kRows;
    plan.shift = 0;
    while (1 << plan.shift < a.page) plan.shift++;
    // a cut query block has a piece more than cuts, and there are fewer cuts than slots
    const size_t pieces = static_cast<size_t>(plan.most_q) + plan.slots, joins = plan.most_q < plan.slots ? plan.most_q : plan.slots, records = 2 * static_cast<size_t>(plan.slots) * a.n_head_kv * plan.slot_rows;
    uintptr_t at = reinterpret_cast<uintptr_t>(a.work);
    const auto take = [&](size_t bytes) {
        char *here = reinterpret_cast<char *>(at);
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    plan.head = reinterpret_cast<int32_t *>(take(kHeadWords * 4));
    plan.first_of = reinterpret_cast<int32_t *>(take((plan.most_blocks + 1) * 4));
    plan.pieces = reinterpret_cast<Piece *>(take(pieces * sizeof(Piece)));
    plan.joins = reinterpret_cast<Join *>(take(joins * sizeof(Join)));
    plan.of = reinterpret_cast<float2 *>(take(records * 8));
    plan.stage = take(static_cast<size_t>(a.max_rows) * a.n_head * D * 4);
    plan.sums = reinterpret_cast<float *>(take(records * D * 4));
    return at;
}

template <int D>
int launch_paged(shv_ctx *ctx, const shv_attn_paged_args &a) {
    Plan plan;
    lay_out(ctx, a, plan);
    using BigSmem = PlanSmem<1024, kMaxSeqs, 8192 + kMaxSeqs>;
    static std::atomic<uint64_t> raised{0};  // by device
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (!(raised.load(std::memory_order_acquire) & bit)) {
        SHV_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(&paged_attn_kernel<D>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(AttnSmem<D>))));
        SHV_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(&paged_plan_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(BigSmem))));
        raised.fetch_or(bit, std::memory_order_release);
    }
    const long long items = static_cast<long long>(a.max_rows) * (a.n_head + a.n_head_kv);
    const unsigned row_blocks = static_cast<unsigned>((items + 3) / 4);
    if (plan.most_q <= kFewBlocks && a.n_seq <= kFewBlocks) {
        SHV_LAUNCH(ctx, (paged_rows_kernel<D, true>), dim3(row_blocks + 1), dim3(256), 0, a, plan);
    } else {
        SHV_LAUNCH(ctx, paged_plan_kernel, dim3(1), dim3(1024), sizeof(BigSmem), a, plan);
        SHV_LAUNCH(ctx, (paged_rows_kernel<D, false>), dim3(row_blocks), dim3(256), 0, a, plan);
    }
    const int g = a.n_head_kv & 7 ? a.n_head_kv & -a.n_head_kv : 8, dies = 8 / g, heads = a.n_head_kv / g;  // Place
    SHV_LAUNCH(ctx, paged_attn_kernel<D>, dim3(static_cast<unsigned>((plan.most_blocks + dies - 1) / dies * heads * 8)), dim3(64 * kWaves), sizeof(AttnSmem<D>), a, plan);
    const long long joins = plan.most_q < plan.slots ? plan.most_q : plan.slots, units = joins * a.n_head_kv * plan.slot_rows;
    SHV_LAUNCH(ctx, paged_join_kernel<D>, dim3(static_cast<unsigned>(units < 2048 ? units : 2048)), dim3(256), 0, a, plan);
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
    *bytes = static_cast<int64_t>(lay_out(ctx, sizes, plan));
    return SHV_OK;
}
