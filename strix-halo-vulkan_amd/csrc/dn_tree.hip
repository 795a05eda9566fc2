// The gated delta rule over a tree of drafted tokens, and the state behind the branch that is kept.
//
// Row i's state would be S_i = g_i S_parent + k_i delta_i^T.  Written out down to the committed state S0, with G_i the sum of
// log g from the root to i,
//     delta_i = beta_i (v_i - e^(G_i) S0^T k_i) - sum over ancestors j of beta_i e^(G_i - G_j) (k_j . k_i) delta_j
//     out_i   = (e^(G_i) S0^T q_i + sum over ancestors j and i itself of e^(G_i - G_j) (k_j . q_i) delta_j) / sqrt(d)
// so no row needs a state of its own: S0 is read once, whatever the tree's shape, and the deltas are a triangular solve whose
// matrix is masked by ancestry.
#include <atomic>

#include "shv_device.hpp"
#include "shv_internal.hpp"
#include "tree.hpp"

namespace {

using namespace shv;

constexpr int kBlock = 256;
constexpr int kD = 128;
constexpr int kRows = SHV_TREE_MAX_ROWS;
constexpr int kCols = 32;  // value columns of a block

__device__ __forceinline__ float softplus_ref(float x) {
    // the add inside the log is float32 on purpose, as in the step's kernels: below about -16.6 it returns exactly 0
    return x > 20.f ? x : logf(1.f + expf(x));
}

struct TreeLds {
    float q[kRows][kD + 4], k[kRows][kD + 4];
    float s[kCols][kD + 4];
    float a[kRows][kRows + 1], m[kRows][kRows + 1];
    float d[kRows][kCols + 1], o[kRows][kCols + 1];
    float G[kRows], beta[kRows];
    uint32_t anc[kRows][2];
    const float *src[kRows][4];  // the rows a row's taps meet, NULL before the sequence's start
};

// grid: (128 / kCols, n_head_v, n_seq)
__global__ __launch_bounds__(kBlock) void dn_tree_kernel(shv_dn_tree_args a) {
    extern __shared__ __align__(16) char raw[];
    TreeLds &L = *reinterpret_cast<TreeLds *>(raw);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int col0 = blockIdx.x * kCols, h = blockIdx.y, seq = blockIdx.z, hk = h % a.n_head_k;
    const int qk = a.n_head_k * kD, vw = a.n_head_v * kD;
    const TreeWords words(a.count, a.pos, a.slot, a.parent, a.conv1d, seq, a.rows, lane);
    const int slot = words.slot, pos = words.pos;
    const TreeRow t = tree_row(words.count, words.parent, a.rows, lane);
    const int n = t.n;
    if (n == 0) return;
    const float *x = a.x + static_cast<size_t>(seq) * a.rows * a.x_stride;
    const float *ring = a.ring + static_cast<size_t>(slot) * a.ring_slots * a.ring_stride;
    {
        // every wave forms the tables, the first one stores them
        int up = lane < n ? lane : -1, above = 0;
        float g = 0.f, b = 0.f;
        if (lane < n) {
            const float *row = x + static_cast<size_t>(lane) * a.x_stride + 2 * qk + 2 * vw;
            g = softplus_ref(row[h] + a.dt_bias[h]) * a.a[h];
            b = sigmoid_exact(row[a.n_head_v + h]);
        }
        const float *src[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (up >= 0) {
                src[k] = x + static_cast<size_t>(up) * a.x_stride;
            } else {
                above++;
                const int p = pos - above;
                src[k] = p >= 0 ? ring + static_cast<size_t>(p % a.ring_slots) * a.ring_stride : nullptr;
            }
            const int next = __shfl(t.parent, up < 0 ? 0 : up, 64);
            up = up < 0 ? -1 : next;
        }
        const float G = tree_sum(t, g, a.rows, lane);
        if (wave == 0) {
            L.G[lane] = G;
            L.beta[lane] = b;
            L.anc[lane][0] = static_cast<uint32_t>(t.ancestors);
            L.anc[lane][1] = static_cast<uint32_t>(t.ancestors >> 32);
#pragma unroll
            for (int k = 0; k < 4; k++) L.src[lane][k] = src[k];
        }
    }
    const int planes = a.n_planes > 1 ? a.n_planes : 1;
    const int cur = a.plane ? static_cast<int>(static_cast<unsigned>(a.plane[slot]) % static_cast<unsigned>(planes)) : 0;
    const float *state = a.state + ((static_cast<size_t>(slot) * planes + cur) * a.n_head_v + h) * kD * kD + static_cast<size_t>(col0) * kD;
    for (int i = tid; i < kCols * kD; i += kBlock) L.s[i / kD][i % kD] = state[i];
    __syncthreads();
    const auto conv = [&](int r, int ch) {
        const float4 tp = *reinterpret_cast<const float4 *>(a.conv1d + static_cast<size_t>(ch) * 4);
        const float w[4] = {tp.w, tp.z, tp.y, tp.x};
        float c = 0.f;
        for (int k = 3; k >= 0; k--) c += (L.src[r][k] ? L.src[r][k][ch] : 0.f) * w[k];
        return c * sigmoid_exact(c);
    };
    for (int r = 0; r < n; r++) (tid < kD ? L.q : L.k)[r][tid & (kD - 1)] = conv(r, tid < kD ? hk * kD + tid : qk + hk * kD + tid - kD);
    __syncthreads();
    for (int v = wave; v < 2 * n; v += 4) {
        float *row = v < n ? L.q[v] : L.k[v - n];
        const float x0 = row[lane], x1 = row[lane + 64];
        const float ss = wave_sum_all(fmaf(x0, x0, x1 * x1));
        const float nrm = a.qk_norm_max ? 1.f / fmaxf(sqrtf(ss), a.eps) : 1.f / sqrtf(ss + a.eps);
        row[lane] = x0 * nrm;
        row[lane + 64] = x1 * nrm;
    }
    __syncthreads();
    if (col0 == 0 && h < a.n_head_k)
        for (int i = tid; i < n * kD; i += kBlock) a.kn[(static_cast<size_t>(seq) * a.rows + i / kD) * qk + hk * kD + i % kD] = L.k[i / kD][i % kD];
    if (col0 == 0 && tid < n) a.decay[(static_cast<size_t>(seq) * a.rows + tid) * a.n_head_v + h] = L.G[tid];
    for (int e = tid; e < n * n; e += kBlock) {
        const int i = e / n, j = e % n;
        float av = 0.f, mv = 0.f;
        if (L.anc[i][j >> 5] >> (j & 31) & 1) {
            float kk = 0.f, kq = 0.f;
            for (int c = 0; c < kD; c++) {
                kk = fmaf(L.k[i][c], L.k[j][c], kk);
                kq = fmaf(L.q[i][c], L.k[j][c], kq);
            }
            const float fall = expf(L.G[i] - L.G[j]);
            av = i == j ? 0.f : L.beta[i] * fall * kk;
            mv = fall * kq;
        }
        L.a[i][j] = av;
        L.m[i][j] = mv;
    }
    for (int e = tid; e < n * kCols; e += kBlock) {
        const int i = e / kCols, c = e % kCols;
        float sk = 0.f, sq = 0.f;
        for (int u = 0; u < kD; u++) {
            sk = fmaf(L.s[c][u], L.k[i][u], sk);
            sq = fmaf(L.s[c][u], L.q[i][u], sq);
        }
        const float fall = expf(L.G[i]);
        L.d[i][c] = L.beta[i] * (conv(i, 2 * qk + h * kD + col0 + c) - fall * sk);
        L.o[i][c] = fall * sq;
    }
    __syncthreads();
    if (tid < kCols) {
        for (int i = 1; i < n; i++) {
            float d = L.d[i][tid];
            for (int j = 0; j < i; j++)
                if (L.anc[i][j >> 5] >> (j & 31) & 1) d = fmaf(-L.a[i][j], L.d[j][tid], d);  // (another row's delta may be NaN)
            L.d[i][tid] = d;
        }
    }
    __syncthreads();
    const float scale = 1.f / sqrtf(static_cast<float>(kD));
    for (int e = tid; e < n * kCols; e += kBlock) {
        const int i = e / kCols, c = e % kCols;
        float o = L.o[i][c];
        for (int j = 0; j <= i; j++)
            if (L.anc[i][j >> 5] >> (j & 31) & 1) o = fmaf(L.m[i][j], L.d[j][c], o);
        const size_t at = (static_cast<size_t>(seq) * a.rows + i) * vw + static_cast<size_t>(h) * kD + col0 + c;
        a.out[at] = o * scale;
        a.delta[at] = L.d[i][c];
    }
}

// grid: (8 slabs of 16 state rows, n_head_v, n_seq): a thread holds eight values of one row.  HBM-bound: the state is read once
// and written once.
constexpr int kKeepRows = 16;
__global__ __launch_bounds__(kBlock) void dn_keep_kernel(shv_dn_keep_args a) {
    __shared__ float fall[kRows];
    __shared__ int row[kRows];
    __shared__ float all;
    __shared__ int used;
    const int tid = threadIdx.x, lane = tid & 63;
    const int slab = blockIdx.x, h = blockIdx.y, seq = blockIdx.z, hk = h % a.n_head_k;
    const int slot = a.slot ? a.slot[seq] : seq;
    const int planes = a.n_planes > 1 ? a.n_planes : 1;
    const int cur = a.plane ? static_cast<int>(static_cast<unsigned>(a.plane[slot]) % static_cast<unsigned>(planes)) : 0;
    const int next = cur + 1 < planes ? cur + 1 : 0;
    const size_t plane_floats = static_cast<size_t>(a.n_head_v) * kD * kD;
    const int j = slab * kKeepRows + tid / 16, i0 = tid % 16 * 4;
    float *at = a.state + static_cast<size_t>(slot) * planes * plane_floats + (static_cast<size_t>(h) * kD + j) * kD + i0;
    float4 s0 = *reinterpret_cast<const float4 *>(at + cur * plane_floats), s1 = *reinterpret_cast<const float4 *>(at + cur * plane_floats + 64);
    const int keep = max(0, min(a.n_keep[seq], a.rows));
    const size_t base = static_cast<size_t>(seq) * a.rows;
    if (tid < 64) {
        const int r = lane < keep ? a.path[base + lane] : -1;
        const bool on = r >= 0 && r < a.rows;
        const float G = on ? a.decay[(base + r) * a.n_head_v + h] : 0.f;
        const uint64_t there = __ballot(on);
        const int n = __popcll(there);
        const float last = n ? __shfl(G, 63 - __clzll(there), 64) : 0.f;
        if (on) {
            const int k = __popcll(there & ((1ull << lane) - 1));
            fall[k] = expf(last - G);
            row[k] = r;
        }
        if (lane == 0) {
            all = expf(last);
            used = n;
        }
    }
    __syncthreads();
    const int n = used;
    const float f = all;
    s0.x *= f; s0.y *= f; s0.z *= f; s0.w *= f;
    s1.x *= f; s1.y *= f; s1.z *= f; s1.w *= f;
    for (int e = 0; e < n; e++) {
        const size_t r = base + row[e];
        const float *k = a.kn + (r * a.n_head_k + hk) * kD + i0;
        const float d = a.delta[(r * a.n_head_v + h) * kD + j] * fall[e];
        const float4 k0 = *reinterpret_cast<const float4 *>(k), k1 = *reinterpret_cast<const float4 *>(k + 64);
        s0.x = fmaf(d, k0.x, s0.x); s0.y = fmaf(d, k0.y, s0.y); s0.z = fmaf(d, k0.z, s0.z); s0.w = fmaf(d, k0.w, s0.w);
        s1.x = fmaf(d, k1.x, s1.x); s1.y = fmaf(d, k1.y, s1.y); s1.z = fmaf(d, k1.z, s1.z); s1.w = fmaf(d, k1.w, s1.w);
    }
    *reinterpret_cast<float4 *>(at + next * plane_floats) = s0;
    *reinterpret_cast<float4 *>(at + next * plane_floats + 64) = s1;
    // the last three rows' conv channels, 256 a block
    const int ch = (h * (kD / kKeepRows) + slab) * kBlock + tid, cw = 2 * a.n_head_k * kD + a.n_head_v * kD;
    const int pos = a.pos ? a.pos[seq] : 0;
    if (ch < cw) {
        float *ring = a.ring + static_cast<size_t>(slot) * a.ring_slots * a.ring_stride;
        for (int e = max(0, keep - (a.conv - 1)); e < keep; e++) {
            const int r = a.path[base + e];
            const long long p = static_cast<long long>(pos) + e;
            if (r >= 0 && r < a.rows && p >= 0) ring[static_cast<size_t>(p % a.ring_slots) * a.ring_stride + ch] = a.x[(base + r) * a.x_stride + ch];
        }
    }
}

}  // namespace

int shv_launch_dn_tree(shv_ctx *ctx, const shv_dn_tree_args *pa) {
    const shv_dn_tree_args &a = *pa;
    SHV_REQUIRE(a.x && a.ring && a.conv1d && a.a && a.dt_bias && a.state && a.out && a.kn && a.delta && a.decay, "dn_tree: NULL argument");
    SHV_REQUIRE(a.rows >= 1 && a.rows <= kRows, "dn_tree: %d rows; 1..%d", a.rows, kRows);
    SHV_REQUIRE(a.n_seq >= 1 && a.n_seq <= 65535, "dn_tree: %d sequences", a.n_seq);
    SHV_REQUIRE(a.head_dim == kD, "dn_tree: head_dim %d; built for %d", a.head_dim, kD);
    SHV_REQUIRE(a.conv == 4, "dn_tree: conv kernel %d; built for 4", a.conv);
    SHV_REQUIRE(a.n_head_k >= 1 && a.n_head_v >= a.n_head_k && a.n_head_v % a.n_head_k == 0 && a.n_head_v <= 1024, "dn_tree: heads %d/%d", a.n_head_k, a.n_head_v);
    const int width = 2 * a.n_head_k * kD + 2 * a.n_head_v * kD + 2 * a.n_head_v, cw = 2 * a.n_head_k * kD + a.n_head_v * kD;
    SHV_REQUIRE(a.x_stride >= width, "dn_tree: x_stride %d < row width %d", a.x_stride, width);
    SHV_REQUIRE(a.ring_stride >= cw && a.ring_slots >= a.conv - 1, "dn_tree: a ring of %d rows %d floats apart", a.ring_slots, a.ring_stride);
    SHV_REQUIRE(a.n_planes >= 0 && a.n_planes <= 64, "dn_tree: %d state planes", a.n_planes);
    SHV_REQUIRE(shv_aligned16(a.x) && shv_aligned16(a.state) && shv_aligned16(a.conv1d) && shv_aligned16(a.ring) && shv_aligned16(a.out) &&
                    shv_aligned16(a.kn) && shv_aligned16(a.delta),
                "dn_tree: x, ring, conv1d, state, out, kn and delta must be 16-byte aligned");
    static std::atomic<bool> raised{false};
    if (!raised.load(std::memory_order_acquire)) {
        SHV_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(&dn_tree_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(TreeLds))));
        raised.store(true, std::memory_order_release);
    }
    SHV_LAUNCH(ctx, dn_tree_kernel, dim3(kD / kCols, a.n_head_v, a.n_seq), dim3(kBlock), sizeof(TreeLds), a);
    return SHV_OK;
}

int shv_launch_dn_keep(shv_ctx *ctx, const shv_dn_keep_args *pa) {
    const shv_dn_keep_args &a = *pa;
    SHV_REQUIRE(a.x && a.kn && a.delta && a.decay && a.state && a.ring && a.path && a.n_keep, "dn_keep: NULL argument");
    SHV_REQUIRE(a.rows >= 1 && a.rows <= kRows, "dn_keep: %d rows; 1..%d", a.rows, kRows);
    SHV_REQUIRE(a.n_seq >= 1 && a.n_seq <= 65535, "dn_keep: %d sequences", a.n_seq);
    SHV_REQUIRE(a.head_dim == kD, "dn_keep: head_dim %d; built for %d", a.head_dim, kD);
    SHV_REQUIRE(a.conv == 4, "dn_keep: conv kernel %d; built for 4", a.conv);
    SHV_REQUIRE(a.n_head_k >= 1 && a.n_head_v >= a.n_head_k && a.n_head_v % a.n_head_k == 0 && a.n_head_v <= 1024, "dn_keep: heads %d/%d", a.n_head_k, a.n_head_v);
    const int cw = 2 * a.n_head_k * kD + a.n_head_v * kD;
    SHV_REQUIRE(a.x_stride >= cw, "dn_keep: x_stride %d < %d conv channels", a.x_stride, cw);
    SHV_REQUIRE(a.ring_stride >= cw && a.ring_slots >= a.conv - 1, "dn_keep: a ring of %d rows %d floats apart", a.ring_slots, a.ring_stride);
    SHV_REQUIRE(a.n_planes >= 0 && a.n_planes <= 64, "dn_keep: %d state planes", a.n_planes);
    SHV_REQUIRE(shv_aligned16(a.state) && shv_aligned16(a.kn), "dn_keep: state and kn must be 16-byte aligned");
    SHV_LAUNCH(ctx, dn_keep_kernel, dim3(kD / kKeepRows, a.n_head_v, a.n_seq), dim3(kBlock), 0, a);
    return SHV_OK;
}
