// Full attention of packed rows over a paged cache.
//
// Row r of a sequence, at position p_r, sees the sequence's cells c <= p_r that lie in a page (with a window those of them below `sinks` or above p_r - window):
//     out_r = sum over them of softmax(q_r . k_c / sqrt(d)) v_c
// q and k normed over a head and rotated at their positions.  One launch writes the rows' keys and values into their cells, a second
// attends: a wave a row and head, cell after cell with a running maximum and sum.
#include "shv_device.hpp"
#include "shv_internal.hpp"

namespace {

using namespace shv;

constexpr int kTile = 32;  // cells of a tile of V

template <int D>
struct Row {  // a lane's dims of one head's row: VEC * lane ..
    static constexpr int VEC = D / 64;
    float x[VEC];
    __device__ __forceinline__ void load(const float *p, int lane) {
#pragma unroll
        for (int v = 0; v < VEC; v++) x[v] = p[VEC * lane + v];
    }
    // The row over its norm, times gamma, rotated by the factors of a row of the table.
    __device__ __forceinline__ void norm_turn(const float *gamma, const float *turn, int rope_dims, float eps, int lane) {
        double ss = 0;
#pragma unroll
        for (int v = 0; v < VEC; v++) ss = fma(static_cast<double>(x[v]), static_cast<double>(x[v]), ss);
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) ss += __shfl_xor(ss, off, 64);
        const double sc = 1.0 / sqrt(ss / D + static_cast<double>(eps));
        const int half = rope_dims / 2;
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            const int e = VEC * lane + v;
            const double y = x[v] * sc * gamma[e];
            const int other = e < half ? e + half : e < rope_dims ? e - half : e;
            const double z = __shfl(y, other / VEC, 64);
            const int i = e < half ? e : e - half;
            x[v] = e >= rope_dims ? static_cast<float>(y) : static_cast<float>(e < half ? y * turn[i] - z * turn[half + i] : y * turn[i] + z * turn[half + i]);
        }
    }
};

// Row and position of a sequence's first row; n 0 where it is left alone.
struct Seq {
    int first, n, pos;
    __device__ __forceinline__ Seq(const shv_attn_paged_args &a, int s) {
        const int from = a.start[s], to = a.start[s + 1];
        first = from;
        n = from >= 0 && to > from && to <= a.max_rows ? to - from : 0;
        pos = n > 0 ? a.row_pos[from] : 0;
        if (pos < 0 || static_cast<long long>(pos) + n > static_cast<long long>(a.max_pages) * a.page) n = 0;
    }
};

// grid: (max_rows, n_head_kv), a wave a row's cell of a KV head
template <int D>
__global__ __launch_bounds__(64) void paged_cells_kernel(shv_attn_paged_args a, int shift) {
    constexpr int VEC = D / 64;
    const int r = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    if (r >= a.start[a.n_seq]) return;
    const int cell = a.row_cell[r];
    const int p = a.row_pos[r];
    if (cell < 0 || cell >= a.n_pages * a.page || p < 0 || p >= a.max_pages * a.page) return;
    const float *src = a.qkv + static_cast<size_t>(r) * a.qkv_stride + static_cast<size_t>(a.n_head) * 2 * D + h * D;
    Row<D> k, v;
    k.load(src, lane);
    v.load(src + a.n_head_kv * D, lane);
    k.norm_turn(a.k_norm, a.rope + static_cast<size_t>(p) * a.rope_dims, a.rope_dims, a.eps, lane);
    const size_t kvw = static_cast<size_t>(a.n_head_kv) * D;
    uint16_t *kd = static_cast<uint16_t *>(a.kpages) + cell * kvw + h * D + VEC * lane;
    uint16_t *vd = static_cast<uint16_t *>(a.vpages) + (cell / kTile * kvw + static_cast<size_t>(h) * D + VEC * lane) * kTile + cell % kTile;
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        kd[e] = __half_as_ushort(__float2half_rn(k.x[e]));
        vd[e * kTile] = __half_as_ushort(__float2half_rn(v.x[e]));
    }
}

// grid: (max_rows, n_head), a wave a row of a head
template <int D>
__global__ __launch_bounds__(64) void paged_attn_kernel(shv_attn_paged_args a, int shift) {
    constexpr int VEC = D / 64;
    const int r = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
    int s = 0;
    while (s < a.n_seq && !(a.start[s] <= r && r < a.start[s + 1])) s++;
    if (s == a.n_seq) return;
    const Seq seq(a, s);
    if (r >= seq.first + seq.n) return;
    const int p = seq.pos + r - seq.first, h = head / (a.n_head / a.n_head_kv);
    Row<D> q;
    q.load(a.qkv + static_cast<size_t>(r) * a.qkv_stride + static_cast<size_t>(head) * 2 * D, lane);
    q.norm_turn(a.q_norm, a.rope + static_cast<size_t>(p) * a.rope_dims, a.rope_dims, a.eps, lane);
    const float scale = 1.f / sqrtf(static_cast<float>(D));
    float o[VEC] = {}, m = -INFINITY, sum = 0.f;
    const size_t kvw = static_cast<size_t>(a.n_head_kv) * D;
    for (int c = 0; c <= p; c++) {
        if (a.window > 0 && c >= a.sinks && p - c >= a.window) continue;
        const int page = a.table[static_cast<size_t>(s) * a.max_pages + (c >> shift)];
        if (page < 0 || page >= a.n_pages) continue;
        const size_t cell = (static_cast<size_t>(page) << shift) + (c & (a.page - 1));
        const uint16_t *kd = static_cast<const uint16_t *>(a.kpages) + cell * kvw + h * D + VEC * lane;
        const uint16_t *vd = static_cast<const uint16_t *>(a.vpages) + (cell / kTile * kvw + static_cast<size_t>(h) * D + VEC * lane) * kTile + cell % kTile;
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < VEC; e++) dot = fmaf(q.x[e], f16_bits_to_f32(kd[e]), dot);
        dot = wave_sum_all(dot) * scale;
        const float top = fmaxf(m, dot), shrink = expf(m - top), w = expf(dot - top);
        m = top;
        sum = fmaf(sum, shrink, w);
#pragma unroll
        for (int e = 0; e < VEC; e++) o[e] = fmaf(o[e], shrink, w * f16_bits_to_f32(vd[e * kTile]));
    }
    float *dst = a.out + (static_cast<size_t>(r) * a.n_head + head) * D + VEC * lane;
#pragma unroll
    for (int e = 0; e < VEC; e++) dst[e] = m == -INFINITY ? 0.f : o[e] / sum;
}

template <int D>
int launch_paged(shv_ctx *ctx, const shv_attn_paged_args &a, int shift) {
    SHV_LAUNCH(ctx, paged_cells_kernel<D>, dim3(a.max_rows, a.n_head_kv), dim3(64), 0, a, shift);
    SHV_LAUNCH(ctx, paged_attn_kernel<D>, dim3(a.max_rows, a.n_head), dim3(64), 0, a, shift);
    return SHV_OK;
}

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
    int shift = 0;
    while (1 << shift < a.page) shift++;
    if (a.head_dim == 256) return launch_paged<256>(ctx, a, shift);
    if (a.head_dim == 128) return launch_paged<128>(ctx, a, shift);
    return launch_paged<64>(ctx, a, shift);
}

extern "C" int shv_attn_paged_work(shv_ctx *ctx, const shv_attn_paged_args *a, int64_t *bytes) {
    SHV_REQUIRE(ctx && a && bytes, "attn_paged_work: NULL argument");
    const int rc = check_sizes(*a);
    if (rc != SHV_OK) return rc;
    *bytes = 16;
    return SHV_OK;
}
