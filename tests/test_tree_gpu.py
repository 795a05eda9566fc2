"""Verification of a tree of drafted tokens on the GPU: attention over cache and ancestors, the gated delta rule over a tree, the choice of the
branch and what keeps it, against float64 forms of the definitions and against the framework's own chain passes."""
import numpy as np
import pytest

import oracle_lib as O
import shv
import tree_oracle as T

pytestmark = pytest.mark.gpu
A = shv.api
EPS = 1e-6
LAYOUTS = {"16/2x256": (16, 2, 256, 64), "32/8x128": (32, 8, 128, 128), "12/2x128": (12, 2, 128, 0), "8/8x64": (8, 8, 64, 32), "5/1x64": (5, 1, 64, 6),
           "32/2x256": (32, 2, 256, 256), "64/1x64": (64, 1, 64, 10), "6/2x256": (6, 2, 256, 24), "9/3x128": (9, 3, 128, 12),
           "32/16x128": (32, 16, 128, 64)}
# Outputs: a score is a sum of d products q k / sqrt(d) of normed vectors, in absolute values at most about sqrt(d) <= 16.  Queries and
# weights enter the products to 22 bits and sums are float32: an error of a score is within 16 * (2^-22 + a few 2^-24) = 1e-5, of a
# weight as much again relative to it, of a weighted mean of the values no more than that.
ATTN_TOL = 2e-5


def v_dev(vc):
    """[slots][cells][nkv][d] to the device's tiles of 32 cells"""
    s, cells, nkv, d = vc.shape
    return np.ascontiguousarray(np.moveaxis(vc.reshape(s, cells // 32, 32, nkv, d), 2, -1))


def v_host(vt):
    s, blocks, nkv, d, _ = vt.shape
    return np.ascontiguousarray(np.moveaxis(vt, -1, 2)).reshape(s, blocks * 32, nkv, d)


class AttnTree:
    """Inputs of one call: sequences of different positions on permuted slots, rows a stride apart wider than they need."""

    def __init__(self, seed, layout, rows, pos, count=None, kind="mixed", parents=None):
        self.rng = rng = np.random.default_rng(seed)
        self.nh, self.nkv, self.d, self.dims = LAYOUTS[layout]
        self.rows, self.pos = rows, np.array(pos, np.int32)
        self.n_seq = len(pos)
        self.count = None if count is None else np.array(count, np.int32)
        self.max_cells = max((int(max(pos)) + rows + 31) // 32 * 32, 32)
        self.width = 2 * self.nh * self.d + 2 * self.nkv * self.d
        self.stride = self.width + 4
        self.parent = np.stack([T.tree(rng, rows, kind) for _ in pos]) if parents is None else np.array(parents, np.int32)
        self.slot = rng.permutation(self.n_seq).astype(np.int32)
        self.qkv = rng.standard_normal((self.n_seq, rows, self.stride)).astype(np.float32)
        self.q_norm = (1 + 0.1 * rng.standard_normal(self.d)).astype(np.float32)
        self.k_norm = (1 + 0.1 * rng.standard_normal(self.d)).astype(np.float32)
        self.table = T.rope_table(self.max_cells, self.dims)
        shape = (self.n_seq, self.max_cells, self.nkv, self.d)
        self.kc, self.vc = (rng.standard_normal(shape, dtype=np.float32).astype(np.float16) for _ in range(2))

    def n(self, s):
        return self.rows if self.count is None else min(max(int(self.count[s]), 0), self.rows)

    def upload(self, c):
        up = c.upload
        self.d_qkv, self.d_qn, self.d_kn, self.d_table = up(self.qkv), up(self.q_norm), up(self.k_norm), up(self.table)
        self.d_kc, self.d_vc = up(self.kc), up(v_dev(self.vc))
        cells = self.n_seq * self.rows * self.nkv * self.d
        self.d_kx, self.d_vx = up(np.full(cells, 0x3555, np.uint16)), up(np.full(cells, 0x3555, np.uint16))
        self.d_out = up(np.full(self.n_seq * self.rows * self.nh * self.d, 77.0, np.float32))
        self.d_pos, self.d_slot, self.d_parent = up(self.pos), up(self.slot), up(self.parent)
        self.d_count = None if self.count is None else up(self.count)

    def args(self, c, n_splits=16, window=0, sinks=0, parent=True):
        part = c.upload(np.full(self.n_seq * self.rows * self.nh * n_splits * (self.d + 2), np.nan, np.float32))
        return A.AttnTreeArgs(self.d_qkv.ptr, self.d_qn.ptr, self.d_kn.ptr, self.d_table.ptr, self.d_kc.ptr, self.d_vc.ptr, self.d_kx.ptr, self.d_vx.ptr, part.ptr,
                              self.d_out.ptr, self.d_pos.ptr, self.d_slot.ptr, self.d_parent.ptr if parent else None, A.ptr(self.d_count), self.n_seq, self.rows,
                              self.nh, self.nkv, self.d, self.dims, self.max_cells, self.stride, n_splits, window, sinks, EPS)

    def results(self):
        shape = (self.n_seq, self.rows, self.nkv, self.d)
        return (self.d_out.read(np.float32, self.n_seq * self.rows * self.nh * self.d).reshape(self.n_seq, self.rows, -1),
                self.d_kx.read(np.float16, int(np.prod(shape))).reshape(shape), self.d_vx.read(np.float16, int(np.prod(shape))).reshape(shape))

    def check(self, window=0, sinks=0):
        out, kx, vx = self.results()
        worst = 0.0
        for s in range(self.n_seq):
            n = self.n(s)
            want, k, v = T.attn_tree(self.qkv[s], self.q_norm, self.k_norm, self.table, self.kc[self.slot[s]], self.vc[self.slot[s]], int(self.pos[s]),
                                     self.parent[s], n, self.nh, self.nkv, self.d, self.dims, EPS, window, sinks)
            assert np.array_equal(kx[s, :n], k, equal_nan=True) and np.array_equal(vx[s, :n].view(np.uint16) & 0x7FFF, v.view(np.uint16) & 0x7FFF)
            fine = np.isfinite(want)
            assert np.array_equal(fine, np.isfinite(out[s, :n]))
            for r in range(n):
                if fine[r].any():
                    worst = max(worst, O.rel_l2(out[s, r][fine[r]], want[r][fine[r]]))
            # rows that are not in use keep what was there
            assert (out[s, n:] == 77.0).all() and (kx[s, n:].view(np.uint16) == 0x3555).all() and (vx[s, n:].view(np.uint16) == 0x3555).all()
        print(f"tree attention {self.n_seq} x {self.rows} behind {self.pos.tolist()}: {worst:.2e}")
        assert worst <= ATTN_TOL
        return out


@pytest.mark.parametrize("layout,rows,pos,n_splits,kind", [
    ("16/2x256", 1, [0], 1, "chain"), ("16/2x256", 1, [1], 16, "chain"), ("16/2x256", 2, [31], 16, "chain"), ("16/2x256", 5, [32], 16, "mixed"),
    ("16/2x256", 3, [700], 64, "star"), ("16/2x256", 17, [33], 16, "mixed"), ("16/2x256", 64, [0], 16, "wide"), ("16/2x256", 64, [1000], 3, "chain"),
    ("16/2x256", 33, [2111], 100, "mixed"), ("16/2x256", 12, [100, 0, 517], 40, "mixed"), ("16/2x256", 9, [4100], 512, "roots"), ("16/2x256", 64, [1500, 90], 20, "star"),
    ("32/8x128", 7, [300, 45], 16, "mixed"), ("32/8x128", 40, [65], 16, "wide"), ("12/2x128", 6, [129], 16, "mixed"), ("12/2x128", 11, [640], 2, "mixed"),
    ("8/8x64", 1, [63], 16, "chain"), ("8/8x64", 21, [500, 1, 64], 8, "mixed"), ("5/1x64", 13, [222], 5, "mixed"), ("5/1x64", 1, [0], 1, "chain"), ("32/2x256", 10, [97], 7, "mixed")])
def test_tree_attention(ctx, layout, rows, pos, n_splits, kind):
    t = AttnTree(100 * rows + pos[0], layout, rows, pos, kind=kind)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_TREE, t.args(ctx, n_splits))
    t.check()


@pytest.mark.parametrize("layout,rows,pos,n_splits", [
    # every query row of a KV head at most: 64 heads of 64 rows; 64 and 65 query rows, on both sides of the line between the two kernels
    ("64/1x64", 64, [700], 9), ("64/1x64", 1, [95, 3], 4), ("16/2x256", 8, [400], 7), ("6/2x256", 22, [64, 200], 6), ("9/3x128", 21, [1000], 12), ("9/3x128", 22, [31], 3),
    # one slice, and the two of which a wide call keeps one for its rows
    ("16/2x256", 64, [1000], 1), ("16/2x256", 40, [70, 0], 2), ("16/2x256", 3, [1000, 40], 1), ("16/2x256", 3, [333], 2), ("32/8x128", 33, [500], 1), ("5/1x64", 64, [129], 2)])
def test_query_rows_and_slices_at_their_lines(ctx, layout, rows, pos, n_splits):
    t = AttnTree(300 + rows + n_splits, layout, rows, pos)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_TREE, t.args(ctx, n_splits))
    t.check()


@pytest.mark.parametrize("rows", [3, 8, 9, 40])
def test_values_left_for_keeping_are_rounded_bit_by_bit(ctx, rows):
    """vcells against the nearest binary16, signs and zeros too: values of either sign, zeros of either, denormals, ties, and what becomes infinite."""
    t = AttnTree(330 + rows, "16/2x256", rows, [70, 5])
    v0 = 2 * t.nh * t.d + t.nkv * t.d
    v = t.qkv[:, :, v0:v0 + t.nkv * t.d]
    odd = np.array([0.0, -0.0, 2.0 ** -24, -2.0 ** -25, 3 * 2.0 ** -25, -6e-8, 1 + 2.0 ** -11, -(1 + 3 * 2.0 ** -11), 65504, -65504, 65519.99, -65520, 7e4], np.float32)
    v[:, :, :40] = t.rng.choice(odd, v[:, :, :40].shape)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_TREE, t.args(ctx))
    with np.errstate(over="ignore"):
        want = v.astype(np.float16).reshape(2, rows, t.nkv, t.d)
    assert (np.signbit(want) & (want == 0)).any() and np.isinf(want).any()
    assert np.array_equal(t.results()[2].view(np.uint16), want.view(np.uint16))


@pytest.mark.parametrize("rows,cells,n_splits,lead", [(3, 3000, 16, 22), (3, 3000, 1, 20), (40, 5000, 9, 22), (40, 9000, 64, 21), (2, 20000, 40, 19)])
def test_small_weights_beside_a_first_cell_that_takes_nearly_all(ctx, rows, cells, n_splits, lead):
    """A first cell with 2^lead times the weight of any other and a value of nothing, as models that rest on their first token have it: the output is what the
    small weights make of their values.  A weight is rounded to the nearest 2^-35 of the largest, by at most 2^-36: of one of 2^-22 that is 2^-14, no two cells alike,
    and of a sum over thousands of them 2^-14 / sqrt(3 * 3000) = 6e-7 is left."""
    t = AttnTree(340 + lead, "12/2x128", rows, [cells], kind="star")
    u = np.sign(t.rng.standard_normal(t.d)).astype(np.float32)
    t.q_norm[:] = t.k_norm[:] = 1
    t.qkv[0, :, :2 * t.nh * t.d].reshape(rows, t.nh, 2, t.d)[:, :, 0] = 3 * u
    away = 1 - lead * np.log(2) / np.sqrt(t.d)
    t.kc[:] = (away * u + 0.05 * t.rng.standard_normal(t.kc.shape)).astype(np.float16)
    t.kc[:, 0] = u
    t.vc[:] = (1 + 0.1 * t.rng.standard_normal(t.vc.shape)).astype(np.float16)
    t.vc[:, 0] = 0
    own = t.qkv[0, :, 2 * t.nh * t.d:]
    own[:, :t.nkv * t.d] = np.tile(-u, t.nkv)
    own[:, t.nkv * t.d:2 * t.nkv * t.d] = 1
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_TREE, t.args(ctx, n_splits))
    t.check()


@pytest.mark.parametrize("rows,n_splits,window", [(2, 16, 0), (9, 5, 0), (12, 16, 40)])
def test_many_sequences_of_which_some_do_not_fit(ctx, rows, n_splits, window):
    """More sequences than a wave has lanes, of lengths from nothing to hundreds of cells, some without rows and some that do not fit the cache."""
    n_seq = 75
    rng = np.random.default_rng(9)
    t = AttnTree(310, "16/2x256", rows, [int(p) for p in rng.choice([0, 1, 31, 32, 33, 64, 150, 700], n_seq)], count=rng.integers(0, rows + 2, n_seq))
    odd = np.arange(5, n_seq, 9)
    t.pos[odd] = np.where(odd % 2, -1 - odd, t.max_cells + odd).astype(np.int32)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_TREE, t.args(ctx, n_splits, window, 3))
    t.pos[odd] = 0
    t.count[odd] = 0  # nothing of these is written
    t.check(window, 3)


@pytest.mark.parametrize("layout,rows,pos,n_splits,window", [
    ("32/16x128", 40, [1500, 3, 700, 1100, 0, 31, 64, 900], 32, 0), ("32/16x128", 3, [2000, 40, 1990, 5, 1, 800], 32, 0), ("8/8x64", 9, [33 * i for i in range(40)], 64, 0),
    ("8/8x64", 9, [0] * 39 + [5000], 512, 0), ("16/2x256", 12, [4000, 4031, 4033, 96], 8, 0), ("32/8x128", 17, [3000, 2999, 17, 1600, 0], 64, 700)])
def test_sequences_of_uneven_lengths_share_the_blocks(ctx, layout, rows, pos, n_splits, window):
    """Lengths for which the slices' common length is looked for among many, with few and many slices a sequence."""
    t = AttnTree(320 + rows, layout, rows, pos)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_TREE, t.args(ctx, n_splits, window, 2 if window else 0))
    t.check(window, 2 if window else 0)


def test_absent_arrays(ctx):
    """pos, slot, parent and count NULL: sequences without a past, slot s, chains, all rows."""
    t = AttnTree(311, "16/2x256", 7, [0, 0, 0], kind="chain")
    t.slot = np.arange(3, dtype=np.int32)
    t.upload(ctx)
    a = t.args(ctx, parent=False)
    a.pos = a.slot = None
    ctx.enqueue(A.OP_ATTN_TREE, a)
    t.check()
    d = DnTree(312, 7, [0, 0, 0], 2, 4, kind="chain", planes=0)
    d.slot = np.arange(3, dtype=np.int32)
    d.upload(ctx)
    a = d.args(parent=False)
    a.pos = a.slot = None
    ctx.enqueue(A.OP_DN_TREE, a)
    states = d.check()
    path = np.tile(np.array([0, 1, 2, 3, -1, -1, -1], np.int32), (3, 1))
    k = d.keep_args(ctx.upload(path), ctx.upload(np.full(3, 4, np.int32)))
    k.pos = k.slot = None
    ctx.enqueue(A.OP_DN_KEEP, k)
    got = d.d_state.read(np.float32, d.state.size).reshape(d.state.shape)
    for s in range(3):
        assert O.rel_l2(got[s, 0], states[s][3]) <= DN_TOL
    p = ctx.upload(path)
    a = A.AttnKeepArgs(t.d_kx.ptr, t.d_vx.ptr, t.d_kc.ptr, t.d_vc.ptr, p.ptr, ctx.upload(np.full(3, 4, np.int32)).ptr, None, None, 3, 7, t.nkv, t.d, t.max_cells)
    ctx.enqueue(A.OP_ATTN_KEEP, a)
    kx = t.results()[1]
    kc = t.d_kc.read(np.float16, t.kc.size).reshape(t.kc.shape)
    assert np.array_equal(kc[:, :4], kx[:, :4]) and np.array_equal(kc[:, 4:], t.kc[:, 4:])


def test_two_contexts_at_once(ctx):
    """The same calls on two streams, nothing waited for between them: a context's scratch is its own."""
    other = shv.pkg.Context(0)
    sets = []
    for c, seed in ((ctx, 320), (other, 321)):
        at, dn, ac = AttnTree(seed, "16/2x256", 17, [300, 700]), DnTree(seed, 17, [300, 700], 4, 8), Accept(seed, 2, 17, 30000)
        at.upload(c)
        dn.upload(c)
        bufs = [c.upload(np.full(34, -7, np.int32)) for _ in range(4)]
        up = [c.upload(x) for x in (ac.logits, ac.ids, ac.parent)]
        acc = A.TreeAcceptArgs(up[0].ptr, up[1].ptr, up[2].ptr, None, bufs[0].ptr, bufs[1].ptr, bufs[2].ptr, bufs[3].ptr, None, None, 2, 17, 30000, 30000)
        sets.append((c, at, dn, ac, at.args(c), dn.args(), acc, bufs, up))
    for _ in range(20):
        for c, _, _, _, a, d, acc, *_ in sets:
            c.enqueue(A.OP_ATTN_TREE, a)
            c.enqueue(A.OP_TREE_ACCEPT, acc)
            c.enqueue(A.OP_DN_TREE, d)
    for c, at, dn, ac, _, _, _, bufs, _ in sets:
        c.sync()
        at.check()
        dn.check()
        ac.check([bufs[0].read(np.int32, 34).reshape(2, -1), bufs[1].read(np.int32, 34).reshape(2, -1), bufs[2].read(np.int32, 2), bufs[3].read(np.int32, 2)])
    other.destroy()


@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (7, 4), (32, 0), (33, 40), (100, 3), (700, 700), (2**31 - 1, 2**31 - 1)])
@pytest.mark.parametrize("layout,rows,pos", [("16/2x256", 9, [640, 5, 31]), ("32/8x128", 23, [1111])])
def test_sliding_window_and_sinks(ctx, layout, rows, pos, window, sinks):
    t = AttnTree(7 + window % 1000, layout, rows, pos)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_TREE, t.args(ctx, 16, window, sinks))
    t.check(window, sinks)


def test_rows_in_use_differ_and_the_others_are_left(ctx):
    t = AttnTree(3, "16/2x256", 20, [70, 400, 0, 33, 64], count=[20, 1, 7, 0, -3])
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_TREE, t.args(ctx))
    t.check()
    t.count = np.array([99, 2**31 - 1, 3, -2**31, 64], np.int32)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_TREE, t.args(ctx))
    t.check()


def test_a_sequence_that_does_not_fit_is_left_alone(ctx):
    t = AttnTree(4, "16/2x256", 6, [50, 58, 59, 3])
    assert t.max_cells == 96
    t.upload(ctx)
    args = t.args(ctx)
    args.max_cells = 64  # the same memory as fewer cells: only what is refused is looked at
    t.pos = np.array([59, 64, -1, 2**31 - 4], np.int32)
    t.d_pos.write(t.pos)
    ctx.enqueue(A.OP_ATTN_TREE, args)
    out, kx, vx = t.results()
    assert (out == 77.0).all() and (kx.view(np.uint16) == 0x3555).all() and (vx.view(np.uint16) == 0x3555).all()


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 2)])
def test_what_a_row_does_not_see_may_hold_anything(ctx, window, sinks):
    """NaN and infinities in cells behind the sequence's end and outside the window, and in rows that are no ancestors."""
    parents = [[-1, 0, 0, 1, 2, 2, 5, 1, -1]]
    for bad in (np.nan, np.inf, -np.inf, 1e6):
        t = AttnTree(11, "16/2x256", 9, [103], parents=parents)
        t.kc[:, 103:] = t.vc[:, 103:] = bad
        if window:
            t.kc[:, 2:103 - window + 1] = t.vc[:, 2:103 - window + 1] = bad  # the first row sees positions above 103 - 40, and two sinks
        v0 = 2 * t.nh * t.d + t.nkv * t.d
        t.qkv[0, 4, v0 + 3:v0 + t.nkv * t.d:5] = bad   # row 4's values: no other row stands on it
        t.qkv[0, 2, v0 + 1] = bad                      # row 2's: rows 4, 5 and 6 stand on it
        if not np.isfinite(bad):
            t.qkv[0, 7, v0 - 9] = bad                  # row 7's key
        t.upload(ctx)
        ctx.enqueue(A.OP_ATTN_TREE, t.args(ctx, 16, window, sinks))
        out = t.check(window, sinks)
        for r in (0, 1, 3, 8):
            assert np.isfinite(out[0, r]).all(), r


def test_infinite_values_inside_the_window_reach_the_rows_that_see_them(ctx):
    """Cells that some rows see and deeper ones no more: an infinite value there is the first ones' alone."""
    t = AttnTree(12, "16/2x256", 12, [200], kind="chain")
    t.vc[:, 200 - 20 + 3, :, 5] = np.inf   # seen by rows 0 .. 2
    t.vc[:, 200 - 20 + 8, 1, 77] = np.nan  # by rows 0 .. 7
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_TREE, t.args(ctx, 16, 20, 0))
    out = t.check(20, 0)
    assert not np.isfinite(out[0, 2]).all() and not np.isfinite(out[0, 7]).all() and np.isfinite(out[0, 8:]).all()


def test_a_chain_is_what_attn_decode_makes_of_it(ctx):
    """parent NULL: the rows of a verification pass, as shv_attn_decode attends them and writes their cells, once these are kept."""
    rows, past = 6, 333
    t = AttnTree(21, "16/2x256", rows, [past])
    t.upload(ctx)
    c, n_splits = ctx, 16
    d_kc, d_vc = c.upload(t.kc), c.upload(v_dev(t.vc))
    d_ref, d_part = c.alloc(rows * t.nh * t.d * 4), c.alloc((rows + 1) * t.nh * n_splits * (t.d + 2) * 4)
    c.enqueue(A.OP_ATTN_DECODE, A.AttnDecodeArgs(t.d_qkv.ptr, t.d_qn.ptr, t.d_kn.ptr, t.d_table.ptr, d_kc.ptr, d_vc.ptr, d_part.ptr, d_ref.ptr, t.d_pos.ptr,
                                                 t.d_slot.ptr, 1, rows, t.nh, t.nkv, t.d, t.dims, t.max_cells, t.stride, n_splits, EPS))
    c.enqueue(A.OP_ATTN_TREE, t.args(c, n_splits, parent=False))
    got, ref = t.results()[0][0], d_ref.read(np.float32, rows * t.nh * t.d).reshape(rows, -1)
    for r in range(rows):
        assert O.rel_l2(got[r], ref[r]) <= 1e-4, r  # a key rounded to the other neighbour moves a score by 16 * 2^-12 / 16
    path, n_keep = c.upload(np.arange(rows, dtype=np.int32)), c.upload(np.array([rows], np.int32))
    c.enqueue(A.OP_ATTN_KEEP, A.AttnKeepArgs(t.d_kx.ptr, t.d_vx.ptr, t.d_kc.ptr, t.d_vc.ptr, path.ptr, n_keep.ptr, t.d_pos.ptr, t.d_slot.ptr, 1, rows, t.nkv, t.d,
                                             t.max_cells))
    k, k_ref = (b.read(np.float16, t.kc.size).astype(np.float32) for b in (t.d_kc, d_kc))
    assert (np.abs(k - k_ref) <= np.abs(k_ref) * 2.0 ** -10 + 1e-5).all()
    assert np.array_equal(t.d_vc.read(np.uint16, t.vc.size), d_vc.read(np.uint16, t.vc.size))


def test_cells_far_behind_32_bits(ctx):
    """A slot whose cells lie more than 2^32 bytes and 2^31 elements into the caches."""
    slots, cells = 70, 65536
    t = AttnTree(31, "16/2x256", 4, [1000])
    big = slots * cells * t.nkv * t.d
    assert (slots - 1) * cells * t.nkv * t.d > 2**31
    t.upload(ctx)
    c = ctx
    kc, vc = c.alloc(big * 2), c.alloc(big * 2)
    at = (slots - 1) * cells * t.nkv * t.d * 2
    kc.write(t.kc[0], at)
    vc.write(v_dev(t.vc), at)
    table = c.upload(T.rope_table(2048, t.dims))
    args = t.args(c)
    args.kcache, args.vcache, args.max_cells, args.rope = kc.ptr, vc.ptr, cells, table.ptr
    args.slot = c.upload(np.array([slots - 1], np.int32)).ptr
    c.enqueue(A.OP_ATTN_TREE, args)
    t.slot[:] = 0
    t.check()
    path, n_keep = c.upload(np.array([[0, 1, 3, -1]], np.int32)), c.upload(np.array([3], np.int32))
    c.enqueue(A.OP_ATTN_KEEP, A.AttnKeepArgs(t.d_kx.ptr, t.d_vx.ptr, kc.ptr, vc.ptr, path.ptr, n_keep.ptr, t.d_pos.ptr, args.slot, 1, 4, t.nkv, t.d, cells))
    row = t.nkv * t.d
    got = kc.read(np.float16, 5 * row, at + 999 * row * 2).reshape(5, row)
    kx = t.results()[1][0].reshape(4, row)
    assert np.array_equal(got[0], t.kc[0, 999].reshape(row)) and np.array_equal(got[1:4], kx[[0, 1, 3]]) and np.array_equal(got[4], t.kc[0, 1003].reshape(row))
    kc.free()
    vc.free()


@pytest.mark.parametrize("layout,rows,pos,lens", [("16/2x256", 12, [29], [5]), ("8/8x64", 7, [0, 31, 200], [7, 1, 0]), ("32/8x128", 64, [64, 90], [64, -4]),
                                                 ("5/1x64", 3, [60, 62, 63], [3, 99, 3])])
def test_kept_cells(ctx, layout, rows, pos, lens):
    """The branch's cells, and only they, move in; path entries that are no row and cells behind the cache's end are passed over."""
    t = AttnTree(41 + rows, layout, rows, pos)
    t.upload(ctx)
    rng, c = t.rng, ctx
    cells = 64 if layout == "5/1x64" else t.max_cells
    kx, vx = (rng.standard_normal((t.n_seq, rows, t.nkv, t.d)).astype(np.float16) for _ in range(2))
    path = np.stack([np.sort(rng.permutation(rows)) for _ in pos]).astype(np.int32)
    if rows == 7:
        path[0, 2], path[0, 4], path[0, 5] = -1, 7, 2**31 - 1
    kc, vc = (rng.standard_normal((t.n_seq, cells, t.nkv, t.d)).astype(np.float16) for _ in range(2))
    d_kc, d_vc, d_kx, d_vx = c.upload(kc), c.upload(v_dev(vc)), c.upload(kx), c.upload(vx)
    d_path, d_n = c.upload(path), c.upload(np.array(lens, np.int32))
    c.enqueue(A.OP_ATTN_KEEP, A.AttnKeepArgs(d_kx.ptr, d_vx.ptr, d_kc.ptr, d_vc.ptr, d_path.ptr, d_n.ptr, t.d_pos.ptr, t.d_slot.ptr, t.n_seq, rows, t.nkv, t.d, cells))
    for s in range(t.n_seq):
        for j in range(min(lens[s], rows)):
            r, at = int(path[s, j]), pos[s] + j
            if 0 <= r < rows and at < cells:
                kc[t.slot[s], at], vc[t.slot[s], at] = kx[s, r], vx[s, r]
    assert np.array_equal(d_kc.read(np.float16, kc.size).reshape(kc.shape), kc)
    assert np.array_equal(v_host(d_vc.read(np.float16, vc.size).reshape(v_dev(vc).shape)), vc)


# ---- the delta rule --------------------------------------------------------------------------

D = 128
# States and deltas are sums of at most 64 terms over the ancestors beside one of 128 products; operands are held to 22 bits and the solve
# is as well conditioned as the rule (norms of keys 1, write strengths below 1): a few hundred roundings of 2^-23 at most.
DN_TOL = 1e-5


class DnTree:
    def __init__(self, seed, rows, pos, hk=16, hv=32, count=None, kind="mixed", planes=2, slots=5):
        self.rng = rng = np.random.default_rng(seed)
        self.rows, self.pos, self.hk, self.hv, self.planes, self.ring_slots = rows, np.array(pos, np.int32), hk, hv, planes, slots
        self.n_seq = len(pos)
        self.count = None if count is None else np.array(count, np.int32)
        self.cw = (2 * hk + hv) * D
        self.width = self.cw + hv * D + 2 * hv
        self.stride, self.ring_stride = self.width + 3, self.width + 5
        self.parent = np.stack([T.tree(rng, rows, kind) for _ in pos])
        self.slot = rng.permutation(self.n_seq).astype(np.int32)
        self.x = rng.standard_normal((self.n_seq, rows, self.stride)).astype(np.float32)
        self.ring = rng.standard_normal((self.n_seq, slots, self.ring_stride)).astype(np.float32)
        self.conv1d = (0.3 * rng.standard_normal((self.cw, 4))).astype(np.float32)
        self.a = (-np.exp(rng.standard_normal(hv))).astype(np.float32)
        self.dt_bias = rng.standard_normal(hv).astype(np.float32)
        self.state = (0.1 * rng.standard_normal((self.n_seq, max(planes, 1), hv, D, D))).astype(np.float32)
        self.plane = rng.integers(0, max(planes, 1), self.n_seq).astype(np.int32)

    n = AttnTree.n

    def upload(self, c):
        up, rows = c.upload, self.n_seq * self.rows
        self.d_x, self.d_ring, self.d_conv, self.d_a, self.d_dt = up(self.x), up(self.ring), up(self.conv1d), up(self.a), up(self.dt_bias)
        self.d_state, self.d_plane, self.d_pos, self.d_slot, self.d_parent = up(self.state), up(self.plane), up(self.pos), up(self.slot), up(self.parent)
        self.d_count = None if self.count is None else up(self.count)
        self.d_out, self.d_delta = (up(np.full(rows * self.hv * D, 77.0, np.float32)) for _ in range(2))
        self.d_kn, self.d_decay = up(np.full(rows * self.hk * D, 77.0, np.float32)), up(np.full(rows * self.hv, 77.0, np.float32))

    def args(self, parent=True, norm_max=0):
        return A.DnTreeArgs(self.d_x.ptr, self.d_ring.ptr, self.d_conv.ptr, self.d_a.ptr, self.d_dt.ptr, self.d_state.ptr, self.d_out.ptr, self.d_kn.ptr,
                            self.d_delta.ptr, self.d_decay.ptr, self.d_pos.ptr, self.d_slot.ptr, self.d_plane.ptr if self.planes else None,
                            self.d_parent.ptr if parent else None, A.ptr(self.d_count), self.n_seq, self.rows, self.hk, self.hv, D, 4, self.stride, self.ring_slots,
                            self.ring_stride, self.planes, norm_max, EPS)

    def keep_args(self, d_path, d_n):
        return A.DnKeepArgs(self.d_x.ptr, self.d_kn.ptr, self.d_delta.ptr, self.d_decay.ptr, self.d_state.ptr, self.d_ring.ptr, d_path.ptr, d_n.ptr, self.d_pos.ptr,
                            self.d_slot.ptr, self.d_plane.ptr if self.planes else None, self.n_seq, self.rows, self.hk, self.hv, D, 4, self.stride, self.ring_slots,
                            self.ring_stride, self.planes)

    def want(self, s, norm_max=0):
        slot = self.slot[s]
        return T.dn_tree(self.x[s], self.ring[slot], self.conv1d, self.a, self.dt_bias, self.state[slot, self.plane[slot]], int(self.pos[s]), self.parent[s], self.n(s),
                         self.hk, self.hv, D, EPS, norm_max)

    def results(self):
        lead = (self.n_seq, self.rows)
        read = lambda b, *shape: b.read(np.float32, int(np.prod(lead + shape))).reshape(lead + shape)  # noqa: E731
        return read(self.d_out, self.hv, D), read(self.d_kn, self.hk, D), read(self.d_delta, self.hv, D), read(self.d_decay, self.hv)

    def check(self, norm_max=0):
        got, states = self.results(), []
        for s in range(self.n_seq):
            n = self.n(s)
            *want, st = self.want(s, norm_max)
            states.append(st)
            for name, g, w in zip(("out", "kn", "delta", "decay"), got, want):
                for r in range(n):
                    e = O.rel_l2(g[s, r], w[r])
                    assert e <= DN_TOL, (s, r, name, e)
                assert (g[s, n:] == 77.0).all(), name
        return states


@pytest.mark.parametrize("rows,pos,heads,kind", [
    (1, [0], (16, 32), "chain"), (1, [9], (16, 32), "chain"), (2, [1], (16, 32), "chain"), (5, [2], (16, 32), "mixed"), (3, [700, 0, 3], (16, 32), "star"),
    (16, [40], (16, 48), "mixed"), (17, [8], (16, 32), "wide"), (31, [5, 100], (16, 16), "mixed"), (33, [77], (2, 2), "chain"), (48, [0], (1, 3), "roots"),
    (49, [12], (3, 6), "mixed"), (64, [30], (16, 32), "chain"), (64, [1, 50], (4, 8), "mixed"), (64, [4], (2, 4), "star"), (63, [2**31 - 70], (2, 2), "wide")])
def test_delta_rule_over_a_tree(ctx, rows, pos, heads, kind):
    t = DnTree(10 * rows + pos[0], rows, pos, *heads, kind=kind)
    t.upload(ctx)
    ctx.enqueue(A.OP_DN_TREE, t.args())
    t.check()
    assert np.array_equal(t.d_state.read(np.float32, t.state.size), t.state.ravel()) and np.array_equal(t.d_ring.read(np.float32, t.ring.size), t.ring.ravel())


@pytest.mark.parametrize("planes,slots,norm_max", [(0, 3, 0), (1, 4, 1), (5, 64, 0)])
def test_planes_rings_and_norms(ctx, planes, slots, norm_max):
    t = DnTree(5, 6, [10, 2], 2, 4, planes=planes, slots=slots)
    t.upload(ctx)
    ctx.enqueue(A.OP_DN_TREE, t.args(norm_max=norm_max))
    t.check(norm_max)


def test_delta_rule_leaves_rows_that_are_not_in_use(ctx):
    t = DnTree(6, 24, [10, 2, 900, 7, 1], 2, 4, count=[24, 1, 0, -5, 17])
    t.upload(ctx)
    ctx.enqueue(A.OP_DN_TREE, t.args())
    t.check()
    t.x[:, 17:] = np.nan  # and reads nothing of them
    t.count = np.array([17, 2, 16, 3, 1], np.int32)
    t.upload(ctx)
    ctx.enqueue(A.OP_DN_TREE, t.args())
    t.check()


def test_rows_with_nan_reach_their_descendants_alone(ctx):
    t = DnTree(8, 20, [10], 2, 4)
    t.parent[0] = [-1, 0, 0, 1, 2, 2, 3, 3, 4, 5, 5, 1, 7, 8, 0, 14, 15, 16, 6, 9]
    t.x[0, 5, 3 * D] = np.nan
    t.upload(ctx)
    ctx.enqueue(A.OP_DN_TREE, t.args())
    out = t.results()[0][0]
    below = {i for i in range(20) if 5 in T.chain(t.parent[0], i)}
    clean = DnTree(8, 20, [10], 2, 4)
    clean.parent[:] = t.parent
    want = clean.want(0)[0]
    for r in set(range(20)) - below:
        assert O.rel_l2(out[r], want[r]) <= DN_TOL, r
    assert all(np.isnan(out[r]).any() for r in below)


@pytest.mark.parametrize("rows", [3, 40])
def test_values_and_states_of_any_size(ctx, rows):
    """Value columns and states from 2^-100 to 2^100, far outside binary16: each column by its own scale."""
    t = DnTree(13, rows, [10], 2, 4)
    size = np.exp2(t.rng.integers(-100, 100, 4 * D)).astype(np.float32)
    v0 = 4 * D
    # (conv and SiLU come before the size does: a value is its channel's size times an ordinary number for large sizes, its square for small)
    t.x[0, :, v0:v0 + 4 * D] *= size
    t.ring[:, :, v0:v0 + 4 * D] *= size
    t.state *= size.reshape(4, D, 1)
    t.upload(ctx)
    ctx.enqueue(A.OP_DN_TREE, t.args())
    got = t.results()
    want = t.want(0)
    for name, g, w in (("out", got[0][0], want[0]), ("delta", got[2][0], want[2])):
        for h in range(4):
            for c in range(0, D, 7):
                # a column of `rows` numbers alone: the tolerance of the whole, with room for a sum of 128 products that cancel in one column
                assert O.rel_l2(g[:, h, c], w[:, h, c]) <= 4 * DN_TOL, (name, h, c)


@pytest.mark.parametrize("rows,far,columns", [(3, 20, None), (20, 40, None), (20, 40, 3), (64, 60, None), (64, 60, 77), (40, 24, 5), (33, -60, None)])
def test_rows_of_one_branch_do_not_cost_the_others_their_places(ctx, rows, far, columns):
    """Two branches behind one root, the values of one (all channels of them, or a single one a head) 2^far times the other's: every row of either is as near
    to its own formula as if it were alone."""
    t = DnTree(14, rows, [10], 2, 4)
    t.parent[0] = np.maximum(np.arange(rows) - 2, 0)  # row 0, then odd rows on odd ones and even rows on even ones
    t.parent[0, 0] = -1
    v = np.arange(4 * D, 8 * D) if columns is None else 4 * D + columns + D * np.arange(4)
    t.x[0, 1::2, v] *= np.float32(2.0 ** far)
    t.upload(ctx)
    ctx.enqueue(A.OP_DN_TREE, t.args())
    t.check()


def test_a_row_that_forgets_everything(ctx):
    """A log decay beyond float32's range (a of -3e38): the state before the row counts nothing, the row itself and those behind it are as ever."""
    t = DnTree(15, 20, [10], 2, 4)
    gates = t.x[0, :, t.cw + 4 * D:t.cw + 4 * D + 4]
    gates[:, 1] = -40  # does not decay at all (log(1 + e^-40) is 0 in float32),
    gates[[3, 8, 9], 1] = 12  # but for three rows
    t.dt_bias[1] = 0
    t.a[1] = -3e38
    t.upload(ctx)
    ctx.enqueue(A.OP_DN_TREE, t.args())
    got = t.results()
    with np.errstate(all="ignore"):
        t.a = t.a.astype(np.float64)
        t.x = t.x.astype(np.float64)
        t.x[0, [r for r in range(20) if r not in (3, 8, 9)], t.cw + 4 * D + 1] = -2000  # (in 64 bits a gate that is 0 all the same)
        want = t.want(0)
    for name, g, w in (("out", got[0][0], want[0]), ("delta", got[2][0], want[2])):
        for r in range(20):
            for h in range(4):
                assert O.rel_l2(g[r, h], w[r, h]) <= 2 * DN_TOL, (name, r, h)


def test_strong_and_weak_decays(ctx):
    """Gates far out: states that vanish in one row (a sum of logs of -1000 and below) and states that do not decay at all."""
    t = DnTree(9, 40, [10], 2, 4)
    t.x[0, :, t.cw + 4 * D:t.cw + 4 * D + 4] = np.array([-40, 40, 0, 12], np.float32)
    t.a = np.array([-1, -30, -1e-6, -8], np.float32)
    t.upload(ctx)
    ctx.enqueue(A.OP_DN_TREE, t.args())
    t.check()


@pytest.mark.parametrize("rows,pos,heads,kind,planes", [(5, [700], (16, 32), "mixed", 2), (64, [3, 50], (4, 8), "chain", 3), (30, [0, 1, 2, 3], (2, 2), "mixed", 1),
                                                       (9, [5], (1, 3), "star", 0), (1, [0], (16, 48), "chain", 2)])
def test_kept_state(ctx, rows, pos, heads, kind, planes):
    """The state behind a branch, and the ring's rows, against the rule along the branch."""
    t = DnTree(20 + rows, rows, pos, *heads, kind=kind, planes=planes)
    t.upload(ctx)
    ctx.enqueue(A.OP_DN_TREE, t.args())
    states = t.check()
    path, lens = np.full((t.n_seq, rows), -1, np.int32), np.zeros(t.n_seq, np.int32)
    for s in range(t.n_seq):
        way = T.chain(t.parent[s], rows - 1 - s % rows)[::-1]
        path[s, :len(way)], lens[s] = way, len(way)
    lens[-1] = 0 if t.n_seq > 2 else lens[-1]
    d_path, d_n = ctx.upload(path), ctx.upload(lens)
    ctx.enqueue(A.OP_DN_KEEP, t.keep_args(d_path, d_n))
    got = t.d_state.read(np.float32, t.state.size).reshape(t.state.shape)
    ring = t.d_ring.read(np.float32, t.ring.size).reshape(t.ring.shape)
    want_ring = t.ring.copy()
    for s in range(t.n_seq):
        slot, n = t.slot[s], int(lens[s])
        cur = t.plane[slot]
        nxt = (cur + 1) % max(planes, 1)
        if n:
            e = O.rel_l2(got[slot, nxt], states[s][path[s, n - 1]])
            assert e <= DN_TOL, (s, e)
        else:
            assert np.array_equal(got[slot, nxt], t.state[slot, cur])
        for p in set(range(max(planes, 1))) - {nxt}:
            assert np.array_equal(got[slot, p], t.state[slot, p])
        for j in range(max(0, n - 3), n):
            want_ring[slot, (pos[s] + j) % t.ring_slots, :t.cw] = t.x[s, path[s, j], :t.cw]
    assert np.array_equal(ring, want_ring)


@pytest.mark.parametrize("kind", ["one row", "twenty rows", "beyond float32", "none"])
def test_kept_state_behind_rows_that_forget(ctx, kind):
    """With log_g the state behind a branch is the rule's, row after row, where a row of it forgets all that was: log g of -1200 and then ordinary rows, twenty
    rows of about -37, one of -3e38 times 12.  A weight is e to a sum of at most 30 ordinary log g of 1 or so, each within 2^-22 of itself: 30 * 2^-22 = 7e-6."""
    rows, hv = 32, 4
    t = DnTree(34, rows, [10, 3], 2, hv, kind="chain")
    gates = t.x[:, :, t.cw + hv * D:t.cw + hv * D + hv]
    t.a[:], t.dt_bias[:] = np.array([-1, -0.3, -1, -2], np.float32), 0
    if kind == "one row":
        gates[:, 4] = 1200
    elif kind == "twenty rows":
        gates[:, :20] = 37
    elif kind == "beyond float32":
        gates[:, :, 0] = -40  # a log g of 0 but for three rows
        gates[:, [2, 3, 9], 0] = 12
        t.a[0] = -3e38
    t.upload(ctx)
    d_log = ctx.upload(np.full(2 * rows * hv, 77.0, np.float32))
    a = t.args()
    a.log_g = d_log.ptr
    ctx.enqueue(A.OP_DN_TREE, a)
    if kind == "beyond float32":
        t.a, t.x = t.a.astype(np.float64), t.x.astype(np.float64)
        t.x[:, [r for r in range(rows) if r not in (2, 3, 9)], t.cw + hv * D] = -2000  # (in 64 bits a log g of 0 all the same)
    path = np.tile(np.arange(rows, dtype=np.int32), (2, 1))
    path[1, [3, 30]] = -1, rows  # passed over; the rule without these rows' products and decays is not the chain's: looked at below
    lens = np.array([rows, 0], np.int32)
    k = t.keep_args(ctx.upload(path), ctx.upload(lens))
    k.log_g, k.decay = d_log.ptr, None
    ctx.enqueue(A.OP_DN_KEEP, k)
    got = t.d_state.read(np.float32, t.state.size).reshape(t.state.shape)
    with np.errstate(all="ignore"):
        want = t.want(0)[-1][-1]
    slot = t.slot[0]
    for h in range(hv):
        assert O.rel_l2(got[slot, 1 - t.plane[slot], h], want[h]) <= DN_TOL, h
    slot = t.slot[1]
    assert np.array_equal(got[slot, 1 - t.plane[slot]], t.state[slot, t.plane[slot]])
    # entries that are no row: as the same path without them
    out = []
    for p, n in ((path[1], rows), (np.delete(path[1], [3, 30]), rows - 2)):
        state = ctx.upload(t.state)
        k = t.keep_args(ctx.upload(np.stack([np.resize(p, rows)] * 2)), ctx.upload(np.array([0, n], np.int32)))
        k.log_g, k.state, k.ring = d_log.ptr, state.ptr, ctx.upload(t.ring).ptr
        ctx.enqueue(A.OP_DN_KEEP, k)
        out.append(state.read(np.float32, t.state.size))
    assert np.array_equal(out[0], out[1])


@pytest.mark.parametrize("heads,count", [((16, 32), [7, 5]), ((2, 6), [0, 3])])
def test_log_decays_of_the_rows(ctx, heads, count):
    """log_g is each row's own, of rows in use alone, and leaves everything else as it is without it."""
    t = DnTree(35, 7, [10, 2], *heads, count=count)
    t.upload(ctx)
    hv = heads[1]
    ctx.enqueue(A.OP_DN_TREE, t.args())
    plain = t.results()
    d_log = ctx.upload(np.full(2 * 7 * hv, 77.0, np.float32))
    a = t.args()
    a.log_g = d_log.ptr
    ctx.enqueue(A.OP_DN_TREE, a)
    t.check()
    assert all(np.array_equal(x, y) for x, y in zip(plain, t.results()))
    got = d_log.read(np.float32, 2 * 7 * hv).reshape(2, 7, hv)
    for s in range(2):
        n, decay = t.n(s), t.want(s)[3]
        for r in range(n):
            way = T.chain(t.parent[s], r)
            assert O.rel_l2(got[s, r], decay[r] - (decay[way[1]] if len(way) > 1 else 0)) <= DN_TOL, (s, r)
        assert (got[s, n:] == 77.0).all()


def test_keeping_passes_over_what_is_no_row(ctx):
    t = DnTree(33, 8, [4, 9], 2, 2)
    t.upload(ctx)
    ctx.enqueue(A.OP_DN_TREE, t.args())
    out = []
    for path, lens in (([[0, -1, 2, 8, 5, 2**31 - 1, -9, 6], [0, 3, 4, 5, 6, 7, 1, 2]], [99, -1]), ([[0, 2, 5, 6, 0, 0, 0, 0], [0] * 8], [4, 0])):
        state = ctx.upload(t.state)
        a = t.keep_args(ctx.upload(np.array(path, np.int32)), ctx.upload(np.array(lens, np.int32)))
        a.state, a.ring = state.ptr, ctx.upload(t.ring).ptr
        ctx.enqueue(A.OP_DN_KEEP, a)
        out.append(state.read(np.float32, t.state.size))
    assert np.array_equal(out[0], out[1])


def test_a_chain_is_what_dn_step_makes_of_it(ctx):
    """parent NULL, then the whole chain kept: outputs and state of shv_dn_step over the same rows."""
    rows, hk, hv = 11, 16, 32
    t = DnTree(44, rows, [50], hk, hv, planes=0, slots=14)
    t.stride = t.ring_stride = t.width
    t.x, t.ring = np.ascontiguousarray(t.x[..., :t.width]), np.ascontiguousarray(t.ring[..., :t.width])
    t.upload(ctx)
    c = ctx
    ring = t.ring.copy()
    for i in range(rows):
        ring[0, (50 + i) % 14] = t.x[0, i]
    d_state, d_out = c.upload(t.state), c.alloc(rows * hv * D * 4)
    c.enqueue(A.OP_DN_STEP, A.DnStepArgs(c.upload(ring).ptr, t.d_conv.ptr, t.d_a.ptr, t.d_dt.ptr, d_state.ptr, d_out.ptr, t.d_pos.ptr, t.d_slot.ptr, 1, rows, hk, hv,
                                         D, 4, 14, t.width, EPS, 0, None, 0, 0, None, 0))
    c.enqueue(A.OP_DN_TREE, t.args(parent=False))
    c.enqueue(A.OP_DN_KEEP, t.keep_args(c.upload(np.arange(rows, dtype=np.int32)), c.upload(np.array([rows], np.int32))))
    assert O.rel_l2(t.results()[0].ravel(), d_out.read(np.float32, rows * hv * D)) <= DN_TOL
    assert O.rel_l2(t.d_state.read(np.float32, t.state.size), d_state.read(np.float32, t.state.size)) <= DN_TOL


# ---- acceptance ------------------------------------------------------------------------------


class Accept:
    def __init__(self, seed, n_seq, rows, n, count=None, stride=0, kind="mixed"):
        self.rng = rng = np.random.default_rng(seed)
        self.n_seq, self.rows, self.n, self.stride = n_seq, rows, n, stride or n
        self.count = None if count is None else np.array(count, np.int32)
        self.parent = np.stack([T.tree(rng, rows, kind) for _ in range(n_seq)])
        self.logits = rng.standard_normal((n_seq, rows, self.stride)).astype(np.float32)
        self.settle(0.7)

    n_of = AttnTree.n

    def settle(self, share):
        self.best = np.array([[T.first_max(self.logits[s, r, :self.n]) for r in range(self.rows)] for s in range(self.n_seq)], np.int32)
        self.ids = np.zeros((self.n_seq, self.rows), np.int32)
        for s in range(self.n_seq):
            for r in range(self.rows):
                p = int(self.parent[s, r])
                agree = 0 <= p < r and self.rng.random() < share
                self.ids[s, r] = self.best[s, p] if agree else self.rng.integers(0, self.n)

    def run(self, c, picks=None, pos=None, graph=0, **kw):
        up = c.upload
        d_best = up(np.full((self.n_seq, self.rows), -7, np.int32) if picks is None else picks)
        d_path, d_n, d_next = up(np.full((self.n_seq, self.rows), -8, np.int32)), up(np.full(self.n_seq, -9, np.int32)), up(np.full(self.n_seq, -9, np.int32))
        d_pos, d_base = (up(pos), up(np.zeros_like(pos))) if pos is not None else (None, None)
        a = A.TreeAcceptArgs(None if picks is not None else up(self.logits).ptr, up(self.ids).ptr, up(self.parent).ptr if kw.get("parent", True) else None,
                             None if self.count is None else up(self.count).ptr, d_best.ptr, d_path.ptr, d_n.ptr, d_next.ptr, A.ptr(d_pos), A.ptr(d_base), self.n_seq,
                             self.rows, self.n, self.stride)
        c.enqueue(A.OP_TREE_ACCEPT, a)
        rows = self.n_seq * self.rows
        got = [d_best.read(np.int32, rows).reshape(self.n_seq, -1), d_path.read(np.int32, rows).reshape(self.n_seq, -1), d_n.read(np.int32, self.n_seq), d_next.read(np.int32, self.n_seq)]
        if pos is not None:
            got += [d_pos.read(np.int32, self.n_seq), d_base.read(np.int32, self.n_seq)]
        return got

    def check(self, got, best=None, parent=None):
        n_best, path, n_keep, nxt = got[:4]
        for s in range(self.n_seq):
            n = AttnTree.n(self, s)
            want = (self.best if best is None else best)[s]
            if best is None:
                assert np.array_equal(n_best[s, :n], want[:n]) and (n_best[s, n:] == -7).all()
            way, after = T.accept(want, self.ids[s], (self.parent if parent is None else parent)[s], n)
            assert path[s].tolist() == way + [-1] * (self.rows - len(way)) and n_keep[s] == len(way) and nxt[s] == after


@pytest.mark.parametrize("n_seq,rows,n,stride", [(1, 1, 1, 0), (1, 2, 3, 0), (1, 5, 151936, 0), (3, 24, 4097, 4099), (1, 64, 50000, 50004), (17, 9, 1000, 1001), (2, 64, 2049, 0),
                                                (250, 64, 65, 0), (1024, 3, 40, 0)])
def test_the_branch_the_model_agrees_with(ctx, n_seq, rows, n, stride):
    t = Accept(n_seq + rows + n, n_seq, rows, n, stride=stride)
    t.check(t.run(ctx))


@pytest.mark.parametrize("kind", ["chain", "star", "roots", "wide"])
def test_branches_of_other_trees(ctx, kind):
    t = Accept(60, 9, 40, 3000, count=[40, 1, 0, -1, 39, 99, 7, 20, 2], kind=kind)
    t.check(t.run(ctx))
    if kind == "chain":
        t.check(t.run(ctx, parent=False))


def test_ties_nan_and_infinities_in_the_logits(ctx):
    t = Accept(61, 1, 12, 9000)
    t.logits[0, 0, [8999, 17, 4096]] = 50           # the first of equals
    t.logits[0, 1] = np.nan                         # nothing but NaN: 0
    t.logits[0, 2] = -np.inf
    t.logits[0, 3, :4000], t.logits[0, 3, 7777] = np.nan, np.inf
    t.logits[0, 4] = np.nan
    t.logits[0, 4, 5000:] = -np.inf                 # -inf behind NaN
    t.logits[0, 5] = 0.0
    t.logits[0, 5, 3] = -0.0
    t.settle(0.9)
    assert t.best[0, :3].tolist() == [17, 0, 0] and t.best[0, 3] == 7777 and t.best[0, 5] == 0
    t.best[0, 4] = 5000  # NaN never wins: the first that is a number
    t.check(t.run(ctx))


def test_of_equal_children_the_lowest_goes_on_and_positions_move(ctx):
    t = Accept(62, 2, 6, 100)
    t.parent = np.array([[-1, 0, 0, 0, 2, 1], [-1, 0, 1, 2, 3, 4]], np.int32)
    picks = np.array([[5, 6, 7, 8, 9, 4], [1, 2, 3, 4, 5, 6]], np.int32)
    t.ids = np.array([[0, 5, 5, 5, 7, 6], [0, 1, 2, 3, 4, 99]], np.int32)
    got = t.run(ctx, picks=picks, pos=np.array([10, 200], np.int32))
    t.check(got, best=picks)
    assert got[1].tolist() == [[0, 1, 5, -1, -1, -1], [0, 1, 2, 3, 4, -1]] and got[3].tolist() == [4, 5]
    assert got[4].tolist() == [13, 205] and got[5].tolist() == [10, 200] and np.array_equal(got[0], picks)


@pytest.mark.parametrize("given", [False, True])
def test_a_sequence_without_room_keeps_nothing(ctx, given):
    """max_cells: by rows in use, on both sides of the line; without it the walk is the tree's."""
    t = Accept(63, 7, 6, 400, count=[6, 6, 5, 6, 1, 0, 6])
    pos = np.array([58, 59, 59, -1, 63, 64, 2**31 - 3], np.int32)
    left = [1, 3, 5, 6]
    for cells in (64, 0):
        up = ctx.upload
        bufs = [up(t.best if given else np.full((7, 6), -7, np.int32)), up(np.full((7, 6), -8, np.int32)), up(np.full(7, -9, np.int32)), up(np.full(7, -9, np.int32)), up(pos),
                up(np.full(7, -9, np.int32))]
        a = A.TreeAcceptArgs(None if given else up(t.logits).ptr, up(t.ids).ptr, up(t.parent).ptr, up(t.count).ptr, *[b.ptr for b in bufs], 7, 6, t.n, t.stride, cells)
        if not cells:
            a.pos = a.base = None
        ctx.enqueue(A.OP_TREE_ACCEPT, a)
        best, path, n_keep, nxt, after, base = [b.read(np.int32, 42 if i < 2 else 7) for i, b in enumerate(bufs)]
        best, path = best.reshape(7, 6), path.reshape(7, 6)
        if not cells:
            t.check([best, path, n_keep, nxt], best=t.best if given else None)
            continue
        assert np.array_equal(base, pos)
        for s in range(7):
            way, want_next = T.accept(t.best[s], t.ids[s], t.parent[s], 0 if s in left else t.n_of(s))
            assert path[s].tolist() == way + [-1] * (6 - len(way)) and n_keep[s] == len(way) and nxt[s] == want_next and after[s] == pos[s] + len(way), s


# ---- as they are used together -----------------------------------------------------------------


def test_rounds_of_a_hybrid_pair_of_layers_recorded_and_replayed(ctx):
    """Trees verified, a branch chosen and kept, round after round through one recorded sequence of ops (attention, delta rule, acceptance, keeping), for two
    sequences: what every round computes is what the float64 forms make of the tokens kept so far, one long chain."""
    rounds, rows, n_seq, vocab = 4, 10, 2, 500
    c = ctx
    at = AttnTree(70, "16/2x256", rows, [45, 130])
    at.max_cells += 64
    at.table = T.rope_table(at.max_cells, at.dims)
    at.kc, at.vc = (np.concatenate([x, np.zeros_like(x[:, :64])], 1) for x in (at.kc, at.vc))
    dn = DnTree(71, rows, [45, 130], 2, 4, slots=6)
    ac = Accept(72, n_seq, rows, vocab)
    dn.slot = at.slot
    at.upload(c)
    dn.upload(c)
    d_ids, d_logits = c.upload(ac.ids), c.upload(ac.logits)
    d_best, d_path, d_n, d_next, d_base = c.alloc(80), c.alloc(80), c.alloc(8), c.alloc(8), c.alloc(8)
    dargs, kargs = dn.args(), dn.keep_args(d_path, d_n)
    dargs.pos, dargs.parent, kargs.pos, kargs.plane = at.d_pos.ptr, at.d_parent.ptr, d_base.ptr, dn.d_plane.ptr
    ops = [A.make_op(A.OP_ATTN_TREE, at.args(c, 8)), A.make_op(A.OP_DN_TREE, dargs),
           A.make_op(A.OP_TREE_ACCEPT, A.TreeAcceptArgs(d_logits.ptr, d_ids.ptr, at.d_parent.ptr, None, d_best.ptr, d_path.ptr, d_n.ptr, d_next.ptr, at.d_pos.ptr,
                                                       d_base.ptr, n_seq, rows, vocab, vocab)),
           A.make_op(A.OP_ATTN_KEEP, A.AttnKeepArgs(at.d_kx.ptr, at.d_vx.ptr, at.d_kc.ptr, at.d_vc.ptr, d_path.ptr, d_n.ptr, d_base.ptr, at.d_slot.ptr, n_seq, rows,
                                                   at.nkv, at.d, at.max_cells)),
           A.make_op(A.OP_DN_KEEP, kargs),
           A.make_op(A.OP_ADVANCE, A.AdvanceArgs(dn.d_plane.ptr, n_seq, 1))]
    rec = c.prerecord(ops)
    pos, plane = at.pos.copy(), dn.plane.copy()
    for k in range(rounds):
        rng = at.rng
        at.qkv = rng.standard_normal(at.qkv.shape).astype(np.float32)
        dn.x = rng.standard_normal(dn.x.shape).astype(np.float32)
        at.parent = dn.parent = ac.parent = np.stack([T.tree(rng, rows) for _ in range(n_seq)])
        ac.logits = rng.standard_normal(ac.logits.shape).astype(np.float32)
        ac.settle(0.8)
        for b, v in ((at.d_qkv, at.qkv), (dn.d_x, dn.x), (at.d_parent, at.parent), (d_ids, ac.ids), (d_logits, ac.logits)):
            b.write(v)
        at.pos = dn.pos = pos
        dn.plane = plane % 2
        if k % 2:
            rec.launch()
        else:
            rec.submit()
        at.check()
        states = dn.check()
        path, n_keep = d_path.read(np.int32, 20).reshape(2, 10), d_n.read(np.int32, 2)
        ac.check([np.where(True, d_best.read(np.int32, 20).reshape(2, 10), 0), path, n_keep, d_next.read(np.int32, 2)])
        # the next round's past
        _, kx, vx = at.results()
        state = dn.d_state.read(np.float32, dn.state.size).reshape(dn.state.shape)
        for s in range(n_seq):
            slot, n = at.slot[s], int(n_keep[s])
            at.kc[slot, pos[s]:pos[s] + n], at.vc[slot, pos[s]:pos[s] + n] = kx[s, path[s, :n]], vx[s, path[s, :n]]
            assert O.rel_l2(state[slot, (plane[slot] + 1) % 2], states[s][path[s, n - 1]]) <= DN_TOL
            for j in range(max(0, n - 3), n):
                dn.ring[slot, (pos[s] + j) % dn.ring_slots, :dn.cw] = dn.x[s, path[s, j], :dn.cw]
        dn.state = state
        assert np.array_equal(at.d_kc.read(np.float16, at.kc.size).reshape(at.kc.shape), at.kc)
        assert np.array_equal(v_host(at.d_vc.read(np.float16, at.vc.size).reshape(v_dev(at.vc).shape)), at.vc)
        assert np.array_equal(dn.d_ring.read(np.float32, dn.ring.size).reshape(dn.ring.shape), dn.ring)
        pos, plane = pos + n_keep, plane + 1
        assert np.array_equal(at.d_pos.read(np.int32, 2), pos)
    rec.destroy()


def test_a_recorded_round_at_the_caches_end(ctx):
    """Rounds of four sequences of which two run out of cells, one at once and one after a round: these stay as they are, round after round, while the others go on."""
    rounds, rows, n_seq, vocab, cells = 4, 8, 4, 300, 96
    c = ctx
    at = AttnTree(90, "16/2x256", rows, [40, 89, 80, 3])
    at.max_cells = cells
    at.table = T.rope_table(cells, at.dims)
    at.kc, at.vc = (at.rng.standard_normal((n_seq, cells, at.nkv, at.d), dtype=np.float32).astype(np.float16) for _ in range(2))
    dn = DnTree(91, rows, [40, 89, 80, 3], 2, 4, slots=5)
    dn.slot = at.slot
    ac = Accept(92, n_seq, rows, vocab)
    at.upload(c)
    dn.upload(c)
    d_ids, d_logits = c.upload(ac.ids), c.upload(ac.logits)
    d_best, d_path, d_n, d_next, d_base = (c.alloc(4 * k) for k in (32, 32, 4, 4, 4))
    dargs, kargs = dn.args(), dn.keep_args(d_path, d_n)
    d_log = c.alloc(n_seq * rows * dn.hv * 4)
    dargs.pos, dargs.parent, kargs.pos, kargs.plane, dargs.log_g, kargs.log_g = at.d_pos.ptr, at.d_parent.ptr, d_base.ptr, dn.d_plane.ptr, d_log.ptr, d_log.ptr
    rec = c.prerecord([
        A.make_op(A.OP_ATTN_TREE, at.args(c, 8)), A.make_op(A.OP_DN_TREE, dargs),
        A.make_op(A.OP_TREE_ACCEPT, A.TreeAcceptArgs(d_logits.ptr, d_ids.ptr, at.d_parent.ptr, None, d_best.ptr, d_path.ptr, d_n.ptr, d_next.ptr, at.d_pos.ptr, d_base.ptr,
                                                     n_seq, rows, vocab, vocab, cells)),
        A.make_op(A.OP_ATTN_KEEP, A.AttnKeepArgs(at.d_kx.ptr, at.d_vx.ptr, at.d_kc.ptr, at.d_vc.ptr, d_path.ptr, d_n.ptr, d_base.ptr, at.d_slot.ptr, n_seq, rows, at.nkv,
                                                 at.d, cells)),
        A.make_op(A.OP_DN_KEEP, kargs), A.make_op(A.OP_ADVANCE, A.AdvanceArgs(dn.d_plane.ptr, n_seq, 1))])
    pos, plane = at.pos.copy(), dn.plane.copy()
    full = 0
    for k in range(rounds):
        at.qkv = at.rng.standard_normal(at.qkv.shape).astype(np.float32)
        dn.x = at.rng.standard_normal(dn.x.shape).astype(np.float32)
        at.parent = dn.parent = ac.parent = np.stack([T.tree(at.rng, rows) for _ in range(n_seq)])
        ac.logits = at.rng.standard_normal(ac.logits.shape).astype(np.float32)
        ac.settle(1.0)
        kx_was, vx_was, out_was = at.results()[1:] + (at.results()[0],)
        for b, v in ((at.d_qkv, at.qkv), (dn.d_x, dn.x), (at.d_parent, at.parent), (d_ids, ac.ids), (d_logits, ac.logits)):
            b.write(v)
        dn.plane = plane % 2
        rec.launch()
        out, kx, vx = at.results()
        state = dn.d_state.read(np.float32, dn.state.size).reshape(dn.state.shape)
        path, n_keep, nxt = d_path.read(np.int32, 32).reshape(4, 8), d_n.read(np.int32, 4), d_next.read(np.int32, 4)
        for s in range(n_seq):
            slot, cur = at.slot[s], plane[at.slot[s]] % 2
            if pos[s] + rows > cells:
                full += 1
                assert n_keep[s] == 0 and nxt[s] == -1 and (path[s] == -1).all()
                assert np.array_equal(out[s], out_was[s]) and np.array_equal(kx[s], kx_was[s]) and np.array_equal(vx[s], vx_was[s])
                assert np.array_equal(state[slot, 1 - cur], dn.state[slot, cur])
                continue
            way, after = T.accept(ac.best[s], ac.ids[s], ac.parent[s], rows)
            n = len(way)
            assert path[s, :n].tolist() == way and n_keep[s] == n and nxt[s] == after
            want = T.attn_tree(at.qkv[s], at.q_norm, at.k_norm, at.table, at.kc[slot], at.vc[slot], int(pos[s]), at.parent[s], rows, at.nh, at.nkv, at.d, at.dims, EPS)[0]
            assert O.rel_l2(out[s], want) <= ATTN_TOL
            states = T.dn_tree(dn.x[s], dn.ring[slot], dn.conv1d, dn.a, dn.dt_bias, dn.state[slot, cur], int(pos[s]), dn.parent[s], rows, dn.hk, dn.hv, D, EPS)[-1]
            assert O.rel_l2(state[slot, 1 - cur], states[way[-1]]) <= DN_TOL
            at.kc[slot, pos[s]:pos[s] + n], at.vc[slot, pos[s]:pos[s] + n] = kx[s, way], vx[s, way]
            for j in range(max(0, n - 3), n):
                dn.ring[slot, (pos[s] + j) % dn.ring_slots, :dn.cw] = dn.x[s, way[j], :dn.cw]
            pos[s] += n
        dn.state = state
        plane = plane + 1
        assert np.array_equal(at.d_pos.read(np.int32, 4), pos)
        assert np.array_equal(at.d_kc.read(np.float16, at.kc.size).reshape(at.kc.shape), at.kc)
        assert np.array_equal(v_host(at.d_vc.read(np.uint16, at.vc.size).reshape(v_dev(at.vc).shape)).view(np.float16), at.vc)
        assert np.array_equal(dn.d_ring.read(np.float32, dn.ring.size).reshape(dn.ring.shape), dn.ring)
    assert rounds < full < 2 * rounds  # one from the start, one from some round on
    rec.destroy()


def test_sequences_that_are_not_there(ctx):
    """One recording for five sequences of which two, then three others, then none are there: slots of -1 and counts of 0.  What belongs to the others is theirs, and
    memory in front of caches, rings and states stays as it is."""
    rows, vocab = 9, 300
    c = ctx
    at, dn = AttnTree(95, "16/2x256", rows, [40, 33, 70, 5, 64], count=[9, 0, 4, 0, 0]), DnTree(96, rows, [40, 33, 70, 5, 64], 2, 4, slots=5, count=[9, 0, 4, 0, 0])
    ac = Accept(97, 5, rows, vocab)
    dn.slot, dn.parent, ac.parent = at.slot, at.parent, at.parent
    ac.settle(0.9)
    at.slot[[1, 3, 4]] = -1
    at.upload(c)
    dn.upload(c)

    def behind_a_wall(v):  # in memory with as much again in front
        n = (v.nbytes + 15) // 16 * 16
        b = c.upload(np.concatenate([np.full(n, 0xA5, np.uint8), np.frombuffer(v.tobytes(), np.uint8)]))
        return b, b.ptr + n, n

    walls = [behind_a_wall(v) for v in (at.kc, v_dev(at.vc), dn.ring, dn.state)]
    (_, kc, _), (_, vc, _), (_, ring, _), (_, state, _) = walls
    bufs = [c.upload(np.full(k, -7, np.int32)) for k in (45, 45, 5, 5, 5)]
    best, path, n_keep, nxt, base = bufs
    aa, da, ka = at.args(c, 6), dn.args(), dn.keep_args(path, n_keep)
    aa.kcache, aa.vcache, da.ring, da.state, ka.ring, ka.state = kc, vc, ring, state, ring, state
    da.slot = ka.slot = at.d_slot.ptr
    da.count = at.d_count.ptr
    da.pos, ka.pos = at.d_pos.ptr, base.ptr
    rec = c.prerecord([A.make_op(A.OP_ATTN_TREE, aa), A.make_op(A.OP_DN_TREE, da),
                       A.make_op(A.OP_TREE_ACCEPT, A.TreeAcceptArgs(c.upload(ac.logits).ptr, c.upload(ac.ids).ptr, at.d_parent.ptr, at.d_count.ptr, best.ptr, path.ptr, n_keep.ptr,
                                                                    nxt.ptr, at.d_pos.ptr, base.ptr, 5, rows, vocab, vocab, at.max_cells)),
                       A.make_op(A.OP_ATTN_KEEP, A.AttnKeepArgs(at.d_kx.ptr, at.d_vx.ptr, kc, vc, path.ptr, n_keep.ptr, base.ptr, at.d_slot.ptr, 5, rows, at.nkv, at.d, at.max_cells)),
                       A.make_op(A.OP_DN_KEEP, ka)])
    for count, slots in (([9, 0, 4, 0, 0], [3, -1, 0, -1, -1]), ([0, 7, 0, 2, 1], [-1, 2, -1, 1, 4]), ([0] * 5, [-1] * 5)):
        pos = at.d_pos.read(np.int32, 5)
        at.count, at.slot = np.array(count, np.int32), np.array(slots, np.int32)
        at.d_count.write(at.count)
        at.d_slot.write(at.slot)
        rec.launch()
        keep = n_keep.read(np.int32, 5)
        kx, vx = at.results()[1:]
        for s in range(5):
            way, after = T.accept(ac.best[s], ac.ids[s], ac.parent[s], count[s])
            assert path.read(np.int32, 45).reshape(5, 9)[s].tolist() == way + [-1] * (9 - len(way)) and keep[s] == len(way) and nxt.read(np.int32, 5)[s] == after
            if slots[s] < 0:
                continue
            j = slots[s]
            want = T.dn_tree(dn.x[s], dn.ring[j], dn.conv1d, dn.a, dn.dt_bias, dn.state[j, dn.plane[j]], int(pos[s]), dn.parent[s], count[s], 2, 4, D, EPS)
            for r in range(count[s]):
                assert O.rel_l2(dn.results()[0][s, r], want[0][r]) <= DN_TOL
            dn.state[j, 1 - dn.plane[j]] = want[-1][way[-1]]
            at.kc[j, pos[s]:pos[s] + len(way)], at.vc[j, pos[s]:pos[s] + len(way)] = kx[s, way], vx[s, way]
            for e in range(max(0, len(way) - 3), len(way)):
                dn.ring[j, (pos[s] + e) % dn.ring_slots, :dn.cw] = dn.x[s, way[e], :dn.cw]
        got = [b.read(np.uint8, b.nbytes) for b, _, n in walls]
        assert all((g[:n] == 0xA5).all() for g, (_, _, n) in zip(got, walls))
        body = [g[n:].tobytes() for g, (_, _, n) in zip(got, walls)]
        assert body[0] == at.kc.tobytes() and body[1] == v_dev(at.vc).tobytes() and body[2] == dn.ring.tobytes()
        got_state = np.frombuffer(body[3], np.float32).reshape(dn.state.shape)
        assert O.rel_l2(got_state.ravel(), dn.state.ravel()) <= DN_TOL
        for j in range(5):
            if j not in slots:
                assert np.array_equal(got_state[j], dn.state[j]), j
        dn.state = got_state.copy()
    rec.destroy()


def test_recorded_rounds_in_place_on_some_of_the_slots(ctx):
    """One state a slot, two sequences on two of five slots: rounds need nothing advanced, and the other slots' states and rings are not touched."""
    rows, vocab, n_seq = 7, 200, 2
    c = ctx
    dn, ac = DnTree(98, rows, [20, 6, 1, 1, 1], 2, 4, planes=1, slots=4), Accept(99, n_seq, rows, vocab)
    dn.n_seq, dn.pos, dn.slot = n_seq, dn.pos[:n_seq].copy(), np.array([4, 1], np.int32)
    dn.x, dn.parent = dn.x[:n_seq], dn.parent[:n_seq]
    ac.parent = dn.parent
    dn.upload(c)
    d_ids, d_logits, d_log = c.upload(ac.ids), c.upload(ac.logits), c.alloc(n_seq * rows * 4 * 4)
    best, path, n_keep, nxt, base = (c.upload(np.zeros(k, np.int32)) for k in (14, 14, 2, 2, 2))
    da, ka = dn.args(), dn.keep_args(path, n_keep)
    da.log_g = ka.log_g = d_log.ptr
    ka.pos, ka.decay = base.ptr, None
    rec = c.prerecord([A.make_op(A.OP_DN_TREE, da),
                       A.make_op(A.OP_TREE_ACCEPT, A.TreeAcceptArgs(d_logits.ptr, d_ids.ptr, dn.d_parent.ptr, None, best.ptr, path.ptr, n_keep.ptr, nxt.ptr, dn.d_pos.ptr,
                                                                    base.ptr, n_seq, rows, vocab, vocab)),
                       A.make_op(A.OP_DN_KEEP, ka)])
    for _ in range(4):
        dn.x = dn.rng.standard_normal(dn.x.shape).astype(np.float32)
        ac.settle(0.9)
        dn.d_x.write(dn.x)
        d_ids.write(ac.ids)
        rec.launch()
        states = dn.check()
        for s in range(n_seq):
            way, _ = T.accept(ac.best[s], ac.ids[s], ac.parent[s], rows)
            assert path.read(np.int32, 14).reshape(2, 7)[s].tolist() == way + [-1] * (7 - len(way))
            got = dn.d_state.read(np.float32, dn.state.size).reshape(dn.state.shape)[dn.slot[s], 0]
            assert O.rel_l2(got, states[s][way[-1]]) <= DN_TOL
            dn.state[dn.slot[s], 0] = got
            for e in range(max(0, len(way) - 3), len(way)):
                dn.ring[dn.slot[s], (dn.pos[s] + e) % dn.ring_slots, :dn.cw] = dn.x[s, way[e], :dn.cw]
            dn.pos[s] += len(way)
        assert np.array_equal(dn.d_state.read(np.float32, dn.state.size), dn.state.ravel()) and np.array_equal(dn.d_ring.read(np.float32, dn.ring.size), dn.ring.ravel())
        assert np.array_equal(dn.d_pos.read(np.int32, 2), dn.pos)
    rec.destroy()


def test_two_recorded_passes_share_a_context(ctx):
    """Two recordings of all five ops with inputs of their own, replayed in turn with eager calls of a third between them: the context's scratch
    carries nothing from one to another."""
    c = ctx
    sets = []
    for i, (rows, pos) in enumerate(((5, [90]), (33, [300, 12]), (1, [7]))):
        at, dn, ac = AttnTree(80 + i, "16/2x256", rows, pos), DnTree(83 + i, rows, pos, 2, 4), Accept(86 + i, len(pos), rows, 20000)
        at.upload(c)
        dn.upload(c)
        d = [c.upload(x) for x in (ac.logits, ac.ids, ac.parent)]
        d_best, d_path, d_n, d_next = (c.upload(np.full(len(pos) * rows, -7, np.int32)) for _ in range(4))
        acc = A.TreeAcceptArgs(d[0].ptr, d[1].ptr, d[2].ptr, None, d_best.ptr, d_path.ptr, d_n.ptr, d_next.ptr, None, None, len(pos), rows, 20000, 20000)
        sets.append((at, dn, ac, [A.make_op(A.OP_ATTN_TREE, at.args(c)), A.make_op(A.OP_TREE_ACCEPT, acc), A.make_op(A.OP_DN_TREE, dn.args())], (d_best, d_path, d_n, d_next)))

    def check(at, dn, ac, _, bufs):
        at.check()
        dn.check()
        q = at.n_seq * at.rows
        ac.check([bufs[0].read(np.int32, q).reshape(at.n_seq, -1), bufs[1].read(np.int32, q).reshape(at.n_seq, -1), bufs[2].read(np.int32, at.n_seq), bufs[3].read(np.int32, at.n_seq)])

    recs = [c.prerecord(s[3]) for s in sets[:2]]
    for _ in range(3):
        recs[0].launch()
        recs[1].launch()
        c.dispatch_multi(sets[2][3])
        recs[0].launch()
        for s in sets:
            check(*s)
            s[0].d_out.write(np.full(s[0].n_seq * s[0].rows * s[0].nh * s[0].d, 77.0, np.float32))
    for r in recs:
        r.destroy()
