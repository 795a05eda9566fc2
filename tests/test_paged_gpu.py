"""A serving batch over a paged cache on the GPU: the pages of a pass, attention of packed rows over them, log probabilities, against plain forms of the
definitions, and the three together as a server's passes."""
import numpy as np
import pytest

import oracle_lib as O
import paged_oracle as P
import shv
import tree_oracle as T

pytestmark = pytest.mark.gpu
A = shv.api
EPS = 1e-6
LAYOUTS = {"16/2x256": (16, 2, 256, 64), "32/8x128": (32, 8, 128, 128), "12/2x128": (12, 2, 128, 0), "8/8x64": (8, 8, 64, 32), "5/1x64": (5, 1, 64, 6), "64/1x64": (64, 1, 64, 10),
           "6/2x256": (6, 2, 256, 24), "9/3x128": (9, 3, 128, 12), "32/16x128": (32, 16, 128, 64), "7/7x256": (7, 7, 256, 256)}
# A score is a sum of d products q k / sqrt(d) of normed vectors, in absolute values at most about sqrt(d) <= 16.  Queries and weights enter the products to 22 bits
# and sums are float32: an error of a score is within 16 * (2^-22 + a few 2^-24) = 1e-5, of a weight as much again relative to it, of a weighted mean of the values
# no more than that.
ATTN_TOL = 2e-5


def v_dev(vp):
    """[pages][page][nkv][d] to the device's tiles of 32 cells"""
    n, page, nkv, d = vp.shape
    return np.ascontiguousarray(np.moveaxis(vp.reshape(n, page // 32, 32, nkv, d), 2, -1))


# ---- the plan ----------------------------------------------------------------------------------


class Plan:
    """Sequences of a pool in a state that passes leave: tables whose pages are nobody else's, a stack of the free ones."""

    def __init__(self, seed, n_seq, page, max_pages, longest, spare, max_rows, odd=True, row_seq=True, shared=True, base=True):
        self.rng = rng = np.random.default_rng(seed)
        self.page, self.max_pages, self.max_rows, self.n_seq = page, max_pages, max_rows, n_seq
        self.pos = rng.integers(0, longest + 1, n_seq).astype(np.int32)
        held = -(-self.pos // page)
        if odd:
            held = held + (rng.random(n_seq) < 0.3) * rng.integers(0, 4, n_seq)  # more than they need
        self.held = np.minimum(held, max_pages).astype(np.int32)
        self.n_pages = int(self.held.sum()) + spare + 7
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((n_seq, max_pages), -99, np.int32)
        at = 0
        for s, h in enumerate(self.held):
            self.table[s, :h] = order[at:at + h]
            at += h
        self.free = np.concatenate([order[at:at + spare], np.full(self.n_pages - spare, -77, np.int32)])
        self.n_free = spare
        self.shared = rng.integers(0, self.held + 1).astype(np.int32) if shared else None
        self.row_seq, self.base = row_seq, base
        if odd and n_seq > 3:
            self.pos[rng.integers(n_seq)] = -3

    def upload(self, c):
        up = c.upload
        self.d = dict(pos=up(self.pos), table=up(self.table), held=up(self.held), free=up(self.free), n_free=up(np.array([self.n_free], np.int32)),
                      shared=None if self.shared is None else up(self.shared), start=up(np.full(self.n_seq + 1, -5, np.int32)),
                      maps=[up(np.full(self.max_rows, -5, np.int32)) for _ in range(3)], base=up(np.full(self.n_seq, -5, np.int32)), rows=c.alloc(self.n_seq * 4))

    def args(self):
        d = self.d
        return A.PagePlanArgs(d["rows"].ptr, d["pos"].ptr, d["table"].ptr, d["held"].ptr, d["free"].ptr, d["n_free"].ptr, A.ptr(d["shared"]), d["start"].ptr,
                              d["maps"][0].ptr if self.row_seq else None, d["maps"][1].ptr, d["maps"][2].ptr, d["base"].ptr if self.base else None, self.n_seq, self.page,
                              self.max_pages, self.n_pages, self.max_rows)

    def check(self, rows, seen):
        """What the device holds against the plan made of the host's state, which moves on; `seen`: the maps as they were."""
        w = P.plan(rows, self.pos, self.table, self.held, self.free, self.n_free, self.shared, self.page, self.max_pages, self.max_rows, self.base)
        d, n = self.d, self.n_seq
        assert np.array_equal(d["start"].read(np.int32, n + 1), w["start"])
        total = int(w["start"][-1])
        for k in range(3):
            if k == 0 and not self.row_seq:
                assert (d["maps"][0].read(np.int32, self.max_rows) == -5).all()
                continue
            seen[k][:total] = w["maps"][:, k]
            assert np.array_equal(d["maps"][k].read(np.int32, self.max_rows), seen[k])  # rows behind the last as they were
        assert np.array_equal(d["held"].read(np.int32, n), w["held"])
        assert np.array_equal(d["pos"].read(np.int32, n), w["pos"])
        if self.base:
            assert np.array_equal(d["base"].read(np.int32, n), w["base"])
        top = d["n_free"].read(np.int32, 1)[0]
        assert top == w["n_free"]
        assert np.array_equal(d["free"].read(np.int32, self.n_pages)[:top], w["free"][:top])
        table = d["table"].read(np.int32, n * self.max_pages).reshape(n, -1)
        for s in range(n):
            assert np.array_equal(table[s, :w["held"][s]], w["table"][s, :w["held"][s]]), s
        self.table, self.held, self.free, self.n_free, self.pos = table, w["held"].astype(np.int32), w["free"], w["n_free"], w["pos"].astype(np.int32)
        return w


@pytest.mark.parametrize("n_seq,page,max_pages,longest,spare,max_rows,kw", [
    (1, 32, 1, 0, 1, 1, {}), (1, 64, 40, 700, 0, 5, {}), (1, 4096, 9, 20000, 3, 9000, {}), (3, 32, 30, 400, 2, 64, {}), (5, 128, 7, 500, 3, 40, dict(base=False)),
    (48, 64, 20, 900, 12, 48, {}), (64, 32, 64, 1500, 4, 200, dict(shared=False)), (65, 256, 9, 1000, 40, 500, dict(row_seq=False)), (256, 32, 40, 600, 100, 4000, {}),
    (257, 32, 40, 600, 30, 700, {}), (900, 32, 200, 3000, 300, 12007, {}), (1024, 64, 33, 1111, 0, 5000, dict(base=False, row_seq=False)), (2047, 32, 20, 333, 900, 20000, {}),
    (2048, 32, 12, 200, 2000, 1 << 20, dict(shared=False))])
def test_plans_of_passes_in_a_row(ctx, n_seq, page, max_pages, longest, spare, max_rows, kw):
    """Passes one behind the other: growth, chunks, what is given back, ends, and sequences that do not fit their table, the pool or the pass."""
    t = Plan(n_seq + page, n_seq, page, max_pages, longest, spare, max_rows, **kw)
    t.upload(ctx)
    seen = [np.full(max_rows, -5, np.int32) for _ in range(3)]
    rng = t.rng
    for step in range(5):
        rows = rng.integers(0, 3, n_seq)
        big = rng.random(n_seq) < 0.1
        rows = np.where(big, rng.integers(0, max(2, max_rows // 3), n_seq), rows)
        rows = np.where(rng.random(n_seq) < 0.08, -1 - rng.integers(0, 9, n_seq), rows).astype(np.int32)
        if step == 3:
            rows[rng.integers(n_seq)] = 2**31 - 1
        if step == 2 and n_seq > 2:
            t.pos = np.where(rng.random(n_seq) < 0.3, t.pos // 2, t.pos).astype(np.int32)  # branches that were not kept
            t.d["pos"].write(t.pos)
        t.d["rows"].write(rows)
        ctx.enqueue(A.OP_PAGE_PLAN, t.args())
        t.check(rows, seen)


def test_pages_stay_one_sequences_each(ctx):
    """Fifty passes of a pool that runs dry and fills again: no page is ever two sequences', none is lost."""
    t = Plan(5, 40, 32, 50, 300, 30, 400, odd=False, shared=False)
    t.upload(ctx)
    seen = [np.full(400, -5, np.int32) for _ in range(3)]
    whole = sorted(t.free[:t.n_free].tolist() + [p for s in range(40) for p in t.table[s, :t.held[s]]])
    dry = 0
    for step in range(50):
        rows = t.rng.integers(0, 30, 40).astype(np.int32)
        rows[t.rng.random(40) < 0.06] = -1
        t.d["rows"].write(rows)
        ctx.enqueue(A.OP_PAGE_PLAN, t.args())
        w = t.check(rows, seen)
        dry += int(((np.diff(w["start"]) == 0) & (rows > 0)).any())
        assert sorted(t.free[:t.n_free].tolist() + [p for s in range(40) for p in t.table[s, :t.held[s]]]) == whole
    assert dry > 3


def test_a_recorded_plan_moves_on_by_itself(ctx):
    """A decode step's plan, replayed: positions move, pages are taken when a page is full, until the pool is empty."""
    t = Plan(6, 30, 32, 20, 200, 25, 30, odd=False, shared=False)
    t.upload(ctx)
    rows = np.ones(30, np.int32)
    t.d["rows"].write(rows)
    rec = ctx.prerecord([A.make_op(A.OP_PAGE_PLAN, t.args())])
    seen = [np.full(30, -5, np.int32) for _ in range(3)]
    for step in range(60):
        rec.submit()
        w = t.check(rows, seen)
    assert w["n_free"] == 0 and w["start"][-1] < 30
    rec.destroy()


# ---- attention ---------------------------------------------------------------------------------


class Paged:
    """Inputs of one call: sequences of n rows behind pos cells on shuffled pages, rows a stride apart wider than they need, and a pool that holds more pages than theirs."""

    def __init__(self, seed, layout, n, pos, page=32, spare_rows=3, extra_pages=5):
        self.rng = rng = np.random.default_rng(seed)
        self.nh, self.nkv, self.d, self.dims = LAYOUTS[layout]
        self.n, self.pos, self.page = list(n), list(pos), page
        pages = [-(-(p + k) // page) for p, k in zip(pos, n)]
        self.max_pages = max(max(pages), 1)
        self.n_pages = sum(pages) + extra_pages
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(n), self.max_pages), -1, np.int32)
        self.start = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        self.total = int(self.start[-1])
        self.max_rows = self.total + spare_rows
        self.row_pos, self.row_cell = np.full(self.max_rows, 7, np.int32), np.full(self.max_rows, 11, np.int32)
        at = 0
        for s, (p, k) in enumerate(zip(pos, n)):
            self.table[s, :pages[s]] = order[at:at + pages[s]]
            at += pages[s]
            where = np.arange(p, p + k)
            self.row_pos[self.start[s]:self.start[s + 1]] = where
            self.row_cell[self.start[s]:self.start[s + 1]] = self.table[s, where // page] * page + where % page
        self.width = 2 * self.nh * self.d + 2 * self.nkv * self.d
        self.stride = self.width + 4
        self.qkv = rng.standard_normal((self.max_rows, self.stride)).astype(np.float32)
        self.q_norm, self.k_norm = ((1 + 0.1 * rng.standard_normal(self.d)).astype(np.float32) for _ in range(2))
        self.rope = T.rope_table(self.max_pages * page, self.dims)
        shape = (self.n_pages, page, self.nkv, self.d)
        self.kp, self.vp = (rng.standard_normal(shape, dtype=np.float32).astype(np.float16) for _ in range(2))

    def cells(self, s, lo, hi):
        """Places of a sequence's cells lo .. hi - 1 in the pool, as (page, cell) indexes."""
        c = np.arange(lo, hi)
        return self.table[s, c // self.page], c % self.page

    def upload(self, c):
        up = c.upload
        self.d_in = [up(x) for x in (self.qkv, self.q_norm, self.k_norm, self.rope)]
        self.d_kp, self.d_vp = up(self.kp), up(v_dev(self.vp))
        self.d_table, self.d_start, self.d_pos, self.d_cell = up(self.table), up(self.start), up(self.row_pos), up(self.row_cell)
        self.d_out = up(np.full(self.max_rows * self.nh * self.d, 77.0, np.float32))

    def args(self, c, window=0, sinks=0, work=None):
        q, qn, kn, rope = self.d_in
        a = A.AttnPagedArgs(q.ptr, qn.ptr, kn.ptr, rope.ptr, self.d_kp.ptr, self.d_vp.ptr, self.d_table.ptr, self.d_start.ptr, self.d_pos.ptr, self.d_cell.ptr, None, self.d_out.ptr, 0,
                            len(self.n), self.max_rows, self.nh, self.nkv, self.d, self.dims, self.page, self.max_pages, self.n_pages, self.stride, window, sinks, EPS)
        a.work_bytes = c.attn_paged_work(a)
        a.work = work if work else c.upload(np.full(a.work_bytes // 4 + 1, np.nan, np.float32)).ptr
        return a

    def results(self):
        kp = self.d_kp.read(np.float16, self.kp.size).reshape(self.kp.shape)
        vt = self.d_vp.read(np.float16, self.vp.size).reshape(self.n_pages, self.page // 32, self.nkv, self.d, 32)
        return self.d_out.read(np.float32, self.max_rows * self.nh * self.d).reshape(self.max_rows, -1), kp, np.ascontiguousarray(np.moveaxis(vt, -1, 2)).reshape(self.vp.shape)

    def check(self, window=0, sinks=0):
        out, kp, vp = self.results()
        want, there, wk, wv = P.attention(self.qkv, self.q_norm, self.k_norm, self.table, self.rope, self.kp, self.vp, self.start, self.row_pos, self.row_cell, self.nh, self.nkv, self.d,
                                          self.dims, EPS, window, sinks)
        assert np.array_equal(kp, wk, equal_nan=True)
        assert np.array_equal(vp, wv, equal_nan=True)
        worst = 0.0
        fine = np.isfinite(want)
        for r in np.flatnonzero(there):
            assert np.array_equal(fine[r], np.isfinite(out[r])), r
            if (want[r] == 0).all():
                assert (out[r] == 0).all(), r
            elif fine[r].any():
                worst = max(worst, O.rel_l2(out[r][fine[r]], want[r][fine[r]]))
        print(f"paged attention of {self.n} behind {self.pos}: {worst:.2e}")
        assert worst <= ATTN_TOL
        assert (out[~there] == 77.0).all()  # rows of no sequence, and of one that is left alone
        return out


@pytest.mark.parametrize("layout,n,pos,page", [
    # single tokens: nothing behind them, tiles and pages that begin and end there, long ones
    ("16/2x256", [1], [0], 32), ("16/2x256", [1], [31], 32), ("16/2x256", [1], [32], 32), ("16/2x256", [1], [900], 32), ("16/2x256", [1], [4095], 4096), ("16/2x256", [1, 1, 1], [5, 700, 64], 64),
    ("32/8x128", [1] * 7, [0, 1, 31, 32, 33, 1000, 257], 64), ("8/8x64", [1, 1], [63, 2000], 32), ("5/1x64", [1], [3000], 128), ("64/1x64", [1, 1], [500, 3], 32), ("7/7x256", [1], [100], 32),
    # chunks
    ("16/2x256", [2], [0], 32), ("16/2x256", [16], [0], 32), ("16/2x256", [17], [15], 32), ("16/2x256", [37], [301], 32), ("16/2x256", [130], [64], 64), ("12/2x128", [100], [0], 256),
    ("12/2x128", [33], [1000], 32), ("32/8x128", [65], [129], 64), ("8/8x64", [150], [50], 32), ("8/8x64", [129], [0], 128), ("5/1x64", [77], [222], 32), ("64/1x64", [9], [33], 32), ("6/2x256", [44], [90], 32),
    ("9/3x128", [43], [1], 32), ("32/16x128", [20], [600], 64), ("7/7x256", [70], [31], 32),
    # both, and sequences without rows
    ("16/2x256", [1, 40, 0, 1, 17], [300, 0, 5, 1, 90], 32), ("32/8x128", [0, 0, 33, 1, 0], [0, 9, 700, 31, 2], 64), ("8/8x64", [3, 0, 200, 1, 1, 5], [0, 0, 10, 64, 1999, 31], 32),
    ("12/2x128", [1] * 70, list(range(70)), 32)])
def test_attention_over_pages(ctx, layout, n, pos, page):
    t = Paged(sum(n) + pos[0], layout, n, pos, page)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    t.check()


@pytest.mark.parametrize("layout,n,pos", [("16/2x256", [300], [700]), ("32/8x128", [150, 1, 1, 260], [0, 1500, 3, 100]), ("8/8x64", [700], [0]), ("64/1x64", [90], [200])])
def test_long_chunks(ctx, layout, n, pos):
    t = Paged(17, layout, n, pos, 64)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    t.check()


@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (31, 4), (32, 0), (33, 40), (100, 3), (700, 700), (2**31 - 1, 2**31 - 1)])
@pytest.mark.parametrize("layout,n,pos", [("16/2x256", [1, 9, 40], [640, 5, 31]), ("32/8x128", [1, 1, 70], [1111, 0, 200])])
def test_sliding_window_and_sinks(ctx, layout, n, pos, window, sinks):
    t = Paged(7 + window % 1000, layout, n, pos)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx, window, sinks))
    t.check(window, sinks)


@pytest.mark.parametrize("n,pos,window", [([1], [700], 0), ([40], [300], 0), ([1, 50, 1], [400, 100, 33], 90)])
def test_table_entries_that_are_no_page(ctx, n, pos, window):
    """Pages taken out of the table, in the middle, at the front and the last: their cells are not seen, and rows whose cell lies in one leave none."""
    for bad in (-1, 10**6, -2**31):
        t = Paged(31, "16/2x256", n, pos)
        for s in range(len(n)):
            last = (pos[s] + n[s] - 1) // 32
            for e in {0, last // 2, last}:
                t.table[s, e] = bad
        for s in range(len(n)):
            for r in range(t.start[s], t.start[s + 1]):
                if t.table[s, t.row_pos[r] // 32] == bad:
                    t.row_cell[r] = -1 if bad != 10**6 else 10**6 * 32
        t.upload(ctx)
        ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx, window, 2 if window else 0))
        t.check(window, 2 if window else 0)


def test_rows_that_see_nothing_are_zeros(ctx):
    t = Paged(32, "32/8x128", [1, 20, 2], [50, 40, 0])
    t.table[:] = -1
    t.row_cell[:t.total] = -1
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    assert (t.check()[:t.total] == 0).all()


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 2)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 6e4])
def test_what_a_row_does_not_see_may_hold_anything(ctx, bad, window, sinks):
    """NaN and infinities in cells behind a sequence's end, outside the window, in pages that are nobody's, and in later rows' keys and values."""
    t = Paged(33, "16/2x256", [1, 21], [103, 203])
    mine = np.zeros((t.n_pages, t.page), bool)
    for s in range(2):
        mine[t.cells(s, 0, t.pos[s])] = True
        if window:
            mine[t.cells(s, sinks, t.pos[s] - window + 1)] = False
    t.kp[~mine] = t.vp[~mine] = bad
    v0 = 2 * t.nh * t.d + t.nkv * t.d
    t.qkv[1 + 9, v0 + 3:v0 + t.nkv * t.d:5] = bad  # a row in the middle of the chunk: only it and those behind it
    if not np.isfinite(bad):
        t.qkv[1 + 15, v0 - 9] = bad
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx, window, sinks))
    out = t.check(window, sinks)
    assert np.isfinite(out[:10]).all()


def test_sequences_that_are_left_alone(ctx):
    """Positions and row numbers that cannot be: no output, whatever the others do."""
    t = Paged(34, "16/2x256", [2, 3, 1, 4], [40, 10, 70, 0], page=32)
    t.row_pos[t.start[1]:t.start[2]] = -2                              # before the sequence's start
    t.row_pos[t.start[2]] = t.max_pages * 32                           # past what a table can name
    t.row_cell[t.start[1]:t.start[3]] = -1
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    out = t.check()
    assert (out[2:6] == 77.0).all() and (out[:2] != 77.0).all()
    t = Paged(35, "16/2x256", [2, 3, 1], [40, 10, 70], spare_rows=0)
    t.start[:] = [0, 2, 9, 9]                                          # past the rows, and what is behind that
    t.row_cell[2:] = -1
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    t.check()


def test_positions_at_the_ends_of_the_table(ctx):
    """The last cells that a table can name; a chunk whose rows would go on behind them is left alone."""
    t = Paged(36, "16/2x256", [5, 6], [32 * 7 - 5, 32 * 7 - 6])
    assert t.max_pages == 7
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    t.check()
    t.row_pos[5:11] += 1
    t.row_cell[5:11] = -1
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    assert (t.check()[5:] == 77.0).all()


def test_pages_shared_by_sequences(ctx):
    """A common prefix: the same pages in several tables, read by all and written by none."""
    t = Paged(37, "32/8x128", [1, 1, 12], [100, 140, 96], page=32)
    t.table[1, :3] = t.table[2, :3] = t.table[0, :3]
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    t.check()


def test_values_are_rounded_bit_by_bit(ctx):
    t = Paged(38, "16/2x256", [1, 40], [70, 5])
    v0 = 2 * t.nh * t.d + t.nkv * t.d
    v = t.qkv[:, v0:v0 + t.nkv * t.d]
    odd = np.array([0.0, -0.0, 2.0 ** -24, -2.0 ** -25, 3 * 2.0 ** -25, -6e-8, 1 + 2.0 ** -11, -(1 + 3 * 2.0 ** -11), 65504, -65504, 65519.99, -65520, 7e4], np.float32)
    v[:, :40] = t.rng.choice(odd, v[:, :40].shape)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    with np.errstate(over="ignore"):
        want = v[:41].astype(np.float16).reshape(41, t.nkv, t.d)
    got = t.results()[2].reshape(-1, t.nkv, t.d)[t.row_cell[:41]]
    assert np.array_equal(got.view(np.uint16), want.view(np.uint16))


@pytest.mark.parametrize("n,cells,lead", [(1, 3000, 22), (3, 3000, 20), (40, 5000, 22), (1, 20000, 19)])
def test_small_weights_beside_a_first_cell_that_takes_nearly_all(ctx, n, cells, lead):
    """A first cell with 2^lead times the weight of any other and a value of nothing, as models that rest on their first token have it: the output is what the
    small weights make of their values.  A weight is rounded to the nearest 2^-35 of the largest, by at most 2^-36: of one of 2^-22 that is 2^-14, no two cells alike,
    and of a sum over thousands of them 2^-14 / sqrt(3 * 3000) = 6e-7 is left."""
    t = Paged(340 + lead, "12/2x128", [n], [cells], 64)
    u = np.sign(t.rng.standard_normal(t.d)).astype(np.float32)
    t.q_norm[:] = t.k_norm[:] = 1
    t.qkv[:, :2 * t.nh * t.d].reshape(-1, t.nh, 2, t.d)[:, :, 0] = 3 * u
    away = 1 - lead * np.log(2) / np.sqrt(t.d)
    t.kp[:] = (away * u + 0.05 * t.rng.standard_normal(t.kp.shape)).astype(np.float16)
    t.vp[:] = (1 + 0.1 * t.rng.standard_normal(t.vp.shape)).astype(np.float16)
    first = (t.table[0, 0], 0)
    t.kp[first], t.vp[first] = u, 0
    own = t.qkv[:, 2 * t.nh * t.d:]
    own[:, :t.nkv * t.d] = np.tile(-u, t.nkv)
    own[:, t.nkv * t.d:2 * t.nkv * t.d] = 1
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    t.check()


def test_pages_far_behind_32_bits(ctx):
    """Pages whose cells lie more than 2^32 bytes into the pool."""
    t = Paged(39, "16/2x256", [1, 33], [200, 90], 64)
    kvw = t.nkv * t.d
    many = (5 << 30) // (64 * kvw * 2)
    kp, vp = ctx.alloc(many * 64 * kvw * 2), ctx.alloc(many * 64 * kvw * 2)
    move = np.arange(t.n_pages) * ((many - 1) // (t.n_pages - 1))  # page i of the small pool lies here in the large one
    assert move[-1] * 64 * kvw * 2 > 1 << 32
    vd = v_dev(t.vp)
    for i, to in enumerate(move):
        kp.write(t.kp[i], int(to) * 64 * kvw * 2)
        vp.write(vd[i], int(to) * 64 * kvw * 2)
    t.upload(ctx)
    t.d_table.write(move[np.maximum(t.table, 0)].astype(np.int32))
    far = np.where(t.row_cell >= 0, move[t.row_cell // 64] * 64 + t.row_cell % 64, -1).astype(np.int32)
    t.d_cell.write(far)
    a = t.args(ctx)
    a.kpages, a.vpages, a.n_pages = kp.ptr, vp.ptr, many
    ctx.enqueue(A.OP_ATTN_PAGED, a)
    for i, to in enumerate(move):  # the pool's pages back to where the check looks for them
        t.d_kp.write(kp.read(np.uint8, 64 * kvw * 2, int(to) * 64 * kvw * 2), i * 64 * kvw * 2)
        t.d_vp.write(vp.read(np.uint8, 64 * kvw * 2, int(to) * 64 * kvw * 2), i * 64 * kvw * 2)
    t.check()
    kp.free()
    vp.free()


def test_one_long_sequence_among_many_short_ones(ctx):
    n = [1] * 40 + [3]
    pos = [int(p) for p in np.random.default_rng(1).integers(0, 90, 40)] + [6000]
    t = Paged(40, "16/2x256", n, pos, 32)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    t.check()


def test_the_most_sequences_a_call_takes(ctx):
    rng = np.random.default_rng(2)
    t = Paged(41, "5/1x64", [int(x) for x in rng.integers(0, 3, 2048)], [int(x) for x in rng.integers(0, 80, 2048)], 32)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    t.check()


def test_too_little_work_is_refused(ctx):
    t = Paged(42, "16/2x256", [1], [5])
    t.upload(ctx)
    a = t.args(ctx)
    a.work_bytes -= 1
    with pytest.raises(shv.pkg.ShvError, match="work"):
        ctx.enqueue(A.OP_ATTN_PAGED, a)


def test_a_recorded_call_and_two_contexts(ctx):
    """Replays between eager calls of other sizes on the same scratch, and the same on another context at once."""
    other = shv.pkg.Context(0)
    sets = []
    for c, seed in ((ctx, 50), (other, 51)):
        t, u = Paged(seed, "16/2x256", [1, 30, 1], [700, 20, 64]), Paged(seed + 9, "32/8x128", [1] * 5, [50 * i for i in range(5)])
        t.upload(c)
        u.upload(c)
        a, b = t.args(c), u.args(c)
        if b.work_bytes > a.work_bytes:
            a.work = b.work
        else:
            b.work = a.work
        sets.append((c, t, u, b, c.prerecord([A.make_op(A.OP_ATTN_PAGED, a)])))
    for _ in range(4):
        for c, _, _, b, rec in sets:
            rec.launch()
            c.enqueue(A.OP_ATTN_PAGED, b)
    for c, t, u, b, rec in sets:
        c.sync()
        t.check()
        u.check()
        t.d_out.write(np.full(t.max_rows * t.nh * t.d, 77.0, np.float32))
        rec.submit()
        t.check()
        rec.destroy()
    other.destroy()


def test_single_tokens_are_what_attn_decode_makes_of_them(ctx):
    """A slot of a contiguous cache is a page of the pool: the same rows by both."""
    pos = [333, 40, 700]
    t = Paged(60, "16/2x256", [1, 1, 1], pos, page=1024, extra_pages=0)
    t.upload(ctx)
    d_kc, d_vc = ctx.upload(t.kp), ctx.upload(v_dev(t.vp))
    n_splits = 16
    d_ref, d_part = ctx.alloc(3 * t.nh * t.d * 4), ctx.alloc(3 * 2 * t.nh * n_splits * (t.d + 2) * 4)
    ctx.enqueue(A.OP_ATTN_DECODE, A.AttnDecodeArgs(t.d_in[0].ptr, t.d_in[1].ptr, t.d_in[2].ptr, t.d_in[3].ptr, d_kc.ptr, d_vc.ptr, d_part.ptr, d_ref.ptr, ctx.upload(np.array(pos, np.int32)).ptr,
                                                   ctx.upload(t.table[:, 0].copy()).ptr, 3, 1, t.nh, t.nkv, t.d, t.dims, 1024, t.stride, n_splits, EPS))
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    got, ref = t.results()[0][:3], d_ref.read(np.float32, 3 * t.nh * t.d).reshape(3, -1)
    for r in range(3):
        assert O.rel_l2(got[r], ref[r]) <= 1e-4  # a key rounded to the other neighbour moves a score by 16 * 2^-12 / 16


@pytest.mark.parametrize("d,dims", [(256, 8), (256, 16), (256, 32), (256, 128), (256, 192), (256, 200), (128, 0), (128, 4), (128, 32), (128, 96), (128, 124), (64, 0), (64, 2), (64, 48), (64, 64)])
def test_rotations(ctx, monkeypatch, d, dims):
    """Pairs of dims in one lane, in two lanes of a wave, and none, in chunks and single tokens."""
    monkeypatch.setitem(LAYOUTS, "own", (6, 2, d, dims))
    t = Paged(80 + dims, "own", [1, 23, 90], [77, 64, 3])
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    t.check()


@pytest.mark.parametrize("d,rep", [(256, 1), (256, 8), (128, 1), (128, 4), (64, 1), (64, 16)])
def test_query_rows_about_the_blocks_sizes(ctx, monkeypatch, d, rep):
    """Numbers of query rows that fill a wave's groups, the waves that share them and a block, one fewer and one more."""
    monkeypatch.setitem(LAYOUTS, "own", (2 * rep, 2, d, 0))
    lines = [max(1, x // rep + e) for x in (16, 32, 48, 64, 80, 128, 192) for e in (-1, 0, 1)]
    t = Paged(90 + rep, "own", lines, [int(x) for x in np.random.default_rng(3).integers(0, 200, len(lines))], 64)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    t.check()


@pytest.mark.parametrize("n,pos,window", [([255], [40], 0), ([256], [40], 0), ([257], [1000], 0), ([300, 1], [50, 900], 0), ([600, 1, 2], [0, 3000, 31], 0), ([600, 1, 40], [500, 700, 64], 300)])
def test_rows_a_sequence_about_those_of_the_larger_blocks(ctx, n, pos, window):
    t = Paged(100 + n[0], "16/2x256", n, pos, 64, spare_rows=0)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx, window, 3 if window else 0))
    t.check(window, 3 if window else 0)


@pytest.mark.parametrize("layout,n,pos", [("5/1x64", [1], [40000]), ("5/1x64", [1, 30, 1], [20000, 9000, 70]), ("16/2x256", [1, 1], [17000, 3]), ("12/2x128", [2, 1], [30000, 4000])])
def test_few_rows_behind_much(ctx, layout, n, pos):
    """A query row's tiles shared by as many blocks as there are, and by a few."""
    t = Paged(110 + n[0], layout, n, pos, 128)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    t.check()


@pytest.mark.parametrize("layout", ["32/8x128", "5/1x64", "12/2x128", "7/7x256"])
@pytest.mark.parametrize("first", [0, 1, 2, 4, 33])
def test_many_rows_cells(ctx, layout, first):
    """Values of rows whose cells begin anywhere in a tile, end with a page, skip a page that is none, and belong to nobody, where rows are many."""
    n, pos = [203, 1, 0, 180, 77, 1, 64], [first, 5, 0, 62 + first, 501, 31, 64]
    t = Paged(170 + first, layout, n, pos, 32, spare_rows=40)
    t.table[3, 4] = -1
    lost = t.row_pos[t.start[3]:t.start[4]] // 32 == 4
    t.row_cell[t.start[3]:t.start[4]][lost] = -1
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    t.check()


@pytest.mark.parametrize("layout", [(1024, 1024, 64, 64), (257, 257, 64, 2), (1024, 16, 256, 64), (48, 24, 128, 32), (39, 13, 128, 128), (640, 10, 64, 0)])
def test_numbers_of_heads(ctx, monkeypatch, layout):
    """More KV heads than units, odd numbers of them, which do not divide the dies, and the most query heads there may be."""
    monkeypatch.setitem(LAYOUTS, "own", layout)
    t = Paged(150 + layout[1], "own", [1, 5, 1], [40, 0, 131])
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    t.check()


def test_positions_near_the_largest(ctx, monkeypatch):
    """A window at the last positions that 32 bits name, without rotation, gives what it gives at the first."""
    monkeypatch.setitem(LAYOUTS, "own", (8, 2, 128, 0))
    window, n, pos, page = 700, [1, 40], [1500, 900], 4096
    t = Paged(140, "own", n, pos, page)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx, window))
    near = t.check(window)
    last = (1 << 31) // page - 1  # pages of the largest table, all but the last one taken out
    table = np.full((2, last), -1, np.int32)
    table[:, -1] = t.table[:, 0]
    by = (last - 1) * page
    t.upload(ctx)
    a = t.args(ctx, window)
    d_table, d_pos = ctx.upload(table), ctx.upload((t.row_pos.astype(np.int64) + by).clip(max=2**31 - 1).astype(np.int32))
    a.table, a.row_pos, a.max_pages, a.rope = d_table.ptr, d_pos.ptr, last, None
    a.work_bytes = ctx.attn_paged_work(a)
    work = ctx.alloc(a.work_bytes)
    a.work = work.ptr
    ctx.enqueue(A.OP_ATTN_PAGED, a)
    far = t.results()[0]
    assert np.array_equal(far[:41], near[:41])


def test_recorded_calls_that_share_scratch(ctx):
    """Two recordings and an eager call, of sizes that lay the same scratch out differently, replayed in turn."""
    sets = [Paged(120, "16/2x256", [1, 1, 1], [900, 5, 300]), Paged(121, "32/8x128", [70, 1, 3], [40, 800, 31], 64), Paged(122, "8/8x64", [1] * 9, [99 * i for i in range(9)])]
    for t in sets:
        t.upload(ctx)
    args = [t.args(ctx) for t in sets]
    work = max(args, key=lambda a: a.work_bytes)
    for a in args:
        a.work, a.work_bytes = work.work, work.work_bytes
    recs = [ctx.prerecord([A.make_op(A.OP_ATTN_PAGED, a)]) for a in args[:2]]
    for _ in range(3):
        for t in sets:
            t.d_out.write(np.full(t.max_rows * t.nh * t.d, 77.0, np.float32))
        recs[0].launch()
        ctx.enqueue(A.OP_ATTN_PAGED, args[2])
        recs[1].launch()
        recs[0].launch()
        ctx.sync()
        for t in sets:
            t.check()
    for rec in recs:
        rec.destroy()


def test_the_same_call_gives_the_same_bits(ctx):
    """Which block takes what is planned, and records are joined in order: no result hangs on who comes first."""
    for layout, n, pos in (("32/8x128", [150, 1, 1, 60], [300, 1500, 3, 100]), ("16/2x256", [1] * 20, [37 * i for i in range(20)]), ("8/8x64", [40, 1], [3000, 900])):
        t = Paged(130, layout, n, pos, 64)
        t.upload(ctx)
        a = t.args(ctx)
        seen = []
        for _ in range(4):
            ctx.enqueue(A.OP_ATTN_PAGED, a)
            seen.append(t.results()[0].tobytes())
        assert len(set(seen)) == 1


# ---- log probabilities ---------------------------------------------------------------------------


def _logprobs(c, logits, ids, top, stride=None, offset=0, entropy=True):
    rows, n = logits.shape
    stride = stride or n
    host = np.full(rows * stride + offset, np.nan, np.float32)
    for r in range(rows):
        host[offset + r * stride:offset + r * stride + n] = logits[r]
    d = c.upload(host)
    out = [c.upload(np.full(max(1, x), 99.0, np.float32)) for x in (rows, rows)]
    d_top = [c.upload(np.full(max(1, rows * top), 99, np.int32)), c.upload(np.full(max(1, rows * top), 99.0, np.float32))]
    a = A.LogprobsArgs(d.at(4 * offset), c.upload(np.array(ids, np.int32)).ptr if ids is not None else None, out[0].ptr if ids is not None else None, out[1].ptr if entropy else None,
                       d_top[0].ptr if top else None, d_top[1].ptr if top else None, rows, n, stride, top)
    return a, lambda: (out[0].read(np.float32, rows), out[1].read(np.float32, rows), d_top[0].read(np.int32, rows * top).reshape(rows, top), d_top[1].read(np.float32, rows * top).reshape(rows, top))


def _check_logprobs(logits, ids, top, got):
    """Z is a sum of n positive terms.  A term e^(x - m) is off by the rounding of its exponent, |x - m| log2(e) 2^-24 of ln 2 each, and two last places of the exponential: within
    4e-6 of itself up to 30 below the maximum, where what matters of Z ends; sums of n / 256 terms by one thread and of 256 threads' by (n / 256 + 256) 2^-24.  log Z is off by
    as much absolutely, a log probability by a rounding of itself more; the entropy's other part, a mean of x - m, is off by as much relative to a mean of |x - m|, which is at
    most log Z + H, both within log n.  What is wanted is float32: a log probability of -6e38, beyond it, is -infinity."""
    n = logits.shape[1]
    z_tol = 4e-6 + (n / 256 + 256) * 2.0 ** -24
    want = list(P.logprobs(logits, ids if ids is not None else [0] * len(logits), top))
    with np.errstate(over="ignore"):
        want[0], want[3] = want[0].astype(np.float32), want[3].astype(np.float32)
    lp, h, ti, tl = got
    if ids is not None:
        assert np.allclose(lp, want[0], rtol=2.0 ** -22, atol=z_tol, equal_nan=True), np.nanmax(np.abs(lp - want[0]))
    assert np.allclose(h, want[1], rtol=2.0 ** -22, atol=z_tol * (2 + 2 * np.log(n)), equal_nan=True), np.nanmax(np.abs(h - want[1]))
    assert np.array_equal(ti, want[2])
    assert np.allclose(tl, want[3], rtol=2.0 ** -22, atol=z_tol, equal_nan=True)


@pytest.mark.parametrize("rows,n,top", [
    (1, 1, 1), (1, 2, 2), (1, 3, 0), (2, 5, 5), (1, 63, 20), (3, 64, 64), (1, 65, 64), (2, 255, 1), (1, 257, 64), (5, 1000, 10), (1, 1023, 3), (1, 4095, 20), (1, 4097, 64), (2, 8191, 5),
    (1, 151936, 0), (1, 151936, 5), (1, 151936, 64), (3, 151937, 20), (24, 151936, 20), (7, 32003, 64), (40, 12345, 33), (1000, 515, 7), (1025, 2049, 20), (1400, 31, 31), (2100, 700, 0)])
def test_log_probabilities(ctx, rows, n, top):
    rng = np.random.default_rng(rows + n + top)
    logits = (3 * rng.standard_normal((rows, n))).astype(np.float32)
    logits[np.arange(rows), rng.integers(0, n, rows)] += rng.choice([0, 9, 25], rows).astype(np.float32)
    ids = rng.integers(0, n, rows)
    a, got = _logprobs(ctx, logits, ids, top)
    ctx.enqueue(A.OP_LOGPROBS, a)
    _check_logprobs(logits, ids, top, got())


@pytest.mark.parametrize("stride,offset", [(5003, 0), (5004, 1), (5001, 2), (5000, 3), (6000, 0)])
def test_rows_that_begin_anywhere(ctx, stride, offset):
    rng = np.random.default_rng(stride + offset)
    logits = rng.standard_normal((6, 5000)).astype(np.float32)
    ids = [0, 4999, 1, 2500, 4998, 3]
    logits[np.arange(6), ids] = 12
    a, got = _logprobs(ctx, logits, ids, 9, stride, offset)
    ctx.enqueue(A.OP_LOGPROBS, a)
    _check_logprobs(logits, ids, 9, got())


@pytest.mark.parametrize("n", [40, 3000, 70001])
@pytest.mark.parametrize("order", ["rising", "falling", "equal", "few values"])
def test_orders_and_ties(ctx, n, order):
    """Rows that put every token in its place anew, and rows in which many are equal: the lower place first."""
    rng = np.random.default_rng(n)
    row = {"rising": np.arange(n) * 1e-3, "falling": -np.arange(n) * 1e-3, "equal": np.zeros(n), "few values": rng.integers(0, 4, n)}[order]
    logits = np.stack([row, np.roll(row, n // 3), row * 0.5]).astype(np.float32)
    for top in (1, 20, 40):
        a, got = _logprobs(ctx, logits, [0, n - 1, n // 2], top)
        ctx.enqueue(A.OP_LOGPROBS, a)
        _check_logprobs(logits, [0, n - 1, n // 2], top, got())


@pytest.mark.parametrize("n,top", [(50, 20), (6000, 20), (151936, 64)])
def test_tokens_that_cannot_come_and_what_is_no_number(ctx, n, top):
    rng = np.random.default_rng(n)
    logits = rng.standard_normal((9, n)).astype(np.float32)
    logits[0, 1:] = -np.inf                     # one token left
    logits[1, rng.random(n) < 0.9] = -np.inf
    logits[2] = -np.inf                         # none
    logits[3, n // 2] = np.nan
    logits[4] = np.nan
    logits[5, 7] = np.inf
    logits[6, rng.random(n) < 0.95] = np.nan    # fewer than asked for, perhaps
    logits[7] = 3e38 * np.sign(logits[7])       # the ends of float32
    logits[8] = -3e38
    ids = [0, 3, 1, 4, 5, 7, 8, 9, -1]
    a, got = _logprobs(ctx, logits, ids, top)
    ctx.enqueue(A.OP_LOGPROBS, a)
    _check_logprobs(logits, ids, top, got())


def test_what_is_not_asked_for(ctx):
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((3, 9000)).astype(np.float32)
    full, got_full = _logprobs(ctx, logits, [1, 2, 9000], 6)
    ctx.enqueue(A.OP_LOGPROBS, full)
    lp, h, ti, tl = got_full()
    assert np.isnan(lp[2])
    a, got = _logprobs(ctx, logits, None, 6, entropy=False)
    ctx.enqueue(A.OP_LOGPROBS, a)
    g = got()
    assert (g[0] == 99).all() and (g[1] == 99).all() and np.array_equal(g[2], ti) and np.array_equal(g[3], tl)
    a, got = _logprobs(ctx, logits, [1, 2, 9000], 0)
    ctx.enqueue(A.OP_LOGPROBS, a)
    assert np.array_equal(got()[0], lp, equal_nan=True) and np.array_equal(got()[1], h)


def test_recorded_log_probabilities(ctx):
    """Replays between eager calls of other shapes: the counters and pieces of one call are not the next one's."""
    rng = np.random.default_rng(4)
    logits, small = rng.standard_normal((3, 151936)).astype(np.float32), rng.standard_normal((40, 5000)).astype(np.float32)
    ids, sids = [5, 100, 151935], rng.integers(0, 5000, 40)
    a, got = _logprobs(ctx, logits, ids, 20)
    b, got_small = _logprobs(ctx, small, sids, 64)
    rec = ctx.prerecord([A.make_op(A.OP_LOGPROBS, a)])
    for _ in range(4):
        rec.launch()
        ctx.enqueue(A.OP_LOGPROBS, b)
        ctx.sync()
        _check_logprobs(logits, ids, 20, got())
        _check_logprobs(small, sids, 64, got_small())
    rec.destroy()


# ---- together --------------------------------------------------------------------------------------


def test_a_servers_passes(ctx):
    """Plan, attention and log probabilities recorded as one pass and replayed: prompts in chunks, then single tokens, one request that ends and another that takes
    its pages.  Every replay against the plain forms, from the state that the one before left."""
    nh, nkv, d, dims = LAYOUTS["32/8x128"]
    n_seq, page, max_pages, n_pages, max_rows, vocab, top = 5, 32, 8, 9, 60, 3001, 4
    rng = np.random.default_rng(70)
    width = 2 * nh * d + 2 * nkv * d
    qn, kn = np.ones(d, np.float32), np.ones(d, np.float32)
    rope = T.rope_table(max_pages * page, dims)
    pos, held, n_free = np.zeros(n_seq, np.int32), np.zeros(n_seq, np.int32), n_pages
    table, free = np.full((n_seq, max_pages), -1, np.int32), rng.permutation(n_pages).astype(np.int32)
    kp, vp = (rng.standard_normal((n_pages, page, nkv, d), dtype=np.float32).astype(np.float16) for _ in range(2))
    up = ctx.upload
    dv = dict(rows=ctx.alloc(n_seq * 4), pos=up(pos), table=up(table), held=up(held), free=up(free), n_free=up(np.array([n_free], np.int32)), start=up(np.zeros(n_seq + 1, np.int32)),
              row_pos=up(np.zeros(max_rows, np.int32)), row_cell=up(np.full(max_rows, -1, np.int32)), base=up(pos), qkv=ctx.alloc(max_rows * width * 4), qn=up(qn), kn=up(kn), rope=up(rope),
              kp=up(kp), vp=up(v_dev(vp)), out=up(np.zeros(max_rows * nh * d, np.float32)), logits=ctx.alloc(max_rows * vocab * 4), ids=ctx.alloc(max_rows * 4),
              lp=up(np.zeros(max_rows, np.float32)), h=up(np.zeros(max_rows, np.float32)), ti=up(np.zeros(max_rows * top, np.int32)), tl=up(np.zeros(max_rows * top, np.float32)))
    plan = A.PagePlanArgs(*(dv[k].ptr for k in ("rows", "pos", "table", "held", "free", "n_free")), None, dv["start"].ptr, None, dv["row_pos"].ptr, dv["row_cell"].ptr, dv["base"].ptr, n_seq,
                          page, max_pages, n_pages, max_rows)
    attn = A.AttnPagedArgs(*(dv[k].ptr for k in ("qkv", "qn", "kn", "rope", "kp", "vp", "table", "start", "row_pos", "row_cell")), None, dv["out"].ptr, 0, n_seq, max_rows, nh, nkv, d, dims,
                           page, max_pages, n_pages, width, 0, 0, EPS)
    attn.work_bytes = ctx.attn_paged_work(attn)
    attn.work = ctx.alloc(attn.work_bytes).ptr
    logp = A.LogprobsArgs(*(dv[k].ptr for k in ("logits", "ids", "lp", "h", "ti", "tl")), max_rows, vocab, vocab, top)
    rec = ctx.prerecord([A.make_op(A.OP_PAGE_PLAN, plan), A.make_op(A.OP_ATTN_PAGED, attn), A.make_op(A.OP_LOGPROBS, logp)])
    out_before = np.zeros((max_rows, nh * d))
    waited = 0
    for step, rows in enumerate([[20, 0, 33, 0, 0], [20, 7, 1, 0, 0], [1, 1, 1, 40, 0], [1, 1, 1, 1, 50], [1, -1, 1, 1, 1], [1, 45, 1, 1, 1], [0, 1, 50, -1, 1], [1, 1, 1, 30, 1], [1, 1, 1, 1, 1]]):
        rows = np.array(rows, np.int32)
        qkv, logits = rng.standard_normal((max_rows, width)).astype(np.float32), rng.standard_normal((max_rows, vocab)).astype(np.float32)
        ids = rng.integers(0, vocab, max_rows).astype(np.int32)
        for k, x in (("rows", rows), ("qkv", qkv), ("logits", logits), ("ids", ids)):
            dv[k].write(x)
        rec.submit()
        w = P.plan(rows, pos, table, held, free, n_free, None, page, max_pages, max_rows, True)
        pos, table, held, free, n_free = w["pos"], w["table"], w["held"], w["free"], w["n_free"]
        total = int(w["start"][-1])
        waited += int((np.diff(w["start"]) < rows).any())
        assert np.array_equal(dv["start"].read(np.int32, n_seq + 1), w["start"]) and np.array_equal(dv["pos"].read(np.int32, n_seq), pos)
        want, there, kp, vp = P.attention(qkv, qn, kn, table, rope, kp, vp, w["start"], w["maps"][:, 1], w["maps"][:, 2], nh, nkv, d, dims, EPS)
        got = dv["out"].read(np.float32, max_rows * nh * d).reshape(max_rows, -1)
        assert there.all() and np.array_equal(got[total:], out_before[total:])
        for r in range(total):
            assert O.rel_l2(got[r], want[r]) <= ATTN_TOL, (step, r)
        out_before = got
        assert np.array_equal(dv["kp"].read(np.float16, kp.size).reshape(kp.shape), kp)
        _check_logprobs(logits, ids, top, (dv["lp"].read(np.float32, max_rows), dv["h"].read(np.float32, max_rows), dv["ti"].read(np.int32, max_rows * top).reshape(max_rows, top),
                                           dv["tl"].read(np.float32, max_rows * top).reshape(max_rows, top)))
    assert waited > 0
    rec.destroy()


def test_each_ops_time_is_told(ctx):
    t, plan = Paged(160, "32/8x128", [1, 40], [300, 20]), Plan(161, 40, 32, 20, 300, 30, 400)
    t.upload(ctx)
    plan.upload(ctx)
    plan.d["rows"].write(np.ones(40, np.int32))
    logits = t.rng.standard_normal((5, 9001)).astype(np.float32)
    a, got = _logprobs(ctx, logits, [1, 2, 3, 4, 5], 7)
    total, each = ctx.dispatch_multi([A.make_op(A.OP_PAGE_PLAN, plan.args()), A.make_op(A.OP_ATTN_PAGED, t.args(ctx)), A.make_op(A.OP_LOGPROBS, a)], per_op=True)
    assert len(each) == 3 and all(x > 0 for x in each) and total > 0
    plan.check(np.ones(40, np.int32), [np.full(400, -5, np.int32) for _ in range(3)])
    t.check()
    _check_logprobs(logits, [1, 2, 3, 4, 5], 7, got())
