"""A serving batch over a paged cache at the ends of what its operators accept: the most query rows, pages that the host has taken out, lists that are nearly full, scores of any
size, against plain forms of the definitions."""
import numpy as np
import pytest

import oracle_lib as O
import paged_oracle as P
import shv
import test_paged_gpu as G
import tree_oracle as T

pytestmark = pytest.mark.gpu
A = shv.api


@pytest.mark.parametrize("rep,n_seq,n", [(64, 2048, 6), (64, 400, 31), (8, 2048, 41)])
def test_more_query_rows_of_256_dims_than_small_blocks_hold(ctx, rep, n_seq, n):
    """Calls whose query rows are close to the most there may be, over many sequences: every row has its output, those of the last sequences too."""
    d, page, dims, pool = 256, 64, 64, 251
    rng = np.random.default_rng(rep + n)
    total, width = n_seq * n, 2 * rep * d + 2 * d
    # rows of a pool, so that the inputs are made quickly; neighbours differ
    few = rng.standard_normal((pool, width)).astype(np.float32)
    which = (np.arange(total) * 97 + rng.integers(pool)) % pool
    pos = rng.integers(0, page - n + 1, n_seq).astype(np.int32)
    table = rng.permutation(n_seq).astype(np.int32)[:, None]
    row_pos = (np.repeat(pos, n) + np.tile(np.arange(n), n_seq)).astype(np.int32)
    row_cell = (np.repeat(table[:, 0], n) * page + row_pos).astype(np.int32)
    start = (np.arange(n_seq + 1) * n).astype(np.int32)
    qn, kn = ((1 + 0.1 * rng.standard_normal(d)).astype(np.float32) for _ in range(2))
    rope = T.rope_table(page, dims)
    kp, vp = (rng.standard_normal((n_seq, page, 1, d), dtype=np.float32).astype(np.float16) for _ in range(2))
    up = ctx.upload
    qkv = ctx.alloc(total * width * 4)
    for r in range(0, total, 4096):
        qkv.write(few[which[r:r + 4096]], r * width * 4)
    out = ctx.alloc(total * rep * d * 4)
    blank = np.full((4096, rep * d), 77.0, np.float32)
    for r in range(0, total, 4096):
        out.write(blank[:total - r], r * rep * d * 4)
    held = [up(x) for x in (qn, kn, rope, kp, G.v_dev(vp), table, start, row_pos, row_cell)]
    a = A.AttnPagedArgs(qkv.ptr, *(b.ptr for b in held), None, out.ptr, 0, n_seq, total, rep, 1, d, dims, page, 1, n_seq, width, 0, 0, G.EPS)
    a.work_bytes = ctx.attn_paged_work(a)
    work = ctx.alloc(a.work_bytes)
    a.work = work.ptr
    ctx.enqueue(A.OP_ATTN_PAGED, a)
    for r in range(0, total, 4096):
        rows = min(4096, total - r)
        got = out.read(np.float32, rows * rep * d, r * rep * d * 4)
        assert not (got == 77.0).any(), (r, np.flatnonzero((got.reshape(rows, -1) == 77.0).any(1))[:4] + r)
    for s in (0, 1, n_seq // 3, n_seq // 2, n_seq - 2, n_seq - 1):
        rows = slice(s * n, s * n + n)
        want, there, _, _ = P.attention(few[which[rows]], qn, kn, np.zeros((1, 1), np.int32), rope, kp[table[s]], vp[table[s]], np.array([0, n]), row_pos[rows], row_pos[rows], rep, 1, d, dims, G.EPS)
        assert there.all()
        got = out.read(np.float32, n * rep * d, s * n * rep * d * 4).reshape(n, -1)
        for r in range(n):
            assert O.rel_l2(got[r], want[r]) <= G.ATTN_TOL, (s, r)
    for b in (qkv, out, work, *held):
        b.free()


@pytest.mark.parametrize("top", [58, 59, 61, 64])
@pytest.mark.parametrize("rows,n,offset", [(1, 65, 0), (40, 66, 3), (3, 67, 1), (200, 71, 2), (9, 8195, 0), (40, 8200, 1), (2, 16390, 3), (3, 151937, 2)])
def test_lists_that_are_nearly_full_and_rows_that_begin_and_end_anywhere(ctx, rows, n, offset, top):
    """The best of a row's body nearly fill the list before what stands before and behind it is added: the largest of them there, and the smallest."""
    rng = np.random.default_rng(n + top)
    logits = rng.standard_normal((rows, n)).astype(np.float32)
    logits[::2, :4], logits[::2, -4:] = 9, 8
    logits[1::2, :4] = logits[1::2, -4:] = -9
    ids = rng.integers(0, n, rows)
    a, got = G._logprobs(ctx, logits, ids, top, n + rows % 4, offset)
    ctx.enqueue(A.OP_LOGPROBS, a)
    G._check_logprobs(logits, ids, top, got())


# ---- pages that the host has taken out of a table ---------------------------------------------


def plan_of_pages(rows, pos, table, held, free, n_free, shared, page, max_pages, max_rows, with_base):
    """The plan, request by request, where entries that are no page are passed over as they are given back."""
    n_pages, n = len(free), len(rows)
    stack, table, held, pos = [int(x) for x in free[:n_free]], table.copy(), list(map(int, held)), list(map(int, pos))
    base, want = list(pos), [0 if r < 0 else -(-(p + int(r)) // page) for r, p in zip(rows, pos)]
    ok = [rows[s] < 0 or (pos[s] >= 0 and want[s] <= max_pages) for s in range(n)]
    for s in range(n):
        if ok[s]:
            keep = min(held[s], max(want[s], min(int(shared[s]), held[s]) if shared is not None else 0))
            stack += [int(e) for e in table[s, keep:held[s]] if 0 <= e < n_pages]
            held[s] = 0 if rows[s] < 0 else keep
    avail, wished, asked, start, maps = len(stack), 0, 0, [0], []
    for s in range(n):
        lot = max(0, int(rows[s])) if ok[s] else 0
        if ok[s] and rows[s] >= 0:
            need = max(0, want[s] - held[s])
            wished, asked = wished + need, asked + lot
            if (need and wished > avail) or asked > max_rows:
                lot = 0
            else:
                for _ in range(need):
                    table[s, held[s]] = stack.pop()
                    held[s] += 1
                for p in range(pos[s], pos[s] + lot):
                    e = int(table[s, p // page])
                    maps.append((s, p, e * page + p % page if 0 <= e < n_pages else -1))
                if with_base:
                    pos[s] += lot
        else:
            lot = 0
            if ok[s] and with_base:
                pos[s] = 0
        start.append(start[-1] + lot)
    after = free.copy()
    after[:len(stack)] = stack
    return dict(table=table, held=np.array(held), free=after, n_free=len(stack), pos=np.array(pos), start=np.array(start), maps=np.array(maps, np.int64).reshape(-1, 3), base=np.array(base))


def take_out(t, chance):
    """Entries of the host's tables that become no page, each at such a chance; what they named is lost, as to another pool."""
    for s in range(t.n_seq):
        out = t.rng.random(t.held[s]) < chance
        t.table[s, :t.held[s]][out] = t.rng.choice([-1, -99, -2**31, t.n_pages, 2**31 - 1], int(out.sum()))


@pytest.mark.parametrize("n_seq,page,max_pages,longest,spare,max_rows,kw", [
    (1, 32, 4, 100, 0, 5, {}), (2, 32, 40, 1200, 1, 100, dict(shared=False)), (48, 64, 20, 900, 0, 48, {}), (64, 32, 190, 6000, 0, 200, dict(shared=False)), (65, 256, 9, 1000, 4, 500, {}),
    (256, 32, 200, 6000, 10, 4000, dict(shared=False)), (900, 32, 200, 3000, 30, 12007, {}), (2048, 32, 12, 200, 100, 20000, dict(shared=False))])
@pytest.mark.parametrize("chance", [0.05, 0.5, 1.0])
def test_pages_that_were_taken_out_are_not_given_back(ctx, monkeypatch, n_seq, page, max_pages, longest, spare, max_rows, kw, chance):
    """Sequences some of whose pages are out of their tables end, go back and grow, in one pass with others that take what came back."""
    monkeypatch.setattr(P, "plan", plan_of_pages)
    t = G.Plan(n_seq + page + 1, n_seq, page, max_pages, longest, spare, max_rows, **kw)
    t.upload(ctx)
    seen = [np.full(max_rows, -5, np.int32) for _ in range(3)]
    for step in range(5):
        take_out(t, chance)
        t.d["table"].write(t.table)
        rows = np.where(t.rng.random(n_seq) < 0.2, t.rng.integers(0, max(2, max_rows // 3), n_seq), t.rng.integers(0, 3, n_seq))
        rows = np.where(t.rng.random(n_seq) < 0.3, -1, rows).astype(np.int32)
        if step == 2:
            t.pos = np.where(t.rng.random(n_seq) < 0.5, t.pos // 2, t.pos).astype(np.int32)
            t.d["pos"].write(t.pos)
        t.d["rows"].write(rows)
        ctx.enqueue(A.OP_PAGE_PLAN, t.args())
        w = t.check(rows, seen)
        stack = w["free"][:w["n_free"]]
        assert ((stack >= 0) & (stack < t.n_pages)).all() and len(set(stack.tolist())) == len(stack)


def test_a_windows_pages_come_back_once(ctx, monkeypatch):
    """A window's pages go from a table to the stack by the host's hand, the sequence ends, another takes all there is: every page is handed out once and no entry that is none."""
    monkeypatch.setattr(P, "plan", plan_of_pages)
    t = G.Plan(9, 2, 32, 20, 0, 0, 700, odd=False, shared=False)
    t.pos[:] = [32 * 9 + 5, 0]
    t.n_pages = 10
    t.table[0, :10] = t.rng.permutation(10)
    t.held[:] = [10, 0]
    t.free = np.full(10, -77, np.int32)
    out = t.table[0, 1:7].copy()
    t.table[0, 1:7] = -1
    t.free[:6], t.n_free = out, 6
    t.upload(ctx)
    rows = np.array([-1, 320], np.int32)
    t.d["rows"].write(rows)
    ctx.enqueue(A.OP_PAGE_PLAN, t.args())
    w = t.check(rows, [np.full(700, -5, np.int32) for _ in range(3)])
    assert list(w["start"]) == [0, 0, 320] and w["n_free"] == 0
    assert sorted(t.table[1, :10].tolist()) == list(range(10)) and (w["maps"][:, 2] >= 0).all()


@pytest.mark.parametrize("n_seq", [4, 70, 300])
@pytest.mark.parametrize("base", [True, False])
def test_a_sequence_without_a_position_ends_and_is_otherwise_left_alone(ctx, n_seq, base):
    """pos below 0: with rows below 0 all its pages come back, with any other rows it keeps them and has no row."""
    t = G.Plan(n_seq, n_seq, 32, 20, 500, 4, 900, odd=False, shared=False, base=base)
    t.pos[::2] = -1 - np.arange(len(t.pos[::2]))
    t.upload(ctx)
    rows = np.ones(n_seq, np.int32)
    rows[::4], rows[2::8] = -3, 0
    t.d["rows"].write(rows)
    held, free, pos = t.held.copy(), t.n_free, t.pos.copy()
    ctx.enqueue(A.OP_PAGE_PLAN, t.args())
    w = t.check(rows, [np.full(900, -5, np.int32) for _ in range(3)])
    assert (w["held"][::4] == 0).all() and np.array_equal(w["held"][2::4], held[2::4]) and (np.diff(w["start"])[::2] == 0).all()
    assert np.array_equal(w["pos"][2::4], pos[2::4])
    assert w["n_free"] == free + held[::4].sum() - (w["held"][1::2] - held[1::2]).sum()


# ---- scores of any size --------------------------------------------------------------------------


@pytest.mark.parametrize("leads", [False, True])
@pytest.mark.parametrize("layout,norm,n,pos", [
    ((16, 2, 256, 0), 1500, [1, 1, 1], [3000, 700, 40]), ((16, 2, 256, 0), 2000, [40, 1], [500, 2000]), ((16, 2, 256, 0), 2000, [300], [100]), ((12, 2, 128, 0), 2000, [1, 90], [2500, 300]),
    ((8, 8, 64, 0), 2000, [1, 200], [2500, 30]), ((16, 2, 256, 0), 4000, [3, 50], [900, 77])])
def test_scores_of_the_largest_norm_weights(ctx, monkeypatch, layout, norm, n, pos, leads):
    """Queries and keys that point one way under large norm weights, scores past 2^24 powers of two, whose last places are several powers of two each: a row's output is a mean of the
    values it sees whatever its weights are, so between their smallest and their largest; where one cell leads by more than all roundings it is that cell's value.  Weights enter to 22
    bits and sums of at most a hundred tiles are float32: 2^-21 + 100 2^-24 < 1e-5 of the largest value."""
    monkeypatch.setitem(G.LAYOUTS, "own", layout)
    t = G.Paged(norm + n[0] + pos[0], "own", n, pos, 64)
    u = np.sign(t.rng.standard_normal(t.d)).astype(np.float32)
    t.q_norm[:] = t.k_norm[:] = norm
    t.qkv[:, :2 * t.nh * t.d].reshape(-1, t.nh, 2, t.d)[:, :, 0] = u
    t.qkv[:, 2 * t.nh * t.d:2 * t.nh * t.d + t.nkv * t.d] = np.tile(np.where(np.arange(t.d) < 8, 1e-3, 1) * u, t.nkv)
    few = (0.03 * t.rng.standard_normal(t.kp.shape)).astype(np.float16)  # a few powers of two by the first dims
    t.kp[:] = np.where(np.arange(t.d) < 8, few, (norm * u).astype(np.float16))
    lead = [int(t.rng.integers(0, p)) for p in pos]
    if leads:
        for s, c in enumerate(lead):
            where = tuple(int(x[0]) for x in t.cells(s, c, c + 1))
            t.kp[where] = (norm * u).astype(np.float16)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    out, _, vp = t.results()
    for s in range(len(n)):
        seen = vp[t.cells(s, 0, pos[s] + n[s])].astype(np.float64)
        for i in range(n[s]):
            got = out[t.start[s] + i].reshape(t.nkv, -1, t.d)
            v = seen[:pos[s] + i + 1]
            tol = 1e-5 * np.abs(v).max()
            low, high = (v[lead[s]], v[lead[s]]) if leads else (v.min(0), v.max(0))
            assert np.isfinite(got).all(), (s, i)
            assert (got >= low[:, None] - tol).all() and (got <= high[:, None] + tol).all(), (s, i)


@pytest.mark.parametrize("n_seq", [1, 3, 70])
def test_long_sequences_of_a_window_end(ctx, monkeypatch, n_seq):
    """Sequences of thirty thousand pages of which a window has left a few: as they end those come back, and others take them."""
    monkeypatch.setattr(P, "plan", plan_of_pages)
    t = G.Plan(n_seq + 3, n_seq, 32, 31000, 0, 3, 5000, odd=False, shared=False)
    long = np.arange(n_seq) % 3 == 0
    t.pos[long], t.held[long] = 32 * 30000 - 7, 30000
    t.n_pages = 66 * n_seq + 20
    order = t.rng.permutation(t.n_pages).astype(np.int32)
    t.table[long] = -1
    for k, s in enumerate(np.flatnonzero(long)):
        t.table[s, [0, *range(30000 - 64, 30000)]] = order[65 * k:65 * k + 65]
    t.free = np.concatenate([order[-3:], np.full(t.n_pages - 3, -77, np.int32)])
    t.upload(ctx)
    rows = np.where(long, -1, 5000 // max(1, int((~long).sum()))).astype(np.int32)
    for step in range(2):
        t.d["rows"].write(rows)
        ctx.enqueue(A.OP_PAGE_PLAN, t.args())
        w = t.check(rows, [np.full(5000, -5, np.int32) if step == 0 else t.d["maps"][k].read(np.int32, 5000) for k in range(3)])
        rows = np.where(long, 40, -1).astype(np.int32)
    assert w["n_free"] + w["held"].sum() == 65 * long.sum() + 3


@pytest.mark.parametrize("layout", [(16, 2, 256, 0), (12, 2, 128, 0), (8, 8, 64, 0)])
@pytest.mark.parametrize("n,pos", [([1, 1], [400, 31]), ([40, 1], [500, 90]), ([300], [480])])
def test_rows_of_large_and_of_ordinary_scores_together(ctx, monkeypatch, layout, n, pos):
    """Keys that grow along the sequence: rows of every second head meet ever larger scores, past 2^24 powers of two at the end, and take the last cell; the others, at right angles to
    the keys, meet ordinary ones beside them in the same group of rows."""
    monkeypatch.setitem(G.LAYOUTS, "own", layout)
    t = G.Paged(900 + n[0], "own", n, pos, 64)
    u = np.sign(t.rng.standard_normal(t.d)).astype(np.float32)
    across = u.copy()
    across[8 + (t.d - 8) // 2:] *= -1  # half of the dims behind the first eight
    t.q_norm[:] = t.k_norm[:] = 2000
    q = t.qkv[:, :2 * t.nh * t.d].reshape(-1, t.nh, 2, t.d)
    q[:, ::2, 0], q[:, 1::2, 0] = u, across
    own = t.qkv[:, 2 * t.nh * t.d:2 * t.nh * t.d + t.nkv * t.d].reshape(-1, t.nkv, t.d)
    own[:] = -u
    few = (0.03 * t.rng.standard_normal(t.kp.shape)).astype(np.float16)
    for s in range(len(n)):
        where = t.cells(s, 0, pos[s])
        grown = (np.round(2000 * (np.arange(pos[s]) + 1) / pos[s])[:, None, None] * u).astype(np.float16)
        t.kp[where] = np.where(np.arange(t.d) < 8, few[where], grown)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_PAGED, t.args(ctx))
    out, _, vp = t.results()
    for s in range(len(n)):
        seen = vp[t.cells(s, 0, pos[s] + n[s])].astype(np.float64)
        for i in range(n[s]):
            v = seen[:pos[s] + i + 1]
            got = out[t.start[s] + i].reshape(t.nh, t.d)
            tol = 1e-5 * np.abs(v).max()
            kv = np.arange(t.nh) // (t.nh // t.nkv)
            assert np.isfinite(got).all(), (s, i)
            assert (np.abs(got - v[pos[s] - 1][kv])[::2] <= tol).all(), (s, i)
            assert (got >= v.min(0)[kv] - tol).all() and (got <= v.max(0)[kv] + tol).all(), (s, i)
