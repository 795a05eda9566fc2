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
