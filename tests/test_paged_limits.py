"""What the host decides for the operators of a serving batch at the ends of the sizes they accept."""
import ctypes as C

import pytest

import shv
import test_paged as B

MOST_BLOCKS = (1 << 20) // 128 + 2048  # query blocks that the plan's launch has room for


def _work(**kw):
    n = C.c_int64(-5)
    return shv.pkg.load().shv_attn_paged_work(B._ctx(), C.byref(B.attn(**kw)), C.byref(n)), n.value


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rep,n_seq,max_rows", [(64, 2048, 16384), (64, 2048, 12288), (64, 400, 12400), (8, 2048, 83968), (8, 1024, 1 << 17), (1, 2048, 1 << 20), (1, 1, 1 << 20), (64, 513, 16384)])
def test_no_accepted_call_has_more_query_blocks_than_a_plan_holds(d, rep, n_seq, max_rows):
    """The scratch of a device with one unit (the context here says none): a block's record and a piece a query block, 64 and 32 bytes, and two records of a block's rows."""
    rc, got = _work(head_dim=d, n_head=rep, n_head_kv=1, n_seq=n_seq, max_rows=max_rows, rope_dims=0)
    assert rc == 0
    assert got <= MOST_BLOCKS * (64 + 32) + 2 * 128 * (d + 2) * 4 + 4096


@pytest.mark.parametrize("heads,rows", [(1024, (1 << 15) + 1), (64, (1 << 19) + 1), (33, 1 << 20)])
def test_more_cells_than_a_launch_has_threads_for_are_refused(heads, rows):
    kw = dict(n_head=heads, n_head_kv=heads, head_dim=64, rope_dims=0, qkv_stride=heads * 256)
    assert _work(**kw, max_rows=rows) == (-1, -5)
    B._refused("shv_attn_paged", B.attn(**kw, max_rows=rows), "KV heads")
    assert _work(**kw, max_rows=(1 << 25) // heads)[0] == 0
