"""Refusals of the tree operators: every argument the kernels do not cover is turned away on the host, before anything is launched."""
import ctypes as C

import pytest

import shv

A = shv.api
P = 1 << 20  # an address that is never followed


def _ctx():
    # the checks come before the context is looked at
    return C.cast(C.create_string_buffer(1 << 16), C.c_void_p)


def attn(**kw):
    return A.AttnTreeArgs(**{**dict(qkv=P, q_norm=P, k_norm=P, rope=P, kcache=P, vcache=P, kcells=P, vcells=P, partial=P, out=P, n_seq=1, rows=4, n_head=16,
                                    n_head_kv=2, head_dim=256, rope_dims=64, max_cells=64, qkv_stride=9216, n_splits=4, eps=1e-6), **kw})


def keep(**kw):
    return A.AttnKeepArgs(**{**dict(kcells=P, vcells=P, kcache=P, vcache=P, path=P, n_keep=P, n_seq=1, rows=4, n_head_kv=2, head_dim=256, max_cells=64), **kw})


def dn(**kw):
    return A.DnTreeArgs(**{**dict(x=P, ring=P, conv1d=P, a=P, dt_bias=P, state=P, out=P, kn=P, delta=P, decay=P, n_seq=1, rows=4, n_head_k=16, n_head_v=32,
                                  head_dim=128, conv=4, x_stride=12352, ring_slots=8, ring_stride=12352, n_planes=2, eps=1e-6), **kw})


def dnkeep(**kw):
    return A.DnKeepArgs(**{**dict(x=P, kn=P, delta=P, decay=P, state=P, ring=P, path=P, n_keep=P, n_seq=1, rows=4, n_head_k=16, n_head_v=32, head_dim=128,
                                  conv=4, x_stride=12352, ring_slots=8, ring_stride=12352, n_planes=2), **kw})


def acc(**kw):
    return A.TreeAcceptArgs(**{**dict(logits=P, ids=P, best=P, path=P, n_keep=P, next=P, n_seq=1, rows=4, n=1000, logits_stride=1000), **kw})


def _refused(fn, args, match):
    L = shv.pkg.load()
    assert getattr(L, fn)(_ctx(), C.byref(args)) == -1
    assert match in L.shv_last_error().decode()


@pytest.mark.parametrize("bad,match", [
    *[({k: None}, "NULL") for k in ("qkv", "q_norm", "k_norm", "rope", "kcache", "vcache", "kcells", "vcells", "partial", "out")],
    *[({k: P + 4}, "aligned") for k in ("rope", "qkv", "q_norm", "k_norm", "kcache", "vcache", "kcells", "vcells", "partial", "out")],
    ({"rows": 0}, "rows"), ({"rows": 65}, "rows"), ({"n_seq": 0}, "sequences"), ({"n_seq": 70000}, "sequences"), ({"head_dim": 96}, "head_dim"),
    ({"head_dim": 512}, "head_dim"), ({"n_head": 15}, "heads"), ({"n_head_kv": 0}, "heads"), ({"n_head": 130}, "heads"), ({"n_head": -16}, "heads"),
    ({"n_head": 1026, "n_head_kv": 1026}, "heads"), ({"rope_dims": 63}, "rope_dims"), ({"rope_dims": 60}, "rope_dims"), ({"rope_dims": 258}, "rope_dims"), ({"rope_dims": -2}, "rope_dims"),
    ({"max_cells": 40}, "max_cells"), ({"max_cells": 0}, "max_cells"), ({"qkv_stride": 9212}, "qkv_stride"), ({"qkv_stride": 9218}, "qkv_stride"),
    ({"n_splits": 0}, "slices"), ({"n_splits": 513}, "slices"), ({"window": -1}, "window"), ({"sinks": -1}, "sinks")])
def test_attn_tree_refuses(bad, match):
    _refused("shv_attn_tree", attn(**bad), match)


@pytest.mark.parametrize("bad,match", [
    *[({k: None}, "NULL") for k in ("kcells", "vcells", "kcache", "vcache", "path", "n_keep")],
    *[({k: P + 8}, "aligned") for k in ("kcells", "vcells", "kcache", "vcache")],
    ({"rows": 0}, "rows"), ({"rows": 65}, "rows"), ({"n_seq": 0}, "sequences"), ({"n_seq": 65536}, "sequences"), ({"head_dim": 32}, "head_dim"),
    ({"n_head_kv": 0}, "heads"), ({"max_cells": 33}, "max_cells")])
def test_attn_keep_refuses(bad, match):
    _refused("shv_attn_keep", keep(**bad), match)


@pytest.mark.parametrize("bad,match", [
    *[({k: None}, "NULL") for k in ("x", "ring", "conv1d", "a", "dt_bias", "state", "out", "kn", "delta", "decay")],
    *[({k: P + 4}, "aligned") for k in ("x", "ring", "conv1d", "state", "out", "kn", "delta")],
    ({"rows": 0}, "rows"), ({"rows": 65}, "rows"), ({"n_seq": 0}, "sequences"), ({"head_dim": 64}, "head_dim"), ({"conv": 3}, "conv"), ({"n_head_k": 0}, "heads"),
    ({"n_head_k": 12}, "heads"), ({"n_head_v": 8}, "heads"), ({"x_stride": 12351}, "x_stride"), ({"ring_slots": 2}, "ring"), ({"ring_stride": 8191}, "ring"),
    ({"n_planes": -1}, "planes"), ({"n_planes": 65}, "planes")])
def test_dn_tree_refuses(bad, match):
    _refused("shv_dn_tree", dn(**bad), match)


@pytest.mark.parametrize("bad,match", [
    *[({k: None}, "NULL") for k in ("x", "kn", "delta", "decay", "state", "ring", "path", "n_keep")],
    *[({k: P + 4}, "aligned") for k in ("kn", "state")],
    ({"rows": 0}, "rows"), ({"rows": 65}, "rows"), ({"n_seq": 0}, "sequences"), ({"head_dim": 256}, "head_dim"), ({"conv": 2}, "conv"), ({"n_head_k": 5}, "heads"),
    ({"x_stride": 8191}, "x_stride"), ({"ring_slots": 2}, "ring"), ({"ring_stride": 8000}, "ring"), ({"n_planes": 65}, "planes")])
def test_dn_keep_refuses(bad, match):
    _refused("shv_dn_keep", dnkeep(**bad), match)


@pytest.mark.parametrize("bad,match", [
    *[({k: None}, "NULL") for k in ("ids", "best", "path", "n_keep", "next")], ({"rows": 0}, "rows"), ({"rows": 65}, "rows"), ({"n_seq": 0}, "sequences"),
    ({"n_seq": 1025}, "sequences"), ({"n_seq": 1000, "rows": 64}, "at most"), ({"n": 0}, "logits"), ({"logits_stride": 999}, "logits"), ({"pos": P}, "together"),
    ({"base": P}, "together"), ({"pos": P, "base": P}, "one array")])
def test_tree_accept_refuses(bad, match):
    _refused("shv_tree_accept", acc(**bad), match)


def test_argument_blocks_fit_the_op_record():
    for t in (A.AttnTreeArgs, A.AttnKeepArgs, A.DnTreeArgs, A.DnKeepArgs, A.TreeAcceptArgs):
        assert C.sizeof(t) <= 248, t
    for kind, args in ((A.OP_ATTN_TREE, attn()), (A.OP_ATTN_KEEP, keep()), (A.OP_DN_TREE, dn()), (A.OP_DN_KEEP, dnkeep()), (A.OP_TREE_ACCEPT, acc())):
        L = shv.pkg.load()
        assert L.shv_enqueue(_ctx(), kind, C.byref(args), C.sizeof(args) - 1) == -1
        assert b"argument block" in L.shv_last_error()


@pytest.mark.parametrize("bad", [{"max_cells": -1}, {"max_cells": 64}, {"max_cells": -64, "pos": P, "base": P + 64}])
def test_tree_accept_refuses_room_it_cannot_look_at(bad):
    _refused("shv_tree_accept", acc(**bad), "max_cells")


@pytest.mark.parametrize("n", [2**31 - 1, 2**31 - 2048, 2**30 + 1])
def test_tree_accept_refuses_rows_its_indexes_cannot_count(n):
    _refused("shv_tree_accept", acc(n=n, logits_stride=2**31 - 1), "logits")
