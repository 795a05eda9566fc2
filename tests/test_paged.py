"""Refusals of the operators of a serving batch over a paged cache: what the kernels do not cover is turned away on the host, before anything is launched."""
import ctypes as C

import pytest

import shv

A = shv.api
P = 1 << 20  # an address that is never followed


def _ctx():
    # the checks come before the context is looked at
    return C.cast(C.create_string_buffer(1 << 16), C.c_void_p)


def plan(**kw):
    return A.PagePlanArgs(**{**dict(rows=P, pos=2 * P, table=P, held=3 * P, free_pages=P, n_free=P, start=P, row_pos=P, row_cell=P, n_seq=4, page=64, max_pages=10,
                                    n_pages=100, max_rows=64), **kw})


def attn(**kw):
    return A.AttnPagedArgs(**{**dict(qkv=P, q_norm=P, k_norm=P, rope=P, kpages=P, vpages=P, table=P, start=P, row_pos=P, row_cell=P, work=P, out=P, work_bytes=1 << 40, n_seq=2,
                                     max_rows=8, n_head=16, n_head_kv=2, head_dim=256, rope_dims=64, page=64, max_pages=10, n_pages=100, qkv_stride=9216, eps=1e-6), **kw})


def logp(**kw):
    return A.LogprobsArgs(**{**dict(logits=P, ids=P, logprob=P, entropy=P, top_ids=P, top_logprobs=P, n_rows=4, n=1000, logits_stride=1000, n_top=5), **kw})


def _refused(fn, args, match):
    L = shv.pkg.load()
    assert getattr(L, fn)(_ctx(), C.byref(args)) == -1
    assert match in L.shv_last_error().decode()


@pytest.mark.parametrize("bad,match", [
    *[({k: None}, "NULL") for k in ("rows", "pos", "table", "held", "free_pages", "n_free", "start", "row_pos", "row_cell")],
    ({"n_seq": 0}, "sequences"), ({"n_seq": 2049}, "sequences"), ({"page": 16}, "page"), ({"page": 48}, "page"), ({"page": 8192}, "page"), ({"page": 0}, "page"), ({"page": -64}, "page"),
    ({"n_pages": 0}, "pages"), ({"n_pages": 1 << 25}, "2^31"), ({"max_pages": 0}, "max_pages"), ({"max_pages": 1 << 25}, "2^31"), ({"max_rows": 0}, "max_rows"),
    ({"max_rows": (1 << 20) + 1}, "max_rows"), ({"base": 2 * P}, "of their own"), ({"rows": 2 * P}, "of their own"), ({"held": 2 * P}, "of their own")])
def test_page_plan_refuses(bad, match):
    _refused("shv_page_plan", plan(**bad), match)


@pytest.mark.parametrize("bad,match", [
    *[({k: None}, "NULL") for k in ("qkv", "q_norm", "k_norm", "rope", "kpages", "vpages", "table", "start", "row_pos", "row_cell", "work", "out")],
    *[({k: P + 4}, "aligned") for k in ("qkv", "q_norm", "k_norm", "rope", "kpages", "vpages", "work", "out")],
    ({"n_seq": 0}, "sequences"), ({"n_seq": 2049}, "sequences"), ({"head_dim": 96}, "head_dim"), ({"n_head": 15}, "heads"), ({"n_head_kv": 0}, "heads"), ({"n_head": 130}, "heads"),
    ({"n_head": 1026, "n_head_kv": 1026}, "heads"), ({"rope_dims": 60}, "rope_dims"), ({"rope_dims": 264}, "rope_dims"), ({"rope_dims": -8}, "rope_dims"), ({"max_rows": 0}, "rows"),
    ({"max_rows": (1 << 17) + 1}, "rows"), ({"page": 33}, "page"), ({"page": 16}, "page"), ({"n_pages": 0}, "pages"), ({"n_pages": 1 << 25}, "2^31"), ({"max_pages": 0}, "max_pages"),
    ({"max_pages": 1 << 25}, "2^31"), ({"qkv_stride": 9212}, "qkv_stride"), ({"qkv_stride": 9218}, "qkv_stride"), ({"window": -1}, "window"), ({"sinks": -1}, "sinks")])
def test_attn_paged_refuses(bad, match):
    _refused("shv_attn_paged", attn(**bad), match)


@pytest.mark.parametrize("bad,match", [
    ({"logits": None}, "NULL"), ({"ids": None}, "together"), ({"logprob": None}, "together"), ({"n_rows": 0}, "rows"), ({"n_rows": 65536}, "rows"), ({"n": 0}, "logits"),
    ({"n": (1 << 30) + 1, "logits_stride": 2**31 - 1}, "logits"), ({"logits_stride": 999}, "logits"), ({"n_top": -1}, "alternatives"), ({"n_top": 65}, "alternatives"),
    ({"n": 4, "n_top": 5}, "alternatives"), ({"top_ids": None}, "top_ids"), ({"top_logprobs": None}, "top_ids"), ({"n_top": 0}, "top_ids"),
    ({"ids": None, "logprob": None, "entropy": None, "n_top": 0, "top_ids": None, "top_logprobs": None}, "nothing")])
def test_logprobs_refuses(bad, match):
    _refused("shv_logprobs", logp(**bad), match)


@pytest.mark.parametrize("bad", [{"n_seq": 0}, {"head_dim": 32}, {"page": 100}, {"max_rows": -1}, {"n_head": 7}, {"n_pages": -1}])
def test_work_of_sizes_that_are_refused(bad):
    n = C.c_int64(-5)
    assert shv.pkg.load().shv_attn_paged_work(_ctx(), C.byref(attn(**bad)), C.byref(n)) == -1
    assert n.value == -5


def test_argument_blocks_fit_the_op_record():
    L = shv.pkg.load()
    for kind, args in ((A.OP_PAGE_PLAN, plan()), (A.OP_ATTN_PAGED, attn()), (A.OP_LOGPROBS, logp())):
        assert C.sizeof(args) <= 248
        assert L.shv_enqueue(_ctx(), kind, C.byref(args), C.sizeof(args) - 1) == -1
        assert b"argument block" in L.shv_last_error()
