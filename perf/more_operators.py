"""A pass of a serving batch over a paged cache, operator by operator, as cases that can be timed.

Requests of uneven length share one pool of cache pages.  A pass first settles which pages each request's new tokens go to
(the plan), attends over the pages with the new tokens' rows packed one request behind the other (a prompt's chunk,
single tokens, both mixed), and answers with log probabilities: of given tokens, with the distribution's entropy and its
most likely tokens.

`run` computes each in its plain form, by elementary torch operations, or through the framework's own entry
points where `own` is set.
"""
import importlib
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-6
ROPE_BASE = 1e7
VOCAB = 151936

# query heads, KV heads, head width, rotated dims: the model's layers, and wider and narrower ones of the same kind
LAYOUTS = {"gqa8_256": (16, 2, 256, 64), "gqa4_128": (32, 8, 128, 128), "gqa6_128": (12, 2, 128, 64), "mha_64": (8, 8, 64, 32)}


def listed():
    return [
        # the step of a small server: one token for each request
        dict(name="plan_48_tokens", op="plan", seqs=48, rows=48, chunks=0, cells=9000, page=64, tight=False),
        # a large server's pass: chunks of prompts among the single tokens, requests that end, and a pool that does not hold them all
        dict(name="plan_900_mixed", op="plan", seqs=900, rows=12007, chunks=24, cells=6000, page=32, tight=True),
        # a short chat's step: latency
        dict(name="attn_1_token_at_900", op="attn", seqs=1, rows=1, chunks=0, cells=900, layout="gqa8_256", page=32, window=0, sinks=0),
        # single tokens of forty requests
        dict(name="attn_40_tokens", op="attn", seqs=40, rows=40, chunks=0, cells=9001, layout="gqa8_256", page=64, window=0, sinks=0),
        # the same where the layers have a sliding window and four sinks
        dict(name="attn_96_tokens_window", op="attn", seqs=96, rows=96, chunks=0, cells=20011, layout="gqa4_128", page=32, window=2048, sinks=4),
        # a follow-up question behind a conversation
        dict(name="attn_37_rows_at_3001", op="attn", seqs=1, rows=37, chunks=1, cells=3001, layout="gqa8_256", page=32, window=0, sinks=0),
        # a prompt's chunk among single tokens
        dict(name="attn_mixed_535", op="attn", seqs=24, rows=535, chunks=1, cells=12000, layout="gqa4_128", page=64, window=0, sinks=0),
        # a prompt from its first token
        dict(name="attn_prompt_4096", op="attn", seqs=1, rows=4096, chunks=1, cells=0, layout="gqa8_256", page=256, window=0, sinks=0),
        # a chunk of a very long document
        dict(name="attn_2048_rows_at_30000", op="attn", seqs=1, rows=2048, chunks=1, cells=30000, layout="gqa8_256", page=128, window=0, sinks=0),
        # the answer's token with five alternatives: latency
        dict(name="logprobs_1_top5", op="logprobs", rows=1, vocab=VOCAB, top=5, banned=0.0),
        # a batch's tokens with twenty, under a grammar that forbids most of the vocabulary
        dict(name="logprobs_40_top20", op="logprobs", rows=40, vocab=VOCAB, top=20, banned=0.7),
        # a prompt scored
        dict(name="logprobs_1500", op="logprobs", rows=1500, vocab=VOCAB, top=0, banned=0.0),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("plan", "attn", "attn", "attn", "attn", "logprobs", "logprobs"))
    page = rng.choice((32, 64, 128, 256))
    if op == "plan":
        seqs = log(1, 900)
        chunks = rng.choice((0, rng.randint(1, max(1, seqs // 8))))
        return dict(op=op, seqs=seqs, rows=seqs + (log(1, 12000) if chunks else 0), chunks=chunks, cells=log(1, 9000), page=page, tight=rng.random() < 0.5)
    if op == "logprobs":
        rows = log(1, 1500)
        return dict(op=op, rows=rows, vocab=rng.choice((VOCAB, log(100, VOCAB))), top=rng.choice((0, 1, rng.randint(2, 20), rng.randint(21, 32))), banned=rng.choice((0.0, rng.uniform(0.1, 0.99))))
    layout = rng.choice(sorted(LAYOUTS))
    kind = rng.choice(("tokens", "chunk", "mixed"))
    seqs = 1 if kind == "chunk" else log(1, 96) if kind == "tokens" else log(2, 40)
    cells = log(1, 30000)
    while seqs * cells > 400000:
        cells //= 2
    rows = seqs + (0 if kind == "tokens" else log(1, 2047))
    chunks = 0 if kind == "tokens" else 1 if kind == "chunk" else rng.randint(1, max(1, seqs // 4))
    heads = LAYOUTS[layout][0] * LAYOUTS[layout][2]
    while rows * (cells + rows) * heads > 2048 * 32000 * 4096:
        cells //= 2
    window = rng.choice((0, 0, log(8, 8192)))
    return dict(op=op, seqs=seqs, rows=rows, chunks=chunks, cells=cells, layout=layout, page=page, window=window, sinks=rng.randint(0, 8) if window else 0)


# ---- inputs ----------------------------------------------------------------------------------


class State:
    pass


def _gen(case, seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 29), random.Random("%d %r" % (seed, sorted((k, v) for k, v in case.items() if k != "name")))


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _rows_of(case, r):
    """New tokens of each request: one, or a chunk's share of what is left of the pass's rows."""
    seqs, chunks = case["seqs"], case["chunks"]
    rows, left = [1] * seqs, case["rows"] - case["seqs"]
    for k, s in enumerate(sorted(r.sample(range(seqs), chunks))):
        share = left if k == chunks - 1 else min(left, int(2 * left / (chunks - k) * r.random()))
        rows[s] += share
        left -= share
    return rows


def _past_of(case, r):
    """Tokens each request has behind it: what the case says of a single one, anything up to it of several."""
    return [case["cells"] if case["seqs"] == 1 else r.randint(case["cells"] // 4, case["cells"]) for _ in range(case["seqs"])]


def _pool(case):
    """Pages of the pool, and of the longest request there may be."""
    page, chunk = case["page"], case["rows"] - case["seqs"]
    return case["seqs"] * (case["cells"] // page + 2) + chunk // page + 9, (case["cells"] + chunk + 1) // page + 2


def _rope_table(cells, dims):
    theta = torch.arange(cells, dtype=torch.float64, device=DEV)[:, None] * ROPE_BASE ** (-2.0 / dims * torch.arange(dims // 2, dtype=torch.float64, device=DEV))
    return torch.cat((theta.cos(), theta.sin()), 1).float()


def _prepare_plan(s, case, r):
    seqs, page = case["seqs"], case["page"]
    rows, pos = _rows_of(case, r), _past_of(case, r)
    held = [-(-p // page) for p in pos]
    # a few requests end, a few stand on a prefix that another one owns
    if seqs > 8:
        for i in range(seqs):
            if rows[i] == 1 and r.random() < 0.05:
                rows[i] = -1
    shared = [r.randint(0, h) if rows[i] > 0 and r.random() < 0.2 else 0 for i, h in enumerate(held)]
    need = sum(max(0, -(-(p + n) // page) - h) for p, n, h in zip(pos, rows, held))
    # of the pool's pages other requests, which are not in this pass, hold those that are neither theirs nor free
    s.n_pages, s.max_pages = _pool(case)
    spare = max(1, need * 3 // 4 if case["tight"] else need + 8)
    order = list(range(s.n_pages))
    r.shuffle(order)
    table = np.full((seqs, s.max_pages), -1, np.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = order[at:at + h]
        at += h
    free = np.array(order[at:at + spare] + [-1] * (s.n_pages - spare), np.int32)
    s.max_rows = case["rows"]
    s.rows, s.pos, s.held, s.shared = _ints(rows), _ints(pos), _ints(held), _ints(shared)
    s.none = torch.zeros_like(s.rows)
    s.table, s.free, s.n_free = torch.from_numpy(table).to(DEV), torch.from_numpy(free).to(DEV), _ints([spare])
    s.start, s.start_after = (torch.zeros(seqs + 1, dtype=torch.int32, device=DEV) for _ in range(2))
    s.row_seq, s.row_pos, s.row_cell = (torch.full((s.max_rows,), -1, dtype=torch.int32, device=DEV) for _ in range(3))


def _prepare_attn(s, case, g, r):
    nh, nkv, d, rope = LAYOUTS[case["layout"]]
    seqs, page = case["seqs"], case["page"]
    s.n_rows, s.n_past = _rows_of(case, r), _past_of(case, r)
    s.pages_of = [-(-(p + n) // page) for p, n in zip(s.n_past, s.n_rows)]
    s.longest = max(s.pages_of)
    s.n_pages, s.max_pages = _pool(case)
    order = list(range(s.n_pages))
    r.shuffle(order)
    table = np.full((seqs, s.max_pages), -1, np.int32)
    start, row_pos, row_cell, at = [0], [], [], 0
    for i, (p, n, h) in enumerate(zip(s.n_past, s.n_rows, s.pages_of)):
        table[i, :h] = order[at:at + h]
        at += h
        start.append(start[-1] + n)
        where = np.arange(p, p + n)
        row_pos += where.tolist()
        row_cell += (table[i, where // page].astype(np.int64) * page + where % page).tolist()
    s.table, s.start, s.row_pos, s.row_cell = torch.from_numpy(table).to(DEV), _ints(start), _ints(row_pos), _ints(row_cell)
    s.first = start
    total = start[-1]
    s.width = 2 * nh * d + 2 * nkv * d
    s.qkv = torch.randn(total, s.width, generator=g, device=DEV)
    s.q_norm, s.k_norm = (1 + 0.1 * torch.randn(d, generator=g, device=DEV) for _ in range(2))
    s.rope = _rope_table(s.max_pages * page, rope)
    s.kpages = torch.empty(s.n_pages, page, nkv, d, dtype=torch.float16, device=DEV).normal_(generator=g)
    s.vpages = torch.empty(s.n_pages, page // 32, nkv, d, 32, dtype=torch.float16, device=DEV).normal_(generator=g)
    s.out = torch.zeros(total, nh * d, device=DEV)


def _prepare_logprobs(s, case, g, r):
    rows, n, top = case["rows"], case["vocab"], case["top"]
    s.logits = 2.5 * torch.randn(rows, n, generator=g, device=DEV)
    # a model is sure of some tokens: one or a few logits stand out
    few = torch.randint(0, n, (rows, 4), generator=g, device=DEV)
    s.logits.scatter_(1, few, 8 + 6 * torch.rand(rows, 4, generator=g, device=DEV))
    if case["banned"] > 0:
        gone = torch.rand(rows, n, generator=g, device=DEV) < case["banned"]
        gone[:, :1] = False
        s.logits.masked_fill_(gone, -math.inf)
    s.ids = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.7, s.logits.argmax(1), few[:, 0]).int()
    s.logprob, s.entropy = (torch.zeros(rows, device=DEV) for _ in range(2))
    s.top_ids, s.top_logprobs = torch.zeros(rows, top, dtype=torch.int32, device=DEV), torch.zeros(rows, top, device=DEV)


def prepare(case, seed):
    g, r = _gen(case, seed)
    s = State()
    s.case, s.calls = case, None
    if case["op"] == "plan":
        _prepare_plan(s, case, r)
    elif case["op"] == "attn":
        _prepare_attn(s, case, g, r)
    else:
        _prepare_logprobs(s, case, g, r)
    return s


# ---- plain forms -----------------------------------------------------------------------------


def _plan_call(s, rows, start):
    page, seqs = s.case["page"], s.case["seqs"]
    r, pos, held, shared = rows.long(), s.pos.long(), s.held.long(), s.shared.long()
    ends, asked = r < 0, r.clamp(min=0)
    want = torch.where(ends, 0, (pos + asked + page - 1) // page)
    fits = want <= s.max_pages
    kept = torch.maximum(want, shared)
    back = torch.where(fits, held - kept, 0).clamp(min=0)
    need = torch.where(fits, want - held, 0).clamp(min=0)
    asked = torch.where(fits, asked, 0)
    avail = s.n_free.long() + back.sum()
    granted = fits & ((need == 0) | (need.cumsum(0) <= avail)) & (asked.cumsum(0) <= s.max_rows)
    take, new = torch.where(granted, need, 0), torch.where(granted, asked, 0)
    j = torch.arange(s.max_pages, device=DEV)
    # the pages given back stand behind the free ones, in the order of the requests
    low = (held - back)[:, None]
    place = s.n_free.long() + (back.cumsum(0) - back)[:, None] + j - low
    leaves = (j >= low) & (j < held[:, None])
    pool = torch.cat((s.free, s.free[:1])).scatter(0, torch.where(leaves, place, s.n_pages).flatten(), s.table.flatten())[:-1]
    # and are taken from the end
    at = avail - 1 - (take.cumsum(0) - take)[:, None] - (j - held[:, None])
    comes = (j >= held[:, None]) & (j < (held + take)[:, None])
    s.table.copy_(torch.where(comes, pool[at.clamp(0, s.n_pages - 1)], s.table))
    s.free.copy_(pool)
    s.n_free.copy_(avail - take.sum())
    s.held.copy_(torch.where(ends, 0, held - back + take))
    start[1:].copy_(new.cumsum(0))
    t = torch.arange(s.max_rows, device=DEV)
    live = t < start[-1]
    seq = (t[:, None] >= start[None, 1:]).sum(1).clamp(max=seqs - 1)
    p = pos[seq] + t - start[seq]
    cell = s.table[seq, (p // page).clamp(max=s.max_pages - 1)] * page + p % page
    s.row_seq.copy_(torch.where(live, seq, s.row_seq))
    s.row_pos.copy_(torch.where(live, p, s.row_pos))
    s.row_cell.copy_(torch.where(live, cell, s.row_cell))


def _plan(s):
    """A pass's pages, and what is given back after it when none of its tokens is kept."""
    _plan_call(s, s.rows, s.start)
    _plan_call(s, s.none, s.start_after)
    return _plan_out(s)


def _plan_out(s):
    return {"table": s.table, "held": s.held, "free": s.free, "n_free": s.n_free, "start": s.start, "start_after": s.start_after,
            "row_seq": s.row_seq, "row_pos": s.row_pos, "row_cell": s.row_cell}


def _turn(x, cos, sin):
    h = cos.shape[-1]
    x0, x1 = x[..., :h], x[..., h:2 * h]
    return torch.cat((x0 * cos - x1 * sin, x0 * sin + x1 * cos, x[..., 2 * h:]), -1)


def _normed(x, gamma):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma


def _attend(q, k, v, c, at, window, sinks):
    """q [seqs][rows][heads][d], k and v [seqs][cells][KV heads][d] at positions c [seqs][cells], at [seqs][rows] the rows' positions."""
    seqs, rows, nh, d = q.shape
    cells, nkv = k.shape[1:3]
    rep = nh // nkv
    qh = q.reshape(seqs, rows, nkv, rep, d).permute(0, 2, 1, 3, 4).reshape(seqs, nkv, rows * rep, d)
    score = (qh @ k.permute(0, 2, 3, 1).contiguous()).div_(math.sqrt(d)).view(seqs, nkv, rows, rep, cells)
    c = c[:, None, :]
    seen = c <= at[:, :, None]
    if window:
        seen = seen & ((c < sinks) | (at[:, :, None] - c < window))
    score.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).view(seqs, nkv, rows * rep, cells)
    o = p @ v.permute(0, 2, 1, 3).contiguous()
    return o.view(seqs, nkv, rows, rep, d).permute(0, 2, 1, 3, 4).reshape(seqs, rows, nh * d)


def _cells(s, table, pages, first):
    """The cells of the first `pages` pages that a table names, or of those that a window behind positions `first` and later leaves of them, in 32 bits, and their positions."""
    nh, nkv, d, rope = LAYOUTS[s.case["layout"]]
    page, window, sinks = s.case["page"], s.case["window"], s.case["sinks"]
    seqs = table.shape[0]
    index = torch.arange(pages, device=DEV).expand(seqs, pages)
    if window:
        rows = s.case["rows"] - s.case["seqs"] + 1
        sink_pages, reach = -(-sinks // page), min(pages, (window + rows) // page + 2)
        low = ((first - window + 1).clamp(min=0) // page).clamp(min=sink_pages)
        index = torch.cat((index[:, :sink_pages], low[:, None] + index[:, :reach]), 1)
    at = table.gather(1, index.clamp(max=table.shape[1] - 1)).clamp(min=0).long()
    cells = at.shape[1] * page
    k = s.kpages[at].reshape(seqs, cells, nkv, d)
    v = s.vpages[at].permute(0, 1, 2, 5, 3, 4).reshape(seqs, cells, nkv, d)
    where = (index[:, :, None] * page + torch.arange(page, device=DEV)).reshape(seqs, cells)
    return k.float(), v.float(), where


def _attn(s):
    case = s.case
    nh, nkv, d, rope = LAYOUTS[case["layout"]]
    page, window, sinks = case["page"], case["window"], case["sinks"]
    total = s.qkv.shape[0]
    at = s.row_pos.long()
    table = s.rope[at][:, None, :]
    cos, sin = table[..., :rope // 2], table[..., rope // 2:]
    q = s.qkv[:, :2 * nh * d].view(total, nh, 2, d)[:, :, 0]
    k = s.qkv[:, 2 * nh * d:2 * nh * d + nkv * d].view(total, nkv, d)
    v = s.qkv[:, 2 * nh * d + nkv * d:].view(total, nkv, d)
    q = _turn(_normed(q, s.q_norm), cos, sin)
    # the cells a row leaves are rounded: their values in 64 bits, so that one next to a border falls where it belongs
    k = _turn(_normed(k.double(), s.k_norm.double()), cos.double(), sin.double()).float().half()
    where = s.row_cell.long()
    s.kpages[where // page, where % page] = k
    s.vpages[where // page, where % page // 32, :, :, where % 32] = v.half()
    if case["rows"] == case["seqs"]:  # one token each: the requests side by side, as long as the longest
        s.out.copy_(_attend(q[:, None], *_cells(s, s.table, s.longest, at), at[:, None], window, sinks)[:, 0])
    else:  # one request after the other: as long as it is
        for i in range(case["seqs"]):
            a, b = s.first[i], s.first[i + 1]
            s.out[a:b] = _attend(q[None, a:b], *_cells(s, s.table[i:i + 1], s.pages_of[i], at[a:a + 1]), at[None, a:b], window, sinks)[0]
    return {"out": s.out, "kpages": s.kpages, "vpages": s.vpages}


def _logprobs(s):
    x, top = s.logits, s.case["top"]
    off = x - x.amax(1, keepdim=True)
    w = torch.exp(off)
    z = w.sum(1, keepdim=True)
    log_z = torch.log(z)
    s.logprob.copy_((off.gather(1, s.ids.long()[:, None]) - log_z)[:, 0])
    s.entropy.copy_((log_z - torch.where(w > 0, w * off, 0).sum(1, keepdim=True) / z)[:, 0])
    if top:
        ranked, place = torch.sort(off, dim=1, descending=True, stable=True)
        s.top_ids.copy_(place[:, :top])
        s.top_logprobs.copy_(ranked[:, :top] - log_z)
    return _logprobs_out(s)


def _logprobs_out(s):
    out = {"logprob": s.logprob, "entropy": s.entropy}
    return {**out, "top_ids": s.top_ids, "top_logprobs": s.top_logprobs} if s.case["top"] else out


# ---- the framework's calls -------------------------------------------------------------------

_handle = []


def _context():
    """One context of the process, as a program keeps one, and the scratch memory its calls share."""
    if not _handle:
        api = importlib.import_module("strix-halo-vulkan_amd").hip_api
        _handle.append([api, api.Context(torch.cuda.current_device()), None])
    return _handle[0]


def _scratch(nbytes):
    h = _context()
    if h[2] is None or h[2].numel() < nbytes:
        h[1].sync()  # calls that are on their way may still use the smaller one
        h[2] = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    return h[2].data_ptr()


def _call(s):
    """The calls' kinds and argument blocks, made once: what the device reads from call to call stands in its memory."""
    api, ctx, _ = _context()
    at = lambda t: t.data_ptr()  # noqa: E731
    case = s.case
    if case["op"] == "plan":
        both = [api.PagePlanArgs(rows=at(rows), pos=at(s.pos), table=at(s.table), held=at(s.held), free_pages=at(s.free), n_free=at(s.n_free), shared=at(s.shared),
                                 start=at(start), row_seq=at(s.row_seq), row_pos=at(s.row_pos), row_cell=at(s.row_cell), n_seq=case["seqs"], page=case["page"],
                                 max_pages=s.max_pages, n_pages=s.n_pages, max_rows=s.max_rows) for rows, start in ((s.rows, s.start), (s.none, s.start_after))]
        return [(api.OP_PAGE_PLAN, a) for a in both], _plan_out(s)
    if case["op"] == "attn":
        nh, nkv, d, rope = LAYOUTS[case["layout"]]
        a = api.AttnPagedArgs(qkv=at(s.qkv), q_norm=at(s.q_norm), k_norm=at(s.k_norm), rope=at(s.rope), kpages=at(s.kpages), vpages=at(s.vpages), table=at(s.table),
                              start=at(s.start), row_pos=at(s.row_pos), row_cell=at(s.row_cell), out=at(s.out), n_seq=case["seqs"], max_rows=s.qkv.shape[0], n_head=nh,
                              n_head_kv=nkv, head_dim=d, rope_dims=rope, page=case["page"], max_pages=s.max_pages, n_pages=s.n_pages, qkv_stride=s.width,
                              window=case["window"], sinks=case["sinks"], eps=EPS)
        a.work_bytes = ctx.attn_paged_work(a)
        a.work = _scratch(a.work_bytes)
        return [(api.OP_ATTN_PAGED, a)], {"out": s.out, "kpages": s.kpages, "vpages": s.vpages}
    top = case["top"]
    a = api.LogprobsArgs(logits=at(s.logits), ids=at(s.ids), logprob=at(s.logprob), entropy=at(s.entropy), top_ids=at(s.top_ids) if top else None,
                         top_logprobs=at(s.top_logprobs) if top else None, n_rows=case["rows"], n=case["vocab"], logits_stride=case["vocab"], n_top=top)
    return [(api.OP_LOGPROBS, a)], _logprobs_out(s)


def run(s):
    if own:
        if s.calls is None:
            s.calls = _call(s)
        ctx = _context()[1]
        if s.case["op"] == "attn":
            s.calls[0][0][1].work = _scratch(s.calls[0][0][1].work_bytes)
        for kind, args in s.calls[0]:
            ctx.enqueue(kind, args)
        return s.calls[1]
    return {"plan": _plan, "attn": _attn, "logprobs": _logprobs}[s.case["op"]](s)


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    if case["op"] == "plan":
        # two calls: four words of every request read, four written and its rows' three words; the tables' new entries are few
        return {"bytes": 2 * case["seqs"] * 8 * 4 + case["rows"] * 12, "flops": 0}
    if case["op"] == "logprobs":
        return {"bytes": case["rows"] * (case["vocab"] * 4 + 12 + 8 * case["top"]), "flops": 0}
    nh, nkv, d, rope = LAYOUTS[case["layout"]]
    seqs, rows, window = case["seqs"], case["rows"], case["window"]
    past = case["cells"] * (0.625 if seqs > 1 else 1.0)  # a batch's are drawn evenly from a quarter of it up
    each = (rows - seqs) / case["chunks"] + 1 if case["chunks"] else 1
    pairs = cells = 0.0  # rows times the cells they see, cells that some row sees
    for m, n in ((seqs - case["chunks"], 1.0), (case["chunks"], each)):
        seen = min(past + (n + 1) / 2, window + case["sinks"]) if window else past + (n + 1) / 2
        pairs += m * n * seen
        cells += m * (min(past + n, window + case["sinks"] + n) if window else past + n)
    return {"bytes": cells * nkv * d * 4 + rows * ((2 * nh + 2 * nkv) * d * 4 + nkv * d * 4), "flops": 4.0 * d * nh * pairs}


# ---- the definitions in 64 bits --------------------------------------------------------------


def _exact_plan(s):
    page, seqs = s.case["page"], s.case["seqs"]
    table, held = s.table.cpu().numpy().copy(), s.held.tolist()
    free, top = s.free.cpu().numpy().copy(), int(s.n_free)
    pos, shared = s.pos.tolist(), s.shared.tolist()
    maps = [np.full(s.max_rows, -1, np.int32) for _ in range(3)]
    starts = []
    for rows in (s.rows.tolist(), [0] * seqs):
        want = [0 if n < 0 else -(-(p + n) // page) for p, n in zip(pos, rows)]
        for i in range(seqs):  # first everything that comes back
            if want[i] > s.max_pages:
                continue
            keep = max(want[i], shared[i])
            for e in range(keep, held[i]):
                free[top] = table[i, e]
                top += 1
            held[i] = min(held[i], keep) if rows[i] >= 0 else 0
        # then what is asked for, request by request
        avail, wished, asked, total, start = top, 0, 0, 0, [0]
        for i in range(seqs):
            n, need = max(rows[i], 0), max(0, want[i] - held[i])
            if rows[i] < 0 or want[i] > s.max_pages:
                start.append(total)
                continue
            wished += need
            asked += n
            if (need and wished > avail) or asked > s.max_rows:
                start.append(total)
                continue
            for _ in range(need):
                top -= 1
                table[i, held[i]] = free[top]
                held[i] += 1
            for q in range(n):
                p = pos[i] + q
                maps[0][total], maps[1][total], maps[2][total] = i, p, table[i, p // page] * page + p % page
                total += 1
            start.append(total)
        starts.append(np.array(start, np.int32))
    return {"table": table, "held": np.array(held, np.int32), "free": free, "n_free": np.array([top], np.int32), "start": starts[0], "start_after": starts[1],
            "row_seq": maps[0], "row_pos": maps[1], "row_cell": maps[2]}


def _exact_attn(s):
    case, page = s.case, s.case["page"]
    nh, nkv, d, rope = LAYOUTS[case["layout"]]
    half, rep = rope // 2, nh // nkv
    out = torch.zeros_like(s.out, dtype=torch.float64)
    kp, vp = s.kpages.double(), s.vpages.double()

    def turned(x, gamma, at):
        x = x / torch.sqrt(torch.mean(x * x, -1, keepdim=True) + EPS) * gamma.double()
        y = x.clone()
        co, si = s.rope[at].double()[:, None, :half], s.rope[at].double()[:, None, half:]
        y[..., :half] = x[..., :half] * co - x[..., half:rope] * si
        y[..., half:rope] = x[..., :half] * si + x[..., half:rope] * co
        return y

    for i in range(case["seqs"]):
        n, past, a = s.n_rows[i], s.n_past[i], s.first[i]
        pages = s.table[i, :s.pages_of[i]].long()
        where = torch.arange(past, past + n, device=DEV)
        x = s.qkv[a:a + n].double()
        kn = turned(x[:, 2 * nh * d:2 * nh * d + nkv * d].reshape(n, nkv, d), s.k_norm, where).float().half().double()
        vn = x[:, 2 * nh * d + nkv * d:].reshape(n, nkv, d).float().half().double()
        kp[pages[where // page], where % page] = kn
        vp[pages[where // page], where % page // 32, :, :, where % 32] = vn
        q = turned(x[:, :2 * nh * d].reshape(n, nh, 2 * d)[:, :, :d], s.q_norm, where)
        keys = kp[pages].reshape(-1, nkv, d)[:past + n]
        values = vp[pages].permute(0, 1, 4, 2, 3).reshape(-1, nkv, d)[:past + n]
        c = torch.arange(past + n, device=DEV)
        hidden = c[None, :] > where[:, None]
        if case["window"]:
            hidden |= (c[None, :] >= case["sinks"]) & (where[:, None] - c[None, :] >= case["window"])
        for e in range(nh):
            w = (q[:, e] @ keys[:, e // rep].T) * d ** -0.5
            w[hidden] = -math.inf
            w = torch.exp(w - w.max(1, keepdim=True).values)
            out[a:a + n, e * d:(e + 1) * d] = (w @ values[:, e // rep]) / w.sum(1, keepdim=True)
    return {"out": out, "kpages": kp, "vpages": vp}


def _exact_logprobs(s):
    rows, top = s.case["rows"], s.case["top"]
    logprob, entropy = np.zeros(rows), np.zeros(rows)
    top_ids, top_logprobs = np.zeros((rows, top), np.int32), np.zeros((rows, top))
    ids = s.ids.tolist()
    for i in range(rows):
        x = s.logits[i].double()
        lse = torch.logsumexp(x, 0)
        lp = x - lse
        logprob[i] = float(lp[ids[i]])
        entropy[i] = -float((lp.exp() * torch.where(torch.isinf(lp), 0.0, lp)).sum())
        if top:
            x = s.logits[i].cpu().numpy()
            best = np.lexsort((np.arange(len(x)), -x))[:top]
            top_ids[i], top_logprobs[i] = best, lp.cpu().numpy()[best]
    out = {"logprob": logprob, "entropy": entropy}
    return {**out, "top_ids": top_ids, "top_logprobs": top_logprobs} if top else out


def exact(case, seed):
    if case["op"] == "logprobs" and case["rows"] * case["vocab"] * (20 if case["top"] else 1) > 3e8:
        return None  # sorted row by row on the host: too long
    s = prepare(case, seed)
    return {"plan": _exact_plan, "attn": _exact_attn, "logprobs": _exact_logprobs}[case["op"]](s)
