"""Verification of a tree of drafted tokens, operator by operator, as cases that can be timed.

A draft proposes several candidates a position; one pass of the model verifies all of them as the rows of a
tree, each row attending to the sequence's committed past and to its own ancestors alone, and the branch the
model agrees with is kept.  The operators are those such a pass consists of beside the projections: the full
attention over the cache (with a sliding window and always-visible first tokens where a layer has them), the gated
delta rule, the choice of the branch, and what writes the kept branch into the cache and the state.

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
TAPS = 4  # of the causal convolution before the delta rule

# query heads, KV heads, head width, rotated dims: the model's layers, and wider and narrower ones of the same kind
LAYOUTS = {"gqa8_256": (16, 2, 256, 64), "gqa4_128": (32, 8, 128, 128), "gqa6_128": (12, 2, 128, 64), "mha_64": (8, 8, 64, 32)}
DN_HEADS = {"16x32": (16, 32), "16x48": (16, 48), "16x16": (16, 16)}
DN_D = 128


def listed():
    return [
        # a short chat's step with one guess beside the certain token: latency
        dict(name="attn_2_rows_at_700", op="attn_tree", seqs=1, rows=2, cells=700, layout="gqa8_256", window=0, sinks=0, ragged=False),
        # a conversation's ordinary verification pass
        dict(name="attn_12_rows_at_9000", op="attn_tree", seqs=1, rows=12, cells=9000, layout="gqa8_256", window=0, sinks=0, ragged=False),
        # a wide tree behind a very long document
        dict(name="attn_64_rows_at_131000", op="attn_tree", seqs=1, rows=64, cells=131000, layout="gqa8_256", window=0, sinks=0, ragged=False),
        # a server's batch of trees of different sizes, layers with a sliding window and four sinks
        dict(name="attn_batch_window", op="attn_tree", seqs=6, rows=21, cells=20011, layout="gqa4_128", window=2048, sinks=4, ragged=True),
        # the kept branch of one tree into the cache, and those of a batch
        dict(name="keep_cells_1", op="attn_keep", seqs=1, rows=12, cells=9000, layout="gqa8_256", ragged=False),
        dict(name="keep_cells_24", op="attn_keep", seqs=24, rows=33, cells=2500, layout="gqa8_256", ragged=True),
        # the delta rule over a small tree, and over a batch of wide ones
        dict(name="dn_5_rows", op="dn_tree", seqs=1, rows=5, heads="16x32", past=700, ragged=False),
        dict(name="dn_batch_64_rows", op="dn_tree", seqs=8, rows=64, heads="16x32", past=9000, ragged=True),
        # the state behind the kept branch
        dict(name="keep_state_1", op="dn_keep", seqs=1, rows=5, heads="16x32", past=700, ragged=False),
        dict(name="keep_state_12", op="dn_keep", seqs=12, rows=40, heads="16x32", past=9000, ragged=True),
        # the branch the model agrees with
        dict(name="accept_5_rows", op="accept", seqs=1, rows=5, vocab=151936, ragged=False),
        dict(name="accept_batch", op="accept", seqs=8, rows=24, vocab=151936, ragged=True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("attn_tree", "attn_tree", "attn_tree", "attn_keep", "dn_tree", "dn_tree", "dn_keep", "accept"))
    seqs = rng.choice((1, 1, rng.randint(2, 8)))
    rows = log(1, 64)
    if op == "attn_tree":
        layout = rng.choice(sorted(LAYOUTS))
        cells = log(1, 131000)
        while seqs * rows * cells > 64 * 131000 or seqs * cells > 262144:
            cells //= 2
        window = rng.choice((0, 0, log(8, 8192)))
        return dict(op=op, seqs=seqs, rows=rows, cells=cells, layout=layout, window=window, sinks=rng.randint(0, 8) if window else 0, ragged=seqs > 1)
    if op == "attn_keep":
        return dict(op=op, seqs=seqs * rng.randint(1, 3), rows=rows, cells=log(1, 8000), layout=rng.choice(sorted(LAYOUTS)), ragged=seqs > 1)
    if op in ("dn_tree", "dn_keep"):
        return dict(op=op, seqs=seqs, rows=rows, heads=rng.choice(sorted(DN_HEADS)), past=rng.choice((rng.randint(0, 4), log(5, 20000))), ragged=seqs > 1)
    return dict(op=op, seqs=seqs, rows=min(rows, 24), vocab=rng.choice((151936, log(100, 151936))), ragged=seqs > 1)


# ---- inputs ----------------------------------------------------------------------------------


class State:
    pass


def _gen(case, seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 13), random.Random("%d %r" % (seed, sorted((k, v) for k, v in case.items() if k != "name")))


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _trees(case, r):
    """Parents of each sequence's rows, and how many of them are in use: mostly children of recent rows, as a
    draft that extends its best candidates leaves them."""
    seqs, rows = case["seqs"], case["rows"]
    parents = [[-1] + [r.randint(max(0, i - 5), i - 1) if r.random() < 0.8 else r.randint(0, i - 1) for i in range(1, rows)] for _ in range(seqs)]
    counts = [r.randint(1, rows) if case["ragged"] else rows for _ in range(seqs)]
    return parents, counts


def _paths(parents, counts, r):
    """A branch of each tree from its first row, as acceptance leaves it: rows in order, -1 behind them."""
    out, lens = [], []
    for par, n in zip(parents, counts):
        at, path = 0, [0]
        while True:
            kids = [i for i in range(at + 1, n) if par[i] == at]
            if not kids or r.random() < 0.15:
                break
            at = r.choice(kids)
            path.append(at)
        out.append(path + [-1] * (len(par) - len(path)))
        lens.append(len(path))
    return out, lens


def _rope_table(cells, dims):
    theta = torch.arange(cells, dtype=torch.float64, device=DEV)[:, None] * ROPE_BASE ** (-2.0 / dims * torch.arange(dims // 2, dtype=torch.float64, device=DEV))
    return torch.cat((theta.cos(), theta.sin()), 1).float()


def prepare(case, seed):
    g, r = _gen(case, seed)
    s = State()
    s.case, s.calls = case, None
    seqs, rows = case["seqs"], case["rows"]
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    parents, counts = _trees(case, r)
    s.parent, s.count = _ints(parents), _ints(counts)
    slots = list(range(seqs))
    r.shuffle(slots)
    s.slot = _ints(slots)
    if case["op"] in ("attn_tree", "attn_keep"):
        nh, nkv, d, rope = LAYOUTS[case["layout"]]
        cells = case["cells"]
        s.max_cells = (cells + rows + 31) // 32 * 32
        pos = [cells if not case["ragged"] else r.randint(cells // 2, cells) for _ in range(seqs)]
        s.pos = _ints(pos)
        s.kcache = torch.empty(seqs, s.max_cells, nkv, d, dtype=torch.float16, device=DEV).normal_(generator=g)
        s.vcache = torch.empty(seqs, s.max_cells // 32, nkv, d, 32, dtype=torch.float16, device=DEV).normal_(generator=g)
        s.kcells, s.vcells = (torch.zeros(seqs, rows, nkv, d, dtype=torch.float16, device=DEV) for _ in range(2))
        if case["op"] == "attn_keep":
            s.kcells.normal_(generator=g)
            s.vcells.normal_(generator=g)
            paths, lens = _paths(parents, counts, r)
            s.path, s.n_keep = _ints(paths), _ints(lens)
            return s
        s.width = 2 * nh * d + 2 * nkv * d
        s.qkv = randn(seqs, rows, s.width)
        s.q_norm, s.k_norm = 1 + 0.1 * randn(d), 1 + 0.1 * randn(d)
        s.rope = _rope_table(s.max_cells, rope)
        s.out = torch.zeros(seqs, rows, nh * d, device=DEV)
        s.n_splits = 256 // max(1, seqs // 2)
        s.partial = torch.empty(seqs * rows * nh * s.n_splits * (d + 2), device=DEV)
        return s
    if case["op"] in ("dn_tree", "dn_keep"):
        hk, hv = DN_HEADS[case["heads"]]
        s.width = 2 * hk * DN_D + 2 * hv * DN_D + 2 * hv
        s.ring_slots = 8
        s.pos = _ints([case["past"] if not case["ragged"] else r.randint(case["past"] // 2, case["past"]) for _ in range(seqs)])
        s.x = randn(seqs, rows, s.width)
        s.ring = randn(seqs, s.ring_slots, s.width)
        s.state = 0.1 * randn(seqs, 2, hv, DN_D, DN_D)
        s.plane = _ints([r.randint(0, 1) for _ in range(seqs)])
        if case["op"] == "dn_tree":
            s.conv1d = 0.3 * randn(2 * hk * DN_D + hv * DN_D, TAPS)
            s.a = -randn(hv).exp()
            s.dt_bias = randn(hv)
            s.out, s.delta = (torch.zeros(seqs, rows, hv, DN_D, device=DEV) for _ in range(2))
            s.kn = torch.zeros(seqs, rows, hk, DN_D, device=DEV)
            s.decay = torch.zeros(seqs, rows, hv, device=DEV)
            return s
        kn = randn(seqs, rows, hk, DN_D)
        s.kn = kn / kn.norm(dim=-1, keepdim=True)
        s.delta = 0.5 * randn(seqs, rows, hv, DN_D)
        # the sum of each path's log decays: smaller down the tree
        s.decay = -randn(seqs, rows, hv).abs() * 0.3
        for i in range(1, rows):
            s.decay[:, i] += s.decay[torch.arange(seqs, device=DEV), s.parent[:, i].long()]
        paths, lens = _paths(parents, counts, r)
        s.path, s.n_keep = _ints(paths), _ints(lens)
        return s
    vocab = case["vocab"]
    s.logits = randn(seqs, rows, vocab)
    top = [[r.randrange(vocab) for _ in range(rows)] for _ in range(seqs)]
    s.logits.scatter_(2, torch.tensor(top, device=DEV)[:, :, None], 12.0)
    s.ids = _ints([[top[b][parents[b][i]] if i and r.random() < 0.6 else r.randrange(vocab) for i in range(rows)] for b in range(seqs)])
    s.best, s.path = (torch.zeros(seqs, rows, dtype=torch.int32, device=DEV) for _ in range(2))
    s.n_keep, s.next = (torch.zeros(seqs, dtype=torch.int32, device=DEV) for _ in range(2))
    return s


# ---- plain forms -----------------------------------------------------------------------------


def _ancestors(parent):
    """[seqs][rows][rows] truth values: row j is row i itself or on its way to the root; and the rows' depths."""
    rows = parent.shape[1]
    i = torch.arange(rows, device=parent.device)
    p = torch.where((parent >= 0) & (parent < i), parent, -1)
    m = (p[:, :, None] == i).float() + torch.eye(rows, device=parent.device)
    m = ((m @ m) > 0).float()  # paths of up to 2, 4, .. 64 steps
    m = ((m @ m) > 0).float()
    m = ((m @ m) > 0).float()
    m = ((m @ m) > 0).float()
    m = ((m @ m) > 0).float()
    m = (m @ m) > 0
    return m, m.sum(2) - 1, p.long()


def _live(s):
    return torch.arange(s.case["rows"], device=DEV) < s.count[:, None]


def _turn(x, cos, sin):
    h = cos.shape[-1]
    x0, x1 = x[..., :h], x[..., h:2 * h]
    return torch.cat((x0 * cos - x1 * sin, x0 * sin + x1 * cos, x[..., 2 * h:]), -1)


def _normed(x, gamma):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma


def _attn_tree(s):
    nh, nkv, d, rope = LAYOUTS[s.case["layout"]]
    seqs, rows, rep = s.case["seqs"], s.case["rows"], nh // nkv
    anc, depth, _ = _ancestors(s.parent)
    live = _live(s)
    at = s.pos[:, None] + depth
    # cos and sin of dead rows are never used: any row of the table
    table = s.rope[at.clamp(max=s.max_cells - 1)]
    cos, sin = table[:, :, None, :rope // 2], table[:, :, None, rope // 2:]
    q = s.qkv[:, :, :2 * nh * d].view(seqs, rows, nh, 2, d)[:, :, :, 0]
    k = s.qkv[:, :, 2 * nh * d:2 * nh * d + nkv * d].view(seqs, rows, nkv, d)
    v = s.qkv[:, :, 2 * nh * d + nkv * d:].view(seqs, rows, nkv, d)
    q = _turn(_normed(q, s.q_norm), cos, sin)
    # the cells a row leaves are rounded: their values in 64 bits, so that one next to a border falls where it belongs
    k = _turn(_normed(k.double(), s.k_norm.double()), cos.double(), sin.double()).float().half()
    here = live[:, :, None, None]
    s.kcells.copy_(torch.where(here, k, s.kcells))
    s.vcells.copy_(torch.where(here, v.half(), s.vcells))
    slot = s.slot.long()
    kc = torch.cat((s.kcache[slot], s.kcells), 1).float()                                      # [seqs][cells + rows][nkv][d]
    vc = torch.cat((s.vcache[slot].permute(0, 1, 4, 2, 3).reshape(seqs, s.max_cells, nkv, d), s.vcells), 1).float()
    qh = q.reshape(seqs, rows, nkv, rep, d).permute(0, 2, 1, 3, 4).reshape(seqs, nkv, rows * rep, d)
    score = qh @ kc.permute(0, 2, 3, 1).contiguous() / math.sqrt(d)
    c = torch.arange(s.max_cells, device=DEV)
    seen = (c < s.pos[:, None])[:, None, :].expand(seqs, rows, s.max_cells)
    tree = anc
    if s.case["window"]:
        seen = seen & ((c < s.case["sinks"]) | (at[:, :, None] - c < s.case["window"]))
        tree = tree & ((at < s.case["sinks"])[:, None, :] | (at[:, :, None] - at[:, None, :] < s.case["window"]))
    mask = torch.cat((seen, tree), 2)[:, None, :, None, :]
    score = score.view(seqs, nkv, rows, rep, -1).masked_fill(~mask, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(seqs, nkv, rows * rep, -1)
    o = (p @ vc.permute(0, 2, 1, 3).contiguous()).view(seqs, nkv, rows, rep, d).permute(0, 2, 1, 3, 4).reshape(seqs, rows, nh * d)
    s.out.copy_(torch.where(live[:, :, None], o, s.out))
    return {"out": s.out, "kcells": s.kcells, "vcells": s.vcells}


def _attn_keep(s):
    seqs, rows = s.path.shape
    j = torch.arange(rows, device=DEV)
    kept = (j < s.n_keep[:, None])[:, :, None, None]
    src = s.path.clamp(min=0).long()
    b = torch.arange(seqs, device=DEV)[:, None]
    slot, cell = s.slot.long()[:, None], (s.pos[:, None] + j).long()
    s.kcache[slot, cell] = torch.where(kept, s.kcells[b, src], s.kcache[slot, cell])
    old = s.vcache[slot, cell // 32, :, :, cell % 32]
    s.vcache[slot, cell // 32, :, :, cell % 32] = torch.where(kept, s.vcells[b, src], old)
    return {"kcache": s.kcache, "vcache": s.vcache}


def _dn_tree(s):
    hk, hv = DN_HEADS[s.case["heads"]]
    seqs, rows = s.case["seqs"], s.case["rows"]
    anc, depth, p0 = _ancestors(s.parent)
    live, slot = _live(s), s.slot.long()
    b = torch.arange(seqs, device=DEV)[:, None]
    cw = (2 * hk + hv) * DN_D
    # the taps' rows: the row, its parent, grandparent and the one above; above the root the ring, zeros before the start
    p1 = torch.where(p0 >= 0, p0[b, p0.clamp(min=0)], -1)
    p2 = torch.where(p1 >= 0, p0[b, p1.clamp(min=0)], -1)

    def tap(p, back):
        before = s.pos[:, None] + depth - back
        past = s.ring[slot[:, None], before.remainder(s.ring_slots).long(), :cw] * (before >= 0)[:, :, None]
        return torch.where((p >= 0)[:, :, None], s.x[b, p.clamp(min=0), :cw], past)

    c = tap(p2, 3) * s.conv1d[:, 0] + tap(p1, 2) * s.conv1d[:, 1] + tap(p0, 1) * s.conv1d[:, 2] + s.x[:, :, :cw] * s.conv1d[:, 3]
    c = c * torch.sigmoid(c)
    q, k, v = c[:, :, :hk * DN_D].view(seqs, rows, hk, DN_D), c[:, :, hk * DN_D:2 * hk * DN_D].view(seqs, rows, hk, DN_D), c[:, :, 2 * hk * DN_D:].view(seqs, rows, hv, DN_D)
    q = q * torch.rsqrt(q.square().sum(-1, keepdim=True) + EPS)
    k = k * torch.rsqrt(k.square().sum(-1, keepdim=True) + EPS)
    gates = s.x[:, :, cw + hv * DN_D:]
    logg = torch.log1p(torch.exp(gates[:, :, :hv] + s.dt_bias)) * s.a
    beta = torch.sigmoid(gates[:, :, hv:2 * hv])
    G = (anc.double() @ logg.double()).float()                                                # [seqs][rows][hv]
    head = torch.arange(hv, device=DEV) % hk
    qh, kh, vh = q[:, :, head].transpose(1, 2).contiguous(), k[:, :, head].transpose(1, 2).contiguous(), v.transpose(1, 2)  # [seqs][hv][rows][d]
    S = s.state[slot, s.plane.long()[slot]].transpose(2, 3).contiguous()                       # [seqs][hv][key][value]
    Gh, bh = G.transpose(1, 2)[..., None], beta.transpose(1, 2)[..., None]
    fall = torch.exp(Gh - Gh.transpose(2, 3)).masked_fill(~anc[:, None], 0.0)                  # [seqs][hv][rows][rows]
    kt = kh.transpose(2, 3).contiguous()
    own_row = torch.eye(rows, dtype=torch.bool, device=DEV)
    L = -(bh * fall * (kh @ kt)).masked_fill(own_row, 0.0).double()                            # nilpotent: no row is its own ancestor
    B = (bh * (vh - torch.exp(Gh) * (kh @ S))).double()
    B = B + L @ B  # (I - L)^-1 B as the product of I + L, I + L^2, .. I + L^32
    L = L @ L
    B = B + L @ B
    L = L @ L
    B = B + L @ B
    L = L @ L
    B = B + L @ B
    L = L @ L
    B = B + L @ B
    L = L @ L
    D = (B + L @ B).float()
    o = (torch.exp(Gh) * (qh @ S) + (fall * (qh @ kt)) @ D) / math.sqrt(DN_D)
    here = live[:, :, None, None]
    s.out.copy_(torch.where(here, o.transpose(1, 2), s.out))
    s.delta.copy_(torch.where(here, D.transpose(1, 2), s.delta))
    s.kn.copy_(torch.where(here, k, s.kn))
    s.decay.copy_(torch.where(live[:, :, None], G, s.decay))
    return {"out": s.out, "kn": s.kn, "delta": s.delta, "decay": s.decay}


def _dn_keep(s):
    hk, hv = DN_HEADS[s.case["heads"]]
    seqs, rows = s.path.shape
    b, slot = torch.arange(seqs, device=DEV)[:, None], s.slot.long()
    j = torch.arange(rows, device=DEV)
    kept = j < s.n_keep[:, None]
    src = s.path.clamp(min=0).long()
    G = s.decay[b, src]
    last = G.gather(1, (s.n_keep.long() - 1)[:, None, None].expand(seqs, 1, hv))               # [seqs][1][hv]
    w = torch.exp(last - G).masked_fill(~kept[:, :, None], 0.0)
    k = s.kn[b, src][:, :, torch.arange(hv, device=DEV) % hk].transpose(1, 2)                  # [seqs][hv][rows][key]
    D = (s.delta[b, src] * w[..., None]).permute(0, 2, 3, 1).contiguous()                      # [seqs][hv][value][rows]
    plane = s.plane.long()[slot]
    s.state[slot, 1 - plane] = torch.exp(last).transpose(1, 2)[..., None] * s.state[slot, plane] + D @ k
    cw = (2 * hk + hv) * DN_D
    # the last three kept rows, where there are as many
    t = s.n_keep[:, None] - TAPS + 1 + torch.arange(TAPS - 1, device=DEV)
    at = (s.pos[:, None] + t).remainder(s.ring_slots).long()
    new = s.x[b, s.path.gather(1, t.clamp(min=0).long()).clamp(min=0).long(), :cw]
    s.ring[slot[:, None], at, :cw] = torch.where((t >= 0)[:, :, None], new, s.ring[slot[:, None], at, :cw])
    return {"state": s.state, "ring": s.ring}


def _accept(s):
    seqs, rows, vocab = s.logits.shape
    live = _live(s)
    i = torch.arange(rows, device=DEV)
    x = torch.where(torch.isnan(s.logits), -math.inf, s.logits)
    first = torch.where(x == x.amax(2, keepdim=True), torch.arange(vocab, device=DEV), vocab).amin(2)
    s.best.copy_(torch.where(live, first, s.best))
    anc, depth, p = _ancestors(s.parent)
    wanted = s.best.gather(1, p.clamp(min=0))
    ok = live & (p >= 0) & (s.ids == wanted)
    # of a row's children that agree the lowest goes on
    rival = ok[:, None, :] & (p[:, :, None] == p[:, None, :]) & (i[None, :] < i[:, None])
    ok = (ok & ~rival.any(2)) | ((i == 0) & live)
    kept = ok & ~(anc & ~ok[:, None, :]).any(2)
    n = kept.sum(1)
    place = torch.where(kept, depth, rows)
    hit = place[:, None, :] == i[:, None]                                                      # [seqs][place][row]
    path = torch.where(hit.any(2), (hit * i).sum(2), -1)
    s.path.copy_(path)
    s.n_keep.copy_(n)
    s.next.copy_(s.best.gather(1, path.gather(1, (n - 1)[:, None])).squeeze(1))
    return {"best": s.best, "path": s.path, "n_keep": s.n_keep, "next": s.next}


# ---- the framework's calls -------------------------------------------------------------------

_handle = []


def _context():
    """One context of the process, as a program keeps one."""
    if not _handle:
        api = importlib.import_module("strix-halo-vulkan_amd").hip_api
        _handle.append((api, api.Context(torch.cuda.current_device())))
    return _handle[0]


def _call(s):
    """The call's kind and argument block, made once: what the device reads from call to call stands in its memory."""
    api, ctx = _context()
    at = lambda t: t.data_ptr()  # noqa: E731
    seqs, rows = s.case["seqs"], s.case["rows"]
    op = s.case["op"]
    if op == "attn_tree":
        nh, nkv, d, rope = LAYOUTS[s.case["layout"]]
        a = api.AttnTreeArgs(qkv=at(s.qkv), q_norm=at(s.q_norm), k_norm=at(s.k_norm), rope=at(s.rope), kcache=at(s.kcache), vcache=at(s.vcache),
                             kcells=at(s.kcells), vcells=at(s.vcells), partial=at(s.partial), out=at(s.out), pos=at(s.pos), slot=at(s.slot),
                             parent=at(s.parent), count=at(s.count), n_seq=seqs, rows=rows, n_head=nh, n_head_kv=nkv, head_dim=d, rope_dims=rope,
                             max_cells=s.max_cells, qkv_stride=s.width, n_splits=s.n_splits, window=s.case["window"], sinks=s.case["sinks"], eps=EPS)
        return api.OP_ATTN_TREE, a, {"out": s.out, "kcells": s.kcells, "vcells": s.vcells}
    if op == "attn_keep":
        nh, nkv, d, rope = LAYOUTS[s.case["layout"]]
        a = api.AttnKeepArgs(kcells=at(s.kcells), vcells=at(s.vcells), kcache=at(s.kcache), vcache=at(s.vcache), path=at(s.path), n_keep=at(s.n_keep),
                             pos=at(s.pos), slot=at(s.slot), n_seq=seqs, rows=rows, n_head_kv=nkv, head_dim=d, max_cells=s.max_cells)
        return api.OP_ATTN_KEEP, a, {"kcache": s.kcache, "vcache": s.vcache}
    if op == "dn_tree":
        hk, hv = DN_HEADS[s.case["heads"]]
        a = api.DnTreeArgs(x=at(s.x), ring=at(s.ring), conv1d=at(s.conv1d), a=at(s.a), dt_bias=at(s.dt_bias), state=at(s.state), out=at(s.out), kn=at(s.kn),
                           delta=at(s.delta), decay=at(s.decay), pos=at(s.pos), slot=at(s.slot), plane=at(s.plane), parent=at(s.parent), count=at(s.count),
                           n_seq=seqs, rows=rows, n_head_k=hk, n_head_v=hv, head_dim=DN_D, conv=TAPS, x_stride=s.width, ring_slots=s.ring_slots,
                           ring_stride=s.width, n_planes=2, qk_norm_max=0, eps=EPS)
        return api.OP_DN_TREE, a, {"out": s.out, "kn": s.kn, "delta": s.delta, "decay": s.decay}
    if op == "dn_keep":
        hk, hv = DN_HEADS[s.case["heads"]]
        a = api.DnKeepArgs(x=at(s.x), kn=at(s.kn), delta=at(s.delta), decay=at(s.decay), state=at(s.state), ring=at(s.ring), path=at(s.path),
                           n_keep=at(s.n_keep), pos=at(s.pos), slot=at(s.slot), plane=at(s.plane), n_seq=seqs, rows=rows, n_head_k=hk, n_head_v=hv,
                           head_dim=DN_D, conv=TAPS, x_stride=s.width, ring_slots=s.ring_slots, ring_stride=s.width, n_planes=2)
        return api.OP_DN_KEEP, a, {"state": s.state, "ring": s.ring}
    a = api.TreeAcceptArgs(logits=at(s.logits), ids=at(s.ids), parent=at(s.parent), count=at(s.count), best=at(s.best), path=at(s.path), n_keep=at(s.n_keep),
                           next=at(s.next), n_seq=seqs, rows=rows, n=s.case["vocab"], logits_stride=s.case["vocab"])
    return api.OP_TREE_ACCEPT, a, {"best": s.best, "path": s.path, "n_keep": s.n_keep, "next": s.next}


def run(s):
    if own:
        if s.calls is None:
            s.calls = _call(s)
        kind, args, out = s.calls
        _context()[1].enqueue(kind, args)
        return out
    return {"attn_tree": _attn_tree, "attn_keep": _attn_keep, "dn_tree": _dn_tree, "dn_keep": _dn_keep, "accept": _accept}[s.case["op"]](s)


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    seqs, rows = case["seqs"], case["rows"]
    # a ragged batch's sizes are drawn evenly: half of the rows, three quarters of the cells
    n = (rows + 1) / 2 if case["ragged"] else rows
    if case["op"] == "attn_tree":
        nh, nkv, d, rope = LAYOUTS[case["layout"]]
        cells = case["cells"] * (0.75 if case["ragged"] else 1.0)
        if case["window"]:
            cells = min(cells, case["window"] - 1 + case["sinks"])
        return {"bytes": seqs * (cells * nkv * d * 4 + n * ((nh + 2 * nkv) * d * 4 + nh * d * 4 + nkv * d * 4)), "flops": seqs * n * nh * 4.0 * d * (cells + 1 + n / 4)}
    keep = min(n, 5.0)  # a branch's usual length
    if case["op"] == "attn_keep":
        nh, nkv, d, rope = LAYOUTS[case["layout"]]
        return {"bytes": seqs * keep * nkv * d * 2 * 4, "flops": 0}
    if case["op"] in ("dn_tree", "dn_keep"):
        hk, hv = DN_HEADS[case["heads"]]
        state = hv * DN_D * DN_D * 4
        if case["op"] == "dn_keep":
            return {"bytes": seqs * (2 * state + keep * (hk + hv) * DN_D * 4 + 2 * 3 * (2 * hk + hv) * DN_D * 4), "flops": seqs * hv * DN_D * DN_D * 2 * (keep + 1)}
        row = (2 * hk + hv) * DN_D * 4 + (2 * hv + hk) * DN_D * 4
        return {"bytes": seqs * (state + n * row), "flops": seqs * n * hv * (4 * DN_D * DN_D + 6 * DN_D * n / 2)}
    return {"bytes": seqs * n * case["vocab"] * 4, "flops": 0}


# ---- the definitions in 64 bits --------------------------------------------------------------


def _chain(par, i):
    """Row i and the rows above it, the row first."""
    rows = []
    while i >= 0:
        rows.append(i)
        i = par[i] if 0 <= par[i] < i else -1
    return rows


def _exact_attn(s):
    nh, nkv, d, rope = LAYOUTS[s.case["layout"]]
    case, half = s.case, rope // 2
    out, kcells, vcells = torch.zeros_like(s.out, dtype=torch.float64), s.kcells.double(), s.vcells.double()
    table = s.rope.double()
    for b in range(case["seqs"]):
        par, n, pos, slot = s.parent[b].tolist(), int(s.count[b]), int(s.pos[b]), int(s.slot[b])
        rows = s.qkv[b, :n].double()
        chains = [_chain(par, i) for i in range(n)]
        at = torch.tensor([pos + len(c) - 1 for c in chains], device=DEV)

        def turned(x, gamma):
            x = x / torch.sqrt(torch.mean(x * x, -1, keepdim=True) + EPS) * gamma.double()
            y = x.clone()
            co, si = table[at][:, None, :half], table[at][:, None, half:]
            y[..., :half] = x[..., :half] * co - x[..., half:rope] * si
            y[..., half:rope] = x[..., :half] * si + x[..., half:rope] * co
            return y

        q = turned(rows[:, :2 * nh * d].reshape(n, nh, 2 * d)[:, :, :d], s.q_norm)
        k = turned(rows[:, 2 * nh * d:2 * nh * d + nkv * d].reshape(n, nkv, d), s.k_norm)
        kcells[b, :n] = k.float().half().double()
        vcells[b, :n] = rows[:, 2 * nh * d + nkv * d:].reshape(n, nkv, d).float().half().double()
        seen = torch.zeros(n, pos + n, dtype=torch.bool, device=DEV)
        seen[:, :pos] = True
        for i, c in enumerate(chains):
            seen[i, [pos + j for j in c]] = True
        if case["window"]:
            where = torch.cat((torch.arange(pos, device=DEV), at))
            seen &= (where < case["sinks"])[None, :] | (at[:, None] - where[None, :] < case["window"])
        kc = s.kcache[slot, :pos]
        vc = s.vcache[slot].permute(0, 3, 1, 2).reshape(s.max_cells, nkv, d)[:pos]
        for h in range(nkv):
            keys = torch.cat((kc[:, h].double(), kcells[b, :n, h]))
            values = torch.cat((vc[:, h].double(), vcells[b, :n, h]))
            for e in range(h * (nh // nkv), (h + 1) * (nh // nkv)):
                w = (q[:, e] @ keys.T) * d ** -0.5
                w = torch.where(seen, w, -math.inf)
                w = torch.exp(w - w.max(1, keepdim=True).values)
                out[b, :n, e * d:(e + 1) * d] = (w @ values) / w.sum(1, keepdim=True)
    return {"out": out, "kcells": kcells, "vcells": vcells}


def _exact_dn(s):
    hk, hv = DN_HEADS[s.case["heads"]]
    out, delta, kn, decay = (torch.zeros_like(t, dtype=torch.float64) for t in (s.out, s.delta, s.kn, s.decay))
    cw = (2 * hk + hv) * DN_D
    taps, of = s.conv1d.double(), torch.arange(hv, device=DEV) % hk
    for b in range(s.case["seqs"]):
        par, n, pos, slot = s.parent[b].tolist(), int(s.count[b]), int(s.pos[b]), int(s.slot[b])
        x, ring = s.x[b, :n].double(), s.ring[slot].double()
        zero = torch.zeros(cw, dtype=torch.float64, device=DEV)
        S0 = s.state[slot, int(s.plane[slot])].double()  # [hv][value][key]
        states = []
        for i in range(n):
            chain = _chain(par, i)
            line = [x[c, :cw] for c in chain[:TAPS]]
            back = pos
            while len(line) < TAPS:
                back -= 1
                line.append(ring[back % s.ring_slots, :cw] if back >= 0 else zero)
            c = sum(line[t] * taps[:, TAPS - 1 - t] for t in range(TAPS))
            c = c / (1 + torch.exp(-c))
            q, k, v = c[:hk * DN_D].view(hk, DN_D), c[hk * DN_D:2 * hk * DN_D].view(hk, DN_D), c[2 * hk * DN_D:].view(hv, DN_D)
            q, k = q / torch.sqrt((q * q).sum(1, keepdim=True) + EPS), k / torch.sqrt((k * k).sum(1, keepdim=True) + EPS)
            log_g = torch.log1p(torch.exp(x[i, cw + hv * DN_D:cw + hv * DN_D + hv] + s.dt_bias.double())) * s.a.double()
            write = 1 / (1 + torch.exp(-x[i, cw + hv * DN_D + hv:cw + hv * DN_D + 2 * hv]))
            S = (states[chain[1]] if len(chain) > 1 else S0) * torch.exp(log_g)[:, None, None]
            dl = write[:, None] * (v - (S * k[of][:, None, :]).sum(2))
            S = S + dl[:, :, None] * k[of][:, None, :]
            states.append(S)
            out[b, i], delta[b, i], kn[b, i] = (S * q[of][:, None, :]).sum(2) / DN_D ** 0.5, dl, k
            decay[b, i] = log_g + (decay[b, chain[1]] if len(chain) > 1 else 0)
    return {"out": out, "kn": kn, "delta": delta, "decay": decay}


def _exact_dn_keep(s):
    hk, hv = DN_HEADS[s.case["heads"]]
    state, ring = s.state.double(), s.ring.double()
    of = torch.arange(hv, device=DEV) % hk
    cw = (2 * hk + hv) * DN_D
    for b in range(s.case["seqs"]):
        n, slot, pos = int(s.n_keep[b]), int(s.slot[b]), int(s.pos[b])
        path, plane = s.path[b, :n].tolist(), int(s.plane[slot])
        S, fell = state[slot, plane].clone(), torch.zeros(hv, dtype=torch.float64, device=DEV)
        for r in path:  # the rule row after row: what is there decays, the row's product is added
            d = s.decay[b, r].double()
            S = S * torch.exp(d - fell)[:, None, None] + s.delta[b, r].double()[:, :, None] * s.kn[b, r].double()[of][:, None, :]
            fell = d
        state[slot, 1 - plane] = S
        for j in range(max(0, n - TAPS + 1), n):
            ring[slot, (pos + j) % s.ring_slots, :cw] = s.x[b, path[j], :cw].double()
    return {"state": state, "ring": ring}


def _exact_keep(s):
    kc, vc = s.kcache.double(), s.vcache.double()
    for b in range(s.case["seqs"]):
        slot, pos = int(s.slot[b]), int(s.pos[b])
        for j in range(int(s.n_keep[b])):
            r, c = int(s.path[b, j]), pos + j
            kc[slot, c] = s.kcells[b, r].double()
            vc[slot, c // 32, :, :, c % 32] = s.vcells[b, r].double()
    return {"kcache": kc, "vcache": vc}


def _exact_accept(s):
    logits, ids, par = s.logits.cpu().numpy(), s.ids.tolist(), s.parent.tolist()
    seqs, rows = len(ids), len(ids[0])
    best, path, keep, nxt = np.zeros((seqs, rows), np.int32), np.full((seqs, rows), -1, np.int32), np.zeros(seqs, np.int32), np.zeros(seqs, np.int32)
    for b in range(seqs):
        n = int(s.count[b])
        best[b, :n] = logits[b, :n].argmax(1)
        at, m = 0, 0
        while at >= 0:
            path[b, m], m = at, m + 1
            at = next((i for i in range(at + 1, n) if par[b][i] == at and ids[b][i] == best[b, at]), -1)
        keep[b], nxt[b] = m, best[b, path[b, m - 1]]
    return {"best": best, "path": path, "n_keep": keep, "next": nxt}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn_tree": _exact_attn, "attn_keep": _exact_keep, "dn_tree": _exact_dn, "dn_keep": _exact_dn_keep, "accept": _exact_accept}[case["op"]](s)
