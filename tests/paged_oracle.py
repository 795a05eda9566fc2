"""Plain forms of the operators of a serving batch over a paged cache: the plan request by request, attention and log probabilities in float64."""
import numpy as np

import tree_oracle as T


def plan(rows, pos, table, held, free, n_free, shared, page, max_pages, max_rows, with_base):
    """All state as it is afterwards (copies), and start, row_seq, row_pos, row_cell, base."""
    table, held, free, pos = table.copy(), list(map(int, held)), free.copy(), list(map(int, pos))
    n_pages, top, n = len(free), int(n_free), len(rows)
    base = list(pos)
    ok, want = [], []
    for s in range(n):
        ends = rows[s] < 0
        w = 0 if ends else -(-(pos[s] + int(rows[s])) // page)
        ok.append(ends or (pos[s] >= 0 and w <= max_pages))
        want.append(w)
        if not ok[s]:
            continue
        keep = max(w, min(int(shared[s]), held[s]) if shared is not None else 0)
        for e in range(keep, held[s]):
            free[top] = table[s, e]
            top += 1
        held[s] = 0 if ends else min(held[s], keep)
    avail, wished, asked, total = top, 0, 0, 0
    start, maps = [0], []
    for s in range(n):
        if ok[s] and rows[s] >= 0:
            need = max(0, want[s] - held[s])
            wished += need
            asked += int(rows[s])
            if (need == 0 or wished <= avail) and asked <= max_rows:
                for _ in range(need):
                    top -= 1
                    table[s, held[s]] = free[top]
                    held[s] += 1
                for i in range(int(rows[s])):
                    p = pos[s] + i
                    at = int(table[s, p // page])
                    maps.append((s, p, at * page + p % page if 0 <= at < n_pages else -1))
                total += int(rows[s])
                if with_base:
                    pos[s] += int(rows[s])
        elif ok[s] and with_base:
            pos[s] = 0
        start.append(total)
    return dict(table=table, held=np.array(held), free=free, n_free=top, pos=np.array(pos), start=np.array(start), maps=np.array(maps, np.int64).reshape(-1, 3), base=np.array(base))


def attention(qkv, q_norm, k_norm, table, rope, kp, vp, start, row_pos, row_cell, nh, nkv, d, dims, eps, window=0, sinks=0):
    """kp, vp [n_pages][page][nkv][d] halves, table the sequences' pages.  out [rows][nh*d] float64 and which rows have one; the pages as the rows leave them."""
    n_pages, page = kp.shape[:2]
    n_seq, max_pages = table.shape
    rows = len(row_pos)
    kp, vp = kp.copy(), vp.copy()
    kf, vf = kp.reshape(-1, nkv, d), vp.reshape(-1, nkv, d)
    x = qkv.astype(np.float64)
    live = [r for r in range(min(int(start[n_seq]), rows)) if 0 <= row_cell[r] < n_pages * page and 0 <= row_pos[r] < max_pages * page]
    if live:
        at = row_pos[live].astype(np.int64)
        k = T.norm_rope(x[live][:, 2 * nh * d:2 * nh * d + nkv * d].reshape(-1, nkv, d), k_norm, rope, at, dims, eps)
        with np.errstate(over="ignore"):
            kf[row_cell[live]] = k.astype(np.float32).astype(np.float16)
            vf[row_cell[live]] = qkv[live][:, 2 * nh * d + nkv * d:2 * nh * d + 2 * nkv * d].reshape(-1, nkv, d).astype(np.float16)
    out, there = np.zeros((rows, nh, d)), np.zeros(rows, bool)
    rep = nh // nkv
    for s in range(n_seq):
        a, b = int(start[s]), int(start[s + 1])
        if not (0 <= a < b <= rows) or row_pos[a] < 0 or int(row_pos[a]) + b - a > max_pages * page:
            continue
        there[a:b] = True
        at = int(row_pos[a]) + np.arange(b - a)
        q = T.norm_rope(x[a:b, :2 * nh * d].reshape(b - a, nh, 2 * d)[:, :, :d], q_norm, rope, at, dims, eps)
        c = np.arange(at[-1] + 1)
        pages = table[s, c // page]
        c = c[(pages >= 0) & (pages < n_pages)]
        cell = table[s, c // page].astype(np.int64) * page + c % page
        keys, values = kf[cell].astype(np.float64), vf[cell].astype(np.float64)
        for i in range(b - a):
            seen = c <= at[i]
            if window:
                seen &= (c < sinks) | (at[i] - c < window)
            if not seen.any():
                continue
            ks, vs = keys[seen], values[seen]
            with np.errstate(invalid="ignore", over="ignore"):
                for h in range(nh):
                    w = ks[:, h // rep] @ q[i, h] / np.sqrt(d)
                    w = np.exp(w - w.max())
                    out[a + i, h] = w @ vs[:, h // rep] / w.sum()
    return out.reshape(rows, nh * d), there, kp, vp


def logprobs(logits, ids, top):
    """logprob, entropy, top_ids, top_logprobs of each row."""
    x = logits.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = np.max(np.where(np.isnan(x), -np.inf, x), 1, keepdims=True)
        off = x - m
        w = np.exp(off)
        z = w.sum(1, keepdims=True)
        lp = off - np.log(z)
        entropy = np.log(z[:, 0]) - np.where(w > 0, w * off, np.where(np.isnan(w), np.nan, 0)).sum(1) / z[:, 0]
    bad = np.isnan(z) | np.isinf(m)
    lp, entropy = np.where(bad, np.nan, lp), np.where(bad[:, 0], np.nan, entropy)
    n = x.shape[1]
    given = np.array([lp[r, i] if 0 <= i < n else np.nan for r, i in enumerate(ids)])
    top_ids, top_lp = np.full((len(x), top), -1), np.full((len(x), top), -np.inf)
    for r in range(len(x)):
        fine = np.flatnonzero(~np.isnan(x[r]))
        best = fine[np.lexsort((fine, -x[r, fine]))][:top]
        top_ids[r, :len(best)], top_lp[r, :len(best)] = best, lp[r, best]
    return given, entropy, top_ids, top_lp
