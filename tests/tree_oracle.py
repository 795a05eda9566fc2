"""Plain float64 forms of the operators that verify a tree of drafted tokens, one sequence at a time, and inputs for them."""
import numpy as np


def chain(parent, i):
    """Row i and the rows it stands on, itself first; a parent that is no lower row ends the way."""
    way = []
    while i >= 0:
        way.append(i)
        i = parent[i] if 0 <= parent[i] < i else -1
    return way


def tree(rng, rows, kind="mixed"):
    """Parents of a tree's rows."""
    if kind == "chain":
        return np.arange(-1, rows - 1).astype(np.int32)
    if kind == "star":
        return np.where(np.arange(rows) == 0, -1, 0).astype(np.int32)
    if kind == "roots":  # parents that are none: themselves, higher rows, far outside
        return rng.choice([-1, -7, rows - 1, rows + 5, 2**31 - 1, 0], rows).astype(np.int32)
    if kind == "wide":  # one row a level that the next level's rows stand on
        return np.maximum(0, (np.arange(rows) - 1) // 4 * 4 - rng.integers(0, 4, rows) % 4 - (np.arange(rows) == 0)).astype(np.int32)
    return np.array([-1] + [int(rng.integers(max(0, i - 6), i)) for i in range(1, rows)], np.int32)


def rope_table(cells, dims, base=1e7):
    if dims == 0:
        return np.zeros((cells, 1), np.float32)
    theta = np.arange(cells, dtype=np.float64)[:, None] * base ** (-2.0 / dims * np.arange(dims // 2))
    return np.concatenate([np.cos(theta), np.sin(theta)], 1).astype(np.float32)


def norm_rope(x, gamma, table, at, dims, eps):
    """x [rows][heads][d] float64"""
    x = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * gamma.astype(np.float64)
    h = dims // 2
    c, s = table[at][:, None, :h].astype(np.float64), table[at][:, None, h:2 * h].astype(np.float64)
    y = x.copy()
    y[..., :h] = x[..., :h] * c - x[..., h:dims] * s
    y[..., h:dims] = x[..., :h] * s + x[..., h:dims] * c
    return y


def attn_tree(qkv, q_norm, k_norm, table, kc, vc, pos, parent, n, nh, nkv, d, dims, eps, window=0, sinks=0):
    """out [n][nh*d] float64, the rows' cells as halves [n][nkv][d]; kc, vc [cells][nkv][d] halves."""
    way = [chain(parent, i) for i in range(n)]
    at = np.array([pos + len(w) - 1 for w in way], np.int64)
    rows = qkv[:n].astype(np.float64)
    q = norm_rope(rows[:, :2 * nh * d].reshape(n, nh, 2 * d)[:, :, :d], q_norm, table, at, dims, eps)
    k = norm_rope(rows[:, 2 * nh * d:2 * nh * d + nkv * d].reshape(n, nkv, d), k_norm, table, at, dims, eps)
    with np.errstate(over="ignore"):
        k = k.astype(np.float32).astype(np.float16)
        v = qkv[:n, 2 * nh * d + nkv * d:2 * nh * d + 2 * nkv * d].reshape(n, nkv, d).astype(np.float16)
    out = np.zeros((n, nh, d))
    rep = nh // nkv
    with np.errstate(invalid="ignore", over="ignore"):
        for i in range(n):
            cells = [c for c in range(pos) if window == 0 or c < sinks or at[i] - c < window]
            mates = [j for j in way[i] if window == 0 or at[j] < sinks or at[i] - at[j] < window]
            keys = np.concatenate([kc[cells], k[mates]]).astype(np.float64)
            values = np.concatenate([vc[cells], v[mates]]).astype(np.float64)
            for h in range(nh):
                w = keys[:, h // rep] @ q[i, h] / np.sqrt(d)
                w = np.exp(w - w.max())
                out[i, h] = w @ values[:, h // rep] / w.sum()
    return out.reshape(n, nh * d), k, v


def dn_tree(x, ring, conv1d, a, dt_bias, S0, pos, parent, n, hk, hv, d, eps, norm_max=0):
    """S0 [hv][value][key]; out, delta [n][hv][d], kn [n][hk][d], decay [n][hv], the rows' states."""
    cw = (2 * hk + hv) * d
    x, ring, taps = x[:n].astype(np.float64), ring.astype(np.float64), conv1d.astype(np.float64)
    out, delta, kn, decay, states = np.zeros((n, hv, d)), np.zeros((n, hv, d)), np.zeros((n, hk, d)), np.zeros((n, hv)), []
    of = np.arange(hv) % hk
    for i in range(n):
        way = chain(parent, i)
        c = np.zeros(cw)
        for t in range(4):  # t steps up
            p = pos + len(way) - 1 - t
            row = x[way[t], :cw] if t < len(way) else ring[p % len(ring), :cw] if p >= 0 else 0.0
            c = c + row * taps[:, 3 - t]
        c = c / (1 + np.exp(-c))
        q, k, v = c[:hk * d].reshape(hk, d), c[hk * d:2 * hk * d].reshape(hk, d), c[2 * hk * d:].reshape(hv, d)
        nrm = (lambda u: np.maximum(np.sqrt((u * u).sum(1, keepdims=True)), eps)) if norm_max else (lambda u: np.sqrt((u * u).sum(1, keepdims=True) + eps))
        q, k = q / nrm(q), k / nrm(k)
        z = x[i, cw + hv * d:cw + hv * d + hv] + dt_bias
        log_g = np.where(z > 20, z, np.log1p(np.exp(np.minimum(z, 20)))) * a
        beta = 1 / (1 + np.exp(-x[i, cw + hv * d + hv:cw + hv * d + 2 * hv]))
        S = (states[way[1]] if len(way) > 1 else S0.astype(np.float64)) * np.exp(log_g)[:, None, None]
        dl = beta[:, None] * (v - np.einsum("hvk,hk->hv", S, k[of]))
        S = S + dl[:, :, None] * k[of][:, None, :]
        states.append(S)
        out[i], delta[i], kn[i] = np.einsum("hvk,hk->hv", S, q[of]) / np.sqrt(d), dl, k
        decay[i] = log_g + (decay[way[1]] if len(way) > 1 else 0)
    return out, kn, delta, decay, states


def accept(best, ids, parent, n):
    """The branch: rows from row 0 on, each the lowest child whose token its parent's row wants."""
    if n == 0:
        return [], -1
    path = [0]
    while True:
        at = path[-1]
        to = [i for i in range(at + 1, n) if parent[i] == at and ids[i] == best[at]]
        if not to:
            return path, int(best[at])
        path.append(to[0])


def first_max(row):
    row = np.where(np.isnan(row), -np.inf, row)
    return int(np.argmax(row))
