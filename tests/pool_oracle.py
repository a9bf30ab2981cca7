"""Plain forms of the serving operators in python integers and 64-bit floats, for the tests."""
import math

import numpy as np


def plan(page, n_pages, cached, new, table, free, n_free, max_tokens):
    """(status, table, n_free, cu_q, kv_len, slots, req_of, positions) of kg_pool_plan_dev."""
    n, width = len(cached), table.shape[1]
    none = -np.ones(max_tokens, np.int64)
    fail = lambda code: (code, table, n_free, np.zeros(n + 1, int), np.zeros(n, int), none, none, none)  # noqa: E731
    if any(c < 0 or a < 0 or c + a >= 2**31 or -(-(c + a) // page) > width for c, a in zip(cached, new)):
        return fail(-1)
    if sum(new) > max_tokens or not 0 <= n_free <= n_pages:
        return fail(-1)
    if any(a and c % page and not 0 <= table[r][c // page] < n_pages for r, (c, a) in enumerate(zip(cached, new))):
        return fail(-1)
    grow = [-(-(c + a) // page) - -(-c // page) for c, a in zip(cached, new)]
    if sum(grow) > n_free:
        return fail(-2)
    if any(not 0 <= x < n_pages for x in free[n_free - sum(grow):n_free]):
        return fail(-1)
    table = table.copy()
    slots, req, pos = none.copy(), none.copy(), none.copy()
    t = 0
    for r, (c, a) in enumerate(zip(cached, new)):
        for j in range(grow[r]):
            n_free -= 1
            table[r][-(-c // page) + j] = free[n_free]
        for x in range(c, c + a):
            slots[t], req[t], pos[t] = table[r][x // page] * page + x % page, r, x
            t += 1
    cu = np.concatenate([[0], np.cumsum(np.asarray(new, int))]).astype(int)
    return 0, table, n_free, cu, np.asarray(cached, int) + np.asarray(new, int), slots, req, pos


def attend(q, k, v, cu, kv, scale, causal):
    """Attention of ragged rows in 64 bits. q [rows][heads][d]; k, v: per request [kv][kv heads][d].
    Returns (out, touched rows, weight sums of |v| per element, score error scale per row and head)."""
    out = np.zeros(q.shape)
    mag = np.zeros(q.shape)
    sco = np.zeros(q.shape[:2])
    mine = np.zeros(q.shape[0], bool)
    heads = q.shape[1]
    for r in range(len(kv)):
        a, b, n = cu[r], cu[r + 1], kv[r]
        mine[a:b] = True
        if a == b or n == 0:
            continue
        group = heads // k[r].shape[1]
        last = np.arange(a, b) - b + n if causal else np.full(b - a, n - 1)
        keep = np.arange(n)[None, :] <= last[:, None]
        for h in range(heads):
            kk, vv = k[r][:n, h // group], v[r][:n, h // group]
            s = np.where(keep, q[a:b, h] @ kk.T * scale, -np.inf)
            top = s.max(-1, keepdims=True)
            w = np.exp(s - np.where(np.isfinite(top), top, 0.0))
            tot = w.sum(-1, keepdims=True)
            w = np.divide(w, tot, out=np.zeros_like(w), where=tot > 0)
            out[a:b, h] = w @ vv
            mag[a:b, h] = w @ np.abs(vv)
            sco[a:b, h] = (np.abs(q[a:b, h]) @ np.abs(kk).T * abs(scale)).max(-1)
    return out, mine, mag, sco


def sample(row, temp, top_k, top_p, min_p, u):
    """The token of one row of logits (python floats), from the definition; -1 if none is left."""
    row = [float(x) for x in row]
    live = [j for j, x in enumerate(row) if x == x and x != -math.inf]
    if not live:
        return -1
    order = sorted(live, key=lambda j: (-row[j], j))
    if not temp > 0:
        return order[0]
    top = row[order[0]]
    w = {j: 1.0 if row[j] == top else 0.0 if math.isinf(top) else math.exp((row[j] - top) / temp) for j in order}
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        want, run, cut = max(top_p, 0.0) * math.fsum(w[j] for j in order), 0.0, []
        for j in order:
            if cut and run >= want:
                break
            cut.append(j)
            run = math.fsum([run, w[j]])
        order = cut
    order = sorted(j for j in order if w[j] >= min(min_p, 1.0)) if min_p > 0 else sorted(order)
    order = [j for j in order if w[j] > 2.0 ** -45]
    total, run = math.fsum(w[j] for j in order), 0.0
    u = min(max(u, 0.0), 1.0)
    for j in order:
        run += w[j]
        if run > u * total:
            return j
    return order[-1]
