"""The operators for several hypotheses of one prompt by lists and in float64, from their definitions."""
import numpy as np

U = 2.0 ** -24                    # half a step of f32, relative


def pages_of(n, page):
    return -(-n // page)


def fork(table, length, parent, rows, n_pages, page):
    """(table, pos, len, status, copies): copies [(source, target, positions)]."""
    n_seq, width = table.shape
    pos = [min(max(int(length[p]), 0), width * page) if 0 <= p < n_seq else 0 for p in parent]
    held = [[int(x) for x in table[p][:pages_of(m, page)]] if m else [] for p, m in zip(parent, pos)]
    ok = lambda p: 0 <= p < n_pages  # noqa: E731
    holders = {}
    for j, row in enumerate(held):
        for s, p in enumerate(row):
            if ok(p):
                holders.setdefault(p, []).append((min(page, pos[j] - s * page), j))
    used = len(holders)
    n = len(parent)
    empty = (np.full((n, width), -1), np.zeros(n, int), np.zeros(n, int))
    wide = sum(pages_of(m + r, page) > width for m, r in zip(pos, rows))
    if wide:
        return *empty, (-wide, used), []
    free = [p for p in range(n_pages) if p not in holders]
    want, copies, out = 0, [], []
    take = iter(free + [None] * sum(pages_of(m + r, page) + 1 for m, r in zip(pos, rows)))
    for j, row in enumerate(held):
        row, part = list(row), pos[j] % page
        if part and rows[j] > 0 and ok(row[-1]):
            most = max(f for f, _ in holders[row[-1]])
            stays = [i for f, i in holders[row[-1]] if f == most and f < page and rows[i] > 0 and held[i][-1] == row[-1] and pos[i] % page == f]
            if not stays or min(stays) != j:
                new = next(take)
                want += 1
                copies.append((row[-1], new, part))
                row[-1] = new
        more = pages_of(pos[j] + rows[j], page) - len(row)
        row += [next(take) for _ in range(more)]
        want += more
        out.append(row + [-1] * (width - len(row)))
    if want > len(free):
        return *empty, (want - len(free), used), []
    return np.array(out).reshape(n, width), np.array(pos), np.array(pos) + rows, (0, used + want), copies


def compact(table, length, n_pages, page):
    """(table, status, moves)."""
    n_seq, width = table.shape
    held = [[int(x) for x in row[:pages_of(min(max(int(m), 0), width * page), page)]] for row, m in zip(table, length)]
    used = sorted({p for row in held for p in row if 0 <= p < n_pages})
    n = len(used)
    moved = dict(zip([p for p in used if p >= n], sorted(set(range(n)) - set(used))))
    out = [[moved.get(p, p) for p in row] + [-1] * (width - len(row)) for row in held]
    return np.array(out).reshape(n_seq, width), (len(moved), n), moved


def gather(pool, row, n, page):
    """Positions 0 .. n of a sequence, [n][heads][dim], and which of them exist."""
    n_pages, heads, _, dim = pool.shape
    out, there = np.zeros((n, heads, dim)), np.zeros(n, bool)
    for s in range(min(pages_of(n, page), len(row))):
        if 0 <= row[s] < n_pages:
            m = min(page, n - s * page)
            out[s * page:s * page + m] = pool[row[s], :, :m].transpose(1, 0, 2)
            there[s * page:s * page + m] = True
    return out, there


def attend(q, k, v, seen, scale, terms):
    """q [n][G * heads][dim] over k, v [positions][heads][dim]; seen [n][positions].  Returns (out, bound): bound on what
    f32 arithmetic with weights that are off by `terms` of themselves may lose."""
    n, hq, dim = q.shape
    heads = k.shape[1]
    g = hq // heads
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(n):
        at = seen[i]
        if not at.any():
            continue
        for h in range(hq):
            kk, vv = k[at, h // g], v[at, h // g]
            s = scale * (kk @ q[i, h])
            e = np.exp(s - s.max())
            w = e / e.sum()
            out[i, h] = w @ vv
            # the score: dim products, three at most of each, summed in any order; the factor and its product, the difference
            # from the maximum (held back by up to 2^8: five steps of ln 2 x 8), the exponential's unit in the last place
            size = abs(scale) * (np.abs(kk) @ np.abs(q[i, h]))
            score = (3 * dim + 8) * U * size + 4 * U * np.abs(s) + 2 * U * (np.abs(s - s.max()) + 6) + 2 * U
            # a weight twice (the sum has it too); the sums: one rounding a product and position at most, the rescalings, the parts
            bound[i, h] = (2 * (score.max() + terms) + (3 * at.sum() + 200) * U) * (w @ np.abs(vv))
    return out, bound


def logprobs(x, targets, k):
    """(logp, entropy, ids, top) of finite or -infinite rows."""
    x = x.astype(np.float64)
    m = x.max(1, keepdims=True)
    e = np.exp(x - m)
    # the sum without the largest term: exact next to a probability of 1
    first = x.argmax(1)
    rest = e.copy()
    rest[np.arange(len(x)), first] = 0
    tail = np.log1p(rest.sum(1))
    lp = x - m - tail[:, None]
    with np.errstate(invalid="ignore"):
        entropy = -np.where(e > 0, np.exp(lp) * lp, 0).sum(1)
    ids = np.argsort(-x, axis=1, kind="stable")[:, :k]
    return lp[np.arange(len(x)), targets], entropy, ids, np.take_along_axis(lp, ids, 1), m[:, 0], first
