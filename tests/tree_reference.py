"""Plain 64-bit forms of the tree-step operators, for the tests: numpy, one
sequence, head and node at a time, straight from the definitions."""

import numpy as np


def chain(batch, nodes):
    return np.tile(np.arange(-1, nodes - 1, dtype=np.int32), (batch, 1))


def random_trees(rng, batch, nodes, forest=False):
    """Parents before their nodes; with `forest` some nodes are roots too."""
    out = np.full((batch, nodes), -1, np.int32)
    for b in range(batch):
        for t in range(1, nodes):
            out[b, t] = rng.integers(max(0, t // 3 - 1), t)
            if forest and rng.random() < 0.2:
                out[b, t] = -1
    return out


def ancestors(parents, t):
    """Node t and its ancestors, or None where a parent does not come before
    its node."""
    line = []
    while t >= 0:
        line.append(t)
        up = int(parents[t])
        if up < -1 or up >= t:
            return None
        t = up
    return line


def tree_attention(q, keys, values, tree_k, tree_v, parents, count, out):
    """One sequence: q [Hq, T, D], history keys / values [Hkv, n, D] and tree
    rows [Hkv, T, D] as the pages hold them.  Fills rows t < count of `out`
    [Hq, T, D] (float64).  Keys that a row does not see take no part."""
    hq, T, d = q.shape
    group = hq // keys.shape[0]
    n = keys.shape[1]
    q = q.astype(np.float64)
    for t in range(min(count, T)):
        line = ancestors(parents, t)
        for h in range(hq):
            if line is None:
                out[h, t] = np.nan
                continue
            line = sorted(line)
            k = np.concatenate([keys[h // group], tree_k[h // group][line]]).astype(np.float64)
            v = np.concatenate([values[h // group], tree_v[h // group][line]]).astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore"):
                s = k @ q[h, t] / np.sqrt(d)
                # exp(s - max) with equal values giving 1, the library's rule
                m = s.max() if not np.isnan(s).any() else np.nan
                p = np.where(s == m, 1.0, np.exp(s - m))
                out[h, t] = np.nan if m == -np.inf else (p @ v) / p.sum()
    assert n == keys.shape[1]
    return out


def verify(target, draft, tokens, parents, count, uniforms, bonus):
    """One sequence: target, draft [T, V] (draft None: certain drafts).
    Returns (path, next token)."""
    if count == 0:
        return [], -1
    V = target.shape[1]
    n, path = 0, [0]
    while True:
        w, mass = np.maximum(target[n].astype(np.float64), 0.0), 1.0
        q = None if draft is None else draft[n].astype(np.float64)
        moved = False
        for c in range(n + 1, count):
            x = int(tokens[c])
            if parents[c] != n or not 0 <= x < V:
                continue
            if float(uniforms[c]) * (mass if q is None else q[x]) < w[x]:
                n, moved = c, True
                path.append(c)
                break
            if q is None:
                mass -= w[x]
                w[x] = 0.0
            else:
                w = np.maximum(w - q, 0.0)
                if w.sum() > 0:
                    w = w / w.sum()
        if not moved:
            break
    if not w.sum() > 0:
        w = np.maximum(target[n].astype(np.float64), 0.0)
    if not w.sum() > 0:
        return path, -1
    sums = np.cumsum(w)
    after = int(np.searchsorted(sums, float(bonus) * sums[-1], side="right"))
    return path, min(after, int(np.flatnonzero(w > 0)[-1]))
