"""Plain 64-bit forms of the serving operators, in numpy, for the tests. Each follows the operator's definition one row at
a time; nothing here is fast."""
import numpy as np


def norm_rope(x, w, eps, table):
    """x [..., D], w [D], table [D] = cos | sin halves: RMSNorm, then the rotation of pairs (i, i + D/2)."""
    D = x.shape[-1]
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    c, s = table[:D // 2].astype(np.float64), table[D // 2:].astype(np.float64)
    a, b = y[..., :D // 2], y[..., D // 2:]
    return np.concatenate([a * c - b * s, a * s + b * c], -1), np.concatenate([np.abs(a) + np.abs(b)] * 2, -1)


def softmax(x):
    m = x.max()
    if not np.isfinite(m):
        return None
    e = np.exp(x - m)
    return e / e.sum()


def verify(logits, row_off, draft, q, temp, u):
    """logits [rows, V] float64 (NaN already -inf): (n_acc, next, p) as the header describes."""
    R = len(row_off) - 1
    V = logits.shape[1]
    n_acc, nxt, shown = [], [], np.zeros(max(len(draft), 1))
    for r in range(R):
        lo, k, i, token = row_off[r], row_off[r + 1] - row_off[r] - 1, 0, None
        while token is None:
            row = logits[lo + i]
            greedy = not temp[r] > 0
            some = np.isfinite(row.max())
            if greedy:
                p = np.zeros(V)
                if some:
                    p[int(np.argmax(row))] = 1.0
            else:
                p = softmax(row / np.float64(temp[r])) if some else np.zeros(V)
            left = p
            if i < k:
                j = lo - r + i
                d = int(draft[j])
                pd = p[d] if 0 <= d < V else 0.0
                shown[j] = pd
                if greedy:
                    keep = pd == 1.0
                else:
                    qd = 0.0 if not 0 <= d < V else 1.0 if q is None else float(q[j, d])
                    keep = qd > 0 and u[lo + i] * qd < pd
                if keep:
                    i += 1
                    continue
                if not greedy:
                    if q is None:
                        left = p.copy()
                        if 0 <= d < V:
                            left[d] = 0.0
                    else:
                        left = np.maximum(p - q[j].astype(np.float64), 0.0)
                    if not left.sum() > 0:
                        left = p
            if not some:
                token = -1
            elif greedy:
                token = int(np.argmax(row))
            else:
                run = np.cumsum(left)
                at = u[lo + i + (1 if i < k else 0)] * run[-1]
                hit = np.nonzero((run >= at) & (left > 0))[0]
                token = int(hit[0]) if len(hit) else int(np.nonzero(left > 0)[0][-1])
        n_acc.append(i)
        nxt.append(token)
    return np.array(n_acc), np.array(nxt), shown
