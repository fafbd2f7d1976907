"""Verification of drafted tokens in 64 bits, each residual made from the one before it, for the tests of wd_verify_drafts."""
import numpy as np


def softmax(x, t):
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore"):
        z = np.where(np.isneginf(x), -np.inf, (x - x.max()) / t)
    e = np.exp(z)
    return e / e.sum()


def lost(x):
    x = np.asarray(x, np.float64)
    return bool(np.isnan(x).any() or np.isposinf(x).any() or np.isneginf(x).all())


def sequence(target, draft, tokens, parents, u, t):
    """Rows of one sequence -> (path, next)."""
    n, vocab = len(tokens), target.shape[1]
    path, at = [0], 0
    while True:
        kids = [j for j in range(at + 1, n) if parents[j] == at]
        greedy = not t >= 1e-6
        drawn = draft is not None and not greedy and kids
        if lost(target[at]) or (drawn and lost(draft[at])):
            return path, -1
        if greedy:
            r = np.zeros(vocab)
            r[int(np.argmax(np.asarray(target[at], np.float64)))] = 1.0
        else:
            r = softmax(target[at], t)
        p, q = r, softmax(draft[at], t) if drawn else None
        to = -1
        for j in kids:
            x = int(tokens[j])
            if not 0 <= x < vocab:
                continue
            if np.float64(u[j]) * (q[x] if drawn else 1.0) < r[x]:
                to = j
                break
            r = r.copy()
            if drawn:
                r = np.maximum(r - q, 0.0)
            else:
                r[x] = 0.0
            r = r / r.sum() if r.sum() > 0 else p
        if to < 0:
            sums = np.cumsum(r)
            above = np.nonzero((sums > np.float64(u[0]) * sums[-1]) & (r > 0))[0]
            return path, int(above[0] if above.size else np.nonzero(r > 0)[0][-1])
        at = to
        path.append(at)
