"""A plain 8-bit key/value cache in 64 bits, page by page, for the tests of wd_kv_*."""
import numpy as np

LIMIT = {0: 127.0, 1: 448.0}


def e4m3_round(z):
    """To the nearest e4m3 number, ties to even: four significant bits down to 2^-6, steps of 2^-9 below."""
    _, e = np.frexp(z)
    u = np.ldexp(1.0, np.maximum(e - 4, -9))
    return np.clip(np.rint(z / u) * u, -448.0, 448.0)


def to_code(z, codes):
    return np.clip(np.rint(z), -127, 127) if codes == 0 else e4m3_round(z)


class Cache:
    """One layer. seqs[i]: list of pages, each a dict of codes [2][page][heads][dim] (as numbers) and scales [2][heads]."""

    def __init__(self, heads, dim, page, codes, max_seqs):
        self.heads, self.dim, self.page, self.codes = heads, dim, page, codes
        self.pages = [[] for _ in range(max_seqs)]
        self.length = [0] * max_seqs

    def blank(self):
        return dict(c=np.zeros((2, self.page, self.heads, self.dim)), s=np.zeros((2, self.heads)))

    def append(self, seq, k, v):
        rows = np.stack([k, v]).astype(np.float64)
        at, n = self.length[seq], rows.shape[1]
        while len(self.pages[seq]) * self.page < at + n:
            self.pages[seq].append(self.blank())
        for p in range(at // self.page, (at + n - 1) // self.page + 1 if n else 0):
            lo, hi = max(at, p * self.page), min(at + n, (p + 1) * self.page)
            a, b = lo - p * self.page, hi - p * self.page
            x = rows[:, lo - at:hi - at]
            g = self.pages[seq][p]
            s0 = g["s"] if a else np.zeros_like(g["s"])
            finite = np.where(np.isfinite(x), np.abs(x), 0.0)
            top = finite.max(axis=(1, 3))
            need = np.where(top > 0, np.maximum((top / LIMIT[self.codes]).astype(np.float32).astype(np.float64), 2.0 ** -100), 0.0)
            s1 = np.maximum(s0, need)
            div = np.where(s1 > 0, s1, 1.0)[:, None, :, None]
            g["c"][:, :a] = to_code(g["c"][:, :a] * s0[:, None, :, None] / div, self.codes)
            x = np.where(np.isnan(x), 0.0, np.where(np.isinf(x), np.sign(x) * LIMIT[self.codes] * div, x))
            g["c"][:, a:b] = to_code(x / div, self.codes)
            g["s"] = s1
        self.length[seq] = at + n

    def numbers(self, seq):
        """[2][length][heads][dim]"""
        if not self.length[seq]:
            return np.zeros((2, 0, self.heads, self.dim))
        x = np.concatenate([g["c"] * g["s"][:, None, :, None] for g in self.pages[seq]], axis=1)
        return x[:, :self.length[seq]]

    def fork(self, src, dst):
        self.pages[dst] = [dict(c=g["c"].copy(), s=g["s"].copy()) for g in self.pages[src]]
        self.length[dst] = self.length[src]

    def truncate(self, seq, length):
        self.length[seq] = length
        self.pages[seq] = self.pages[seq][:-(-length // self.page)]

    def keep(self, seq, first, index):
        old, page = self.pages[seq], self.page
        end = first + len(index)
        new = []
        for p in range(-(-end // page)):
            src = [q if q < first else first + index[q - first] for q in range(p * page, min(end, (p + 1) * page))]
            if all(q == p * page + i for i, q in enumerate(src)):
                new.append(old[p])
                continue
            g = self.blank()
            g["s"] = np.max([old[q // page]["s"] for q in src], axis=0)
            div = np.where(g["s"] > 0, g["s"], 1.0)[:, :, None]
            for i, q in enumerate(src):
                o = old[q // page]
                g["c"][:, i] = to_code(o["c"][:, q % page] * o["s"][:, :, None] / div, self.codes)
            new.append(g)
        self.pages[seq], self.length[seq] = new, end

    def attend(self, seq, q, scale, window, rows=None):
        """q [count][q heads][dim] of the sequence's last tokens, or of some of them: `rows` of the last count ones."""
        k, v = self.numbers(seq)
        n, m, g = self.length[seq], q.shape[0], q.shape[1] // self.heads
        pos = np.arange(n - m, n)
        if rows is not None:
            pos, q = pos[rows], q[rows]
        out = np.zeros(q.shape)
        pos = pos[:, None]
        j = np.arange(n)[None]
        seen = (j <= pos) & ((j > pos - window) if window else True)
        for h in range(q.shape[1]):
            x = np.where(seen, q[:, h].astype(np.float64) @ k[:, h // g].T * scale, -np.inf)
            w = np.exp(x - x.max(axis=1, keepdims=True))
            out[:, h] = w @ v[:, h // g] / w.sum(axis=1, keepdims=True)
        return out
