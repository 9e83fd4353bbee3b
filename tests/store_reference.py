"""A plain statement of the 4-bit key/value store's formulas (include/base2.h), number by number, in Python's whole
numbers where 64 bits could overflow. Test infrastructure only."""
import numpy as np

HD, TOP, LIM = 64, 1 << 47, (1 << 30) - 1


def rnd(x: int, s: int) -> int:
    return (x + (1 << (s - 1))) >> s if s > 0 else x


def clamp(x):
    return np.clip(np.asarray(x, np.int64), -TOP, TOP - 1)


def shift4(x) -> int:
    return min(max(max(int(abs(int(t))).bit_length() for t in x) - 3, 0), 44)


def codes(x, s: int):
    return [min(max(rnd(int(t), s), -8), 7) for t in x]


def hold_key(x):
    """(64 codes, the halves' shifts) of one head row."""
    x = clamp(x)
    s = [shift4(x[:32]), shift4(x[32:])]
    s = [max(t, max(s) - 3) for t in s]
    return codes(x[:32], s[0]) + codes(x[32:], s[1]), s


def hold_value(x):
    x = clamp(x)
    s = shift4(x)
    return codes(x, s), s


def read_key(held):
    c, s = held
    return np.array([t << s[i // 32] for i, t in enumerate(c)], dtype=np.int64)


def read_value(held):
    c, s = held
    return np.array([t << s for t in c], dtype=np.int64)


def score(q, key) -> int:
    """q.k / 8 at 2^-10, q at 15 bits, held between -LIM and LIM."""
    q = [int(t) for t in clamp(q)]
    u = max(max(abs(t).bit_length() for t in q) - 14, 0)
    q15 = [rnd(t, u) for t in q]
    c, s = key
    S = max(s)
    dot = sum(a * (b << (s[i // 32] - S + 3)) for i, (a, b) in enumerate(zip(q15, c)))
    e = u + S - 28
    return min(max(dot << e if e >= 0 else rnd(dot, -e), -LIM), LIM)


def log2fix(z: int, LOG2) -> int:
    t = z.bit_length() - 1
    return t * 65536 + int(LOG2[(z >> (t - 16) if t >= 16 else z << (16 - t)) & 65535])


def power(x: int, F: int, EXP2) -> int:
    y, s = x * int(EXP2[F & 65535]), 16 - (F >> 16)
    return rnd(y, s) if s >= 0 else y << -s


def attend(q, keys, values, T):
    """One row over its visible keys (held pairs, in any order): 64 numbers."""
    if not keys:
        return np.zeros(HD, np.int64)
    sc = [score(q, k) for k in keys]
    start, M = max(sc), max(s for _, s in values)
    ARR = T["arrival"]
    a = [int(ARR[start - t]) if start - t < len(ARR) else 0 for t in sc]
    Z = sum(a)
    num = [0] * HD
    for t, (c, s) in zip(a, values):
        w = rnd(t, 1 + M - s)
        if w:
            num = [n + w * x for n, x in zip(num, c)]
    F = 65536 * (M + 1) - log2fix(Z, T["log2"])
    return np.array([power(n, F, T["exp2"]) for n in num], dtype=np.int64)


class Store:
    """The whole store in plain Python: rows as b2_store_* take them."""

    def __init__(self, T, n_head):
        self.T, self.H, self.k, self.v = T, n_head, {}, {}

    @staticmethod
    def places(pos, cu):
        n = len(pos)
        cu = list(range(n + 1)) if cu is None else [int(c) for c in cu]
        return [(s, int(pos[s]) + r - cu[s], r) for s in range(n) for r in range(cu[s], cu[s + 1])]

    def write(self, k, v, pos, cu=None, layer=0):
        for s, p, r in self.places(pos, cu):
            for h in range(self.H):
                self.k[layer, s, p, h], self.v[layer, s, p, h] = hold_key(k[r, h]), hold_value(v[r, h])

    def read(self, pos, cu=None, layer=0):
        at = self.places(pos, cu)
        k = np.zeros((len(at), self.H, HD), np.int64)
        v = np.zeros_like(k)
        for s, p, r in at:
            for h in range(self.H):
                if (layer, s, p, h) in self.k:
                    k[r, h], v[r, h] = read_key(self.k[layer, s, p, h]), read_value(self.v[layer, s, p, h])
        return k, v

    def attend(self, q, pos, cu=None, window=0, first=None, layer=0):
        at = self.places(pos, cu)
        out = np.zeros((len(at), self.H, HD), np.int64)
        nothing = ([0] * HD, [0, 0]), ([0] * HD, 0)
        for s, p, r in at:
            lo = max(0, int(first[s]) if first is not None else 0, p - window + 1 if window else 0)
            for h in range(self.H):
                ids = [(layer, s, j, h) for j in range(lo, p + 1)]
                out[r, h] = attend(q[r, h], [self.k.get(i, nothing[0]) for i in ids],
                                   [self.v.get(i, nothing[1]) for i in ids], self.T)
        return out


class FastStore:
    """The same store for values of ordinary size, with numpy's 64-bit whole numbers (products as float64 matrix products
    that stay below 2^53): one layer, a run of positions per stream written from 0 on. Checked against Store."""

    def __init__(self, T, heads, streams):
        self.T, self.H, self.held = T, heads, [[] for _ in range(streams)]

    @staticmethod
    def _bits(x):
        return np.frexp(np.abs(x).max(axis=-1).astype(np.float64))[1].astype(np.int64)

    @staticmethod
    def _rnd(x, s):
        return np.where(s > 0, ((x >> np.maximum(s - 1, 0)) + 1) >> 1, x)

    def _hold(self, x, halves):
        x = x.reshape(*x.shape[:2], halves, HD // halves)
        s = np.maximum(self._bits(x) - 3, 0)
        s = np.maximum(s, s.max(-1, keepdims=True) - 3)
        return np.clip(self._rnd(x, s[..., None]), -8, 7).reshape(*x.shape[:2], HD), s

    def write(self, s, k, v):
        """Rows [n, heads, 64] at stream s's next positions."""
        self.held[s].append((*self._hold(k, 2), *self._hold(v, 1)))

    def attend(self, s, q, p0, window=0, first=0):
        """Rows [n, heads, 64] of stream s at positions p0 .."""
        kc, ks, vc, vs = (np.concatenate(x)[:p0 + len(q)] for x in zip(*self.held[s]))
        out, at = np.zeros(q.shape, np.int64), np.arange(p0 + len(q))[None]
        me = p0 + np.arange(len(q))[:, None]
        seen = (at <= me) & (at >= np.maximum(first, me - window + 1 if window else 0))
        ARR, LOG2, EXP2 = (self.T[k] for k in ("arrival", "log2", "exp2"))
        for h in range(self.H):
            u = np.maximum(self._bits(q[:, h]) - 14, 0)
            S = ks[:, h].max(-1)
            k8 = kc[:, h] << np.repeat(ks[:, h] - S[:, None] + 3, 32, axis=1)
            dot = (self._rnd(q[:, h], u[:, None]).astype(np.float64) @ k8.T.astype(np.float64)).astype(np.int64)
            r = 28 - u[:, None] - S[None]
            assert (r >= -30).all()                                # |dot| <= 2^26: nothing below passes 64 bits
            sc = np.where(r >= 0, self._rnd(dot, np.maximum(r, 0)), np.clip(dot << np.maximum(-r, 0), -LIM, LIM))
            d = np.where(seen, sc, np.iinfo(np.int64).min).max(1, keepdims=True) - sc
            a = np.where(seen & (d < len(ARR)), ARR[np.clip(d, 0, len(ARR) - 1)], 0)
            M = np.where(seen, vs[None, :, h, 0], 0).max(1)
            w = self._rnd(a, np.where(seen, 1 + M[:, None] - vs[None, :, h, 0], 1))
            num = (w.astype(np.float64) @ vc[:, h].astype(np.float64)).astype(np.int64)
            for i in np.flatnonzero(seen.any(1)):
                F = 65536 * (int(M[i]) + 1) - log2fix(int(a[i].sum()), LOG2)
                out[i, h] = [power(int(n), F, EXP2) for n in num[i]]
        return out
