"""The 8-bit key/value cache in plain float64, on the CPU: what the tests of fl_kv8_* compare with.

A stored value's roundings are part of the definition (a rotated key is fma(x0, c, -(x1 s)) in 32 bits, then fp16; scale =
absmax/127, integer = rint(x * (127/absmax)), each step in 32 bits), so rows, scales and tails are compared bit for bit; a
product or quotient rounded once to 32 bits is formed in 64 bits and rounded."""
import math

import numpy as np

U = 2.0 ** -24  # half a step of a 32-bit float, relative


def f32(x):
    return np.asarray(x, np.float64).astype(np.float32).astype(np.float64)


def rotate_key(x, row):
    """[..., D] by table rows [..., D], with the definition's roundings."""
    x, row = np.asarray(x, np.float64), np.asarray(row, np.float64)
    a, b, c, s = x[..., 0::2], x[..., 1::2], row[..., 0::2], row[..., 1::2]
    with np.errstate(invalid="ignore", over="ignore"):
        o = np.stack([f32(a * c - f32(b * s)), f32(b * c + f32(a * s))], -1)
    return o.reshape(x.shape)


def rotate(x, row):
    z = (np.asarray(x, np.float64)[..., 0::2] + 1j * np.asarray(x, np.float64)[..., 1::2]) * (row[..., 0::2].astype(np.float64) + 1j * row[..., 1::2])
    return np.stack([z.real, z.imag], -1).reshape(x.shape)


def stored(x):
    x = np.asarray(x, np.float64)
    return np.where(np.isfinite(x), np.clip(x, -65504.0, 65504.0), 0.0).astype(np.float16)


class Cache:
    """Arrays as the library's; `junk` fills what has not been written yet."""

    def __init__(self, B, H, D, L, T, weights=False, junk=True, seed=0):
        r = np.random.RandomState(seed)
        n = L // T
        self.B, self.H, self.D, self.L, self.T = B, H, D, L, T
        self.k, self.v = (r.randint(-127, 128, (B, H, L, D)).astype(np.int8) for _ in range(2))
        self.k_scale, self.v_scale = (np.full((B, H, n), np.nan if junk else 0.0, np.float32) for _ in range(2))
        self.k_tail, self.v_tail = (np.full((B, H, T, D), np.nan if junk else 0.0, np.float16) for _ in range(2))
        self.weights = np.full((B, H, n), np.nan if junk else 0.0, np.float32) if weights else None

    def names(self):
        return [n for n in ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail", "weights") if getattr(self, n) is not None]

    def copy(self):
        c = Cache.__new__(Cache)
        c.__dict__.update({n: (x.copy() if isinstance(x, np.ndarray) else x) for n, x in self.__dict__.items()})
        return c

    def fill(self, rows, seed=1):
        """`rows` [B] rows of N(0,1) values, as earlier calls would have left them."""
        r = np.random.RandomState(seed)
        for b, n in enumerate(rows):
            for s in range(int(n)):
                self.put(b, s, r.randn(self.H, self.D).astype(np.float16), r.randn(self.H, self.D).astype(np.float16))
        if self.weights is not None:
            for b, n in enumerate(rows):
                m = -(-int(n) // self.T)
                self.weights[b, :, :m] = r.rand(self.H, m)
        return self

    def put(self, b, row, k16, v16):
        T = self.T
        blk, at = row // T, row % T
        self.k_tail[b, :, at], self.v_tail[b, :, at] = k16, v16
        if at == T - 1:
            for q, sc, tail in ((self.k, self.k_scale, self.k_tail), (self.v, self.v_scale, self.v_tail)):
                x = tail[b].astype(np.float64)
                top = np.abs(x).max((-1, -2))
                per = np.where(top > 0, f32(127.0 / np.where(top > 0, top, 1.0)), 0.0)
                q[b, :, blk * T:(blk + 1) * T] = np.rint(f32(x * per[:, None, None])).astype(np.int8)
                sc[b, :, blk] = (top / 127.0).astype(np.float32)

    def values(self, b, rows):
        T, out = self.T, []
        for q, sc, tail in ((self.k, self.k_scale, self.k_tail), (self.v, self.v_scale, self.v_tail)):
            x = np.zeros((self.H, rows, self.D))
            whole = rows // T * T
            x[:, :whole] = q[b, :, :whole] * sc[b, :, :whole // T].astype(np.float64).repeat(T, -1)[..., None]
            x[:, whole:] = tail[b, :, :rows - whole]
            out.append(x)
        return out

    def step(self, q, k_new, v_new, table, start, mask=None, rope=None, scale=None, weight_queries=0, lens=None):
        """S tokens [B,S,H,D] at rows start[b] .., lens[b] of them the sequence's own; returns out [B,H,S,D] and how far a 32-bit computation may be off it
        [B,1,1,1] (see tolerance()).  A position outside the cache: NaN, nothing stored."""
        B, S_all, H, D = q.shape
        scale = scale or 1.0 / math.sqrt(D)
        out, tol = np.full((B, H, S_all, D), np.nan), np.zeros((B, 1, 1, 1))
        for b in range(B):
            P, S = int(start[b]), S_all if lens is None else int(lens[b])
            if P < 0 or P + S > self.L or S < 0 or S > S_all:
                continue
            out[b] = 0.0
            if S == 0:
                continue
            rr = P if rope is None else int(rope[b])
            rows = table[rr:rr + S][:, None]
            kk, vv = stored(rotate_key(k_new[b, :S], rows)), stored(v_new[b, :S])
            for s in range(S):
                self.put(b, P + s, kk[s], vv[s])
            k, v = self.values(b, P + S)
            qq = rotate(q[b, :S], rows).transpose(1, 0, 2)
            z = qq @ k.transpose(0, 2, 1) * scale
            with np.errstate(invalid="ignore", over="ignore"):
                if mask is not None:
                    z = z + mask[P:P + S, :P + S].astype(np.float64)
                e = np.exp(z - np.maximum(z.max(-1, keepdims=True), -1e9))
                p = e / e.sum(-1, keepdims=True)
                out[b, :, :S] = p @ v
            tol[b] = self.tolerance(qq, k, v, scale, P + S)
            if self.weights is not None:
                W = min(weight_queries or S, S)
                ok = p[:, -W:]
                ok = np.where(np.isnan(ok), 0.0, ok).sum(1)
                n, first = -(-(P + S) // self.T), -(-P // self.T)
                per = np.pad(ok, ((0, 0), (0, n * self.T - P - S))).reshape(H, n, self.T).sum(-1)
                old = self.weights[b, :, :n].astype(np.float64)
                old[:, first:] = 0.0
                self.weights[b, :, :n] = (old + per).astype(np.float32)
        return out, tol

    @staticmethod
    def tolerance(q, k, v, scale, rows):
        """32-bit arithmetic, U = 2^-24 per rounding.  A score's operand and product errors are at most U each on terms that
        add up to A = scale * max|q| * sum|k|; they are of random sign, so a score is off by about 2 U A (four times the
        deviation of a dozen roundings along a sum), and a weight relatively by as much, numerator and denominator: 4 U A.
        The sums over the rows add sqrt(rows) U, the exponential, scales and quotient a few U: 64 U holds them.  Relative to
        the largest |v|."""
        A = scale * np.abs(q[np.isfinite(q)]).max() * np.abs(k).sum(-1).max() if q.size else 0.0
        return np.abs(v).max() * U * (4 * A + math.sqrt(rows) + 64)


def evict(c, rows, keep, recent, into=None):
    """Returns (kept, rows after), and moves blocks in `into` (c itself where it is None)."""
    to, T = into if into is not None else c, c.T
    src = c.copy()
    kept, after = np.full((c.B, c.H, keep), -1, np.int32), np.full(c.B, -1, np.int32)
    for b in range(c.B):
        if rows[b] < 0 or rows[b] > c.L:
            continue
        n, open_ = int(rows[b]) // T, int(rows[b]) % T
        m = min(keep, n)
        sure = min(recent, m)
        after[b] = m * T + open_
        for h in range(c.H):
            w = src.weights[b, h, :n - sure].astype(np.float64)
            key = np.where(np.isnan(w), -np.inf, w)
            order = sorted(range(n - sure), key=lambda i: (bool(np.isnan(w[i])), -key[i], i))
            stay = sorted(order[:m - sure]) + list(range(n - sure, n))
            kept[b, h, :m] = stay
            for r, i in enumerate(stay):
                for x, y in ((src.k, to.k), (src.v, to.v)):
                    y[b, h, r * T:(r + 1) * T] = x[b, h, i * T:(i + 1) * T]
                for x, y in ((src.k_scale, to.k_scale), (src.v_scale, to.v_scale), (src.weights, to.weights)):
                    y[b, h, r] = x[b, h, i]
            if open_ and m < to.L // T:
                to.weights[b, h, m] = src.weights[b, h, n]
        if into is not None:
            to.k_tail[b, :, :open_], to.v_tail[b, :, :open_] = src.k_tail[b, :, :open_], src.v_tail[b, :, :open_]
    return kept, after
