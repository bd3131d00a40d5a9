"""The 8-bit paged cache restated in 64 bits for the tests: pages of values per
(page, head, side) with an exponent, append, attention, mass and eviction as
include/draftkv_b200.h defines them (dkv_q8_*)."""
import math

import numpy as np

E_MIN, E_MAX = -120, 119


def round_e4m3(x):
    """Nearest e4m3 number (3 fraction bits, exponents from -6, |x| <= 448), ties to even."""
    mag = np.maximum(np.abs(x), 2.0 ** -30)
    _, k = np.frexp(mag)
    step = np.ldexp(1.0, np.maximum(k - 1, -6) - 3)
    return np.round(x / step) * step


def exponent_of(amax):
    if amax == 0:
        return E_MIN
    f, k = math.frexp(amax)
    return min(max(k - 9 if f <= 0.875 else k - 8, E_MIN), E_MAX)


def decode(codes, page, d, index):
    """uint8 [..., 2, page*d] -> code values [..., 2, page, d] (NaN codes as NaN)."""
    b = codes.reshape(codes.shape[:-2] + (2 * page * d,))[..., index.reshape(-1)].astype(np.int64)
    e, f = (b >> 3) & 15, b & 7
    mag = np.where(e == 0, f / 8 * 2.0 ** -6, np.ldexp(1 + f / 8, e - 7))
    mag = np.where((b & 127) == 127, np.nan, mag)
    return np.where(b >= 128, -mag, mag).reshape(codes.shape[:-2] + (2, page, d))


def page_index(page, d):
    """[2, page, d]: byte of (side, token, dim) in a page of one head, from the header's words."""
    at = np.full((2, page, d), -1)
    for tile in range(page // 16):
        for j in range(d // 32):
            for lane in range(32):
                g, t = lane // 4, lane % 4
                for w in range(4):
                    for i, c in enumerate((2 * t, 2 * t + 1, 2 * t + 8, 2 * t + 9)):
                        byte = tile * 16 * d + j * 512 + lane * 16 + w * 4 + i
                        at[0, tile * 16 + g + 8 * (w & 1), 32 * j + 16 * (w >> 1) + c] = byte
                        at[1, tile * 16 + c, 32 * j + 16 * (w >> 1) + 8 * (w & 1) + g] = page * d + byte
    assert (at >= 0).all() and len(np.unique(at)) == at.size
    return at


class RefCache:
    """Values [n_pages, kv, 2, page, d] under exponents [n_pages, kv, 2]."""

    def __init__(self, codes, scale, table, page, d):
        self.page, self.d = page, d
        self.index = page_index(page, d)
        self.vals = decode(codes, page, d, self.index)
        self.exp = np.round(np.log2(scale.astype(np.float64))).astype(np.int64)
        self.table = table

    def append(self, layer, k, v, entry0, n_rows):
        for b in range(k.shape[0]):
            for p in range(entry0[b] // self.page, -(-(entry0[b] + n_rows[b]) // self.page) if n_rows[b] else 0):
                pid = self.table[b, layer, p]
                lo = max(entry0[b] - p * self.page, 0)
                r0 = p * self.page + lo - entry0[b]
                cnt = min(n_rows[b] - r0, self.page - lo)
                for i, x in ((0, k), (1, v)):
                    for h in range(k.shape[2]):
                        self._put(pid, h, i, lo, x[b, r0:r0 + cnt, h].astype(np.float64))

    def _put(self, pid, h, i, lo, rows):
        e = exponent_of(np.abs(rows).max())
        vals = self.vals[pid, h, i]
        if lo:
            e_old = int(self.exp[pid, h, i])
            e = max(e, e_old)
            vals[:lo] = round_e4m3(np.ldexp(vals[:lo], e_old - e))
        vals[lo:lo + len(rows)] = round_e4m3(np.clip(np.ldexp(rows, -e), -448, 448))
        self.exp[pid, h, i] = e

    def entries(self, b, layer, h, n):
        """(k, v) [n, d] of one head's first n entries."""
        pid = self.table[b, layer, : -(-n // self.page)]
        x = self.vals[pid, h] * np.ldexp(1.0, self.exp[pid, h])[..., None, None]
        return x[:, 0].reshape(-1, self.d)[:n], x[:, 1].reshape(-1, self.d)[:n]

    def attention(self, layer, q, entry0, n_rows=None):
        """(out, mass added [batch, kv, capacity], score bound): rows past n_rows are NaN; the bound is
        max over rows and keys of sum |q k| / sqrt(d)."""
        B, T, HQ, d = q.shape
        kv = self.vals.shape[1]
        G = HQ // kv
        out = np.full(q.shape, np.nan)
        mass = np.zeros((B, kv, self.table.shape[2] * self.page))
        bound = 0.0
        for b in range(B):
            for t in range(T if n_rows is None else n_rows[b]):
                n = entry0[b] + t + 1
                for h in range(kv):
                    if n <= 0:
                        out[b, t, h * G:(h + 1) * G] = 0.0
                        continue
                    k, v = self.entries(b, layer, h, n)
                    qq = q[b, t, h * G:(h + 1) * G].astype(np.float64)
                    s = qq @ k.T / math.sqrt(d)
                    bound = max(bound, (np.abs(qq) @ np.abs(k).T).max() / math.sqrt(d))
                    p = np.exp(s - s.max(-1, keepdims=True))
                    p /= p.sum(-1, keepdims=True)
                    out[b, t, h * G:(h + 1) * G] = p @ v
                    mass[b, h, :n] += p.sum(0)
        return out, mass, bound


def evict(mass, n, budget, sink, recent):
    """Kept indices (ascending) of one head."""
    m = min(n, max(budget, sink + recent))
    idx = np.arange(n)
    free = idx[(idx >= sink) & (idx < n - recent)]
    drop = free[np.lexsort((free, mass[free]))][: n - m]
    return np.setdiff1d(idx, drop)


def attention_tolerance(d, n, bound, vmax, out_eps):
    """(relative, absolute) bound of an output element's error.

    Scores are fp32 sums of d products (each addition off by at most 2^-23 of
    the sum of magnitudes `bound`, tensor-core additions truncate), queries
    enter with 2^-22, ex2 is good to 2^-21: a probability is off by the factor
    1 +- delta.  Numerator and denominator each carry delta, and the sums over
    n keys in tiles of 16 with a merge of key groups and splits at most
    (n / 16 + 128) roundings of 2^-23.  A probability is the sum of two f16
    numbers (2^-22).  Then one rounding to the output type."""
    delta = (d + 8) * 2.0 ** -23 * bound + 2.0 ** -20
    return out_eps / 2, 2 * vmax * (delta + (n / 16 + 128) * 2.0 ** -23)


def prompt_tolerance(d, n, bound, vmax, out_eps):
    """The same for more than 64 rows: queries are one f16 number (2^-11 of a
    value, at least 2^-25 of the row's largest: bound * 2^-11 covers both),
    probabilities too (2^-11 of the numerator's terms, and 2^-31 of the max
    for each key)."""
    rel, ab = attention_tolerance(d, n, bound, vmax, out_eps)
    return rel, ab + 2 * vmax * (2.0 ** -11 * bound) + vmax * (2.0 ** -11 + n * 2.0 ** -31)
