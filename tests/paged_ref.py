"""Plain 64-bit (and plain Python) counterparts of the token-paged cache's operators, for the tests."""
import math

import numpy as np
import torch

E_MIN, E_MAX = -60, 60


# ---------------------------------------------------------------------------------------- e4m3
def all_codes():
    """Value of every e4m3 code, from the format's definition (bias 7, no infinities, 0x7f / 0xff NaN)."""
    out = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.nan if (c & 0x7f) == 0x7f else (m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        out[c] = -v if c & 0x80 else v
    return out


CODES = all_codes()
_POS = CODES[:0x7f]  # ascending


def to_code(y):
    """Codes nearest to y (float64 array), ties to the even mantissa, magnitudes above 448 to 448, NaN to NaN."""
    y = np.asarray(y, dtype=np.float64)
    a = np.minimum(np.abs(np.nan_to_num(y, nan=0.0, posinf=1e300, neginf=-1e300)), 448.0)
    hi = np.searchsorted(_POS, a)  # first code >= a
    lo = np.maximum(hi - 1, 0)
    up, down = _POS[hi] - a, a - _POS[lo]
    c = np.where(up < down, hi, np.where(up > down, lo, np.where(hi % 2 == 0, hi, lo)))
    c = np.where(_POS[hi] == a, hi, c)
    return np.where(np.isnan(y), 0x7f, c | (np.signbit(y) * 0x80)).astype(np.uint8)


def scale_for(amax):
    """Smallest power of two that keeps amax within 448, in [2^-60, 2^60]."""
    e = E_MIN
    while e < E_MAX and 448.0 * 2.0 ** e < amax:
        e += 1
    return 2.0 ** e


# ---------------------------------------------------------------------------------------- the cache
class Books:
    """The cache in plain Python: one layer of codes and scales per (page, head), tables as lists."""

    def __init__(self, cache):
        self.P, self.n_pages, self.per_row, self.max_seqs = cache.page_tokens, cache.n_pages, cache.max_pages_per_seq, cache.max_seqs
        self.pull(cache)

    def pull(self, cache):
        self.table = [[int(p) for p in row if p >= 0] for row in cache.page_table.cpu().tolist()]
        self.lens = cache.seq_lens.cpu().tolist()
        self.refs = cache.page_refs.cpu().tolist()
        self.k8, self.v8 = [t.view(torch.uint8).cpu().numpy().copy() for t in (cache.k8, cache.v8)]
        self.ks, self.vs = [t.double().cpu().numpy().copy() for t in (cache.k_scale, cache.v_scale)]

    def same(self, cache):
        """None, or what differs (codes and scales of pages in use only)."""
        other = Books.__new__(Books)
        other.pull(cache)
        if other.lens != self.lens:
            return f"seq_lens {other.lens} != {self.lens}"
        if other.table != self.table:
            return f"page_table {other.table} != {self.table}"
        if other.refs != self.refs:
            return f"page_refs {other.refs} != {self.refs}"
        for row, n in zip(self.table, self.lens):
            for slot, p in enumerate(row):
                held = min(n - slot * self.P, self.P)
                for name in ("k8", "v8"):
                    if not np.array_equal(getattr(self, name)[:, p, :, :held], getattr(other, name)[:, p, :, :held]):
                        return f"{name} of page {p}"
                for name in ("ks", "vs"):
                    if not np.array_equal(getattr(self, name)[:, p], getattr(other, name)[:, p]):
                        return f"{name} of page {p}"
        return None

    def _take(self, n):
        free = [p for p in range(self.n_pages) if self.refs[p] == 0]
        return free[:n] if len(free) >= n else None

    def reserve(self, seqs, n_new):
        if len(set(seqs)) < len(seqs) or any(s < 0 or s >= self.max_seqs or a < 0 for s, a in zip(seqs, n_new)):
            return None
        if any(self.lens[s] + a > self.per_row * self.P for s, a in zip(seqs, n_new)):
            return None
        need = [-(-(self.lens[s] + a) // self.P) - -(-self.lens[s] // self.P) for s, a in zip(seqs, n_new)]
        ids = self._take(sum(need))
        if ids is None:
            return None
        starts = []
        for s, a, k in zip(seqs, n_new, need):
            mine, ids = ids[:k], ids[k:]
            for p in mine:
                self.refs[p] = 1
            self.table[s] += mine
            starts.append(self.lens[s])
            self.lens[s] += a
        return starts

    def branch(self, src, dst, share):
        bad = any(s < 0 or s >= self.max_seqs for s in src + dst) or len(set(dst)) < len(dst) or set(src) & set(dst)
        if bad or any(self.lens[d] for d in dst):
            return False
        first = [self.lens[s] // self.P if share else 0 for s in src]
        ids = self._take(sum(len(self.table[s]) - f for s, f in zip(src, first)))
        if ids is None:
            return False
        for s, d, f in zip(src, dst, first):
            row = list(self.table[s][:f])
            for p in row:
                self.refs[p] += 1
            for p in self.table[s][f:]:
                new, ids = ids[0], ids[1:]
                self.refs[new] = 1
                self._move(p, new)
                row.append(new)
            self.table[d], self.lens[d] = row, self.lens[s]
        return True

    def _move(self, old, new):
        for a in (self.k8, self.v8, self.ks, self.vs):
            a[:, new] = a[:, old]

    def free(self, seqs):
        if len(set(seqs)) < len(seqs) or any(s < 0 or s >= self.max_seqs for s in seqs):
            return False
        for s in seqs:
            for p in self.table[s]:
                self.refs[p] -= 1
            self.table[s], self.lens[s] = [], 0
        return True

    def compact(self):
        live = [p for p in range(self.n_pages) if self.refs[p] > 0]
        n = len(live)
        holes, movers = [p for p in range(n) if self.refs[p] == 0], [p for p in live if p >= n]
        to = dict(zip(movers, holes))
        for old, new in to.items():
            self._move(old, new)
            self.refs[new], self.refs[old] = self.refs[old], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]

    def append(self, layer, seq, start, k, v):
        """k, v float64 [tokens, heads, 128] at positions start.. of a sequence whose length counts them."""
        for codes, scales, x in ((self.k8, self.ks, k), (self.v8, self.vs, v)):
            for slot in range(start // self.P, -(-(start + len(x)) // self.P)):
                p, base = self.table[seq][slot], slot * self.P
                lo, hi = max(start, base) - base, min(start + len(x), base + self.P) - base
                held = min(self.lens[seq] - base, self.P)
                rows = [r for r in range(held) if not lo <= r < hi]
                for h in range(x.shape[1]):
                    new = x[base + lo - start:base + hi - start, h]
                    fin = np.abs(new[np.isfinite(new)])
                    after = scale_for(fin.max() if fin.size else 0.0)
                    if rows:
                        before = scales[layer, p, h]
                        after = max(after, before)
                        codes[layer, p, h, rows] = to_code(CODES[codes[layer, p, h, rows]] * (before / after))
                    scales[layer, p, h] = after
                    codes[layer, p, h, lo:hi] = to_code(new / after)

    def kv(self, layer, seq, head):
        """(k, v) float64 [len, 128] of one sequence and kv head, as the codes and scales say."""
        out = []
        for codes, scales in ((self.k8, self.ks), (self.v8, self.vs)):
            parts = [CODES[codes[layer, p, head]] * scales[layer, p, head] for p in self.table[seq]]
            out.append(np.concatenate(parts)[:self.lens[seq]] if parts else np.zeros((0, 128)))
        return out


# ---------------------------------------------------------------------------------------- attention
def attention(books, layer, q, seqs, cu, hkv, scale=None, causal=True, window=0):
    """fp64 (out, lse, tol_out, tol_lse) of q [total, Hq, 128] (float64 values of its bf16 entries); rows that no entry
    owns are NaN in out.

    tol bounds what the kernel's own roundings may do to an exact computation:
      * P as e4m3 plus residual as e5m2: the first rounding leaves at most 2^-4 of the value, the second is off by at most
        2^-3 of that: 2^-7, and fp16 in between by 2^-11.  Where the first term is subnormal it leaves at most 2^-10, of which
        the second loses 2^-13, and the largest weight of a row is at least 2^5: 2^-18 of it.
        |do| <= (2^-7 + 2^-11) sum p|v| + 2^-18 sum |v| / l, where l is the sum of the weights relative to the largest;
      * Q in two e4m3 terms, each row scaled so that its largest entry lies in (224, 448]: 16 (two 4-bit) significand bits
        hold bf16's 8 exactly, except that what lies below 2^-10 / 224 < 2^-17 of the row's largest entry is lost:
        |ds| <= scale * 2^-17 max|q| * sum_d |k_d|, which changes a weight by a factor of at most exp(2 |ds|);
      * fp32 sums over at most 2^17 keys in parts of 128 and the fp32 exponent of a score of size s: 2^-14 in all here;
      * the result rounded to bf16: 2^-8 |o|."""
    total, hq, _ = q.shape
    group = hq // hkv
    scale = scale if scale else 1 / math.sqrt(128)
    out, lse = np.full(q.shape, np.nan), np.full(q.shape[:2], np.nan)
    tol, tol_l = np.zeros(q.shape), np.zeros(q.shape[:2])
    for i, s in enumerate(seqs):
        n, nq = books.lens[s], cu[i + 1] - cu[i]
        for h in range(hkv):
            k, v = books.kv(layer, s, h)
            for r in range(nq):
                pos = n - nq + r
                end, begin = (pos + 1 if causal else n), (max(0, pos - window + 1) if window else 0)
                heads = slice(h * group, (h + 1) * group)
                qq = q[cu[i] + r, heads]
                if end <= begin:
                    out[cu[i] + r, heads], lse[cu[i] + r, heads] = 0.0, -math.inf
                    continue
                kk, vv = k[begin:end], v[begin:end]
                with np.errstate(all="ignore"):
                    sc = qq @ kk.T * scale
                    top = sc.max(1, keepdims=True)
                    w = np.exp(sc - top)
                    l = w.sum(1, keepdims=True)
                    o = w @ vv / l
                    ds = scale * 2.0 ** -17 * np.abs(qq).max(1, keepdims=True) * np.abs(kk).sum(1).max()
                    a = w @ np.abs(vv) / l
                    out[cu[i] + r, heads], lse[cu[i] + r, heads] = o, (top + np.log(l))[:, 0]
                    tol[cu[i] + r, heads] = 2.0 ** -8 * np.abs(o) + (2.0 ** -7 + 2.0 ** -11 + 2 * ds + 2.0 ** -14) * a + 2.0 ** -18 * np.abs(vv).sum(0) / l
                    tol_l[cu[i] + r, heads] = (ds + 2.0 ** -16 + 2.0 ** -20 * np.abs(top))[:, 0]
    return out, lse, tol, tol_l


# ---------------------------------------------------------------------------------------- rotary
def rotary(x, positions, inv_freq, layout, mscale=1.0, inverse=False):
    """fp64 [T, H, D]."""
    x, half = np.array(x, dtype=np.float64), len(inv_freq)
    angle = np.asarray(positions, dtype=np.float64)[:, None] * np.asarray(inv_freq)
    c, s = np.cos(angle)[:, None] * mscale, np.sin(angle)[:, None] * mscale * (-1 if inverse else 1)
    a, b = (slice(0, half), slice(half, 2 * half)) if layout == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    first, second = x[..., a].copy(), x[..., b].copy()
    x[..., a], x[..., b] = first * c - second * s, second * c + first * s
    return x
