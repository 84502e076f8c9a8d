"""The paged 4-bit KV cache in numpy, from its definition: the values that stored rows stand for, attention
over them in 64 bits, and a model of the page tables."""
import numpy as np


def kv4_values(x):
    """f16 values of rows x (f16, last axis a multiple of 32) after quantization."""
    a = np.ascontiguousarray(x, np.float16).reshape(-1, 32)
    with np.errstate(all="ignore"):
        lo, hi = a.min(1).astype(np.float64), a.max(1).astype(np.float64)
        d = ((hi - lo) / 15).astype(np.float16)  # numpy rounds 64 bits to 16 once, ties to even
        over = lo + 15 * d.astype(np.float64) > 65504
        d[over] = np.nextafter(d[over], np.float16(0))
        step = d.astype(np.float64)[:, None]
        t = np.divide(a.astype(np.float64) - lo[:, None], step, out=np.zeros(a.shape), where=step > 0)
        v = (lo[:, None] + np.minimum(np.rint(t), 15) * step).astype(np.float16)
    v[~np.isfinite(a).all(1)] = np.nan
    return v.reshape(np.shape(x))


def attention64(q, K, V, nq, nkv, hd):
    """Last len(q) positions of K and V (values) attended to by rows q: the output, the bound's ingredients
    (sum of probability times |V|, largest score magnitude) per output, all in 64 bits."""
    rows, S, G = len(q), len(K), nq // nkv
    out = np.empty((rows, nq, hd))
    mass = np.empty((rows, nq, hd))
    top = np.empty((rows, nq, 1))
    Kd, Vd = (x.astype(np.float64).reshape(S, nkv, hd) for x in (K, V))
    for r in range(rows):
        n = S - rows + r + 1
        for h in range(nq):
            qv = q[r].astype(np.float64).reshape(nq, hd)[h]
            s = Kd[:n, h // G] @ qv / np.sqrt(hd)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[r, h] = p @ Vd[:n, h // G]
            mass[r, h] = p @ np.abs(Vd[:n, h // G])
            top[r, h] = (np.abs(Kd[:n, h // G]) @ np.abs(qv)).max() / np.sqrt(hd)
    return out.reshape(rows, -1), mass.reshape(rows, -1), np.repeat(top, hd, 2).reshape(rows, -1)


def attention_bound(want, mass, top, S, hd, vmax):
    """How far an f16 output may be off: its own rounding (an f16 step), each probability's rounding to f16
    (2^-11 of it, against a sum of unrounded ones), the f32 rounding of dot products (hd 2^-24 of the sum of
    |products| each), exponentials and sums, doubled, and probabilities under 2^-39 of the largest that a
    scaled f16 can round by 2^-40."""
    ulp = np.spacing(np.abs(want).astype(np.float16)).astype(np.float64)
    return ulp + mass * (2.0 ** -11 + ((hd + 16) * (1 + top) + S) * 2.0 ** -23) + S * 2.0 ** -39 * vmax


class Book:
    """Sequences as lists of page ids, lowest free page first; `rows` model what positions hold."""

    def __init__(self, pages, page):
        self.page, self.total, self.seqs = page, pages, {}

    def owners(self):
        n = {}
        for pages, _ in self.seqs.values():
            for p in pages:
                n[p] = n.get(p, 0) + 1
        return n

    def free(self):
        used = self.owners()
        return [p for p in range(self.total) if p not in used]

    def begin(self, ids, rows):
        """False (nothing changed) without enough pages; else the (source, copy) pairs."""
        saved = {i: (list(p), n) for i, (p, n) in self.seqs.items()}
        copies = []
        try:
            for i, r in zip(ids, rows):
                pages, n = self.seqs.setdefault(i, ([], 0))
                if r and n % self.page and self.owners()[pages[-1]] > 1:
                    new = self.free()[0]
                    copies.append((pages[-1], new))
                    pages[-1] = new
                self.seqs[i] = (pages, n + r)
                while len(pages) * self.page < n + r:
                    pages.append(self.free()[0])
        except IndexError:
            self.seqs = saved
            return False
        return copies

    def length(self, i):
        return self.seqs.get(i, ([], 0))[1]

    def pages(self, i):
        return self.seqs.get(i, ([], 0))[0]

    def fork(self, i, j):
        self.seqs[j] = (list(self.pages(i)), self.length(i))

    def copy(self, i, j):
        if len(self.pages(i)) > len(self.free()):
            return False
        self.seqs[j] = ([], self.length(i))
        for _ in self.pages(i):
            self.seqs[j][0].append(self.free()[0])
        return True

    def truncate(self, i, n):
        self.seqs[i] = (self.pages(i)[: -(-n // self.page)], n)

    def compact(self):
        used = len(self.owners())
        for p in sorted(q for q in self.owners() if q >= used):
            to = self.free()[0]
            for i, (pages, n) in self.seqs.items():
                self.seqs[i] = ([to if x == p else x for x in pages], n)
        return used
