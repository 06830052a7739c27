"""Paged KV caches and batches of the many-request tests: device copies, and
the definitions in float64 that the calls are held to."""
import numpy as np

EPS32 = 2.0 ** -24                # half a step of float32 relative to the value
EPS16 = 2.0 ** -11                # of binary16


class Pool:
    """One layer's page pool. order: 'head' [page][head][slot], 'slot'
    [page][slot][head], 'outer' [head][page][slot]; pad: extra elements (a
    multiple of 8) between rows."""

    def __init__(self, pkg, r, kv, order, num_pages, page, KVH, hd, pad=0, fill=None):
        self.pkg, self.kv, self.num_pages, self.page, self.KVH, self.hd = pkg, kv, num_pages, page, KVH, hd
        self.dtype = np.float16 if kv == "f16" else np.float32
        row = hd + pad
        n = num_pages * page * KVH
        st = {"head": (KVH * page * row, page * row, row), "slot": (KVH * page * row, row, KVH * row),
              "outer": (page * row, num_pages * page * row, row)}[order]
        self.strides = st
        self.k, self.v = ((r.normal(size=n * row) if fill is None else np.full(n * row, fill)).astype(self.dtype)
                          for _ in range(2))

    def at(self, page, head, slot):
        b = page * self.strides[0] + head * self.strides[1] + slot * self.strides[2]
        return slice(b, b + self.hd)

    def put(self, d):
        self.dk, self.dv = d.put(self.k), d.put(self.v)
        return self.pkg.PagedKV(self.dk, self.dv, 1 if self.kv == "f16" else 0, self.num_pages, self.page, self.KVH,
                                self.hd, *self.strides)


class Batch:
    """seqs: (new rows, positions cached with them) of each sequence. Pages are
    handed out in random order; `bad` maps (sequence, entry) to a page id."""

    def __init__(self, r, seqs, page, spare=3, pad_rows=0, bad=None):
        self.seqs, self.page = seqs, page
        need = [max(0, -(-max(L, 0) // page)) for _, L in seqs]
        self.num_pages = sum(need) + spare
        perm = r.permutation(self.num_pages)
        self.max_pages = max(max(need), 1)
        self.pages = np.full((len(seqs), self.max_pages), 2 ** 31 - 1, dtype=np.int32)   # unused entries: no page
        at = 0
        for s, n in enumerate(need):
            self.pages[s, :n] = perm[at:at + n]
            at += n
        for (s, e), p in (bad or {}).items():
            self.pages[s, e] = p
        self.row_start = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int32)
        self.kv_len = np.array([L for _, L in seqs], dtype=np.int32)
        self.used = int(self.row_start[-1])
        self.rows = self.used + pad_rows

    def put(self, pkg, d, max_new=0):
        self.d = [d.put(self.row_start), d.put(self.kv_len), d.put(self.pages)]
        return pkg.PagedBatch(*self.d, len(self.seqs), self.max_pages, self.rows, max_new)

    def place(self, s, pos):
        """(page, slot) of a position, or None."""
        if pos < 0 or pos >= self.max_pages * self.page:
            return None
        p = int(self.pages[s, pos // self.page])
        return (p, pos % self.page) if 0 <= p < self.num_pages else None

    def row_places(self):
        """(row, sequence, position) of every row in use."""
        for s, (n, L) in enumerate(self.seqs):
            for i in range(n):
                yield int(self.row_start[s]) + i, s, L - n + i


def rotate64(x, cos, sin, half):
    """apply_rope_raw (gemv.rs:757-778) on [..., hd] in float64."""
    y = np.array(x, dtype=np.float64)
    a, b = y[..., :half].copy(), y[..., half:2 * half].copy()
    y[..., :half] = a * cos - b * sin
    y[..., half:2 * half] = b * cos + a * sin
    return y


def attention64(pool, batch, q, H):
    """(out, tolerance) [rows in use][H][hd] in float64.

    The tolerance counts, per row and head, with S = sum |q k| scale of the
    largest score: a score's float32 products, their sum of hd terms and the 22
    bits q and an f32 k are held to (2^-22 each) move it by (hd + 16) S half
    steps, twice that reaches a weight ratio; the weighted sum of n values and
    the division add n + 64 half steps, all relative to the largest |v|."""
    hd, G = pool.hd, H // pool.KVH
    out = np.zeros((batch.used, H, hd))
    tol = np.zeros((batch.used, H, 1))
    cache = {}
    for row, s, pos in batch.row_places():
        if (s not in cache):
            pl = [(j, batch.place(s, j)) for j in range(batch.seqs[s][1])]
            pl = [(j, p) for j, p in pl if p is not None]
            cache[s] = (np.array([j for j, _ in pl], dtype=np.int64),
                        [np.array([pool.k[pool.at(p[0], h, p[1])] for _, p in pl], dtype=np.float64).reshape(-1, hd)
                         for h in range(pool.KVH)],
                        [np.array([pool.v[pool.at(p[0], h, p[1])] for _, p in pl], dtype=np.float64).reshape(-1, hd)
                         for h in range(pool.KVH)])
        js, ks, vs = cache[s]
        n = int(np.searchsorted(js, pos, side="right"))
        if n == 0:
            continue
        for h in range(H):
            k, v, qq = ks[h // G][:n], vs[h // G][:n], q[row, h].astype(np.float64)
            sc = k @ qq / np.sqrt(hd)
            e = np.exp(sc - sc.max())
            out[row, h] = e @ v / e.sum()
            S = (np.abs(k) @ np.abs(qq)).max() / np.sqrt(hd)
            tol[row, h] = EPS32 * (2 * (hd + 16) * S + n + 64) * np.abs(v).max()
    return out, tol
