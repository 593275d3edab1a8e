"""A plain model of a cache of pages: the table's rules one sequence and page after another, what pages hold, and
attention in 64 bits."""
import numpy as np

from tests.helpers import attention_f64, rng_for, rope_f32


def held(rows, hd, q8):
    """What a cache holds of fp32 rows."""
    if not q8:
        return np.asarray(rows, np.float64)
    x = np.asarray(rows, np.float32).reshape(-1, hd)
    a = np.maximum(np.abs(x).max(axis=1, keepdims=True), np.float32(2.0 ** -100))
    q = np.rint(x * (np.float32(127) / a)).astype(np.float64)
    return (q * (a / np.float32(127)).astype(np.float64)).reshape(np.shape(rows))


class Pages:
    """The tables and the pages' contents, [layers][pages][2][page_rows][kv_dim]."""

    def __init__(self, n_seq, width, n_pages, page_rows, layers, kv_dim):
        self.table = np.full((n_seq, width), -1, np.int32)
        self.refs = np.zeros(n_pages, np.int32)
        self.R = page_rows
        self.rows = np.zeros((layers, n_pages, 2, page_rows, kv_dim))

    def pages_of(self, rows):
        return -(-rows // self.R)

    def reserve(self, begin, end):
        """False, with nothing changed, where the pool is too small."""
        table, refs, copies = self.table.copy(), self.refs.copy(), []
        for i, (b, e) in enumerate(zip(begin, end)):
            for j in range(b // self.R, self.pages_of(e) if b < e else 0):
                p = table[i, j]
                if p >= 0 and refs[p] == 1:
                    continue
                free = np.flatnonzero(refs == 0)
                if not free.size:
                    return False
                if p >= 0:
                    refs[p] -= 1
                    copies.append((p, free[0]))
                refs[free[0]] = 1
                table[i, j] = free[0]
        for p, to in copies:
            self.rows[:, to] = self.rows[:, p]
        self.table, self.refs = table, refs
        return True

    def fork(self, parent, rows):
        new = [self.table[i if parent is None else parent[i]].copy() for i in range(len(rows))]
        for t, r in zip(new, rows):
            t[self.pages_of(r):] = -1
        self.table[:len(new)] = new
        self.refs[:] = np.bincount(self.table[self.table >= 0], minlength=self.refs.size)

    def compact(self):
        used = int((self.refs > 0).sum())
        to = np.flatnonzero(self.refs[:used] == 0)
        source = used + np.flatnonzero(self.refs[used:] > 0)
        for s, t in zip(source, to):
            self.rows[:, t] = self.rows[:, s]
            self.refs[t], self.refs[s] = self.refs[s], 0
            self.table[self.table == s] = t
        return used

    def row(self, layer, seq, pos):
        return self.rows[layer, self.table[seq, pos // self.R], :, pos % self.R]

    def of(self, layer, seq, rows):
        """K and V of the first rows, or of those listed."""
        at = np.arange(rows) if np.isscalar(rows) else np.asarray(rows)
        x = self.rows[layer, self.table[seq, at // self.R], :, at % self.R]
        return x[:, 0], x[:, 1]


class Model:
    """A handle and its model.  Sequences' pages come scattered over the pool."""

    def __init__(self, nh, nkv, hd, seq_len, n_seq, cache="f32", page_rows=16, layers=1, spare=9, bounds=False, key=0, n_pages=None):
        from leap_amd.attention import PagedAttention
        self.nh, self.nkv, self.hd, self.n_seq, self.q8, self.layers = nh, nkv, hd, n_seq, cache == "q8", layers
        width = -(-seq_len // page_rows)
        n_pages = n_seq * width + spare if n_pages is None else n_pages
        self.h = PagedAttention(nh, nkv, hd, seq_len, n_pages, page_rows, n_layers=layers, max_batch=n_seq, cache=cache, bounds=bounds)
        self.p = Pages(n_seq, width, n_pages, page_rows, layers, nkv * hd)
        self.seq_len = seq_len
        from leap_amd.attention import HipAttention
        with HipAttention(nh, nkv, hd, seq_len) as t:  # (the tables are the same)
            self.cos, self.sin = t.rope_download()
        self.rng = rng_for(0x70616765, nh, nkv, hd, seq_len, n_seq, page_rows, key)

    def held(self, rows):
        return held(rows, self.hd, self.q8)

    def reserve(self, begin, end):
        ok = self.p.reserve(begin, end)
        assert ok
        self.h.reserve(begin, end)

    def fork(self, parent, rows):
        self.p.fork(parent, rows)
        self.h.fork(parent, rows)

    def scatter(self, lens):
        """Pages for lens rows of the sequences, in turns."""
        at = [0] * len(lens)
        while at != list(lens):
            to = [min(n, a + int(self.rng.integers(1, 2 + n // 3))) for a, n in zip(at, lens)]
            self.reserve(at, to)
            at = to

    def write(self, seq, layer, begin, k, v):
        self.h.write(seq, layer, begin, k, v)
        for i in range(len(k)):
            row = self.p.row(layer, seq, begin + i)
            row[0], row[1] = self.held(k[i]), self.held(v[i])

    def fill(self, lens, scale=1.0):
        """Random rows, their pages scattered."""
        self.scatter([max(n, 0) for n in lens])
        for i, n in enumerate(lens):
            for l in range(self.layers):
                if n > 0:
                    k, v = (self.rng.standard_normal((n, self.nkv * self.hd)).astype(np.float32) * np.float32(scale) for _ in range(2))
                    self.write(i, l, 0, k, v)

    def tokens(self, n):
        f = lambda w, s: (s * self.rng.standard_normal((n, w))).astype(np.float32)  # noqa: E731
        return f(self.nh * self.hd, 2.0), f(self.nkv * self.hd, 1.0), f(self.nkv * self.hd, 1.0)

    def store(self, layer, pos, k, v):
        """The new rows into the model."""
        for i, p in enumerate(pos):
            row = self.p.row(layer, i, p)
            row[0] = self.held(rope_f32(k[i], self.cos[p], self.sin[p]))
            row[1] = self.held(v[i])

    def turned(self, q, p):
        c, s = self.cos[p].astype(np.float64), self.sin[p].astype(np.float64)
        x = q.astype(np.float64).reshape(-1, self.hd)
        y = np.empty_like(x)
        y[:, 0::2], y[:, 1::2] = x[:, 0::2] * c - x[:, 1::2] * s, x[:, 1::2] * c + x[:, 0::2] * s
        return y.reshape(-1)

    def want(self, layer, pos, q, k, v):
        """Outputs in 64 bits, the rows stored."""
        self.store(layer, pos, k, v)
        return np.stack([attention_f64(self.turned(q[i], p), *self.p.of(layer, i, p + 1), self.nh, self.nkv, self.hd)
                         for i, p in enumerate(pos)])

    def choose(self, layer, seq, p, keep, q):
        """The pages that each KV head attends to, from the definition."""
        R, n = self.p.R, p // self.p.R
        x = rope_f32(q, self.cos[p], self.sin[p]).astype(np.float64).reshape(self.nkv, -1, self.hd)
        out = []
        for g in range(self.nkv):
            score = []
            for j in range(n):
                keys = self.p.rows[layer, self.p.table[seq, j], 0][:, g * self.hd:(g + 1) * self.hd]
                if self.q8:  # (bounds are of the values as fp32)
                    keys = keys.astype(np.float32).astype(np.float64)
                lo, hi = keys.min(axis=0), keys.max(axis=0)
                score.append(np.maximum(x[g] * lo, x[g] * hi).sum())
            order = sorted(range(n), key=lambda j: (-score[j] if score[j] == score[j] else -np.inf, j))[:keep - 1]
            out.append(sorted(order) + [n])
        return out

    def want_sparse(self, layer, pos, keep, q, k, v):
        """Outputs and chosen pages; the rows stored."""
        self.store(layer, pos, k, v)
        out = np.empty((len(pos), self.nh * self.hd))
        picked = np.full((len(pos), self.nkv, keep), -1, np.int32)
        group = self.nh // self.nkv
        for i, p in enumerate(pos):
            y = self.turned(q[i], p).reshape(self.nkv, -1)
            for g, pages in enumerate(self.choose(layer, i, p, keep, q[i])):
                picked[i, g, :len(pages)] = pages
                rows = [r for j in pages for r in range(j * self.p.R, min(p + 1, (j + 1) * self.p.R))]
                K, V = (x[:, g * self.hd:(g + 1) * self.hd] for x in self.p.of(layer, i, rows))
                out[i].reshape(self.nkv, -1)[g] = attention_f64(y[g], K, V, group, 1, self.hd)
        return out, picked

    def check_state(self):
        table, refs = self.h.state()
        assert np.array_equal(table, self.p.table)
        assert np.array_equal(refs, self.p.refs)

    def check_rows(self, lens):
        for i, n in enumerate(lens):
            for l in range(self.layers):
                for got, want in zip(self.h.read(i, l, 0, n), self.p.of(l, i, n)):
                    # (fp32: the rows as they were stored; 8 bits: value * scale rounded once)
                    np.testing.assert_allclose(got, want, rtol=2.0 ** -24 if self.q8 else 0, atol=0)


def begin_of(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
