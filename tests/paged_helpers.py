"""Inputs, float64 definitions and tolerances of the tests of rotation and of the paged cache."""
import numpy as np

import cache_helpers as C

U = C.U32


def turned(x, pos, freq, half, rot, amplitude=1.0, inverse=False):
    """x [B][heads][T][D] with its pairs turned by pos [B][T] times freq, in float64; and, for
    tolerances, each element's pair's |x1| + |x2| (0 where nothing turns)."""
    x = x.astype(np.float64)
    y, size = x.copy(), np.zeros_like(x)
    angle = np.asarray(pos, np.float64)[:, None, :, None] * freq.astype(np.float64)
    c, s = amplitude * np.cos(angle), amplitude * np.sin(angle) * (-1 if inverse else 1)
    i = np.arange(rot // 2)
    i1, i2 = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
    a, b = x[..., i1], x[..., i2]
    y[..., i1], y[..., i2] = a * c - b * s, a * s + b * c
    size[..., i1] = size[..., i2] = np.abs(a) + np.abs(b)
    return y, size


def turned_tol(dtype, want, size, pos, freq, amplitude=1.0):
    """Half a step of the type, and of fp32: the angle's last rounding (half turns of at most 1 to
    half a step, 2^-25 pi, so 1.6 U), the sine's own error (2 steps of at most 1: 4 U), the
    product with the amplitude (1 U, and 1 U of the amplitude's own), the two products and their sum
    (2 U): 10 U of |x1| + |x2| times the amplitude.  fp64: four roundings of the turns, here and
    there, 2^-53 of up to |pos| max(freq) / 2 pi turns each."""
    far = np.abs(np.asarray(pos, np.float64)).max() * float(freq.max()) * 4 * 2.0 ** -53
    return (10 * U + far) * amplitude * size * 1.001 + C.HALF[dtype] * np.abs(want) + 1e-37


def deal_pages(rng, lens, counts, page, slots=None, spare=3):
    """A table [B][slots] of pages in no order (-1 where there is none) and the number of pages."""
    need = [-(-(l + n) // page) for l, n in zip(lens, counts)]
    slots = max(need + [1]) + 1 if slots is None else slots
    order = rng.permutation(sum(need) + spare)
    table = np.full((len(lens), slots), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        n = min(n, slots)
        table[b, :n] = order[at:at + n]
        at += n
    return table, int(len(order))


def share(table, first, rows, page):
    """The members of each group get its first sequence's pages below `rows` (whole ones)."""
    for i in range(len(rows)):
        for b in range(first[i] + 1, first[i + 1]):
            table[b, :rows[i] // page] = table[first[i], :rows[i] // page]


def rows_at(pool, table, b, upto, page):
    """Rows 0 .. upto - 1 of sequence b [heads][rows][D]."""
    r = np.arange(upto)
    return pool[table[b, r // page], :, r % page].transpose(1, 0, 2)


class Paged:
    """An attention call on random pages: rows in use random, all others `fill`."""

    def __init__(self, am, dtype, B, Hq, G, T, D, page, lens, counts=None, first=None, rows=None,
                 order="heads", offset=0, pad=0, seed=1, sigma=1.5, fill=np.nan, slots=None):
        rng = np.random.default_rng(seed)
        self.am, self.dtype, self.D, self.page = am, dtype, D, page
        self.lens, self.counts = list(lens), [T] * B if counts is None else list(counts)
        self.first, self.rows = first, rows
        table, pages = deal_pages(rng, self.lens, self.counts, page, slots)
        pools = [np.full((pages, G, page, D), fill, np.float32) for _ in range(2)]
        if first is not None:
            share(table, first, rows, page)
        self.table = table
        for b in range(B):
            r = np.arange(min(self.lens[b] + self.counts[b], table.shape[1] * page))
            for x in pools:
                x[table[b, r // page], :, r % page] = rng.standard_normal((len(r), G, D))
        if first is not None:  # (copies of the rows of a last page that is shared in part)
            for i, n in enumerate(rows):
                r = np.arange(n // page * page, n)
                for b in range(first[i] + 1, first[i + 1]):
                    for x in pools:
                        x[table[b, r // page], :, r % page] = \
                            x[table[first[i], r // page], :, r % page]
        q = rng.standard_normal((B, Hq, T, D)).astype(np.float32) * np.float32(sigma)
        for b in range(B):
            q[b, :, self.counts[b]:] = fill
        lay = dict(order=order, offset=offset, pad=pad)
        self.Q, self.K, self.V = (C.Tensor(x, dtype, **lay) for x in (q, *pools))
        self.out = C.Tensor(np.full(q.shape, 7.0, np.float32), dtype, **lay)
        self.lse = C.floats(np.full((B, Hq, T), 7.0))
        self.len, self.tab = C.ints(self.lens), C.ints(table)
        self.cache = am.PagedCache(self.K.dev, self.V.dev, self.tab, self.len)
        self.drafts = am.Drafts(self.Q.dev, count=None if counts is None else C.ints(counts))
        self.prefix = None if first is None else am.SharedPrefix(C.ints(first), C.ints(rows))

    def want(self, lens=None, scale=None, table=None, K=None, V=None):
        lens = self.lens if lens is None else lens
        table = self.table if table is None else table
        B, Hq, T, D = self.Q.host.shape
        G, page, cap = self.K.host.shape[1], self.page, table.shape[1] * self.page
        top = max(lens) + T
        x = []
        for pool in (self.K.host if K is None else K, self.V.host if V is None else V):
            old, new = np.zeros((B, G, max(lens), D)), np.zeros((B, G, T, D))
            for b in range(B):
                got = rows_at(pool, table, b, min(lens[b] + self.counts[b], cap), page)
                old[b, :, :lens[b]] = got[:, :lens[b]]
                new[b, :, :self.counts[b]] = got[:, lens[b]:]
            x += [old, new]
        assert top > 0
        return C.attend64(self.Q.host, x[0], x[2], x[1], x[3], lens, self.counts, None, scale)

    def check(self, want=None):
        want, lse, info = self.want() if want is None else want
        got, got_lse = self.out.numpy(), self.lse.numpy()
        C.attend_close(self.dtype, self.D, got, got_lse, want, lse, info, self.counts)
        for b, n in enumerate(self.counts):  # rows past count: as they were
            assert (got[b, :, n:] == 7.0).all() and (got_lse[b, :, n:] == 7.0).all()
