"""Append of keys and values to the pages of a cache on the GPU: rows where they belong and nowhere
else, keys and queries turned by their positions, and the lengths."""
import numpy as np
import pytest

import cache_helpers as C
import paged_helpers as P

pytestmark = pytest.mark.gpu


class Append:
    def __init__(self, am, dtype, B, Hq, G, T, D, page, lens, counts=None, pairing="half", rot=0,
                 order="heads", offset=0, pad=0, seed=1, slots=None, amplitude=1.0, edit=None):
        rng = np.random.default_rng(seed)
        self.dtype, self.page, self.rot, self.half, self.amplitude = dtype, page, rot, \
            pairing == "half", amplitude
        self.lens, self.counts = list(lens), [T] * B if counts is None else list(counts)
        self.table, pages = P.deal_pages(rng, self.lens, self.counts, page, slots)
        if edit:
            edit(self.table)
        lay = dict(order=order, offset=offset, pad=pad)
        self.K, self.V = (C.Tensor(rng.standard_normal((pages, G, page, D)), dtype, **lay)
                          for _ in range(2))
        self.Q, self.Kd, self.Vd = (C.Tensor(rng.standard_normal((B, h, T, D)), dtype, **lay)
                                    for h in (Hq, G, G))
        self.q_out = C.Tensor(np.full((B, Hq, T, D), 7.0), dtype, **lay)
        self.tab, self.len = C.ints(self.table), C.ints(self.lens)
        self.cache = am.PagedCache(self.K.dev, self.V.dev, self.tab, self.len)
        self.drafts = am.Drafts(self.Q.dev, self.Kd.dev, self.Vd.dev,
                                count=None if counts is None else C.ints(counts))
        self.rotary = None
        if rot:
            self.freq, _ = am.rope_frequencies(rot)
            self.rotary = am.Rotary(C.floats(self.freq), pairing, rot, amplitude)

    def check(self, pos=None, lens=None, q_out=None):
        lens = self.lens if lens is None else lens
        T, page = self.Kd.host.shape[2], self.page
        cap = self.table.shape[1] * page
        at = np.asarray(lens)[:, None] + np.arange(T)[None]
        pos = at if pos is None else pos
        K, V = self.K.host.astype(np.float64), self.V.host.copy()
        tol = np.zeros_like(K)
        q, k = ((x.host, 0 * x.host) if not self.rot else
                P.turned(x.host, pos, self.freq, self.half, self.rot, self.amplitude)
                for x in (self.Q, self.Kd))
        tols = [0 * x[0] if not self.rot else
                P.turned_tol(self.dtype, *x, pos, self.freq, self.amplitude) for x in (q, k)]
        for b, n in enumerate(self.counts):
            for t in range(n):
                r = at[b, t]
                p = self.table[b, r // page] if r < cap else -1
                if 0 <= p < K.shape[0]:
                    K[p, :, r % page], tol[p, :, r % page] = k[0][b, :, t], tols[1][b, :, t]
                    V[p, :, r % page] = self.Vd.host[b, :, t]
        assert (np.abs(self.K.numpy() - K) <= tol).all()
        assert np.array_equal(self.V.numpy(), V)
        got = (self.q_out if q_out is None else q_out).numpy()
        for b, n in enumerate(self.counts):
            assert (np.abs(got[b, :, :n] - q[0][b, :, :n]) <= tols[0][b, :, :n]).all()
            rest = self.Q.host[b, :, n:] if q_out is self.Q else 7.0
            assert (got[b, :, n:] == rest).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [1, 5, 16, 64])
@pytest.mark.parametrize("order,offset,pad", [("heads", 0, 0), ("rows", 0, 0), ("rows", 3, 1),
                                              ("heads", 8, 8)])
def test_append(am, dev, dtype, page, order, offset, pad):
    a = Append(am, dtype, 4, 6, 2, 9, 48, page, [0, 3, 15, 77], [9, 0, 1, 5], rot=32, order=order,
               offset=offset, pad=pad, amplitude=1.5)
    am.paged_append_ex(a.cache, a.drafts, a.rotary, q_out=a.q_out.dev)
    a.check()


@pytest.mark.parametrize("pairing", ["interleaved", "half"])
@pytest.mark.parametrize("D,rot", [(128, 128), (80, 20), (7, 6), (512, 512), (8192, 256), (64, 0)])
def test_dims(am, dev, pairing, D, rot):
    for dtype in ("f32", "bf16"):
        a = Append(am, dtype, 2, 4, 2, 3, D, 16, [5, 100], pairing=pairing, rot=rot)
        am.paged_append_ex(a.cache, a.drafts, a.rotary, q_out=a.q_out.dev)
        a.check()


def test_positions_given(am, dev):
    a = Append(am, "f32", 3, 4, 4, 6, 64, 16, [10, 0, 31], [6, 2, 6], rot=64)
    pos = np.random.default_rng(2).integers(0, 1 << 20, (3, 6)).astype(np.int32)
    am.paged_append_ex(a.cache, a.drafts, a.rotary, pos=C.ints(pos), q_out=a.q_out.dev)
    a.check(pos)


@pytest.mark.parametrize("rot", [0, 32])
def test_queries_in_place_or_left_out(am, dev, rot):
    a = Append(am, "bf16", 2, 4, 2, 5, 32, 16, [3, 18], [5, 4], rot=rot)
    am.paged_append_ex(a.cache, a.drafts, a.rotary, q_out=a.Q.dev)
    a.check(q_out=a.Q)
    a = Append(am, "bf16", 2, 4, 2, 5, 32, 16, [3, 18], [0, 0], rot=rot)
    am.paged_append_ex(a.cache, a.drafts, a.rotary)
    a.check()  # (no query is written, nor any row)


def test_rows_that_the_table_does_not_hold(am, dev):
    """Past its end, of entries that name no page, and of lengths out of range."""
    def edit(table):
        table[1, 1], table[2, 1] = -1, 1 << 30

    a = Append(am, "f32", 4, 2, 2, 30, 16, 8, [10, 0, 3, 20], rot=16, slots=4, edit=edit)
    am.paged_append_ex(a.cache, a.drafts, a.rotary, q_out=a.q_out.dev)
    a.check()
    am.paged_advance_ex(a.cache, a.drafts)
    assert a.len.numpy().tolist() == [32, 30, 32, 32]
    a = Append(am, "f32", 3, 2, 2, 3, 16, 8, [0, 0, 0], rot=16, slots=2)
    a.len.upload(np.array([-5, 1000, 1 << 30]))
    am.paged_append_ex(a.cache, a.drafts, a.rotary, q_out=a.q_out.dev)
    a.check(lens=[0, 16, 16])
    am.paged_advance_ex(a.cache, a.drafts)
    assert a.len.numpy().tolist() == [3, 16, 16]


def test_counts_out_of_range(am, dev):
    a = Append(am, "f32", 3, 2, 2, 3, 16, 8, [1, 2, 3], [3, 0, 3], rot=16)
    import attn_mi355x
    a.drafts = attn_mi355x.Drafts(a.Q.dev, a.Kd.dev, a.Vd.dev, count=C.ints([1 << 30, -7, 4]))
    am.paged_append_ex(a.cache, a.drafts, a.rotary, q_out=a.q_out.dev)
    a.check()
    am.paged_advance_ex(a.cache, a.drafts)
    assert a.len.numpy().tolist() == [4, 2, 6]


@pytest.mark.parametrize("B,T", [(300, 1), (1, 1500), (257, 3)])
def test_many_tokens(am, dev, B, T):
    lens = [(37 * b) % 90 for b in range(B)]
    a = Append(am, "bf16", B, 4, 2, T, 64, 16, lens, [max(0, T - b % 3) for b in range(B)], rot=64)
    am.paged_append_ex(a.cache, a.drafts, a.rotary, q_out=a.q_out.dev)
    a.check()
    am.paged_advance_ex(a.cache, a.drafts)
    assert a.len.numpy().tolist() == [l + n for l, n in zip(lens, a.counts)]
    a.drafts.desc.count = None  # (all T tokens of each)
    am.paged_advance_ex(a.cache, a.drafts)
    cap = a.table.shape[1] * 16
    assert a.len.numpy().tolist() == [min(cap, l + n + T) for l, n in zip(lens, a.counts)]


@pytest.mark.parametrize("order", ["rows", "heads"])
@pytest.mark.parametrize("B,T", [(3, 1), (33, 1), (2, 4)])
def test_columns_of_one_buffer(am, dev, order, B, T):
    """Queries, keys and values as columns of a projection's rows (or heads of one buffer), the queries
    turned where they are; a token each, as in a step of decoding, and several."""
    import types

    import hip_rt
    Hq, G, D = 6, 2, 32
    a = Append(am, "bf16", B, Hq, G, T, D, 16, [(11 * b) % 40 for b in range(B)], rot=D)
    n = Hq + 2 * G
    x = np.concatenate([a.Q.host, a.Kd.host, a.Vd.host], axis=1)  # [B][n][T][D]
    lie = (0, 2, 1, 3) if order == "rows" else (0, 1, 2, 3)
    base = hip_rt.DeviceArray.from_numpy(np.ascontiguousarray(x.transpose(lie)), "bf16")
    s = (n * T * D, D, n * D, 1) if order == "rows" else (n * T * D, T * D, D, 1)
    step = s[1]

    def view(first, heads):
        return hip_rt.DeviceArray.wrap(base.ptr + 2 * first * step, (B, heads, T, D), "bf16", strides=s,
                                       keep=base)

    q = view(0, Hq)
    am.paged_append_ex(a.cache, am.Drafts(q, view(Hq, G), view(Hq + G, G)), a.rotary, q_out=q)
    got = base.numpy().transpose(lie)
    a.check(q_out=types.SimpleNamespace(numpy=lambda: got[:, :Hq]))
    assert np.array_equal(got[:, Hq:], x[:, Hq:])
