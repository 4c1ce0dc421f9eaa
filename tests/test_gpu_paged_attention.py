"""Attention over a paged cache on the GPU against the definition in float64: head sizes, pages that
end inside a tile, lengths from zero, shared prefixes, anything in rows that no token attends,
tables and groups of any content, workspaces, streams and captured graphs."""
import numpy as np
import pytest

import cache_helpers as C
import paged_helpers as P

pytestmark = pytest.mark.gpu


def run(am, p, **kw):
    am.paged_attention_ex(p.cache, p.drafts, p.out.dev, p.lse, prefix=p.prefix, **kw)


DIMS = [1, 3, 4, 7, 16, 40, 63, 64, 65, 80, 127, 128, 129, 160, 192, 200, 255, 256]
WIDE = [257, 260, 320, 511, 512, 513, 777, 1024, 1025, 1032, 2048, 2050, 3000, 4096, 4100, 8192]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", DIMS + WIDE)
def test_head_sizes(am, dev, dtype, D):
    p = P.Paged(am, dtype, 3, 4, 2, 2, D, 16, [0, 37, 130], [1, 2, 2])
    run(am, p)
    p.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [16, 64, 80, 128, 192, 256, 320, 1000, 2048, 4096])
@pytest.mark.parametrize("page", [16, 20])
def test_head_sizes_under_a_prefix(am, dev, dtype, D, page):
    p = P.Paged(am, dtype, 5, 6, 2, 1, D, page, [100, 117, 90, 33, 250], first=[0, 3, 5], rows=[83, 32])
    run(am, p)
    p.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [1, 2, 7, 8, 15, 16, 17, 32, 48, 100, 256])
@pytest.mark.parametrize("D", [72, 384])
def test_pages(am, dev, dtype, page, D):
    p = P.Paged(am, dtype, 4, 3, 3, 1, D, page, [0, 1, 99, 301], first=[0, 2, 4], rows=[0, 77])
    run(am, p)
    p.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Hq,G", [(1, 1), (5, 1), (8, 8), (16, 2), (40, 1), (12, 4)])
@pytest.mark.parametrize("T", [1, 3, 17, 70])
def test_rows_of_a_tile(am, dev, dtype, Hq, G, T):
    for D in (128, 300):
        p = P.Paged(am, dtype, 2, Hq, G, T, D, 32, [45, 201], [T, max(1, T - 5)])
        run(am, p)
        p.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("T", [1, 5, 33])
def test_rows_of_a_prefix_tile(am, dev, dtype, D, T):
    """A group's members are rows of one tile, or of several."""
    lens = [150 + 11 * b for b in range(9)]
    p = P.Paged(am, dtype, 9, 8, 2, T, D, 16, lens, [max(0, T - b % 2) for b in range(9)],
                first=[1, 3, 9], rows=[140, 155])
    run(am, p)
    p.check()


@pytest.mark.parametrize("T", [1, 100, 300])
@pytest.mark.parametrize("lens", [[0], [1], [31], [32], [33], [1000]])
def test_lengths(am, dev, T, lens):
    for dtype in ("f32", "bf16"):
        p = P.Paged(am, dtype, 1, 2, 1, T, 64, 16, lens)
        run(am, p)
        p.check()


@pytest.mark.parametrize("order,offset,pad", [("rows", 0, 0), ("heads", 1, 0), ("rows", 3, 5),
                                              ("heads", 8, 8), ("rows", 0, 2)])
@pytest.mark.parametrize("D", [80, 128, 512])
def test_strides(am, dev, order, offset, pad, D):
    for dtype in ("f32", "bf16"):
        p = P.Paged(am, dtype, 3, 4, 2, 3, D, 16, [60, 70, 99], first=[0, 3], rows=[50], order=order,
                    offset=offset, pad=pad)
        run(am, p)
        p.check()


@pytest.mark.parametrize("B,groups", [(70, 0), (130, 65), (200, 3), (65, 1)])
@pytest.mark.parametrize("D", [64, 260])
def test_many_sequences(am, dev, B, groups, D):
    rng = np.random.default_rng(B)
    lens = [int(x) for x in rng.integers(40, 90, B)]
    counts = [int(x) for x in rng.integers(0, 3, B)]
    first = rows = None
    if groups:
        first = [i * B // groups for i in range(groups + 1)]
        rows = [int(x) for x in rng.integers(0, 41, groups)]
    p = P.Paged(am, "bf16", B, 2, 2, 2, D, 16, lens, counts, first=first, rows=rows)
    run(am, p)
    p.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [128, 1024])
def test_long(am, dev, dtype, D):
    """Ranges that cut sequences, and parts that a merge adds up."""
    p = P.Paged(am, dtype, 3, 4, 2, 1, D, 64, [3000, 777, 2500], first=[0, 2], rows=[700])
    run(am, p, max_len=3200)
    p.check()
    p.prefix = None
    run(am, p)
    p.check()


def test_scales(am, dev):
    for D in (64, 300):
        for scale in (0.3, -0.2, 1e-3):
            p = P.Paged(am, "bf16", 2, 4, 2, 3, D, 16, [50, 90], first=[0, 2], rows=[40])
            run(am, p, scale=scale)
            p.check(p.want(scale=scale))


def test_max_len_bounds_what_is_attended(am, dev):
    for D in (64, 512):
        p = P.Paged(am, "f32", 2, 2, 2, 1, D, 16, [99, 20])
        run(am, p, max_len=64)
        # sequence 0 attends rows 0 .. 63
        want = p.want(lens=[63, 20])
        p.check(want)


def test_tokens_that_attend_nothing(am, dev):
    """A table that names no page: zeros, and an lse of -infinity."""
    for D in (64, 512):
        for first in (None, [0, 2]):
            p = P.Paged(am, "bf16", 2, 2, 2, 2, D, 16, [40, 40], first=first,
                        rows=None if first is None else [32])
            p.tab.upload(np.full(p.table.shape, -1))
            run(am, p)
            assert (p.out.numpy() == 0).all() and np.isneginf(p.lse.numpy()).all()


@pytest.mark.parametrize("bad", [-1, 1 << 30, -(1 << 31)])
@pytest.mark.parametrize("page", [16, 7])
def test_rows_without_a_page(am, dev, bad, page):
    """Rows of an entry that names no page are not attended; the others are."""
    for D in (80, 384):
        p = P.Paged(am, "f32", 2, 2, 1, 1, D, page, [100, 64])
        table = p.table.copy()
        table[0, 2] = bad
        table[1, 0] = bad
        p.tab.upload(table)
        run(am, p)
        got, got_lse = p.out.numpy(), p.lse.numpy()
        for b in range(2):
            r = np.arange(p.lens[b] + 1)
            r = r[(table[b, r // page] >= 0) & (table[b, r // page] < p.K.host.shape[0])]
            k, v = (x.host[table[b, r // page], 0, r % page].astype(np.float64) for x in (p.K, p.V))
            one = np.zeros((1, 1, len(r), D))
            want, lse, info = C.attend64(p.Q.host[b:b + 1], one + k, one + v, None, None, [len(r)], [1])
            tol, tol_lse = C.attend_tol("f32", D, want, info)
            assert (np.abs(got[b] - want[0]) <= tol[0]).all()
            assert (np.abs(got_lse[b] - lse[0]) <= tol_lse[0] + 4 * C.U32 * np.abs(lse[0])).all()


@pytest.mark.parametrize("D", [64, 128, 512])
@pytest.mark.parametrize("fill", [np.inf, -np.inf, 3e38])
def test_what_no_token_attends(am, dev, D, fill):
    for dtype in ("f32", "bf16"):
        p = P.Paged(am, dtype, 3, 4, 2, 5, D, 16, [40, 71, 33], [5, 3, 0], first=[0, 2], rows=[35],
                    fill=fill)
        run(am, p)
        p.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [48, 128, 256, 400, 2048])
def test_not_finite_values_reach_their_rows_alone(am, dev, dtype, D):
    """Tokens that come after a value's row have it in that dim; those before it do not change."""
    T, lens = 6, [50, 61]
    p = P.Paged(am, dtype, 2, 4, 2, T, D, 16, lens)
    run(am, p)
    p.check()
    before, lse = p.out.numpy(), p.lse.numpy()
    V = p.V.host.copy()
    put = [(0, 2, 3, np.inf), (0, 4, 3, -np.inf), (0, 1, D - 1, -np.inf), (1, 0, 5, np.nan),
           (1, 5, 0, np.inf)]  # sequence, token, dim
    for b, t, d, x in put:
        r = lens[b] + t
        V[p.table[b, r // 16], :, r % 16, d] = x
    p.V.base.upload(p.V._flat(V))
    run(am, p)
    got = p.out.numpy()
    hit = np.zeros(got.shape, bool)
    for b, t, d, x in put:
        hit[b, :, t:, d] = True
    assert np.array_equal(got[~hit], before[~hit]) and np.array_equal(p.lse.numpy(), lse)
    assert np.isposinf(got[0, :, 2:4, 3]).all() and np.isnan(got[0, :, 4:, 3]).all()
    assert np.isneginf(got[0, :, 1:, D - 1]).all() and np.isnan(got[1, :, :, 5]).all()
    assert np.isposinf(got[1, :, 5:, 0]).all()


def test_not_finite_values_in_whole_blocks(am, dev):
    """Of rows that every token attends, prefix or own: infinite or NaN in their dim, no other."""
    for dtype in ("f32", "bf16"):
        for D in (64, 128, 512):
            p = P.Paged(am, dtype, 3, 2, 1, 1, D, 16, [200, 210, 190], first=[0, 3], rows=[100])
            V = p.V.host.copy()
            V[p.table[0, 2], 0, 5, 9] = np.inf        # row 37 of all
            V[p.table[1, 8], 0, 0, 11] = np.nan       # row 128 of sequence 1
            p.V.base.upload(p.V._flat(V))
            run(am, p)
            got = p.out.numpy()
            bad = np.zeros(got.shape, bool)
            bad[..., 9] = True
            bad[1, ..., 11] = True
            assert np.array_equal(~np.isfinite(got), bad) and np.isfinite(p.lse.numpy()).all()


def test_scores_that_are_not_finite(am, dev):
    """Attended keys of -infinity weigh nothing; of NaN make the rows that attend them NaN."""
    for D in (64, 512):
        p = P.Paged(am, "f32", 2, 2, 1, 3, D, 16, [40, 50], seed=6)
        q = np.abs(p.Q.host)
        p.Q.base.upload(p.Q._flat(q))
        p.Q.host = q
        K = p.K.host.copy()
        K[p.table[0, 0], 0, 3] = -np.inf
        r = 51  # token 1's row of sequence 1
        K[p.table[1, r // 16], 0, r % 16, 0] = np.nan
        p.K.base.upload(p.K._flat(K))
        run(am, p)
        got, lse = p.out.numpy(), p.lse.numpy()
        assert np.isnan(got[1, :, 1:]).all() and np.isnan(lse[1, :, 1:]).all()
        assert np.isfinite(got[1, :, 0]).all()
        rows = [i for i in range(41) if i != 3]
        k, v = (x[p.table[0, np.array(rows) // 16], :, np.array(rows) % 16].transpose(1, 0, 2)[None]
                for x in (K, p.V.host))
        want, wl, info = C.attend64(q[:1, :, :1], k.astype(np.float64), v.astype(np.float64), None, None,
                                    [40], [1])
        tol, _ = C.attend_tol("f32", D, want, info)
        assert (np.abs(got[:1, :, :1] - want) <= tol).all()


def test_large_logits(am, dev):
    for dtype in ("f32", "bf16"):
        for D in (128, 512):
            p = P.Paged(am, dtype, 2, 4, 2, 2, D, 16, [300, 410], first=[0, 2], rows=[256], sigma=30.0)
            run(am, p)
            p.check()


@pytest.mark.parametrize("D", [64, 128, 300])
def test_lists_of_any_content(am, dev, D):
    """Groups that do not ascend or pass the batch, lengths and tables out of range: nothing outside
    the outputs is written, and calls on good lists are as before."""
    rng = np.random.default_rng(7)
    p = P.Paged(am, "bf16", 6, 4, 2, 2, D, 16, [50, 60, 70, 80, 90, 40], first=[0, 3, 6], rows=[48, 33])
    run(am, p)
    p.check()
    first, rows = p.prefix.first, p.prefix.rows
    for f, n in (([5, 0, 9], [1 << 30, -4]), ([-3, 1 << 30, 0], [1 << 30, 1 << 30]),
                 ([0, 6, 0], [64, 64]), ([6, 6, 6], [10, 10]), ([0, 6, 6], [1 << 30, 5])):
        first.upload(np.array(f))
        rows.upload(np.array(n))
        run(am, p)
        p.out.numpy()
        p.tab.upload(rng.integers(-(1 << 31), 1 << 31, p.table.shape))
        p.len.upload(rng.integers(-(1 << 31), 1 << 31, 6))
        run(am, p)
        p.out.numpy()
        p.tab.upload(p.table)
        p.len.upload(np.array(p.lens))
    first.upload(np.array([0, 3, 6]))
    rows.upload(np.array([48, 33]))
    run(am, p)
    p.check()


def test_same_bits_every_time(am, dev):
    for D in (128, 512):
        p = P.Paged(am, "bf16", 4, 8, 2, 1, D, 16, [900, 1500, 700, 650], first=[0, 4], rows=[600])
        run(am, p)
        first, lse = p.out.base.bits(), p.lse.bits()
        for _ in range(4):
            run(am, p)
            assert np.array_equal(p.out.base.bits(), first) and np.array_equal(p.lse.bits(), lse)


@pytest.mark.parametrize("D", [128, 512])
def test_workspaces(am, dev, D):
    """The caller's, with anything behind it; fewer kv heads a launch where it is small."""
    import hip_rt
    p = P.Paged(am, "f32", 3, 8, 4, 2, D, 16, [700, 800, 600], first=[0, 3], rows=[500])
    need = am.paged_attention_workspace_bytes(p.cache, p.drafts, p.prefix)
    ws = hip_rt.DeviceArray((need + 4096,), "bf16", fill=0)
    guard = np.full(2048, 3, np.uint16)
    tail = hip_rt.DeviceArray.view(ws, need // 2, (2048,))
    tail.upload(guard)
    full = hip_rt.DeviceArray.wrap(ws.ptr, (need // 2,), "bf16", keep=ws)
    run(am, p, workspace=full)
    p.check()
    assert np.array_equal(tail.bits(), guard)
    # the smallest that runs: a kv head at a time, or whole items
    size, ran = need, 0
    while size > 40960:
        size = 40960 + (size - 40960) // 2 // 16 * 16
        small = hip_rt.DeviceArray.wrap(ws.ptr, (size // 2,), "bf16", keep=ws)
        p.out.base.upload(p.out._flat(np.full(p.out.host.shape, 7.0, np.float32)))
        try:
            run(am, p, workspace=small)
        except am.AtnError as e:
            assert e.status == -8
            break
        ran += 1
        p.check()
        assert np.array_equal(tail.bits(), guard)
    assert ran >= 1
    # none at all without a prefix, but for the scores of one kv head where head_d > 256
    p.prefix = None
    if D > 256:
        one = 3 * (1024 // 32 + 1) * 16 * 32 * 4  # sequences, blocks of a table's rows, rows, keys
        with pytest.raises(am.AtnError):
            run(am, p, workspace=hip_rt.DeviceArray.wrap(ws.ptr, (20480,), "bf16", keep=ws))
        small = 40960 + one * 2
    else:
        small = 40960
    run(am, p, workspace=hip_rt.DeviceArray.wrap(ws.ptr, (small // 2,), "bf16", keep=ws))
    p.check()


def test_streams_and_captured(am, dev):
    """Captured calls replay with what lengths, tables, counts and prefixes hold; two graphs share a
    workspace."""
    import hip_rt
    a = P.Paged(am, "bf16", 3, 8, 2, 1, 128, 16, [300, 420, 350], [1, 1, 1], first=[0, 3], rows=[256],
                slots=40)
    b = P.Paged(am, "bf16", 3, 8, 2, 1, 128, 16, [500, 320, 400], [1, 1, 0], first=[0, 3], rows=[300],
                slots=40, seed=3)
    for p in (a, b):  # rows for the lengths to come
        rng = np.random.default_rng(11)
        for x in (p.K, p.V):
            y = C.rounded(rng.standard_normal(x.host.shape), "bf16")
            for i in range(3):
                r = np.arange(256 // 16 * 16, p.rows[0])
                y[p.table[i, r // 16], :, r % 16] = y[p.table[0, r // 16], :, r % 16]
            x.host = y
            x.base.upload(x._flat(y))
    need = max(am.paged_attention_workspace_bytes(p.cache, p.drafts, p.prefix) for p in (a, b))
    ws = hip_rt.DeviceArray((need // 2 + 8,), "bf16", fill=0)
    s = hip_rt.Stream()
    calls = [am.paged_attention_call(p.cache, p.drafts, p.out.dev, p.lse, prefix=p.prefix,
                                     workspace=ws) for p in (a, b)]
    graphs = [hip_rt.Graph(s, lambda c=c: c(s)) for c in calls]
    for step in range(3):
        for g in graphs:
            g.launch()
        s.synchronize()
        for p in (a, b):
            p.check()
        calls[0]()  # eager work between the replays
        hip_rt.synchronize()
        a.lens = [n - 7 for n in a.lens]
        a.len.upload(np.array(a.lens))
        a.prefix.rows.upload(np.array([[0], [31], [200]][step]))
        b.table = b.table[:, :]
        b.lens = [300 + step, 310, 333]
        b.len.upload(np.array(b.lens))
    for g in graphs:
        g.destroy()
    # without a workspace of its own, a call that has run before may be captured
    s2 = hip_rt.Stream()
    call = am.paged_attention_call(a.cache, a.drafts, a.out.dev, a.lse, prefix=a.prefix)
    call(s2)
    s2.synchronize()
    g = hip_rt.Graph(s2, lambda: call(s2))
    for _ in range(2):
        g.launch()
        s2.synchronize()
        a.check()
    g.destroy()
    for x in (s, s2):
        x.destroy()


def test_two_streams_at_once(am, dev):
    import hip_rt
    ps = [P.Paged(am, "bf16", 4, 8, 2, 1, 128, 16, [1500, 1200, 1100, 1300], first=[0, 4], rows=[1024],
                  seed=i) for i in range(2)]
    wants = [p.want() for p in ps]
    ss = [hip_rt.Stream() for _ in ps]
    for _ in range(5):
        for p, s in zip(ps, ss):
            run(am, p, stream=s)
    for p, s, w in zip(ps, ss, wants):
        s.synchronize()
        p.check(w)
        s.destroy()


def test_half_a_pool_past_4_gib(am, dev):
    """Pages whose offsets pass 32 bits, in bytes and in elements."""
    import hip_rt
    G, page, D, pages = 8, 64, 256, 18000  # 4.7 GB a pool of bf16
    rng = np.random.default_rng(2)
    pools = [hip_rt.DeviceArray((pages, G, page, D), "bf16") for _ in range(2)]
    table = np.array([[pages - 1, 3, pages - 2]], np.int32)
    host = rng.standard_normal((2, 3, G, page, D)).astype(np.float32)
    for x, h in zip(pools, host):
        for i, p in enumerate(table[0]):
            hip_rt.DeviceArray.view(x, int(p) * G * page * D, (G, page, D)).upload(h[i])
    h16 = C.rounded(host, "bf16")
    q = C.Tensor(rng.standard_normal((1, 16, 1, D)), "bf16")
    out = C.Tensor(np.zeros((1, 16, 1, D)), "bf16")
    lse = C.floats(np.zeros((1, 16, 1)))
    cache = am.PagedCache(*pools, C.ints(table), C.ints([150]))
    am.paged_attention_ex(cache, am.Drafts(q.dev), out.dev, lse)
    k, v = (x.transpose(1, 0, 2, 3).reshape(1, G, 3 * page, D) for x in h16)
    want, wl, info = C.attend64(q.host, k, v, None, None, [151], [1])
    C.attend_close("bf16", D, out.numpy(), lse.numpy(), want, wl, info, [1])


@pytest.mark.parametrize("D", [64, 128, 300])
def test_groups_that_overlap(am, dev, D):
    """A list that does not ascend shares nothing: every sequence's rows are read as its own."""
    for B, first in ((6, [0, 6, 0, 6]), (6, [0, 4, 2, 6]), (6, [3, 6, 0, 6, 0, 6]),
                     (70, [0, 70] * 33 + [0]), (70, list(range(68)) + [0, 70])):
        p = P.Paged(am, "bf16", B, 4, 2, 1, D, 16, [90 + b % 7 for b in range(B)], first=[0, B], rows=[80])
        groups = len(first) - 1
        p.prefix = am.SharedPrefix(C.ints(first), C.ints([80] * groups))
        run(am, p)
        p.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,T", [(64, 1), (128, 90), (512, 2)])
def test_without_lse(am, dev, dtype, D, T):
    """The same output; in place of the queries is refused, as the library's other calls do it."""
    for first in (None, [0, 3]):
        p = P.Paged(am, dtype, 3, 4, 2, T, D, 16, [900, 700, 810], first=first,
                    rows=None if first is None else [650])
        run(am, p)
        p.check()
        out = p.out.base.bits()
        p.out.base.upload(p.out._flat(np.full(p.out.host.shape, 7.0, np.float32)))
        am.paged_attention_ex(p.cache, p.drafts, p.out.dev, None, prefix=p.prefix)
        assert np.array_equal(p.out.base.bits(), out)
    with pytest.raises(am.AtnError) as e:
        am.paged_attention_ex(p.cache, p.drafts, p.Q.dev, None)
    assert e.value.status == -5


@pytest.mark.parametrize("D", [64, 512])
def test_prefix_that_passes_a_member(am, dev, D):
    """Rows behind a member's own: unspecified results for it, the others' as they should be."""
    p = P.Paged(am, "f32", 4, 2, 1, 1, D, 16, [300, 310, 20, 305], first=[0, 2, 4], rows=[280, 16])
    p.prefix = am.SharedPrefix(C.ints([0, 2, 4]), C.ints([280, 1 << 30]))
    run(am, p)
    want, lse, info = p.want()
    got = p.out.numpy()
    tol, _ = C.attend_tol("f32", D, want, info)
    assert (np.abs(got[:2] - want[:2]) <= tol[:2]).all() and np.isfinite(p.lse.numpy()[:2]).all()


@pytest.mark.parametrize("D", [64, 128, 384])
def test_the_same_page_many_times(am, dev, D):
    """A table may name a page in several places; max_len may be less than the prefix."""
    p = P.Paged(am, "bf16", 3, 4, 2, 1, D, 16, [200, 190, 210], first=[0, 3], rows=[160])
    table = p.table.copy()
    table[:, 1:10] = table[0, 0]
    p.tab.upload(table)
    p.table = table
    run(am, p)
    p.check()
    run(am, p, max_len=100)
    p.check(p.want(lens=[99, 99, 99]))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [2, 16, 64, 72, 128, 160, 192, 256])
@pytest.mark.parametrize("page", [16, 24])
def test_few_and_many_items(am, dev, dtype, D, page):
    """Items whole by 8 waves or by 4, or in ranges, by how many there are and how long they may be."""
    rng = np.random.default_rng(D)
    for B, rows in ((2, 160), (2, 9000), (150, 160), (150, 9000), (600, 300)):
        lens = [int(x) for x in rng.integers(0, 150, B)]
        p = P.Paged(am, dtype, B, 4, 2, 1, D, page, lens, [int(x > 0) for x in rng.integers(0, 9, B)],
                    slots=-(-rows // page))
        run(am, p)
        p.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [2, 7, 40, 64, 72, 128, 160, 192, 250, 256])
@pytest.mark.parametrize("page", [16, 24])
def test_few_and_many_items_of_several_rows(am, dev, dtype, D, page):
    rng = np.random.default_rng(D)
    for B, T, rows in ((2, 15, 200), (2, 9, 9000), (20, 10, 600), (2, 45, 200), (140, 11, 170)):
        lens = [int(x) for x in rng.integers(0, 150, B)]
        p = P.Paged(am, dtype, B, 4, 2, T, D, page, lens, [int(x) for x in rng.integers(0, T + 1, B)],
                    slots=-(-rows // page))
        run(am, p)
        p.check()


@pytest.mark.parametrize("dtype,D,T,page", [("bf16", 128, 40, 16), ("bf16", 128, 6, 20), ("f32", 80, 12, 16),
                                            ("bf16", 512, 4, 16), ("f32", 2048, 4, 20)])
def test_prefixes_that_no_workspace_holds(am, dev, tuner, dtype, D, T, page):
    """A prefix whose parts the library's workspace does not hold: its rows are the sequences' own. The
    size that a query gives runs, and so does a larger one, which holds the parts."""
    import hip_rt
    p = P.Paged(am, dtype, 4, 16, 2, T, D, page, [1200, 1100, 1300, 1000], [T, T, 1, T], first=[0, 4],
                rows=[990])
    whole = am.paged_attention_workspace_bytes(p.cache, p.drafts, p.prefix)
    ws = hip_rt.DeviceArray((whole // 2,), "bf16", fill=0)
    tuner.set(workspace_cap_mib=1)
    need = am.paged_attention_workspace_bytes(p.cache, p.drafts, p.prefix)
    assert need <= (1 << 20) + 40960 < whole
    run(am, p)
    p.check()
    for n in (need, whole):
        p.out.base.upload(p.out._flat(np.full(p.out.host.shape, 7.0, np.float32)))
        run(am, p, workspace=hip_rt.DeviceArray.wrap(ws.ptr, (n // 2,), "bf16", keep=ws))
        p.check()


@pytest.mark.parametrize("dtype,D,T", [("bf16", 64, 48), ("f32", 80, 31), ("bf16", 512, 31)])
def test_prefixes_of_too_few_rows_need_no_room(am, dev, dtype, D, T):
    """Rows that no group reads once, whatever its list says: a workspace for the call without it."""
    import hip_rt
    p = P.Paged(am, dtype, 3, 8, 2, T, D, 16, [150, 140, 160], first=[0, 3], rows=[130])
    most = 256
    need = am.paged_attention_workspace_bytes(p.cache, p.drafts, None, most)
    ws = hip_rt.DeviceArray((need // 2,), "bf16", fill=0)
    run(am, p, workspace=ws, max_len=most)
    p.check()


@pytest.mark.parametrize("dtype,D", [("f32", 2048), ("bf16", 8192), ("f32", 8192)])
@pytest.mark.parametrize("rows", [None, [700]])
def test_fewer_shares_and_ranges(am, dev, dtype, D, rows):
    """Workspaces from what the library asks for down to the least: fewer shares of the dims, fewer ranges."""
    import hip_rt
    p = P.Paged(am, dtype, 2, 2, 1, 1, D, 16, [800, 730], first=None if rows is None else [0, 2],
                rows=rows)
    need = am.paged_attention_workspace_bytes(p.cache, p.drafts, p.prefix)
    ws = hip_rt.DeviceArray((need + 4096,), "bf16", fill=0)
    tail = hip_rt.DeviceArray.view(ws, need // 2, (2048,))
    tail.upload(np.full(2048, 3, np.uint16))
    ran = 0
    for i in range(16):
        size = 40960 + (need - 40960) * (16 - i) // 16 // 16 * 16
        small = hip_rt.DeviceArray.wrap(ws.ptr, (size // 2,), "bf16", keep=ws)
        p.out.base.upload(p.out._flat(np.full(p.out.host.shape, 7.0, np.float32)))
        try:
            run(am, p, workspace=small)
        except am.AtnError as e:
            assert e.status == -8
            break
        ran += 1
        p.check()
    assert ran >= 4 and (tail.bits() == 3).all()


@pytest.mark.parametrize("dtype,D,T,page,order", [("bf16", 512, 30, 16, "heads"), ("bf16", 320, 21, 20, "rows"),
                                                  ("f32", 1025, 13, 16, "rows"), ("f32", 512, 40, 16, "heads")])
def test_sequences_in_turn(am, dev, tuner, dtype, D, T, page, order):
    """head_d > 256 where the scores of all sequences pass the workspace: some sequences a launch, the
    last ones fewer; on a stream and from a graph too, with a prefix that is left out."""
    import hip_rt
    B = 7
    rng = np.random.default_rng(D)
    lens = [int(x) for x in rng.integers(40, 1100, B)]
    counts = [T, 0, T - 3, 1, T, 7, T]
    p = P.Paged(am, dtype, B, 8, 2, T, D, page, lens, counts, first=[0, 3, 7], rows=[30, 20], order=order,
                offset=3, pad=5, slots=70)
    tuner.set(workspace_cap_mib=1)
    want = p.want()
    for prefix in (p.prefix, None):
        p.prefix = prefix
        p.out.base.upload(p.out._flat(np.full(p.out.host.shape, 7.0, np.float32)))
        run(am, p)
        p.check(want)
    need = am.paged_attention_workspace_bytes(p.cache, p.drafts)
    assert need <= (1 << 20) + 40960
    ws = hip_rt.DeviceArray((need // 2 + 2048,), "bf16", fill=0)
    tail = hip_rt.DeviceArray.view(ws, need // 2, (2048,))
    tail.upload(np.full(2048, 3, np.uint16))
    ws = hip_rt.DeviceArray.wrap(ws.ptr, (need // 2,), "bf16", keep=ws)
    call = am.paged_attention_call(p.cache, p.drafts, p.out.dev, p.lse, workspace=ws)
    s = hip_rt.Stream()
    g = hip_rt.Graph(s, lambda: call(s))
    for _ in range(3):
        p.out.base.upload(p.out._flat(np.full(p.out.host.shape, 7.0, np.float32)))
        g.launch()
        s.synchronize()
        p.check(want)
        run(am, p)  # eager work between the replays
        hip_rt.synchronize()
    assert (tail.bits() == 3).all()
    g.destroy()
    s.destroy()
